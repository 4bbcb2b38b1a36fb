"""Attention over the quantised cache on the matrix units (single tokens, prompt portions) against 64 bits."""

import pytest
import torch

from . import e4m3_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from shrike_amd.kernels import ops

    return ops


# heads, kv heads, head size, page size
FORMS = [(14, 2, 64, 16), (28, 4, 128, 16), (40, 8, 128, 64), (6, 6, 32, 16), (24, 8, 96, 32), (16, 1, 128, 48), (36, 2, 64, 16),
         (4, 2, 160, 16), (4, 1, 192, 32), (5, 1, 224, 16), (8, 1, 256, 16), (128, 1, 32, 16), (33, 1, 96, 16)]


def poisoned(step, k_pool, v_pool, scales):
    """The pools on the device with NaN codes and bytes of 255 (an infinite unit) in every slot that no token of the step has."""
    used = torch.zeros(step.pages, step.ps, dtype=torch.bool)
    for i, n in enumerate(step.ctx_lens.tolist()):
        at = torch.arange(n)
        used[step.tables[i].long()[at // step.ps], at % step.ps] = True
    free = ~used
    k = k_pool.view(torch.uint8).transpose(2, 3).clone()  # [pages, kv, slot, slab, 32]
    k.transpose(1, 2)[free] = 0x7f
    v = v_pool.view(torch.uint8).transpose(2, 3).clone()
    v.transpose(1, 2)[free] = 0x7f
    s = scales.permute(0, 3, 1, 2).clone()
    s[free] = 0xff
    return (k.transpose(2, 3).contiguous().view(plain.E4M3).cuda(), v.transpose(2, 3).contiguous().view(plain.E4M3).cuda(),
            s.permute(0, 2, 3, 1).contiguous().cuda())


def setup(step, form, gain=2.0):
    heads, kv, dim, ps = form
    k_pool, v_pool, scales, keys, values = plain.random_pools(step.pages, kv, dim, ps, step.gen)
    q = (gain * torch.randn(step.n, heads * dim, generator=step.gen)).bfloat16()
    return poisoned(step, k_pool, v_pool, scales), keys, values, q


def check(step, form, got, q, keys, values, window, chunk, rows=slice(None)):
    heads, _, dim, _ = form
    want, size, reach = plain.attention(step, q, keys, values, heads, dim ** -0.5, window, chunk)
    limit = plain.allowed(want, size, reach, dim, max(step.ctx_lens.tolist()), True)
    off = (got.cpu().double().view_as(want) - want).abs()
    assert (off <= limit)[rows].all(), f"{(off / limit)[rows].max().item():.3g} of what is allowed"


DECODES = [([0], None, None), ([15, 16, 17, 0], None, None), ([62, 63, 64, 65, 127, 128, 129], None, None), ([255, 256, 700], None, None),
           ([300, 5, 64], 1, None), ([300, 1000, 64], 100, None), ([300, 191, 192], None, 64), ([500, 90], 70, 48)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("starts, window, chunk", DECODES)
@pytest.mark.parametrize("nsplit", [1, 3, 64])
def test_single_tokens(ops, form, starts, window, chunk, nsplit):
    heads, kv, dim, ps = form
    step = plain.Step(starts, [1] * len(starts), ps, seed=dim + len(starts))
    pools, keys, values, q = setup(step, form)
    out = torch.full((step.n + 1, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    partial = torch.full((step.n * heads * nsplit * (dim + 2),), float("nan"), device="cuda")
    ops.attention_decode_e4m3(q.cuda(), out, step.n, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, window,
                              dim ** -0.5, partial, nsplit, chunk=chunk)
    assert (out[step.n] == 9).all()
    check(step, form, out[: step.n], q, keys, values, window, chunk)


PORTIONS = [
    # tokens before, new tokens, sequences with one token in front of them, window, chunk
    ([0], [1], 0, None, None), ([0], [2], 0, None, None), ([0, 17, 5], [16, 1, 33], 0, None, None), ([63, 64, 65], [65, 64, 1], 0, None, None),
    ([1000], [5], 0, None, None), ([40, 300, 0], [1, 70, 20], 1, None, None), ([7, 9, 0, 130], [1, 1, 0, 140], 2, None, None),
    ([200], [100], 0, 30, None), ([200, 0], [40, 90], 0, None, 64), ([100], [200], 0, 90, 128), ([500], [3], 0, 1, None),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("starts, news, singles, window, chunk", PORTIONS)
@pytest.mark.parametrize("nsplit", [1, 4])
def test_portions(ops, form, starts, news, singles, window, chunk, nsplit):
    heads, kv, dim, ps = form
    step = plain.Step(starts, news, ps, seed=dim + len(starts))
    pools, keys, values, q = setup(step, form)
    wide = torch.zeros(step.n, heads * dim + 24, dtype=torch.bfloat16, device="cuda")
    wide[:, : heads * dim] = q.cuda()
    out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    partial = torch.full(((step.n - singles) * heads * nsplit * (dim + 2),), float("nan"), device="cuda")
    ops.attention_prefill_e4m3(wide[:, : heads * dim], out, singles, len(starts) - singles, heads, kv, dim, step.cu_q.cuda(),
                               step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps, window, dim ** -0.5, partial, nsplit, chunk=chunk)
    assert (out[:singles] == 9).all()
    check(step, form, out, q, keys, values, window, chunk, slice(singles, None))


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16), (16, 16, 128, 32), (8, 1, 96, 16)])
@pytest.mark.parametrize("starts, news", [([0], [1500]), ([3000], [300]), ([0] * 70, [29 + 3 * (i % 5) for i in range(70)])])
def test_many_rows_take_workgroups_of_256(ops, form, starts, news):
    heads, kv, dim, ps = form
    step = plain.Step(starts, news, ps, seed=1)
    pools, keys, values, q = setup(step, form, 1.0)
    for nsplit in (1, 2):
        out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
        partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
        ops.attention_prefill_e4m3(q.cuda(), out, 0, len(starts), heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(),
                                   step.tables.cuda(), *pools, ps, None, dim ** -0.5, partial, nsplit)
        check(step, form, out, q, keys, values, None, None)


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16)])
def test_long_contexts(ops, form):
    heads, kv, dim, ps = form
    step = plain.Step([20000, 9000, 31], [1, 1, 1], ps, seed=2)
    pools, keys, values, q = setup(step, form, 3.0)
    keys[step.tables[0, 0].long(), :, 0] *= 1.0  # (the first key as it is)
    for nsplit in (1, 16, 64):
        out = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
        partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
        ops.attention_decode_e4m3(q.cuda(), out, step.n, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None,
                                  dim ** -0.5, partial, nsplit)
        check(step, form, out, q, keys, values, None, None)


def test_one_large_weight_before_many_small_ones(ops):
    """A first token that takes most of the weight, and thousands whose weights are 2^-17 of it: they count."""
    heads, kv, dim, ps = 2, 1, 64, 16
    step = plain.Step([16000, 16000 - 7], [1, 7], ps, seed=3)
    k = torch.zeros(step.pages, kv, ps, dim, dtype=torch.float64)
    v = torch.full_like(k, 1.0)
    for i in range(2):
        k[step.tables[i, 0].long(), :, 0] = 17 * 0.6875 / 8  # times 64 elements of 1 / 8: 2^17 in the end
        v[step.tables[i, 0].long(), :, 0] = -1.0
    (kq, ke), (vq, ve) = plain.quantised(k), plain.quantised(v)
    codes = [(x / 2.0 ** e.double()[..., None]).float().to(plain.E4M3).view(torch.uint8) for x, e in ((kq, ke), (vq, ve))]
    pools = (codes[0].view(step.pages, kv, ps, 2, 32).transpose(2, 3).contiguous().view(plain.E4M3),
             codes[1].transpose(2, 3).contiguous().view(plain.E4M3), torch.stack([ke + 127, ve + 127], 2).to(torch.uint8).contiguous())
    q = torch.ones(step.n, heads * dim).bfloat16()
    pools = tuple(t.cuda() for t in pools)
    out = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    partial = torch.empty(step.n * heads * 8 * (dim + 2), device="cuda")
    for nsplit in (1, 8):
        ops.attention_decode_e4m3(q.cuda(), out, 1, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.125,
                                  partial, nsplit)
        ops.attention_prefill_e4m3(q.cuda(), out, 1, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools,
                                   ps, None, 0.125, partial, nsplit)
        want, size, reach = plain.attention(step, q, kq, vq, heads, 0.125)
        limit = plain.allowed(want, size, reach, dim, 16001, True)
        assert ((out.cpu().double().view_as(want) - want).abs() <= limit).all()


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16), (8, 1, 256, 32)])
@pytest.mark.parametrize("sizes", [[-30, 0, 20], [-60, 60], [-100, -99], [70, 72], [0, -117], [None, 0], [None]])
def test_values_of_very_different_sizes(ops, form, sizes):
    """Rows of values times 2^size, None: zeros.  (Beyond 40 either way the portions' kernel multiplies the codes themselves.)"""
    heads, kv, dim, ps = form
    step = plain.Step([200, 90], [1, 70], ps, seed=8)
    k_pool, v_pool, scales, keys, values = plain.random_pools(step.pages, kv, dim, ps, step.gen)
    pick = torch.randint(0, len(sizes), (step.pages, kv, ps), generator=step.gen)
    by = torch.tensor([0.0 if x is None else 2.0 ** x for x in sizes], dtype=torch.float64)[pick]
    values, e = plain.quantised(values * by[..., None])
    codes = (values / 2.0 ** e.double()[..., None]).float().to(plain.E4M3).view(torch.uint8)
    scales = scales.clone()
    scales[:, :, 1] = (e + 127).to(torch.uint8)
    pools = poisoned(step, k_pool, codes.transpose(2, 3).contiguous().view(plain.E4M3), scales)
    q = (2 * torch.randn(step.n, heads * dim, generator=step.gen)).bfloat16()
    out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    for nsplit in (1, 3):
        partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
        ops.attention_decode_e4m3(q.cuda(), out, 1, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None, dim ** -0.5,
                                  partial, nsplit)
        ops.attention_prefill_e4m3(q.cuda(), out, 1, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps,
                                   None, dim ** -0.5, partial, nsplit)
        want, size, reach = plain.attention(step, q, keys, values, heads, dim ** -0.5)
        # (2^-126: below that bfloat16 numbers and their products have fewer bits)
        limit = plain.allowed(want, size, reach, dim, 201, True) + 2.0 ** -126
        assert ((out.cpu().double().view_as(want) - want).abs() <= limit).all()


@pytest.mark.parametrize("gain", [30.0, 300.0])
def test_scores_of_hundreds(ops, gain):
    """Weights that overflow a type relative to an earlier reference, rising and falling along the keys."""
    form = heads, kv, dim, ps = 8, 2, 64, 16
    step = plain.Step([700, 400], [1, 60], ps, seed=9)
    pools, keys, values, _ = setup(step, form)
    q = (gain * torch.randn(step.n, heads * dim, generator=step.gen)).bfloat16()
    out = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    for nsplit in (1, 3):
        partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
        ops.attention_decode_e4m3(q.cuda(), out, 1, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.125, partial,
                                  nsplit)
        ops.attention_prefill_e4m3(q.cuda(), out, 1, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps,
                                   None, 0.125, partial, nsplit)
        check(step, form, out, q, keys, values, None, None)


def test_tokens_and_pages_that_are_not_there(ops):
    form = heads, kv, dim, ps = 14, 2, 64, 16
    step = plain.Step([40, 100, 33], [1, 1, 50], ps, seed=4)
    pools, keys, values, q = setup(step, form)
    out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    positions = step.positions.clone()
    positions[1] = -1  # padding
    for nsplit in (1, 2):
        partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
        ops.attention_decode_e4m3(q.cuda(), out, 2, heads, kv, dim, positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.125, partial,
                                  nsplit)
        assert (out[1] == 0).all()
        check(step, form, out, q, keys, values, None, None, slice(0, 1))
        # entries outside the pool and positions beyond the table are not followed (what comes out is no sequence's)
        bad = torch.full_like(step.tables, 2 ** 31 - 1).cuda()
        ops.attention_decode_e4m3(q.cuda(), out, 2, heads, kv, dim, step.positions.cuda(), bad, *pools, ps, None, 0.125, partial, nsplit)
        ops.attention_decode_e4m3(q.cuda(), out, 2, heads, kv, dim, step.positions.cuda() + 1000, step.tables.cuda(), *pools, ps, None, 0.125,
                                  partial, nsplit)
        ops.attention_prefill_e4m3(q.cuda(), out, 2, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), bad, *pools, ps, None, 0.125,
                                   partial, nsplit)
        ops.attention_prefill_e4m3(q.cuda(), out, 2, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda() + 999, step.tables.cuda(),
                                   *pools, ps, None, 0.125, partial, nsplit)
        short = step.ctx_lens.clone()
        short[2] = 20  # a run of 50 tokens at the end of 20: the first 30 are before the sequence
        out.fill_(9.0)
        ops.attention_prefill_e4m3(q.cuda(), out, 2, 1, heads, kv, dim, step.cu_q.cuda(), short.cuda(), step.tables.cuda(), *pools, ps, None,
                                   0.125, partial, nsplit)
        assert (out[:2] == 9).all() and (out[2:32] == 0).all() and out.isfinite().all()
        # no sequences, no rows
        ops.attention_prefill_e4m3(q.cuda(), out, 2, 0, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps,
                                   None, 0.125, partial, nsplit)
        ops.attention_decode_e4m3(q.cuda(), out, 0, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.125,
                                  partial, nsplit)


def test_a_nan_in_a_key_reaches_the_rows_that_read_it_and_no_others(ops):
    form = heads, kv, dim, ps = 4, 2, 64, 16
    step = plain.Step([40, 45, 100], [1, 1, 40], ps, seed=5)
    pools, keys, values, q = setup(step, form)
    k = pools[0].view(torch.uint8)
    k[step.tables[0, 1].long(), 1, :, 3] = 0x7f  # key 19 of sequence 0, head 1
    k[step.tables[2, 7].long(), 0, :, 8] = 0x7f  # key 120 of sequence 2, head 0
    out = torch.zeros(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    ops.attention_decode_e4m3(q.cuda(), out, 2, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.125)
    ops.attention_prefill_e4m3(q.cuda(), out, 2, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps,
                               None, 0.125)
    bad = out.cpu().view(step.n, heads, dim).isnan()
    want = torch.zeros(step.n, heads, dtype=torch.bool)
    want[0, 2:] = True
    want[2 + 20:, :2] = True
    assert torch.equal(bad.any(-1), want) and torch.equal(bad.all(-1), want)


def test_offsets_beyond_32_bits(ops):
    """Pages whose codes begin past 2^32 bytes in the pools."""
    form = heads, kv, dim, ps = 28, 4, 128, 16
    step = plain.Step([70, 30], [1, 40], ps, seed=6, spare=0)
    pages = (1 << 32) // (kv * dim * ps) + 50
    small = plain.Step([70, 30], [1, 40], ps, seed=6, spare=0)
    (k, v, s), keys, values, q = setup(small, form)
    far = pages - step.pages  # page p of the small pools lies at far + p
    big_k = torch.empty(pages, *k.shape[1:], dtype=torch.uint8, device="cuda")
    big_v = torch.empty(pages, *v.shape[1:], dtype=torch.uint8, device="cuda")
    big_s = torch.empty(pages, *s.shape[1:], dtype=torch.uint8, device="cuda")
    big_k[far:], big_v[far:], big_s[far:] = k.view(torch.uint8), v.view(torch.uint8), s
    pools = (big_k.view(plain.E4M3), big_v.view(plain.E4M3), big_s)
    tables = torch.where(step.tables >= 0, step.tables + far, step.tables).to(torch.int32).cuda()
    out = torch.zeros(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    ops.attention_decode_e4m3(q.cuda(), out, 1, heads, kv, dim, step.positions.cuda(), tables, *pools, ps, None, dim ** -0.5)
    ops.attention_prefill_e4m3(q.cuda(), out, 1, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), tables, *pools, ps, None, dim ** -0.5)
    check(step, form, out, q, keys, values, None, None)
    out.zero_()
    ops.attention_e4m3(q.cuda(), out, heads, kv, dim, step.positions.cuda(), step.token_seq.cuda(), tables, *pools, ps, None, dim ** -0.5)
    check(step, form, out, q, keys, values, None, None)
    # written and read there too
    qkv = torch.randn(step.n, (heads + 2 * kv) * dim, generator=step.gen).bfloat16().cuda()
    ops.rope_kv_store_e4m3(qkv, heads, kv, dim, 0, None, step.positions.cuda(), step.token_seq.cuda(), tables, *pools, ps)
    got = [torch.empty(step.n, kv * dim, device="cuda") for _ in range(2)]
    ops.kv_read_e4m3(*got, kv, dim, step.positions.cuda(), step.token_seq.cuda(), tables, *pools, ps)
    rows = qkv.cpu().double().view(step.n, heads + 2 * kv, dim)
    for have, base in zip(got, (heads, heads + kv)):
        assert torch.equal(have.cpu().double().view(step.n, kv, dim), plain.quantised(rows[:, base:base + kv])[0])


def test_refusals_of_the_matrix_kernels(ops):
    from shrike_amd.kernels.lib import KernelError

    form = heads, kv, dim, ps = 14, 2, 64, 16
    step = plain.Step([40, 20], [1, 9], ps, seed=7)
    pools, _, _, q = setup(step, form)
    q, out = q.cuda(), torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    single = (step.positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.1)
    runs = (step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps, None, 0.1)
    with pytest.raises(KernelError, match="scratch"):
        ops.attention_decode_e4m3(q, out, 1, heads, kv, dim, *single, None, 2)
    with pytest.raises(KernelError, match="scratch"):
        ops.attention_prefill_e4m3(q, out, 1, 1, heads, kv, dim, *runs, torch.empty(5, device="cuda"), 2)
    with pytest.raises(KernelError, match="shares"):
        ops.attention_decode_e4m3(q, out, 1, heads, kv, dim, *single, torch.empty(100000, device="cuda"), 65)
    with pytest.raises(KernelError, match="bfloat16"):
        ops.attention_decode_e4m3(q.float(), out.float(), 1, heads, kv, dim, *single)
    with pytest.raises(KernelError, match="fewer rows"):
        ops.attention_decode_e4m3(q, out, 11, heads, kv, dim, *single)
    with pytest.raises(KernelError, match="tables of"):
        ops.attention_decode_e4m3(q, out, 3, heads, kv, dim, *single)
    with pytest.raises(KernelError, match="aligned"):
        shifted = torch.empty(step.n * heads * dim + 1, dtype=torch.bfloat16, device="cuda")[1:].view(step.n, -1)
        ops.attention_decode_e4m3(shifted, out, 1, heads, kv, dim, *single)
    with pytest.raises(KernelError, match="cu_q|rows"):
        ops.attention_prefill_e4m3(q, out, 1, 5, heads, kv, dim, *runs)
    with pytest.raises(KernelError, match="scale must be positive"):
        ops.attention_prefill_e4m3(q, out, 1, 1, heads, kv, dim, *runs[:-1], 0.0)
    assert not ops.attention_e4m3_supports_mfma(14, 2, 80, 16, 14 * 80)
    assert not ops.attention_e4m3_supports_mfma(14, 2, 64, 8, 14 * 64)
    assert not ops.attention_e4m3_supports_mfma(129, 1, 64, 16, 129 * 64)
    assert not ops.attention_e4m3_supports_mfma(14, 2, 64, 16, 14 * 64 + 4)


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16), (8, 1, 256, 32)])
@pytest.mark.parametrize("nsplit", [1, 2, 5])
def test_rows_that_belong_to_no_sequence_stay(ops, form, nsplit):
    """A batch padded at its end, and one whose last sequences are not asked for."""
    heads, kv, dim, ps = form
    step = plain.Step([0, 70, 200, 5], [1, 40, 33, 20], ps, seed=8)
    pools, keys, values, q = setup(step, form)
    padded = torch.cat([q, torch.randn(37, heads * dim, generator=step.gen).bfloat16()]).cuda()
    partial = torch.empty(padded.shape[0] * heads * nsplit * (dim + 2), device="cuda")
    for count, rows in ((3, step.n), (2, step.n - 20), (1, 41)):
        out = torch.full((step.n + 37, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
        partial.fill_(float("nan"))
        ops.attention_prefill_e4m3(padded, out, 1, count, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools,
                                   ps, None, dim ** -0.5, partial, nsplit)
        assert (out[:1] == 9).all() and (out[rows:] == 9).all()
        check(step, form, out[:step.n], q, keys, values, None, None, slice(1, rows))


@pytest.mark.parametrize("form", [(4, 2, 64, 16), (6, 2, 128, 32), (4, 2, 96, 16), (4, 2, 256, 16)])
@pytest.mark.parametrize("window, chunk", [(None, None), (30, None), (None, 70)])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_a_nan_in_a_value_reaches_the_rows_that_read_it_and_no_others(ops, form, window, chunk, nsplit):
    """Also where a neighbouring query of the same workgroup reads it."""
    heads, kv, dim, ps = form
    step = plain.Step([40, 45, 100], [1, 1, 150], ps, seed=9)
    pools, keys, values, q = setup(step, form)
    v = pools[1].view(torch.uint8)
    at = {0: 40, 1: 20, 2: 137}
    for seq, key in at.items():
        v[step.tables[seq, key // ps].long(), seq % 2, :, key % ps] = 0x7f if seq else 0xff
        values[step.tables[seq, key // ps].long(), seq % 2, key % ps] = 0.0
    partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
    out = torch.zeros(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    where = (step.tables.cuda(), *pools, ps, window, dim ** -0.5)
    ops.attention_decode_e4m3(q.cuda(), out, 2, heads, kv, dim, step.positions.cuda(), *where, partial, nsplit, chunk=chunk)
    ops.attention_prefill_e4m3(q.cuda(), out, 2, 1, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), *where, partial, nsplit, chunk=chunk)
    want = torch.zeros(step.n, heads, dtype=torch.bool)
    for t in range(step.n):
        seq, pos = int(step.token_seq[t]), int(step.positions[t])
        key = at[seq]
        if key <= pos and (not window or pos - key < window) and (not chunk or key // chunk == pos // chunk):
            want[t, seq % 2 * heads // 2:(seq % 2 + 1) * heads // 2] = True
    bad = out.cpu().view(step.n, heads, dim).isnan()
    assert torch.equal(bad.any(-1), want) and torch.equal(bad.all(-1), want)
    clean = torch.where(bad, 0.0, out.cpu().float().view(step.n, heads, dim)).bfloat16().view(step.n, -1)
    want_off, size, reach = plain.attention(step, q, keys, values, heads, dim ** -0.5, window, chunk)
    off = (clean.double().view_as(want_off) - want_off).abs()
    limit = plain.allowed(want_off, size, reach, dim, 250, True)
    assert (off <= limit)[~want].all()
    general = torch.empty_like(out)
    ops.attention_e4m3(q.cuda(), general, heads, kv, dim, step.positions.cuda(), step.token_seq.cuda(), *where, chunk=chunk)
    assert torch.equal(general.cpu().view(step.n, heads, dim).isnan().any(-1), want)


def test_refusals_of_what_is_not_aligned(ops):
    from shrike_amd.kernels.lib import KernelError

    form = heads, kv, dim, ps = 14, 2, 64, 16
    step = plain.Step([40, 20], [1, 9], ps, seed=10)
    pools, _, _, q = setup(step, form)
    q = q.cuda()
    scratch = torch.empty(step.n * heads * 2 * (dim + 2) + 1, device="cuda")
    shifted = torch.empty(step.n * heads * dim + 1, dtype=torch.bfloat16, device="cuda")[1:].view(step.n, -1)
    out = torch.empty(step.n, heads * dim, dtype=torch.bfloat16, device="cuda")
    single = (step.positions.cuda(), step.tables.cuda(), *pools, ps, None, 0.1)
    runs = (step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(), *pools, ps, None, 0.1)
    for args in ((shifted, scratch[:-1]), (out, scratch[1:])):
        with pytest.raises(KernelError, match="aligned"):
            ops.attention_decode_e4m3(q, args[0], 1, heads, kv, dim, *single, args[1], 2)
        with pytest.raises(KernelError, match="aligned"):
            ops.attention_prefill_e4m3(q, args[0], 1, 1, heads, kv, dim, *runs, args[1], 2)


@pytest.mark.parametrize("news", [[1] * 70, [300, 1, 129, 2], [128] * 9])
@pytest.mark.parametrize("form", [(64, 1, 32, 16), (128, 1, 32, 16), (3, 1, 64, 16), (2, 2, 64, 16)])
def test_runs_of_queries_of_every_length(ops, form, news):
    """Groups that do not divide 128, runs of one query, sequences that end inside a run and with it."""
    heads, kv, dim, ps = form
    step = plain.Step([(37 * i) % 90 for i in range(len(news))], news, ps, seed=11)
    pools, keys, values, q = setup(step, form)
    for nsplit in (1, 3):
        out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
        partial = torch.empty(step.n * heads * nsplit * (dim + 2), device="cuda")
        ops.attention_prefill_e4m3(q.cuda(), out, 0, len(news), heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda(),
                                   *pools, ps, None, dim ** -0.5, partial, nsplit)
        check(step, form, out, q, keys, values, None, None)


def test_more_runs_than_a_grid_is_deep(ops):
    """70,000 runs of one query: the same bits as in two calls."""
    form = heads, kv, dim, ps = 128, 1, 32, 16
    step = plain.Step([0] * 700, [100] * 700, ps, seed=12)
    k_pool, v_pool, scales, _, _ = plain.random_pools(step.pages, kv, dim, ps, step.gen)
    pools = (k_pool.cuda(), v_pool.cuda(), scales.cuda())
    q = torch.randn(step.n, heads * dim, device="cuda").bfloat16()
    cu_q, ctx_lens, tables = step.cu_q.cuda(), step.ctx_lens.cuda(), step.tables.cuda()
    whole, halves = (torch.full_like(q, 9.0) for _ in range(2))
    ops.attention_prefill_e4m3(q, whole, 0, 700, heads, kv, dim, cu_q, ctx_lens, tables, *pools, ps, None, dim ** -0.5)
    for first in (0, 350):
        rows = slice(100 * first, 100 * first + 35000)
        ops.attention_prefill_e4m3(q[rows], halves[rows], 0, 350, heads, kv, dim, cu_q[:351], ctx_lens[first:first + 350],
                                   tables[first:first + 350], *pools, ps, None, dim ** -0.5)
    assert whole.isfinite().all() and torch.equal(whole, halves) and not (whole == 9.0).all(1).any()
