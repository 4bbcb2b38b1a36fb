"""Writing the quantised cache, reading it back, and attention over it in the kernel for any sizes, against 64 bits."""

import math

import pytest
import torch

from . import e4m3_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from shrike_amd.kernels import ops

    return ops


def empty_pools(ops, pages, kv, dim, ps, fill=0x55):
    """Pools and scales with every byte `fill`."""
    k = torch.full(ops.key_pool_shape(pages, kv, ps, dim), fill, dtype=torch.uint8, device="cuda").view(plain.E4M3)
    v = torch.full((pages, kv, dim, ps), fill, dtype=torch.uint8, device="cuda").view(plain.E4M3)
    return k, v, torch.full(ops.e4m3_scales_shape(pages, kv, ps), fill, dtype=torch.uint8, device="cuda")


def read(ops, step, pools, kv, dim, dtype=torch.float32):
    k, v = (torch.empty(step.n, kv * dim, dtype=dtype, device="cuda") for _ in range(2))
    ops.kv_read_e4m3(k, v, kv, dim, step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(), *pools, step.ps)
    return k.cpu().double().view(step.n, kv, dim), v.cpu().double().view(step.n, kv, dim)


def inv_freqs(rot):
    return (1e4 ** (-torch.arange(0, max(rot, 2), 2, dtype=torch.float64) / max(rot, 2))).float()[: rot // 2]


FORMS = [
    # heads, kv heads, head size, rotated, page size
    (14, 2, 64, 64, 16), (28, 4, 128, 128, 16), (6, 3, 32, 32, 64), (24, 8, 96, 96, 32), (4, 1, 256, 256, 16),
    (4, 4, 80, 80, 4), (3, 1, 17, 16, 5), (5, 5, 48, 20, 16), (2, 2, 128, 0, 16), (8, 1, 160, 64, 48), (1, 1, 1, 0, 1),
]
STEPS = [([0], [1]), ([5, 0, 31], [1, 1, 1]), ([16], [40]), ([3, 40, 0, 7], [1, 33, 16, 95]), ([37], [130]), ([15990], [25])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("starts, news", STEPS)
def test_rows_come_back_as_the_nearest_codes(ops, form, starts, news, dtype):
    heads, kv, dim, rot, ps = form
    step = plain.Step(starts, news, ps, seed=dim)
    x = torch.randn(step.n, (heads + 2 * kv) * dim, generator=step.gen) * torch.exp(torch.randn(step.n, 1, generator=step.gen))
    x = x.to(dtype)
    freq = inv_freqs(rot)
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    qkv = x.cuda()
    ops.rope_kv_store_e4m3(qkv, heads, kv, dim, rot, freq.cuda(), step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(),
                           *pools, ps)
    rows = x.double().view(step.n, heads + 2 * kv, dim)
    turned = plain.rotate(rows[:, : heads + kv], step.positions, freq, rot)
    # a rotated element is two products and a sum in float32 of cosines good to 2^-22
    slack = 2.0 ** -20 * turned.abs().amax(-1, keepdim=True) + 2.0 ** -20 * rows[:, : heads + kv].abs().amax(-1, keepdim=True)
    got_q = qkv.cpu().double().view(step.n, heads + 2 * kv, dim)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    assert ((got_q[:, :heads] - turned[:, :heads]).abs() <= half * turned[:, :heads].abs() + slack[:, :heads]).all()
    assert torch.equal(got_q[:, heads:], rows[:, heads:])  # the other columns stay
    k, v = read(ops, step, pools, kv, dim)
    assert torch.equal(v, plain.quantised(rows[:, heads + kv:])[0])  # values are not rotated: every bit
    want = turned[:, heads:]
    unit = 2.0 ** plain.exponents(want).double()[..., None]
    border = (want.abs().amax(-1, keepdim=True) / (448 * unit) - 1).abs() < 1e-5  # (the other power of two there)
    limit = plain.half_step(want / unit) * unit * torch.where(border, 2.0, 1.0) + slack[:, heads:]
    assert ((k - want).abs() <= limit).all()
    if rot == 0:
        assert torch.equal(k, plain.quantised(want)[0])
    kb, vb = read(ops, step, pools, kv, dim, torch.bfloat16)  # bfloat16 holds the values exactly
    assert torch.equal(kb, k) and torch.equal(vb, v)
    # pages that belong to nobody are as they were
    for t in pools:
        assert (t.view(torch.uint8)[step.free.cuda()] == 0x55).all()


@pytest.mark.parametrize("adjacent, v_from_k, splits, magnitude", [(True, False, 0, 1.0), (False, True, 0, 1.0), (True, True, 3, 1.0),
                                                                  (False, False, 2, 1.25), (False, False, 9, 1.0)])
@pytest.mark.parametrize("news", [[1, 1, 1], [150, 1]])
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_ways_of_rotating_and_of_getting_the_projections(ops, adjacent, v_from_k, splits, magnitude, news, dim):
    heads, kv, ps = 6, 2, 16
    step = plain.Step([20 + i for i in range(len(news))], news, ps, seed=splits)
    width = (heads + (1 if v_from_k else 2) * kv) * dim
    freq = inv_freqs(dim)
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    qkv = torch.zeros(step.n, width, dtype=torch.bfloat16)
    sums = None
    if splits:
        parts = torch.randn(splits, step.n, width, generator=step.gen)
        bias = torch.randn(width, generator=step.gen)
        x = parts.double().sum(0) + bias.double()
        sums = ops.SplitSum(parts.cuda(), bias.cuda())
    else:
        qkv = torch.randn(step.n, width, generator=step.gen).bfloat16()
        x = qkv.double()
    q_out = torch.full((step.n, heads * dim + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    given = qkv.cuda()
    ops.rope_kv_store_e4m3(given, heads, kv, dim, dim, freq.cuda(), step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(),
                           *pools, ps, split_sum=sums, adjacent_pairs=adjacent, values_from_keys=v_from_k, magnitude=magnitude,
                           q_out=q_out[:, : heads * dim])
    assert torch.equal(given.cpu(), qkv) and (q_out[:, heads * dim:] == 7).all()
    rows = x.view(step.n, -1, dim)
    turned = plain.rotate(rows[:, : heads + kv], step.positions, freq, dim, adjacent, magnitude)
    slack = (2.0 ** -20 + splits * 2.0 ** -23) * (rows.abs().amax() + turned.abs().amax())
    got = q_out[:, : heads * dim].cpu().double().view(step.n, heads, dim)
    assert ((got - turned[:, :heads]).abs() <= 2.0 ** -8 * turned[:, :heads].abs() + slack).all()
    k, v = read(ops, step, pools, kv, dim)
    for have, want in ((k, turned[:, heads:]), (v, rows[:, heads:heads + kv] if v_from_k else rows[:, heads + kv:])):
        unit = 2.0 ** plain.exponents(want).double()[..., None]
        border = (want.abs().amax(-1, keepdim=True) / (448 * unit) - 1).abs() < 1e-5
        limit = plain.half_step(want / unit) * unit * torch.where(border, 2.0, 1.0) + slack
        assert ((have - want).abs() <= limit).all()


@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_zeros_of_extreme_sizes_and_with_infinities(ops, dtype, n):
    kv, dim, ps = 8, 64, 16
    step = plain.Step([3], [n], ps)
    x = torch.randn(n, 3 * kv, dim, generator=step.gen)
    x[:, kv:] = torch.randn(1, 2 * kv, dim, generator=step.gen)
    big = float(torch.finfo(dtype).max)
    for base in (kv, 2 * kv):  # keys (not rotated here) and values alike
        x[:, base] = 0.0
        x[:, base + 1] *= 1e-41  # below the smallest unit: zeros or its smallest codes
        x[:, base + 2, 5] = math.inf
        x[:, base + 3, 9] = math.nan
        x[:, base + 4, 0] = big
        x[:, base + 5] *= 2.0 ** 100
        x[:, base + 6] = 448.0
        x[:, base + 7, 3] = 448.0 * 2 ** 10 * (1 + 2.0 ** -7)  # just beyond a power of two's range
    x = x.to(dtype)
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    qkv = x.view(n, -1).cuda()
    ops.rope_kv_store_e4m3(qkv, kv, kv, dim, 0, None, step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(), *pools, ps)
    k, v = read(ops, step, pools, kv, dim)
    for got, want in ((k, x[:, kv:2 * kv].double()), (v, x[:, 2 * kv:].double())):
        assert got[:, 2].isnan().all() and got[:, 3].isnan().all()
        fine = [0, 1, 4, 5, 6, 7]
        assert torch.equal(got[:, fine], plain.quantised(want[:, fine])[0])
        assert got[:, fine].isfinite().all()


def test_tokens_that_are_not_there(ops):
    heads, kv, dim, ps = 4, 2, 64, 16
    step = plain.Step([0, 5], [30, 9], ps)
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    before = [t.clone() for t in pools]
    qkv = torch.randn(step.n, (heads + 2 * kv) * dim, generator=step.gen).bfloat16().cuda()
    freq = inv_freqs(dim).cuda()
    positions = torch.full((step.n,), -1, dtype=torch.int32, device="cuda")
    ops.rope_kv_store_e4m3(qkv, heads, kv, dim, dim, freq, positions, step.token_seq.cuda(), step.tables.cuda(), *pools, ps)
    for entry in (-1, step.pages, 2 ** 31 - 1):  # an id outside the pool is never followed
        bad = torch.full_like(step.tables, entry).cuda()
        ops.rope_kv_store_e4m3(qkv, heads, kv, dim, dim, freq, step.positions.cuda(), step.token_seq.cuda(), bad, *pools, ps)
    beyond = torch.full((step.n,), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    ops.rope_kv_store_e4m3(qkv, heads, kv, dim, dim, freq, beyond, step.token_seq.cuda(), step.tables.cuda(), *pools, ps)
    strange = torch.full((step.n,), 2, dtype=torch.int32, device="cuda")  # there are two sequences
    ops.rope_kv_store_e4m3(qkv, heads, kv, dim, dim, freq, step.positions.cuda(), strange, step.tables.cuda(), *pools, ps)
    for t, b in zip(pools, before):
        assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))
    k, v = (torch.zeros(step.n, kv * dim, device="cuda") for _ in range(2))
    ops.kv_read_e4m3(k, v, kv, dim, positions, step.token_seq.cuda(), step.tables.cuda(), *pools, ps)
    assert k.isnan().all() and v.isnan().all()
    q = torch.randn(step.n, heads * dim, generator=step.gen).cuda()
    out = torch.full_like(q, 3.0)
    ops.attention_e4m3(q, out, heads, kv, dim, positions, step.token_seq.cuda(), step.tables.cuda(), *pools, ps, None, 0.1)
    assert (out == 0).all()  # no key to read
    out.fill_(3.0)
    ops.attention_e4m3(q, out, heads, kv, dim, step.positions.cuda(), step.token_seq.cuda(),
                       torch.full_like(step.tables, step.pages).cuda(), *pools, ps, None, 0.1)
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", [(14, 2, 64, 16), (4, 4, 80, 4), (3, 1, 17, 5), (40, 1, 128, 32), (4, 2, 256, 16), (2, 1, 1, 3)])
@pytest.mark.parametrize("starts, news, window, chunk", [([0], [1], None, None), ([300, 0, 700], [1, 1, 1], None, None),
                                                        ([40, 3, 0], [1, 30, 18], None, None), ([600], [20], 100, None),
                                                        ([500, 30], [9, 40], None, 64), ([500], [3], 1, None), ([90], [60], 50, 32)])
def test_attention_of_any_sizes(ops, form, starts, news, window, chunk, dtype):
    heads, kv, dim, ps = form
    step = plain.Step(starts, news, ps, seed=dim + heads)
    k_pool, v_pool, scales, keys, values = plain.random_pools(step.pages, kv, dim, ps, step.gen)
    k_pool.view(torch.uint8)[step.free] = 0x7f  # pages that belong to nobody hold NaN
    v_pool.view(torch.uint8)[step.free] = 0x7f
    q = (2 * torch.randn(step.n, heads * dim + 8, generator=step.gen)).to(dtype)
    out = torch.empty(step.n, heads * dim, dtype=dtype, device="cuda")
    scale = dim ** -0.5
    ops.attention_e4m3(q.cuda()[:, : heads * dim], out, heads, kv, dim, step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(),
                       k_pool.cuda(), v_pool.cuda(), scales.cuda(), ps, window, scale, chunk=chunk)
    want, size, reach = plain.attention(step, q[:, : heads * dim], keys, values, heads, scale, window, chunk)
    limit = plain.allowed(want, size, reach, dim, max(step.ctx_lens.tolist()), dtype == torch.bfloat16)
    assert ((out.cpu().double().view_as(want) - want).abs() <= limit).all()


def test_refusals_of_the_faces(ops):
    from shrike_amd.kernels.lib import KernelError

    step = plain.Step([0], [8], 16)
    kv, dim, ps = 2, 64, 16
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    where = (step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda())
    q = torch.zeros(step.n, 4 * dim, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    k = torch.zeros(step.n, kv * dim, device="cuda")
    with pytest.raises(KernelError, match="float8_e4m3fn"):
        ops.kv_read_e4m3(k, k, kv, dim, *where, pools[0].view(torch.uint8), *pools[1:], ps)
    with pytest.raises(KernelError, match="key pool"):
        ops.kv_read_e4m3(k, k, kv, dim, *where, *pools, 32)
    with pytest.raises(KernelError, match="scales"):
        ops.kv_read_e4m3(k, k, kv, dim, *where, *pools[:2], pools[2][:, :, :1].contiguous(), ps)
    with pytest.raises(KernelError, match="k_out and v_out"):
        ops.kv_read_e4m3(k[:, 1:], k[:, 1:], kv, dim, *where, *pools, ps)
    with pytest.raises(KernelError, match="rows"):
        ops.kv_read_e4m3(k, k, kv, dim, where[0][:3], *where[1:], *pools, ps)
    with pytest.raises(KernelError, match="scale must be positive"):
        ops.attention_e4m3(q, out, 4, kv, dim, *where, *pools, ps, None, -0.1)
    with pytest.raises(KernelError, match="multiple of kv_heads"):
        ops.attention_e4m3(q[:, : 3 * dim], out[:, : 3 * dim].contiguous(), 3, kv, dim, *where, *pools, ps, None, 0.1)
    with pytest.raises(KernelError, match="out must be"):
        ops.attention_e4m3(q, out[:, ::2], 4, kv, dim, *where, *pools, ps, None, 0.1)
    with pytest.raises(KernelError, match="qkv must be"):
        ops.rope_kv_store_e4m3(q, 4, kv, dim, dim, inv_freqs(dim).cuda(), *where, *pools, ps)
    qkv = torch.zeros(step.n, 8 * dim, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KernelError, match="frequencies"):
        ops.rope_kv_store_e4m3(qkv, 4, kv, dim, dim, inv_freqs(dim)[:-1].cuda(), *where, *pools, ps)
    with pytest.raises(KernelError, match="q_out"):
        ops.rope_kv_store_e4m3(qkv, 4, kv, dim, dim, inv_freqs(dim).cuda(), *where, *pools, ps, q_out=out.float())
