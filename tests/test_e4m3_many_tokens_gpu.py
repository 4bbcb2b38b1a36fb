"""Writing the quantised cache for so many tokens and heads that rows travel in vectors (more wavefronts than the chip holds, one a head)."""

import pytest
import torch

from . import e4m3_plain as plain
from .test_e4m3_cache_gpu import empty_pools, inv_freqs, read
from .test_e4m3_cache_gpu import test_rows_come_back_as_the_nearest_codes as rows_come_back

pytestmark = pytest.mark.gpu

WAVES = 256 * 32


@pytest.fixture(scope="module")
def ops():
    from shrike_amd.kernels import ops

    return ops


def waves(tokens, heads, kv, dim):
    return tokens * (heads + 2 * kv) * -(-dim // 128)


FORMS = [(14, 2, 64, 64, 16), (28, 4, 128, 128, 16), (40, 40, 32, 32, 64), (24, 8, 96, 96, 32), (24, 8, 160, 160, 16), (20, 4, 256, 256, 48),
         (28, 4, 128, 128, 5), (28, 4, 128, 128, 4), (16, 16, 128, 128, 12)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("starts, news", [([37], [600]), ([3, 40, 0, 7, 64], [1, 333, 16, 120, 64]), ([0] * 40, [11 + i % 7 for i in range(40)])])
def test_rows(ops, form, starts, news):
    heads, kv, dim, rot, _ = form
    assert waves(sum(news), heads, kv, dim) > WAVES
    rows_come_back(ops, form, starts, news, torch.bfloat16)


@pytest.mark.parametrize("splits, magnitude", [(2, 1.25), (9, 1.0)])
@pytest.mark.parametrize("news", [[300], [150, 1, 149]])
@pytest.mark.parametrize("dim", [64, 128])
def test_parts_of_a_product(ops, splits, magnitude, news, dim):
    heads, kv, ps = 24, 3, 16
    step = plain.Step([20 + i for i in range(len(news))], news, ps, seed=splits)
    assert waves(step.n, heads, kv, dim) > WAVES
    width = (heads + 2 * kv) * dim
    freq = inv_freqs(dim)
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    parts, bias = torch.randn(splits, step.n, width, generator=step.gen), torch.randn(width, generator=step.gen)
    q_out = torch.full((step.n, heads * dim + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    given = torch.zeros(step.n, width, dtype=torch.bfloat16, device="cuda")
    ops.rope_kv_store_e4m3(given, heads, kv, dim, dim, freq.cuda(), step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(), *pools,
                           ps, split_sum=ops.SplitSum(parts.cuda(), bias.cuda()), magnitude=magnitude, q_out=q_out[:, : heads * dim])
    assert (given == 0).all() and (q_out[:, heads * dim:] == 7).all()
    rows = (parts.double().sum(0) + bias.double()).view(step.n, -1, dim)
    turned = plain.rotate(rows[:, : heads + kv], step.positions, freq, dim, False, magnitude)
    # (as for few tokens: two products and a sum of cosines good to 2^-22, sums of the parts)
    slack = (2.0 ** -20 + splits * 2.0 ** -23) * (rows.abs().amax() + turned.abs().amax())
    got = q_out[:, : heads * dim].cpu().double().view(step.n, heads, dim)
    assert ((got - turned[:, :heads]).abs() <= 2.0 ** -8 * turned[:, :heads].abs() + slack).all()
    k, v = read(ops, step, pools, kv, dim)
    for have, want in ((k, turned[:, heads:]), (v, rows[:, heads + kv:])):
        unit = 2.0 ** plain.exponents(want).double()[..., None]
        border = (want.abs().amax(-1, keepdim=True) / (448 * unit) - 1).abs() < 1e-5
        assert ((have - want).abs() <= plain.half_step(want / unit) * unit * torch.where(border, 2.0, 1.0) + slack).all()


def test_rows_of_extreme_sizes_and_tokens_that_are_not_there(ops):
    heads, kv, dim, ps, n = 8, 8, 64, 16, 400
    step = plain.Step([3], [n], ps)
    assert waves(n, heads, kv, dim) > WAVES
    x = torch.randn(n, 3 * kv, dim, generator=step.gen)
    big = float(torch.finfo(torch.bfloat16).max)
    for base in (kv, 2 * kv):
        x[:, base] = 0.0
        x[:, base + 1] *= 1e-41
        x[:, base + 2, 5] = float("inf")
        x[:, base + 3, 9] = float("nan")
        x[:, base + 4, 0] = big
        x[:, base + 5] *= 2.0 ** 100
    x = x.bfloat16()
    positions, still = step.positions.clone(), torch.full((dim // 2,), 0.0)  # rates of 0: nothing turns
    gone = torch.arange(n) % 5 == 3
    positions[gone] = -1
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    ops.rope_kv_store_e4m3(x.view(n, -1).cuda(), heads, kv, dim, dim, still.cuda(), positions.cuda(), step.token_seq.cuda(), step.tables.cuda(),
                           *pools, ps)
    k, v = read(ops, step, pools, kv, dim)
    at = torch.arange(n) + 3
    page, slot = step.tables[0].long()[at // ps], at % ps
    for got, want in ((k, x[:, kv:2 * kv].double()), (v, x[:, 2 * kv:].double())):
        assert got[~gone][:, 2:4].isnan().all()
        fine = [0, 1, 4, 5, 6, 7]
        assert torch.equal(got[~gone][:, fine], plain.quantised(want[:, fine])[0][~gone])
    # a token that is not there leaves its slots alone
    for t in (pools[0].view(torch.uint8).transpose(2, 3), pools[1].view(torch.uint8).transpose(2, 3)):
        assert (t.cpu()[page[gone], :, slot[gone]] == 0x55).all()
    assert (pools[2].cpu()[page[gone], :, :, slot[gone]] == 0x55).all()


@pytest.mark.parametrize("ps", [16, 8, 7])
def test_runs_of_every_length(ops, ps):
    """Blocks of 16 neighbouring tokens of a step whose slots are neighbours, or not, in every way."""
    heads, kv, dim = 24, 4, 64
    gen = torch.Generator().manual_seed(ps)
    # 40 sequences of 1 .. 20 tokens, each from another slot on
    news = [1 + i % 20 for i in range(40)]
    starts = [int(torch.randint(0, 40, (1,), generator=gen)) for _ in news]
    step = plain.Step(starts, news, ps, seed=ps)
    assert waves(step.n, heads, kv, dim) > WAVES
    x = torch.randn(step.n, (heads + 2 * kv) * dim, generator=gen).bfloat16()
    pools = empty_pools(ops, step.pages, kv, dim, ps)
    # tokens in any order too
    for order in (torch.arange(step.n), torch.arange(step.n).flip(0), torch.randperm(step.n, generator=gen)):
        pools = empty_pools(ops, step.pages, kv, dim, ps)
        ops.rope_kv_store_e4m3(x[order].cuda(), heads, kv, dim, dim, inv_freqs(dim).cuda(), step.positions[order].cuda(), step.token_seq[order].cuda(),
                               step.tables.cuda(), *pools, ps)
        _, v = read(ops, step, pools, kv, dim)
        assert torch.equal(v, plain.quantised(x.double().view(step.n, -1, dim)[:, heads + kv:])[0])
