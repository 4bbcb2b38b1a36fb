"""Attention over a quantised cache with pages of thousands of tokens, at positions whose page a quotient by 2^32 / page_size misses."""

import pytest
import torch

from . import e4m3_plain as plain

pytestmark = pytest.mark.gpu


def rounded_up(page, x):
    """x / page as the product with ceil(2^32 / page) has it."""
    return x * -(-2 ** 32 // page) >> 32


@pytest.mark.parametrize("page, last", [(32752, 163759), (65520, 131039), (16384, 163839)])
@pytest.mark.parametrize("window", [None, 100])
def test_the_last_token_of_a_page(page, last, window):
    from shrike_amd.kernels import ops

    assert last % page == page - 1 and (rounded_up(page, last) != last // page or page == 16384)
    heads, kv, dim = 2, 1, 32
    # single tokens at the page's last slot and the next one's first, portions that end there
    starts, news = [last, last + 1, last - 19, last - 40], [1, 1, 20, 70]
    step = plain.Step(starts, news, page, seed=page, spare=0)
    gen = torch.Generator().manual_seed(page)
    # codes as bytes, of which none is a NaN; powers of two around 1
    shapes = (step.pages, kv, dim // 32, page, 32), (step.pages, kv, dim, page)
    k, v = (torch.randint(0, 127, s, generator=gen, dtype=torch.uint8) | torch.randint(0, 2, s, generator=gen, dtype=torch.uint8) << 7 for s in shapes)
    scales = torch.randint(119, 122, (step.pages, kv, 2, page), generator=gen, dtype=torch.uint8)
    unit = torch.ldexp(torch.ones(1, dtype=torch.float64), scales.int() - 127)
    keys = k.view(plain.E4M3).double()[:, :, 0] * unit[:, :, 0, :, None]
    values = v.view(plain.E4M3).double().transpose(2, 3) * unit[:, :, 1, :, None]
    q = torch.randn(step.n, heads * dim, generator=gen).bfloat16()
    out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    pools = (k.view(plain.E4M3).cuda(), v.view(plain.E4M3).cuda(), scales.cuda())
    tables, positions = step.tables.cuda(), step.positions.cuda()
    want, size, reach = plain.attention(step, q, keys, values, heads, dim ** -0.5, window)
    limit = plain.allowed(want, size, reach, dim, min(window or last + 100, last + 100), True)
    for nsplit in (1, 7):
        partial = torch.full((step.n * heads * nsplit * (dim + 2),), float("nan"), device="cuda")
        ops.attention_decode_e4m3(q.cuda(), out, 2, heads, kv, dim, positions, tables, *pools, page, window, dim ** -0.5, partial, nsplit)
        ops.attention_prefill_e4m3(q.cuda(), out, 2, 2, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(), tables, *pools, page, window,
                                   dim ** -0.5, partial, nsplit)
        assert ((out.cpu().double().view_as(want) - want).abs() <= limit).all()
