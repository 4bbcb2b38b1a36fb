"""Attention over a quantised cache where scores are so large that one key has all the weight, or the scale is as far from 1 as the
kernels take: results are finite, and the value of the largest score."""

import pytest
import torch

from . import e4m3_plain as plain
from .test_e4m3_attention_gpu import setup

pytestmark = pytest.mark.gpu

STARTS, NEWS, SINGLES = [150, 700, 333, 90], [1, 1, 40, 70], 2


def both(form, step, pools, q, scale, nsplit):
    """Results of the step's single tokens and portions [n, heads, dim], on the CPU."""
    from shrike_amd.kernels import ops

    heads, kv, dim, ps = form
    out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    partial = torch.full((step.n * heads * nsplit * (dim + 2),), float("nan"), device="cuda")
    ops.attention_decode_e4m3(q.cuda(), out, SINGLES, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, None, scale,
                              partial, nsplit)
    ops.attention_prefill_e4m3(q.cuda(), out, SINGLES, len(STARTS) - SINGLES, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(),
                               step.tables.cuda(), *pools, ps, None, scale, partial, nsplit)
    return out.cpu().double().view(step.n, heads, dim)


def the_largest_score_s_value(form, step, got, keys, values, q, scale):
    heads, kv, dim, _ = form
    assert torch.isfinite(got).all()
    seen, t = 0, 0
    for i, (start, new) in enumerate(zip(step.starts, step.news)):
        k, v = step.rows(keys, i, start + new), step.rows(values, i, start + new)
        for h in range(heads):
            g = h * kv // heads
            rows = q.double().view(step.n, heads, dim)[t:t + new, h]
            hidden = torch.arange(start + new)[None] > torch.arange(start, start + new)[:, None]
            s = (rows @ k[:, g].t()).masked_fill(hidden, -float("inf"))
            # a score is a sum of dim products in float32, begun with at most 40 / scale
            error = (dim + 4) * 2.0 ** -24 * (rows.abs() @ k[:, g].abs().t()).amax(-1) + 64 / scale
            top, at = s.topk(2, -1)
            clear = (top[:, 0] - top[:, 1] - 2 * error) * scale > 100  # the others' weights are below 2^-140
            want = v[at[:, 0], g]
            # (a value of the cache is a bfloat16 number; 2^-8 for the rounding of what is divided)
            assert ((got[t:t + new, h] - want).abs() <= 2.0 ** -8 * want.abs())[clear].all()
            seen += int(clear.sum())
        t += new
    assert seen > step.n * heads * 0.9


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16), (8, 1, 256, 32)])
@pytest.mark.parametrize("gain, scale", [(2.0 ** 20, None), (2.0 ** 30, None), (2.0 ** 34, None), (2.0 ** 60, None), (2.0 ** 100, None), (1.0, 2.0 ** 100),
                                         (2.0 ** 10, 2.0 ** 100)])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_one_key_has_all_the_weight(form, gain, scale, nsplit):
    heads, kv, dim, ps = form
    scale = dim ** -0.5 if scale is None else scale
    step = plain.Step(STARTS, NEWS, ps, seed=5)
    pools, keys, values, q = setup(step, form, gain)
    got = both(form, step, pools, q, scale, nsplit)
    the_largest_score_s_value(form, step, got, keys, values, q, scale)


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16), (8, 1, 256, 32)])
@pytest.mark.parametrize("gain, scale", [(2.0 ** 98, 2.0 ** -100), (2.0 ** -102, 2.0 ** 100)])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_scales_far_from_one(form, gain, scale, nsplit):
    heads, kv, dim, ps = form
    step = plain.Step(STARTS, NEWS, ps, seed=6)
    pools, keys, values, q = setup(step, form, gain)
    want, size, reach = plain.attention(step, q, keys, values, heads, scale)
    off = (both(form, step, pools, q, scale, nsplit) - want).abs()
    assert (off <= plain.allowed(want, size, reach, dim, max(step.ctx_lens.tolist()), True)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gain, scale", [(2.0 ** 34, 0.125), (2.0 ** 100, 0.125), (1.0, 2.0 ** 110)])
def test_the_kernel_for_any_sizes(dtype, gain, scale):
    from shrike_amd.kernels import ops

    form = heads, kv, dim, ps = 6, 2, 48, 8
    step = plain.Step(STARTS, NEWS, ps, seed=5)
    pools, keys, values, q = setup(step, form, gain)
    out = torch.full((step.n, heads * dim), 9.0, dtype=dtype, device="cuda")
    ops.attention_e4m3(q.to(dtype).cuda(), out, heads, kv, dim, step.positions.cuda(), step.token_seq.cuda(), step.tables.cuda(), *pools, ps, None,
                       scale)
    the_largest_score_s_value(form, step, out.cpu().double().view(step.n, heads, dim), keys, values, q, scale)
