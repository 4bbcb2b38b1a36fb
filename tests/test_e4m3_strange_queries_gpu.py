"""Attention over a quantised cache where some queries hold a NaN or an infinity, and rows that lie apart: the others' results stay."""

import pytest
import torch

from . import e4m3_plain as plain
from .test_e4m3_attention_gpu import setup

pytestmark = pytest.mark.gpu

STARTS, NEWS, SINGLES = [150, 700, 333, 90], [1, 1, 40, 70], 2


@pytest.mark.parametrize("form", [(14, 2, 64, 16), (28, 4, 128, 16), (24, 8, 96, 32), (8, 1, 256, 32)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("nsplit", [1, 3])
@pytest.mark.parametrize("window", [None, 50])
def test_a_query_s_nan_stays_its_own(form, what, nsplit, window):
    from shrike_amd.kernels import ops

    heads, kv, dim, ps = form
    step = plain.Step(STARTS, NEWS, ps, seed=7)
    pools, keys, values, q = setup(step, form)
    want, size, reach = plain.attention(step, q, keys, values, heads, dim ** -0.5, window)
    limit = plain.allowed(want, size, reach, dim, max(step.ctx_lens.tolist()), True)
    strange = torch.rand(step.n, heads, generator=step.gen) < 0.2
    rows = q.view(step.n, heads, dim).clone()
    rows[strange, 3] = what
    wide = torch.zeros(step.n, (heads + 3) * dim, dtype=torch.bfloat16, device="cuda")
    wide[:, : heads * dim] = rows.view(step.n, -1).cuda()
    apart = wide[:, : heads * dim]
    out = torch.full((step.n, heads * dim), 9.0, dtype=torch.bfloat16, device="cuda")
    partial = torch.full((step.n * heads * nsplit * (dim + 2),), float("nan"), device="cuda")
    ops.attention_decode_e4m3(apart, out, SINGLES, heads, kv, dim, step.positions.cuda(), step.tables.cuda(), *pools, ps, window, dim ** -0.5,
                              partial, nsplit)
    ops.attention_prefill_e4m3(apart, out, SINGLES, len(STARTS) - SINGLES, heads, kv, dim, step.cu_q.cuda(), step.ctx_lens.cuda(),
                               step.tables.cuda(), *pools, ps, window, dim ** -0.5, partial, nsplit)
    got = out.cpu().double().view(step.n, heads, dim)
    assert ((got - want).abs() <= limit)[~strange].all()
    if what != what:  # (an infinite element's products have either sign: which weights that leaves is not said here)
        assert got[strange].isnan().all()
