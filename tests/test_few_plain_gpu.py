"""Products of few rows that are still to be divided by their root mean square, left in float32 for a cache write of its own."""

import pytest
import torch

from .test_few_products_gpu import scaled_rows, sums_bound

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 7, 16, 17, 50, 64])
@pytest.mark.parametrize("m, k", [(16, 8), (1152, 896), (768, 1000), (4608, 3584), (272, 904)])
@pytest.mark.parametrize("scaled, biased", [(True, True), (False, True), (True, False)])
def test_rows_against_64_bits(m, k, n, scaled, biased):
    from shrike_amd.kernels import ops

    torch.manual_seed(m + k + n)
    x, r, rms = scaled_rows(n, k, k // (8 if k <= 2048 else 16))  # (as many sums as few_stream leaves)
    if not scaled:
        x, rms = r, torch.ones(n, 1, device="cuda", dtype=torch.float64)
    w, bias = (torch.randn(m, k, device="cuda") / k**0.5).bfloat16(), torch.randn(m, device="cuda")
    out = torch.full((n + 1, m), 5.0, device="cuda")
    ops.few_plain(x, ops.retile_weight(w), k, out[:n], bias=bias if biased else None)
    want = (r.double() @ w.double().t()) * rms
    size = (r.double().abs() @ w.double().abs().t()) * rms
    if biased:
        want, size = want + bias.double(), size + bias.double().abs()
    # sums of k products, of the squares, the root, the product with it and the bias
    assert bool(((out[:n].double() - want).abs() <= (sums_bound(k) + (k // 8 + 12) * 2.0**-24) * size + 1e-7).all())
    assert bool((out[n:] == 5.0).all())


def test_refusals():
    from shrike_amd.kernels import ops
    from shrike_amd.kernels.lib import KernelError

    w = torch.randn(32, 64, device="cuda").bfloat16()
    wt, a = ops.retile_weight(w), torch.randn(3, 64, device="cuda").bfloat16()
    with pytest.raises(KernelError, match="contiguous"):
        ops.few_plain(a, wt, 64, torch.empty(2, 32, device="cuda"))
    with pytest.raises(KernelError, match="expected torch.float32"):
        ops.few_plain(a, wt, 64, torch.empty(3, 32, device="cuda").bfloat16())
    with pytest.raises(KernelError, match="weights"):
        ops.few_plain(a, wt, 64, torch.empty(3, 48, device="cuda"))
    with pytest.raises(KernelError, match="rows must be"):
        ops.few_plain(torch.randn(65, 64, device="cuda").bfloat16(), wt, 64, torch.empty(65, 32, device="cuda"))
    with pytest.raises(KernelError, match="aligned"):
        ops.few_plain(torch.randn(3 * 64 + 1, device="cuda").bfloat16()[1:].view(3, 64), wt, 64, torch.empty(3, 32, device="cuda"))


@pytest.mark.parametrize("n", [1, 5, 16, 40, 64])
@pytest.mark.parametrize("name", ["B", "D"])
def test_a_quantised_step_takes_rows_that_are_still_to_be_divided(name, n, tmp_path, monkeypatch):
    """The layers' norms before the projections are no kernels of their own, and logits are as with them."""
    from shrike_amd.cache import CacheManager
    from shrike_amd.engine.loading import load_model
    from shrike_amd.engine.runner import ModelRunner, StepEntry
    from shrike_amd.kernels import ops

    from .tiny import make_model_dir

    model_dir = make_model_dir(name, tmp_path, dtype="bfloat16", mode="unit")
    model, runtime, cfg = load_model(model_dir, "bfloat16", cache_dtype="e4m3")
    calls, few = [], ops.few_plain
    monkeypatch.setattr(ops, "few_plain", lambda x, *a, **k: (calls.append(isinstance(x, ops.ScaledRows)), few(x, *a, **k))[1])

    def run():
        calls.clear()
        cache = CacheManager(model.cache_specs(), 16, 80, enable_prefix_caching=False)
        cache.allocate(runtime.dtype, runtime.device)
        runner = ModelRunner(model, cache, runtime, graphs=False)
        ids = [(11 * i + 5) % cfg.vocab_size for i in range(n)]
        seq = cache.new_sequence()
        cache.append(seq, 0, n)
        logits = [runner.step([StepEntry(seq, ids, 0, [n - 1])]).double()]
        cache.append(seq, n, 1)
        return torch.cat([*logits, runner.step([StepEntry(seq, [3], n, [0])]).double()]), list(calls)

    got, used = run()
    monkeypatch.setattr(ops, "few_plain_takes", lambda *sizes: False)
    want, unused = run()
    assert any(used) and not unused
    # Some twenty roundings to bfloat16 a path on either side, of 2^-9 at random: sqrt(40) * 2^-9.  And rows that differ by 2^-8 have 1 in 32 of
    # their codes a step of 2^-3 apart: 2^-5.5 of keys and of values in every layer.
    assert float((got - want).norm() / want.norm()) <= 0.0125 + (2 * len(model.blocks)) ** 0.5 * 2.0**-5.5
