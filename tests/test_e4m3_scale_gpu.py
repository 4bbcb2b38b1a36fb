"""Attention over a quantised cache at scales outside of 2^-100 to 2^100, which the kernels on the matrix units refuse."""

from dataclasses import replace

import pytest
import torch

from .compare import TOL

pytestmark = pytest.mark.gpu


def rows(scale):
    """Logits of two sequences, a prompt's portion and single tokens, of a model whose second layer has `scale`."""
    from shrike_amd.config import AttentionSpec, BlockSpec, ModelSpec, RMSNormSpec, RotarySpec, SwiGLUSpec
    from shrike_amd.engine.runner import StepEntry

    from .test_parts_gpu import cpu_weights, make_runner

    norm = RMSNormSpec(eps=1e-5)
    mixer = AttentionSpec(num_heads=4, num_kv_heads=2, head_dim=64, qkv_bias=True, out_bias=False, scale=0.125,
                          position=RotarySpec(theta=1e4, rotary_dim=64), cache_dtype="e4m3")
    blocks = tuple(BlockSpec(name=f"model.layers.{i}", mixer=replace(mixer, scale=s), ffn=SwiGLUSpec(intermediate_size=88),
                             mixer_norm=norm, ffn_norm=norm) for i, s in enumerate((0.125, scale)))
    spec = ModelSpec(architecture="toy", hidden_size=48, vocab_size=97, blocks=blocks, final_norm=norm, tie_word_embeddings=False)
    runner, _, cache = make_runner(spec, cpu_weights(spec), torch.bfloat16, page_size=16)
    a, b = cache.new_sequence(), cache.new_sequence()
    out = []
    cache.append(a, 0, 40)
    out.append(runner.step([StepEntry(a, [(7 * i + 3) % 97 for i in range(40)], 0, list(range(40)))]).cpu().clone())
    cache.append(a, 40, 1)
    cache.append(b, 0, 20)
    out.append(runner.step([StepEntry(a, [5], 40, [0]), StepEntry(b, [(11 * i + 1) % 97 for i in range(20)], 0, list(range(20)))]).cpu().clone())
    cache.append(a, 41, 1)
    cache.append(b, 20, 1)
    out.append(runner.step([StepEntry(a, [9], 41, [0]), StepEntry(b, [8], 20, [0])]).cpu().clone())
    return torch.cat(out).double()


@pytest.mark.parametrize("near, far", [(2.0 ** -100, 2.0 ** -101), (2.0 ** -100, 2.0 ** -120), (2.0 ** 100, 2.0 ** 101)])
def test_scales_outside_the_matrix_kernels_range(near, far):
    """All weights are equal there (2^-100 and below), or one key has all of them (2^100 and above), so that the last scale
    which the matrix kernels take is the same model."""
    want, got = rows(near), rows(far)
    assert torch.isfinite(got).all()
    assert (got - want).abs().max() <= TOL["bfloat16"] * want.abs().max()


@pytest.mark.parametrize("scale", [0.0, -0.125, float("inf"), float("nan")])
def test_scales_that_are_none(scale):
    with pytest.raises(ValueError, match="a positive scale"):
        rows(scale)
