"""Mofarax with a quantised cache, attention without a value projection inside blocks of positions, heads rotated by neighbours (whole, in part, not
at all), runs that read another run's cache, against the plain model whose keys (rotated) and values (the keys as projected) are
quantised by the definition.  How near: as in test_e4m3_engine_gpu.py."""

import random

import pytest
import torch

from . import e4m3_plain
from .plain import mofarax as plain_mofarax
from .test_e4m3_engine_gpu import compare
from .tiny_mofarax import CONFIGS, make_model_dir

pytestmark = pytest.mark.gpu


def quantised_mixer(h, positions, w, prefix, m):
    n, heads, groups, dim = h.shape[0], m["heads"], m["kv_heads"], m["dim"]
    rot = m.get("rot") or {"dims": 0, "base": 1.0}
    q = plain_mofarax.rotate_interleaved((h @ w[prefix + ".q"].T).view(n, heads, dim), positions, float(rot["base"]), int(rot["dims"]))
    k = (h @ w[prefix + ".k"].T).view(n, groups, dim)
    v = e4m3_plain.quantised(k)[0]
    k = e4m3_plain.quantised(plain_mofarax.rotate_interleaved(k, positions, float(rot["base"]), int(rot["dims"])))[0]
    return plain_mofarax.block_local_attention(q, k, v, m["scale"], int(m["mask"]["size"])).reshape(n, heads * dim) @ w[prefix + ".o"].T


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits(name, dtype, monkeypatch, tmp_path):
    from shrike_amd.cache import CacheManager
    from shrike_amd.engine.loading import load_model
    from shrike_amd.engine.runner import ModelRunner, StepEntry

    model_dir = make_model_dir(name, tmp_path, dtype=dtype)
    rng = random.Random(11)
    seqs = {f"r{i}": [rng.randrange(CONFIGS[name]["vocab"]) for _ in range(n)] for i, n in enumerate((75, 40))}
    plain = plain_mofarax.PlainMofarax(model_dir)
    exact = {rid: plain.logits(ids).numpy() for rid, ids in seqs.items()}
    with monkeypatch.context() as m:
        m.setattr(plain_mofarax, "attention_mixer", quantised_mixer)
        quantised = {rid: plain.logits(ids).numpy() for rid, ids in seqs.items()}
    model, rt, _ = load_model(model_dir, dtype, cache_dtype="e4m3")
    cache = CacheManager(model.cache_specs(), 16, 30, enable_prefix_caching=False)
    cache.allocate(rt.dtype, rt.device)
    runner = ModelRunner(model, cache, rt)
    held = {rid: cache.new_sequence() for rid in seqs}
    at, got = dict.fromkeys(seqs, 0), {}
    # both sequences in one step, single tokens and portions side by side
    for news in ((50, 1), (1, 17), (1, 1), (20, 1), (1, 19), (2, 1)):
        entries = []
        for (rid, ids), n in sorted(zip(seqs.items(), news), key=lambda x: x[1]):
            cache.append(held[rid], at[rid], n)
            entries.append((rid, n, StepEntry(held[rid], ids[at[rid]:at[rid] + n], at[rid], list(range(n)))))
        rows = runner.step([e for *_, e in entries]).cpu().double().numpy()
        first = 0
        for rid, n, _ in entries:
            for i in range(n):
                got[("x_" + rid, at[rid] + i)] = rows[first + i]
            first, at[rid] = first + n, at[rid] + n
            cache.trim(held[rid], at[rid])
    assert at == {"r0": 75, "r1": 40}
    compare(got, quantised, exact, dtype)


def test_the_oracle_without_quantising(monkeypatch, tmp_path):
    """The mixer above is the plain one where nothing is quantised."""
    plain = plain_mofarax.PlainMofarax(make_model_dir("P", tmp_path, dtype="float32"))
    want = plain.logits(range(40))
    monkeypatch.setattr(e4m3_plain, "quantised", lambda x: (x, None))
    monkeypatch.setattr(plain_mofarax, "attention_mixer", quantised_mixer)
    assert (plain.logits(range(40)) - want).abs().max() <= 1e-12 * want.abs().max()
