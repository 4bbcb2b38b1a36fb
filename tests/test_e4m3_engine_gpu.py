"""The engine with its keys and values in 8-bit codes: logits against the plain model whose keys and values are quantised by the
definition, the cuttings of the replay tool over poisoned pages, graphs, preemption and prefix sharing, the command line.

How near: the engine's rows and the plain model's differ by float32 (or bfloat16) rounding before they are quantised, which puts a
few elements on the next code.  Both are quantisations of the same model, so with d the distance of the plain model's logits
with and without quantising, the engine lies within 2 d of them besides the type's own tolerance; in float32, where a code in some
hundred thousand moves, within d, and a tenth of it in the mean."""

import io
import json
import random
import sys

import numpy as np
import pytest
import torch

from . import e4m3_plain
from .compare import TOL
from .plain import model as plain_model
from .plain import mofarax as plain_mofarax
from .plain.model import PlainModel
from .tiny import CONFIGS, PAGE_SIZES, make_model_dir
from .traces import TraceBuilder, changing_portions, check_pages, last_one_by_one, mixed, read_pages, whole

pytestmark = pytest.mark.gpu

LENGTHS = {"A": [5, 17, 70], "B": [1, 30, 100], "C": [3, 40, 97], "D": [6, 130, 190]}


@pytest.fixture(scope="module")
def model_root(tmp_path_factory):
    return tmp_path_factory.mktemp("models")


def requests_for(name):
    rng = random.Random(sum(map(ord, name)))
    return {f"r{i}": [rng.randrange(CONFIGS[name]["vocab_size"]) for _ in range(n)] for i, n in enumerate(LENGTHS[name])}


def quantised_attention(original):
    def attention(q, k, v, *args, **kw):
        return original(q, e4m3_plain.quantised(k)[0], e4m3_plain.quantised(v)[0], *args, **kw)
    return attention


@pytest.fixture
def plain_logits(monkeypatch):
    """(quantised, as they are) logits of a model folder's sequences, {id: [n, vocab]}."""
    def both(model_dir, seqs):
        plain = PlainModel(model_dir)
        exact = {rid: plain.logits(ids).numpy() for rid, ids in seqs.items()}
        with monkeypatch.context() as m:
            m.setattr(plain_model, "causal_attention", quantised_attention(plain_model.causal_attention))
            return {rid: plain.logits(ids).numpy() for rid, ids in seqs.items()}, exact
    return both


def compare(got, quantised, exact, dtype):
    top = max(np.abs(x).max() for x in exact.values())
    d = max(np.abs(quantised[r] - exact[r]).max() for r in exact) / top
    assert d > 3 * 1e-4  # quantising shows
    worst, total, count = 0.0, 0.0, 0
    for (rid, pos), row in got.items():
        off = np.abs(row - quantised[rid[2:]][pos]) / top
        worst, total, count = max(worst, off.max()), total + off.mean(), count + 1
    mean = np.mean([np.abs(quantised[r] - exact[r]).mean() for r in exact]) / top
    if dtype == "float32":
        assert worst <= TOL[dtype] + d and total / count <= TOL[dtype] + 0.1 * mean
    else:
        assert worst <= TOL[dtype] + 2 * d
    # it did run on codes: nearer to the quantised model than to the other one
    assert total < sum((np.abs(row - exact[rid[2:]][pos]) / top).mean() for (rid, pos), row in got.items())


def replay(monkeypatch, capsys, model_dir, dtype, tb, budget, out, vocab, page):
    from shrike_amd.replay import trace

    with monkeypatch.context() as m:
        m.setattr(sys, "stdin", io.StringIO("".join(json.dumps(s) + "\n" for s in tb.steps)))
        assert trace.main(["--model", str(model_dir), "--dtype", dtype, "--cache-dtype", "e4m3", "--out", str(out), "--max-tokens",
                           str(budget), "--block-size", str(page), "--poison", "--pages"]) == 0
    capsys.readouterr()
    outputs = {}
    for s in tb.steps:
        wanted = sum(len(e.get("want", [])) for e in s["entries"])
        if wanted:
            outputs[s["step"]] = np.fromfile(out / f"{s['step']}.f32", dtype="<f4").reshape(wanted, vocab)
    return outputs


# (A and C have pages or heads that the matrix-unit kernels do not take)
@pytest.mark.parametrize("name, page", [("A", 4), ("B", 16), ("B", 8), ("C", 16), ("D", 16), ("D", 32)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_four_cuttings_agree_with_the_quantised_plain_model(name, page, dtype, model_root, tmp_path, monkeypatch, capsys, plain_logits):
    model_dir = make_model_dir(name, model_root, dtype=dtype, mode="unit")
    vocab, seqs = CONFIGS[name]["vocab_size"], requests_for(name)
    quantised, exact = plain_logits(model_dir, seqs)
    tb = TraceBuilder()
    budget = max(-(-len(ids) // 64) * 64 for ids in seqs.values()) + 128
    whole(tb, "w_", seqs)
    last_one_by_one(tb, "d_", seqs)
    changing_portions(tb, "p_", seqs)
    mixed(tb, "m_", seqs, budget, seed=3)
    outputs = replay(monkeypatch, capsys, model_dir, dtype, tb, budget, tmp_path / "out", vocab, page)
    assert all(np.isfinite(rows).all() for rows in outputs.values())
    assert check_pages(tb.steps, read_pages(tmp_path / "out", tb.steps), page, budget // page) > 0
    got = tb.collect(outputs)
    compare(got, quantised, exact, dtype)
    if dtype == "float32":  # one order of summation whatever the step holds, and so the same codes: the same bits
        for (rid, pos), row in got.items():
            assert np.array_equal(row, got[("w_" + rid[2:], pos)])


def test_blocks_of_positions_values_from_keys_and_runs_that_share_a_cache(monkeypatch, tmp_path):
    """Mofarax: attention without a value projection inside blocks of positions, heads rotated by neighbours, wholly, in part or not."""
    from shrike_amd.cache import CacheManager
    from shrike_amd.engine.loading import load_model
    from shrike_amd.engine.runner import ModelRunner, StepEntry

    from .tiny_mofarax import CONFIGS as MOFARAX
    from .tiny_mofarax import make_model_dir as make_mofarax

    rng = random.Random(5)
    for name in ("P", "Q", "R"):
        model_dir = make_mofarax(name, tmp_path, dtype="float32")
        ids = [rng.randrange(MOFARAX[name]["vocab"]) for _ in range(75)]
        exact = plain_mofarax.PlainMofarax(model_dir).logits(ids).numpy()
        for dtype in ("float32", "bfloat16"):
            model, rt, _ = load_model(model_dir, dtype, cache_dtype="e4m3")
            cache = CacheManager(model.cache_specs(), 16, 20, enable_prefix_caching=False)
            cache.allocate(rt.dtype, rt.device)
            runner = ModelRunner(model, cache, rt)
            seq = cache.new_sequence()
            rows, at = [], 0
            for n in (50, 1, 1, 1, 20, 1, 1):
                cache.append(seq, at, n)
                rows.append(runner.step([StepEntry(seq, ids[at:at + n], at, list(range(n)))]).cpu().clone())
                at += n
                cache.trim(seq, at)
            got = torch.cat(rows).double().numpy()
            # quantising moves an element by up to 2^-4 of itself; through the layers of these models a logit by less than that of
            # the largest one
            off = np.abs(got - exact).max() / np.abs(exact).max()
            assert 1e-4 < off < 2.0 ** -4 * 4 and np.isfinite(got).all()


@pytest.mark.parametrize("name", ["B", "D"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graph_replays_equal_eager_steps(name, dtype, model_root):
    from shrike_amd.cache import CacheManager
    from shrike_amd.engine.loading import load_model
    from shrike_amd.engine.runner import ModelRunner, StepEntry

    model_dir = make_model_dir(name, model_root, dtype=dtype, mode="unit")
    model, rt, cfg = load_model(model_dir, dtype, cache_dtype="e4m3")

    def run(graphs):
        cache = CacheManager(model.cache_specs(), 16, 60, enable_prefix_caching=False)
        cache.allocate(rt.dtype, rt.device)
        runner = ModelRunner(model, cache, rt, graphs=graphs)
        rng = random.Random(1)
        live, outs = [], []
        for step in range(40):
            if step in (0, 3, 9, 10, 20):
                ids = [rng.randrange(cfg.vocab_size) for _ in range(rng.choice([5, 40, 90]))]
                seq = cache.new_sequence()
                cache.append(seq, 0, len(ids))
                outs.append(runner.step([StepEntry(seq, ids, 0, [len(ids) - 1])]).cpu().clone())
                live.append([seq, len(ids)])
            entries = []
            for item in live:
                cache.append(item[0], item[1], 1)
                entries.append(StepEntry(item[0], [rng.randrange(cfg.vocab_size)], item[1], [0]))
                item[1] += 1
            outs.append(runner.step(entries).cpu().clone())
        return outs, runner.graph_replays

    eager, n0 = run(False)
    graphed, n1 = run(True)
    assert n0 == 0 and n1 > 20
    assert all(torch.equal(a, b) for a, b in zip(eager, graphed))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_preemption_and_prefix_sharing(dtype, model_root):
    from shrike_amd import SamplingParams
    from shrike_amd.engine.llm_engine import LLMEngine

    model_dir = make_model_dir("B", model_root, dtype=dtype, mode="unit")
    rng = random.Random(6)
    common = [rng.randrange(500) for _ in range(40)]
    prompts = [common + [rng.randrange(500) for _ in range(n)] for n in (3, 9, 20)]
    sp = SamplingParams(max_new_tokens=16, ignore_eos=True)
    options = dict(dtype=dtype, cache_dtype="fp8", block_size=16)
    roomy = LLMEngine(str(model_dir), num_kv_blocks=64, enable_prefix_caching=False, **options)
    assert roomy.cache.groups[0].tensors["k"].dtype == torch.float8_e4m3fn
    want = roomy.generate(prompts, sp)
    sharing = LLMEngine(str(model_dir), num_kv_blocks=64, **options)
    got = [sharing.generate([p], sp)[0] for p in prompts]
    assert sharing.cache.cache_hit_blocks > 0
    tight = LLMEngine(str(model_dir), num_kv_blocks=12, enable_prefix_caching=False, **options)  # 11 for the prompts, 14 in the end
    pressed = tight.generate(prompts, sp)
    assert tight.metrics()["preemptions"] > 0 and tight.cache.num_free == 12
    assert all(len(o) == 16 for o in want + got + pressed)
    if dtype == "float32":  # the same codes and the same sums however the steps are cut
        assert got == want and pressed == want


def test_twice_the_pages_in_the_same_memory(model_root):
    from shrike_amd.cache import CacheManager
    from shrike_amd.engine.loading import load_model

    model_dir = make_model_dir("D", model_root, dtype="bfloat16", mode="unit")
    sizes = []
    for cache_dtype in (None, "e4m3"):
        model, _, _ = load_model(model_dir, "bfloat16", cache_dtype=cache_dtype)
        sizes.append(CacheManager(model.cache_specs(), 16, 1).bytes_per_page(2))
    assert sizes[1] * 4 * 64 == sizes[0] * (2 * 64 + 2)  # a byte an element and one of 64 elements


def test_command_line(model_root, capsys):
    from shrike_amd.__main__ import main

    model_dir = make_model_dir("B", model_root, dtype="bfloat16", mode="unit")
    assert main(["--model", str(model_dir), "--cache-dtype", "e4m3", "--prompt-ids", "5,6,7,8", "--max-tokens", "5", "--num-kv-blocks", "8"]) == 0
    assert len(capsys.readouterr().out.split()) == 5
    assert main(["--random-config", "qwen2.5-0.5b", "--cache-dtype", "fp8", "--prompt-len", "20", "--max-tokens", "3", "--num-kv-blocks", "8"]) == 0


def test_a_model_that_was_built_without_is_refused(model_root):
    from shrike_amd.config import EngineConfig
    from shrike_amd.engine.llm_engine import LLMEngine
    from shrike_amd.engine.loading import load_model

    model_dir = make_model_dir("B", model_root, dtype="bfloat16", mode="unit")
    model, rt, _ = load_model(model_dir, "bfloat16")
    with pytest.raises(ValueError, match="built without"):
        LLMEngine(None, EngineConfig(cache_dtype="e4m3", num_kv_blocks=8), model=model, runtime=rt)
