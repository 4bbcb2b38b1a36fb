"""The engine with a quantised cache at page sizes whose bytes a layer are no multiple of 16, at odd and even numbers of pages."""

import random

import pytest

from .tiny import CONFIGS, make_model_dir

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page", [1, 2, 4, 12])
def test_page_sizes_and_page_counts(page, dtype, tmp_path):
    """The same tokens whatever the number of pages, in float32 whatever the page size too (one order of summation)."""
    from shrike_amd import SamplingParams
    from shrike_amd.engine.llm_engine import LLMEngine

    model_dir = make_model_dir("B", tmp_path, dtype="float32", mode="unit")  # (one key/value head, three layers)
    rng = random.Random(3)
    prompts = [[rng.randrange(CONFIGS["B"]["vocab_size"]) for _ in range(n)] for n in (5, 21)]
    sp = SamplingParams(max_new_tokens=4, ignore_eos=True)

    def generate(page, pages):
        engine = LLMEngine(str(model_dir), dtype=dtype, cache_dtype="e4m3", block_size=page, num_kv_blocks=pages)
        return engine.generate(prompts, sp)

    even = -(-40 // page) // 2 * 2 + 4
    got = generate(page, even)
    assert got == generate(page, even + 1)
    if dtype == "float32":
        assert got == generate(16, 8)
