"""What the launchers of the quantised cache refuse (nothing is launched), and the 64-bit oracle against torch's conversion."""

import pytest
import torch

from . import e4m3_plain as plain


def test_the_oracle_rounds_as_the_type_does():
    codes = torch.arange(256, dtype=torch.uint8).view(plain.E4M3).float().double()
    codes = codes[codes.isfinite()]
    assert codes.numel() == 254
    assert torch.equal(plain.rounded(codes), codes)
    x = torch.randn(100000, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 50
    x = torch.cat([x, x * 2.0 ** -10, (codes[1:] + codes[:-1]) / 2]).clamp(-448, 448)
    assert torch.equal(plain.rounded(x), x.float().to(plain.E4M3).double())


def test_the_oracle_s_exponents():
    x = torch.tensor([[0.0], [448.0], [449.0], [224.0], [1e-300], [1e300], [448 * 2.0 ** 119]], dtype=torch.float64)
    assert plain.exponents(x).tolist() == [-117, 0, 1, -1, -117, 119, 119]


@pytest.fixture(scope="module")
def lib():
    from shrike_amd.kernels.lib import load

    return load()


def refused(lib, name, args, part):
    assert getattr(lib, name)(*args) != 0
    assert part in lib.shk_last_error().decode()


def test_refusals_before_any_launch(lib):
    P = None

    def store(dtype=1, n=4, heads=4, kv=2, dim=64, rot=64, ps=16, pages=9, stride=3, seqs=2, splits=0, pairing=0, q_ld=512, bias=P):
        return (P, dtype, n, heads, kv, dim, rot, P, P, P, P, stride, seqs, P, P, P, ps, pages, 1, P, splits, bias, pairing, 0, 1.0, P,
                q_ld, P)

    name = "shk_rope_kv_store_e4m3"
    assert getattr(lib, name)(*store(n=0)) == 0
    for args, part in ((store(dtype=2), "dtype"), (store(n=-1), "n=-1"), (store(dim=257), "head_dim=257"), (store(rot=66), "rot_dim"),
                       (store(rot=63), "rot_dim"), (store(pairing=2), "pairing"), (store(q_ld=255), "queries"),
                       (store(splits=2), "parts"), (store(heads=0), "heads=0"), (store(), "null pointer")):
        refused(lib, name, args, part)

    def read(dtype=1, n=4, kv=2, dim=64, ps=16, pages=9, stride=3, seqs=2):
        return (P, P, dtype, n, kv, dim, P, P, P, stride, seqs, P, P, P, ps, pages, P)

    name = "shk_kv_read_e4m3"
    assert getattr(lib, name)(*read(n=0)) == 0
    for args, part in ((read(dtype=5), "dtype"), (read(kv=0), "kv_heads=0"), (read(ps=0), "page_size=0"), (read(pages=0), "num_pages=0"),
                       (read(), "null pointer")):
        refused(lib, name, args, part)

    def attend(dtype=1, n=4, heads=4, kv=2, dim=64, q_ld=256, ps=16, pages=9, scale=0.1):
        return (P, q_ld, P, dtype, n, heads, kv, dim, P, P, P, 3, 2, P, P, P, ps, pages, 0, 0, scale, P)

    name = "shk_attention_e4m3"
    assert getattr(lib, name)(*attend(n=0)) == 0
    for args, part in ((attend(dtype=3), "dtype"), (attend(heads=3), "multiple"), (attend(dim=300), "head_dim"), (attend(q_ld=255), "q_stride"),
                       (attend(ps=0), "page_size=0"), (attend(scale=0.0), "positive"), (attend(scale=float("nan")), "positive"),
                       (attend(n=70000), "65535"), (attend(), "null pointer")):
        refused(lib, name, args, part)


def test_names_of_the_cache_dtype():
    from shrike_amd.config import EngineConfig, canonical_cache_dtype

    assert EngineConfig().cache_dtype is None and EngineConfig(cache_dtype="auto").cache_dtype is None
    assert {canonical_cache_dtype(n) for n in ("e4m3", "fp8", "fp8_e4m3", "float8_e4m3fn", torch.float8_e4m3fn)} == {"e4m3"}
    with pytest.raises(ValueError, match="e5m2"):
        EngineConfig(cache_dtype="e5m2")


def test_models_that_a_quantised_cache_is_not_built_for_are_refused():
    from dataclasses import replace

    from shrike_amd.config import architecture_name, get_architecture
    from shrike_amd.config.specs import with_cache_dtype
    from shrike_amd.models import DecoderModel

    from .tiny import CONFIGS
    from .tiny_bevovik import CONFIGS as BEVOVIK
    from .tiny_fozedra import CONFIGS as FOZEDRA
    from .tiny_minilorn import CONFIGS as MINILORN
    from .tiny_mofarax import CONFIGS as MOFARAX

    def spec_of(raw):
        arch = get_architecture(architecture_name(raw))
        return arch.build_spec(arch.config_cls.from_dict(raw))

    for raw in (*CONFIGS.values(), *MOFARAX.values()):
        spec = with_cache_dtype(spec_of(raw), "e4m3")
        model = DecoderModel(spec)
        for need in model.cache_specs():
            assert [t.dtype for t in need.tensors] == ["float8_e4m3fn", "float8_e4m3fn", "uint8"]
        for block in model.blocks:
            block.mixer.check(None)
        assert with_cache_dtype(spec_of(raw), None) == spec_of(raw)
    for raw in (*BEVOVIK.values(), *FOZEDRA.values(), *MINILORN.values()):
        spec = spec_of(raw)
        try:
            model = DecoderModel(with_cache_dtype(spec, "e4m3"))
        except ValueError as e:
            assert "is built for paged attention" in str(e)
            continue
        with pytest.raises(ValueError, match="is built for attention that rotates"):
            for block in model.blocks:
                block.mixer.check(None)
    first = spec_of(CONFIGS["A"]).blocks[0].mixer
    from shrike_amd.parts.attention import PagedAttention

    with pytest.raises(ValueError, match="must be None or e4m3"):
        PagedAttention(replace(first, cache_dtype="int4"), 64, "x").check(None)


@pytest.mark.parametrize("heads, kv", [(14, 2), (28, 4), (16, 16), (40, 1), (128, 1)])
def test_launch_plans(heads, kv):
    from shrike_amd.parts.attention import e4m3_decode_splits, e4m3_portion_splits

    for seqs in (1, 2, 7, 64, 300):
        for ctx in (1, 63, 256, 257, 5000, 131072):
            n = e4m3_decode_splits(seqs, heads, kv, 128, ctx)
            assert 1 <= n <= min(64, -(-ctx // 256))
            # a batch that is padded to the next power of two takes the same
            assert n == e4m3_decode_splits(1 << (seqs - 1).bit_length(), heads, kv, 128, ctx)
    for lens, starts in (([2], [0]), ([512], [16000]), ([17] * 4, [700, 800, 900, 1900]), ([2048], [0]), ([1, 0, 30], [5, 0, 9])):
        longest = max(a + n for a, n in zip(starts, lens))
        assert 1 <= e4m3_portion_splits(lens, starts, heads, kv, 128, 1 << 40) <= min(64, -(-longest // 256))
        assert e4m3_portion_splits(lens, starts, heads, kv, 128, 100) == 1  # a window of 100 keys is not shared


def test_refusals_of_the_matrix_kernels_before_any_launch(lib):
    P = None

    def decode(seqs=2, heads=4, kv=2, dim=64, q_ld=256, ps=16, pages=9, stride=3, rows=2, scale=0.1, nsplit=1):
        return (P, q_ld, P, seqs, heads, kv, dim, P, P, stride, rows, P, P, P, ps, pages, 0, 0, scale, P, nsplit, P)

    def portions(n=9, first=1, seqs=1, heads=4, kv=2, dim=64, q_ld=256, ps=16, pages=9, stride=3, rows=2, scale=0.1, nsplit=1):
        return (P, q_ld, P, n, first, seqs, heads, kv, dim, P, P, P, stride, rows, P, P, P, ps, pages, 0, 0, scale, P, nsplit, P)

    for name, args in (("shk_attention_decode_e4m3", decode), ("shk_attention_prefill_e4m3", portions)):
        assert getattr(lib, name)(*args(seqs=0)) == 0
        for bad, part in ((args(dim=80), "not built"), (args(ps=24), "not built"), (args(kv=3), "not built"), (args(q_ld=260), "not built"),
                          (args(pages=0), "num_pages=0"), (args(stride=0), "table_stride=0"), (args(nsplit=0), "shares"),
                          (args(nsplit=65), "shares"), (args(rows=0), "tables of 0"), (args(scale=0.0), "positive"),
                          (args(scale=1e-38), "positive"), (args(scale=1e38), "positive"), (args(scale=float("nan")), "positive"),
                          (args(), "null pointer")):
            refused(lib, name, bad, part)
