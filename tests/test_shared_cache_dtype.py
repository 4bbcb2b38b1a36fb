"""Runs that read another run's cache keep to its dtype: anything else is refused when the model is described."""

from dataclasses import replace

import pytest

import shrike_amd.models  # noqa: F401  (registers the architectures)
from shrike_amd.config.specs import ParallelMixerSpec, ScheduleEntry, with_cache_dtype

from .tiny import CONFIGS


def spec_of(raw):
    from shrike_amd.config import architecture_name, get_architecture

    arch = get_architecture(architecture_name(raw))
    return arch.build_spec(arch.config_cls.from_dict(raw))


def with_mixers(spec, *mixers):
    return replace(spec, blocks=tuple(replace(b, mixer=m) for b, m in zip(spec.blocks, mixers)),
                   schedule=(ScheduleEntry(0), ScheduleEntry(1, cache_of=0)))


@pytest.mark.parametrize("owner, reader", [(None, "e4m3"), ("e4m3", None)])
def test_a_reader_of_another_dtype_is_refused(owner, reader):
    spec = spec_of(CONFIGS["A"])
    one = spec.blocks[0].mixer
    first, second = replace(one, cache_dtype=owner), replace(one, cache_dtype=reader)
    with pytest.raises(ValueError, match=r"schedule\[1\] keeps its keys and values .* position 0"):
        with_mixers(spec, first, second)
    with pytest.raises(ValueError, match=r"schedule\[1\] keeps its keys and values .* position 0"):
        with_mixers(spec, ParallelMixerSpec((("a", one), ("b", first)), 1e-6), ParallelMixerSpec((("b", second), ("c", first)), 1e-6))


@pytest.mark.parametrize("dtype", [None, "e4m3"])
def test_a_reader_of_the_same_dtype_is_not(dtype):
    spec = spec_of(CONFIGS["A"])
    one = replace(spec.blocks[0].mixer, cache_dtype=dtype)
    with_mixers(spec, one, one)
    # branches of other names read nothing of each other
    with_mixers(spec, ParallelMixerSpec((("a", one),), 1e-6), ParallelMixerSpec((("b", replace(one, cache_dtype=None)),), 1e-6))
    shared = replace(spec, schedule=(ScheduleEntry(0), ScheduleEntry(1, cache_of=0)))
    assert [b.mixer.cache_dtype for b in with_cache_dtype(shared, dtype).blocks] == [dtype] * 2
