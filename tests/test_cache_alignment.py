"""Every layer's part of a group's pools starts on 16 bytes, whatever a page holds and however many pages there are: kernels that
move 16 bytes at a time refuse pools that do not."""

import itertools

import pytest
import torch

from shrike_amd.cache import CacheManager
from shrike_amd.parts import kv_cache_spec


@pytest.mark.parametrize("cache_dtype", [None, "e4m3"])
@pytest.mark.parametrize("kv, dim", [(1, 64), (2, 32), (3, 64), (1, 9), (4, 24)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layers_start_on_16_bytes(kv, dim, cache_dtype, dtype):
    for page, pages in itertools.product((1, 2, 4, 12, 16), (5, 20, 21)):
        cache = CacheManager([kv_cache_spec(kv, dim, cache_dtype=cache_dtype)] * 3, page, pages, enable_prefix_caching=False)
        cache.allocate(dtype, "cpu")
        group, = cache.groups
        names = {"k", "v"} | ({"scales"} if cache_dtype else set())
        layers = [cache.layer_cache(i).pools for i in range(3)]
        for name in names:
            spec = next(t for t in group.spec.tensors if t.name == name)
            for i, pools in enumerate(layers):
                pool = pools[name]
                assert tuple(pool.shape) == (pages + 1, *spec.shape(page)) and pool.is_contiguous()
                assert pool.data_ptr() % 16 == 0
                assert not pool.view(torch.uint8).any()
                # the group's tensor is the same memory
                assert group.tensors[name][i].data_ptr() == pool.data_ptr()
            for i, pools in enumerate(layers):  # each of them its own memory
                pools[name].view(torch.uint8).fill_(i + 1)
            assert all((pools[name].view(torch.uint8) == i + 1).all() for i, pools in enumerate(layers))


def test_poison_reaches_every_layer():
    from shrike_amd.replay.poison import PagePoisoner

    cache = CacheManager([kv_cache_spec(1, 9, cache_dtype="e4m3")] * 3, 1, 6, enable_prefix_caching=False)
    cache.allocate(torch.float32, "cpu")
    poisoner = PagePoisoner(cache)
    poisoner.poison_pages(0, [2, 4])
    for name in ("k", "v"):
        t = cache.groups[0].tensors[name].float()
        assert t[:, [2, 4]].isnan().all() and (t[:, [0, 1, 3, 5, 6]] == 0).all()
    poisoner.poison_everything()
    assert all(cache.groups[0].tensors[name].float().isnan().all() for name in ("k", "v"))
