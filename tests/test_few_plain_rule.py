"""Which projections of few tokens leave in float32 for a cache write of its own (CPU)."""

import pytest

from shrike_amd.kernels import ops


@pytest.mark.parametrize("n, m, k, takes", [(1, 1152, 896, True), (16, 2560, 2048, True), (1, 4608, 3584, False), (64, 1152, 896, True),
                                             (65, 1152, 896, False), (8, 1144, 896, False), (8, 1152, 900, False)])
def test_sizes(n, m, k, takes):
    assert ops.few_plain_takes(n, m, k) is takes


def test_alike_for_every_row_count_of_a_graph_bucket():
    for m, k in ((1152, 896), (4608, 3584), (2560, 2048), (7168, 5120)):
        for lo, hi in ((1, 16), (17, 32), (33, 64), (65, 128)):
            assert len({ops.few_plain_takes(n, m, k) for n in range(lo, hi + 1)}) == 1
