"""Where projections of few tokens leave in float32 for a quantised cache's write: of more than 16 tokens smaller matrices alone (CPU)."""

import pytest

from shrike_amd.kernels import ops


@pytest.mark.parametrize("m, k, sixteen, more", [(1152, 896, True, True), (1536, 1024, True, True), (1792, 1280, True, True), (2048, 1536, True, False),
                                                 (2560, 2048, True, False), (2816, 2304, False, False)])
def test_lines(m, k, sixteen, more):
    assert all(ops.few_plain_takes(n, m, k) is sixteen for n in range(1, 17))
    assert all(ops.few_plain_takes(n, m, k) is more for n in range(17, 65))
