"""Borders of the logarithmic distance buckets, by whole numbers."""
from __future__ import annotations

import pytest

from oss_cuda import log_position_buckets

CASES = [(243, 144), (16, 60), (32, 128), (8, 9), (6, 2), (2, 1), (64, 2047), (24, 144), (16, 1024), (12, 216), (200, 128), (4, 625)]


@pytest.mark.parametrize("side,most", CASES)
@pytest.mark.parametrize("causal", [False, True])
def test_every_distance_is_in_its_bucket(side, most, causal):
    """Bucket near + k begins at the first distance r with (most / near)^k <= (r / near)^(side - near)."""
    near = side // 2
    if most <= near:
        with pytest.raises(ValueError):
            log_position_buckets(side if causal else 2 * side, most, causal=causal)
        return
    past = log_position_buckets(side if causal else 2 * side, most, causal=causal).flatten()[:most + 1].flip(0).tolist()
    n = side - near
    for r, b in enumerate(past):
        if r < near:
            assert b == r
        elif r == most:
            assert b == side - 1
        else:
            k = b - near
            assert most**k * near ** (n - k) <= r**n
            assert k + 1 == n or most ** (k + 1) * near ** (n - k - 1) > r**n
