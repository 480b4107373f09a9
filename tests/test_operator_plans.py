"""Which kernels a call of the window attention goes to, as far as its scratch shows it (CPU only)."""
from __future__ import annotations

import pytest

from oss_cuda import _lib


@pytest.mark.parametrize("entries,listed", [(0, True), (961, True), (4095, False)])
def test_few_keys_are_listed_where_their_kernel_takes_them(entries, listed):
    """Two lists of windows: not where the biases of a group leave the kernels for long windows everything."""
    need = [_lib.lib().oss_window_attention_backward_scratch_bytes(1, 100, 0, w, 4, 2, 32, 0, entries, 0) for w in (1, 1 << 20)]
    assert (need[1] - need[0] > 8_000_000) == listed
