"""Addresses that the C entry points of the window attention refuse (CPU only: before any device work)."""
from __future__ import annotations

import pytest

from oss_cuda import _lib


@pytest.mark.parametrize("at", [65, 68, 72])
@pytest.mark.parametrize("dtype", [0, 1, 2, 17])
def test_scratch_off_16_bytes_is_refused(dtype, at):
    """It holds vectors of four floats and doubles."""
    lib = _lib.lib()
    need = lib.oss_window_attention_scratch_bytes(dtype, 1, 100000, 1, 4, 2, 32, 0, 0)
    assert need > 0
    rc = lib.oss_window_attention_forward(dtype, 1, 100000, 1, 4, 2, 32, 64, 128, 32, 64, 64, 32, 64, 64, 32, 64, 64, 1.0, 0, None, 0, 0,
                                          None, 0, 0, None, None, 1, 64, None, None, at, need, None)
    assert rc == 1 and "aligned" in lib.oss_last_error().decode()
    need = lib.oss_window_attention_backward_scratch_bytes(dtype, 4, 5, 1, 4, 2, 32, 0, 0, 0)
    rc = lib.oss_window_attention_backward(dtype, 4, 5, 1, 4, 2, 32, 64, 128, 32, 64, 64, 32, 64, 64, 32, 64, 64, 1.0, 0, None, 0, 0, None,
                                           0, 0, None, None, 1, 64, 64, None, 64, 128, 32, 64, 64, 64, None, at, need, None)
    assert rc == 1 and "aligned" in lib.oss_last_error().decode()
