"""The largest scale of the window attention (CPU only)."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oss_cuda import _lib, fused_window_cross_attention


@pytest.mark.parametrize("scale", [2.0e38, 2.9e38])
def test_scale_whose_base_2_form_is_infinite_is_refused(scale):
    """Times log2(e) it would make 0 times infinity of a score of 0."""
    with FakeTensorMode(), pytest.raises(ValueError, match="scale"):
        q, k = (torch.empty(n, 2, 16, device="cuda") for n in (3, 5))
        off = torch.empty(2, dtype=torch.int32, device="cuda")
        fused_window_cross_attention(q, k, k, off, off, scale=scale)
    lib = _lib.lib()
    rc = lib.oss_window_attention_forward(0, 4, 5, 1, 4, 2, 32, 64, 128, 32, 64, 64, 32, 64, 64, 32, 64, 64, scale, 0, None, 0, 0, None, 0, 0,
                                          None, None, 1, 64, None, None, None, 0, None)
    assert rc == 1 and "scale" in lib.oss_last_error().decode()
