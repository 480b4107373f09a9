"""Forward-mode derivatives of the window attention and the gated residual norm: refused, not dropped (fake CUDA tensors)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

from oss_cuda import fused_window_cross_attention, gated_residual_norm


def fake(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("which", ["q", "k", "v", "bias_table"])
@pytest.mark.parametrize("no_grad", [False, True])
def test_attention_refuses_a_tangent(which, no_grad):
    with FakeTensorMode(), forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        a = dict(q=fake(6, 4, 32), k=fake(9, 2, 32), v=fake(9, 2, 32), bias_table=fake(9, 4))
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        off = fake(4, dtype=torch.int32)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fused_window_cross_attention(a["q"], a["k"], a["v"], off, off, bias_table=a["bias_table"], buckets=fake(3, 3, dtype=torch.int32),
                                         q_pos=fake(6, 2, dtype=torch.int32), k_pos=fake(9, 2, dtype=torch.int32))


@pytest.mark.parametrize("which", ["x", "h", "gate", "weight", "scale", "bias", "next_weight", "next_bias"])
def test_norm_refuses_a_tangent(which):
    with FakeTensorMode(), forward_ad.dual_level():
        a = {n: fake(6, 48) for n in ("x", "h", "gate")} | {n: fake(48) for n in ("weight", "scale", "bias", "next_weight", "next_bias")}
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_residual_norm(a.pop("x"), a.pop("h"), a.pop("weight"), kind="layer", **a)
