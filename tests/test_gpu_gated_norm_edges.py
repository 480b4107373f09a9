"""The gated residual norm at values where single ones could go wrong, against float64."""
from __future__ import annotations

import pytest
import torch

from attention_reference import F32, gated_norm
from test_gpu_gated_norm import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("c", [32, 181])
def test_far_gates_in_fp32(cuda_device, act, c):
    """Gates far on either side of 0 keep fp32's relative precision: nothing of x hides what they let through."""
    g = torch.Generator().manual_seed(c)
    rows = 64
    gate = torch.linspace(-102, 40, rows * c).view(rows, c)
    a = {"x": torch.zeros(rows, c), "h": torch.randn(rows, c, generator=g) + 2.0, "weight": torch.ones(c), "scale": None, "gate": gate}
    dy = torch.randn(rows, c, generator=g)
    got = run(cuda_device, a, act=act, dy=dy)
    want = gated_norm(a["x"], a["h"], a["weight"], gate=gate, act=act, dy=dy)
    # a row's sum of c squares and some ten roundings in y; its slope is a sum of two terms
    f = (16 + c / 8) * F32
    s = torch.sigmoid(gate.double())
    n = (want["y"] / (s * (gate.double() if act == "silu" else 1.0))).abs()
    size = {"y": want["y"].abs(), "dgate": (dy.double().abs() * n) * s * (1 + gate.double().abs() * (1 - s) if act == "silu" else 1.0)}
    for name, most in size.items():
        off = (got[name].cpu().double() - want[name]).abs()
        # 1 - s is a difference in fp32: half a step of 1 in the slope; results below 2^-126 have a fixed step
        allowed = f * most + 2.0**-140 * (1 + n)
        if name == "dgate":
            allowed = allowed + F32 * dy.double().abs() * n * s * (1 + gate.double().abs())
        assert (off <= allowed).all(), (name, float((off / allowed).max()))
