"""Refusals of the window attention, its bucket maps and the gated residual norm.

CPU only: the Python checks see fake CUDA tensors (shapes, types and strides without memory), and every
C-ABI call here is refused, or has nothing to do, before any device work.
"""
from __future__ import annotations

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import oss_cuda
from oss_cuda import _lib

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def fake(shape, dtype=BF16, device="cuda"):
    return torch.empty(shape, dtype=dtype, device=device)


def attention(**change):
    a = dict(q=fake((6, 4, 32)), k=fake((9, 2, 32)), v=fake((9, 2, 32)), q_offsets=fake(4, I32), k_offsets=fake(4, I32))
    a.update({n: c() if callable(c) else c for n, c in change.items()})
    return oss_cuda.fused_window_cross_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("q_offsets"), a.pop("k_offsets"), **a)


def bias(**change):
    b = dict(bias_table=lambda: fake((9, 4), F32), buckets=lambda: fake((3, 3), I32), q_pos=lambda: fake((6, 2), I32),
             k_pos=lambda: fake((9, 2), I32))
    b.update(change)
    return b


ATTENTION = {
    "q on the CPU": (dict(q=lambda: fake((6, 4, 32), device="cpu")), RuntimeError, "q must be CUDA"),
    "k on the CPU": (dict(k=lambda: fake((9, 2, 32), device="cpu")), RuntimeError, "k must be CUDA"),
    "two axes": (dict(q=lambda: fake((6, 32))), RuntimeError, "tokens, heads, head dim"),
    "mixed types": (dict(k=lambda: fake((9, 2, 32), F16)), RuntimeError, "one type"),
    "fp64": (dict(q=lambda: fake((6, 4, 32), torch.float64)), RuntimeError, "one type"),
    "k and v differ": (dict(v=lambda: fake((8, 2, 32))), RuntimeError, "same shape"),
    "other head dim": (dict(q=lambda: fake((6, 4, 16))), RuntimeError, "q's head dim"),
    "head dim 136": (dict(q=lambda: fake((6, 4, 136)), k=lambda: fake((9, 2, 136)), v=lambda: fake((9, 2, 136))),
                     RuntimeError, r"head dim must be in \[1, 128\]"),
    "head dim 0": (dict(q=lambda: fake((6, 4, 0)), k=lambda: fake((9, 2, 0)), v=lambda: fake((9, 2, 0))),
                   RuntimeError, r"head dim must be in \[1, 128\]"),
    "heads not a multiple": (dict(q=lambda: fake((6, 5, 32))), RuntimeError, "multiple"),
    "no heads": (dict(q=lambda: fake((6, 0, 32))), RuntimeError, "multiple"),
    "too many tokens": (dict(q=lambda: fake((1, 1, 4)).expand(2**30, 4, 4), k=lambda: fake((9, 2, 4)), v=lambda: fake((9, 2, 4))),
                        RuntimeError, "tokens"),
    "int64 offsets": (dict(q_offsets=lambda: fake(4, torch.int64)), RuntimeError, "q_offsets must be int32"),
    "offsets on the CPU": (dict(k_offsets=lambda: fake(4, I32, "cpu")), RuntimeError, "k_offsets must be CUDA"),
    "strided offsets": (dict(k_offsets=lambda: fake(8, I32)[::2]), RuntimeError, "k_offsets must be contiguous"),
    "offsets of two axes": (dict(k_offsets=lambda: fake((2, 2), I32)), RuntimeError, "windows"),
    "no offsets": (dict(q_offsets=lambda: fake(0, I32), k_offsets=lambda: fake(0, I32)), RuntimeError, "windows"),
    "offsets differ": (dict(k_offsets=lambda: fake(5, I32)), RuntimeError, "same length"),
    "scale 0": (dict(scale=0.0), ValueError, "scale"),
    "scale negative": (dict(scale=-1.0), ValueError, "scale"),
    "scale infinite": (dict(scale=math.inf), ValueError, "scale"),
    "scale NaN": (dict(scale=math.nan), ValueError, "scale"),
    "buckets alone": (dict(buckets=lambda: fake((3, 3), I32)), ValueError, "bias_table only"),
    "positions alone": (dict(q_pos=lambda: fake((6, 2), I32)), ValueError, "bias_table only"),
    "table alone": (dict(bias_table=lambda: fake((9, 4), F32)), ValueError, "needs buckets"),
    "table on the CPU": (bias(bias_table=lambda: fake((9, 4), F32, "cpu")), RuntimeError, "q's device"),
    "table of another type": (bias(bias_table=lambda: fake((9, 4), F16)), RuntimeError, "fp32 or of q's type"),
    "table of other heads": (bias(bias_table=lambda: fake((9, 2), F32)), RuntimeError, "num_buckets"),
    "table without rows": (bias(bias_table=lambda: fake((0, 4), F32)), RuntimeError, "num_buckets"),
    "int64 buckets": (bias(buckets=lambda: fake((3, 3), torch.int64)), RuntimeError, "buckets must be int32"),
    "even map": (bias(buckets=lambda: fake((3, 4), I32)), RuntimeError, "reach"),
    "large map": (bias(buckets=lambda: fake((65, 65), I32)), RuntimeError, "4096"),
    "positions of other tokens": (bias(q_pos=lambda: fake((7, 2), I32)), RuntimeError, "q_pos"),
    "positions of three axes": (bias(k_pos=lambda: fake((9, 3), I32)), RuntimeError, "k_pos"),
    "axes differ": (bias(k_pos=lambda: fake(9, I32)), RuntimeError, "number of axes"),
    "one axis, square map": (bias(q_pos=lambda: fake(6, I32), k_pos=lambda: fake(9, I32)), RuntimeError, "one axis"),
}


@pytest.mark.parametrize("case", ATTENTION)
def test_attention_refuses(case):
    change, error, message = ATTENTION[case]
    with FakeTensorMode(), pytest.raises(error, match=message):
        attention(**change)


def norm(**change):
    a = dict(x=lambda: fake((6, 48)), h=lambda: fake((6, 48)), weight=lambda: fake(48, F32))
    a.update(change)
    a = {n: c() if callable(c) else c for n, c in a.items()}
    return oss_cuda.gated_residual_norm(a.pop("x"), a.pop("h"), a.pop("weight"), **a)


NORM = {
    "kind": (dict(kind="batch"), ValueError, "kind"),
    "activation": (dict(gate=lambda: fake((6, 48)), gate_act="relu"), ValueError, "gate_act"),
    "eps negative": (dict(eps=-1e-6), ValueError, "eps"),
    "eps NaN": (dict(eps=math.nan), ValueError, "eps"),
    "eps infinite": (dict(eps=math.inf), ValueError, "eps"),
    "bias of rms": (dict(bias=lambda: fake(48, F32)), ValueError, "layer"),
    "next bias of rms": (dict(next_weight=lambda: fake(48, F32), next_bias=lambda: fake(48, F32)), ValueError, "layer"),
    "next bias alone": (dict(kind="layer", next_bias=lambda: fake(48, F32)), ValueError, "next_weight"),
    "x on the CPU": (dict(x=lambda: fake((6, 48), device="cpu")), RuntimeError, "x must be CUDA"),
    "h of another type": (dict(h=lambda: fake((6, 48), F16)), RuntimeError, "one type"),
    "fp64": (dict(x=lambda: fake((6, 48), torch.float64)), RuntimeError, "one type"),
    "h of another shape": (dict(h=lambda: fake((5, 48))), RuntimeError, "x's shape"),
    "no channels": (dict(x=lambda: fake((6, 0)), h=lambda: fake((6, 0)), weight=lambda: fake(0, F32)), RuntimeError, "8192"),
    "8193 channels": (dict(x=lambda: fake((6, 8193)), h=lambda: fake((6, 8193)), weight=lambda: fake(8193, F32)),
                      RuntimeError, "8192"),
    "scalar": (dict(x=lambda: fake(()), h=lambda: fake(()), weight=lambda: fake(1, F32)), RuntimeError, "C"),
    "gate of other channels": (dict(gate=lambda: fake((6, 24))), RuntimeError, "gate must be"),
    "gate of other rows": (dict(gate=lambda: fake((1, 48))), RuntimeError, "gate must be"),
    "no weight": (dict(weight=None), RuntimeError, "weight"),
    "weight of another size": (dict(weight=lambda: fake(47, F32)), RuntimeError, "weight must be"),
    "weight on the CPU": (dict(weight=lambda: fake(48, F32, "cpu")), RuntimeError, "weight must be"),
    "weight of another type": (dict(weight=lambda: fake(48, F16)), RuntimeError, "fp32 or x's"),
    "scale of another type": (dict(scale=lambda: fake(48, BF16)), RuntimeError, "one type"),
}


@pytest.mark.parametrize("case", NORM)
def test_norm_refuses(case):
    change, error, message = NORM[case]
    with FakeTensorMode(), pytest.raises(error, match=message):
        norm(**change)


def test_bucket_maps():
    m = oss_cuda.window_position_buckets(2, 1)
    assert m.shape == (5, 3) and m.dtype == I32 and m.flatten().tolist() == list(range(15))
    assert oss_cuda.window_position_buckets(0, 0).tolist() == [[0]]
    for reaches in ((-1, 2), (2, -1), (32, 32), (0, 2048)):
        with pytest.raises(ValueError):
            oss_cuda.window_position_buckets(*reaches)
    m = oss_cuda.log_position_buckets(8, 16).flatten()
    assert m.numel() == 33 and m.min() == 0 and m.max() == 7
    assert m[16] == 0 and m[15] == 1 and m[14] == 2 and m[0] == 3  # behind: 0 .. 3, the first two one each
    assert m[17] == 5 and m[32] == 7  # ahead: 4 .. 7
    assert (m[:17].flip(0).diff() >= 0).all() and (m[17:].diff() >= 0).all()
    m = oss_cuda.log_position_buckets(8, 64, causal=True).flatten()
    assert m[64:].eq(0).all() and m[:65].flip(0)[:4].tolist() == [0, 1, 2, 3] and m[0] == 7
    for args in ((1, 16), (2, 1), (32, 8), (32, 2048)):
        with pytest.raises(ValueError):
            oss_cuda.log_position_buckets(*args)


def last_error():
    return _lib.lib().oss_last_error().decode()


def c_forward(dtype=1, tq=4, tk=5, windows=1, heads=4, kv=2, dim=32, q=64, scale=1.0, table=None, tdtype=0, rows=9, bmap=64,
              ry=1, rx=1, pos=64, axes=2, out=64, offsets=64, scratch=None, nbytes=0):
    return _lib.lib().oss_window_attention_forward(
        dtype, tq, tk, windows, heads, kv, dim, q, heads * dim, dim, q, kv * dim, dim, q, kv * dim, dim, offsets, offsets, scale, 0,
        table, tdtype, rows, bmap, ry, rx, pos, pos, axes, out, None, None, scratch, nbytes, None)


@pytest.mark.parametrize("change, rc, message", [
    (dict(dtype=3), 1, "dtype"), (dict(tq=-1), 1, "non-negative"), (dict(windows=-1), 1, "non-negative"),
    (dict(heads=5), 1, "multiple"), (dict(heads=0), 1, "multiple"), (dict(kv=0), 1, "multiple"),
    (dict(dim=0), 1, "head dim"), (dict(dim=129), 1, "head dim"), (dict(heads=65536, kv=65536), 3, "65535"),
    (dict(tq=1 << 31), 3, "2^30"), (dict(tk=1 << 31), 3, "2^30"), (dict(windows=1 << 31), 3, "2^30"),
    (dict(scale=0.0), 1, "scale"), (dict(scale=math.inf), 1, "scale"), (dict(scale=math.nan), 1, "scale"),
    (dict(q=None), 1, "non-null"), (dict(out=None), 1, "non-null"), (dict(offsets=None), 1, "offsets"),
    (dict(table=64, tdtype=3), 1, "table dtype"), (dict(table=64, rows=0), 1, "table needs rows"),
    (dict(table=64, axes=3), 1, "axes"), (dict(table=64, rx=2048), 3, "4096"), (dict(table=64, ry=-1), 3, "4096"),
    (dict(table=64, bmap=None), 1, "bucket map"), (dict(table=64, pos=None), 1, "positions"),
])
def test_c_attention_refuses(change, rc, message):
    assert c_forward(**change) == rc and message in last_error()


def test_c_attention_scratch():
    lib = _lib.lib()
    assert c_forward(tq=0) == 0  # nothing to do
    need = lib.oss_window_attention_scratch_bytes(1, 1, 100000, 1, 4, 2, 32, 0, 0)
    assert need > 0  # a long axis is split
    assert c_forward(tq=1, tk=100000, scratch=64, nbytes=need - 1) == 4 and "scratch" in last_error()
    assert c_forward(tq=1, tk=100000, scratch=None, nbytes=need) == 4
    assert lib.oss_window_attention_scratch_bytes(7, 1, 100000, 1, 4, 2, 32, 0, 0) == 0
    assert lib.oss_window_attention_backward_scratch_bytes(7, 1, 100000, 1, 4, 2, 32, 0, 0, 0) == 0

    def backward(**change):
        a = dict(lse=64, dtable=None, dq=64, dk=64, scratch=64, nbytes=0)
        a.update(change)
        return lib.oss_window_attention_backward(
            1, 4, 5, 1, 4, 2, 32, 64, 128, 32, 64, 64, 32, 64, 64, 32, 64, 64, 1.0, 0, None, 0, 0, None, 0, 0, None, None, 1,
            64, a["lse"], None, 64, 128, 32, a["dq"], a["dk"], 64, a["dtable"], a["scratch"], a["nbytes"], None)

    assert backward(dtable=64) == 1 and "bias table" in last_error()
    assert backward(lse=None) == 1 and "lse" in last_error()
    assert backward(dq=None) == 1 and backward(dk=None) == 1
    assert backward(nbytes=lib.oss_window_attention_backward_scratch_bytes(1, 4, 5, 1, 4, 2, 32, 0, 0, 0) - 1) == 4
    assert "scratch" in last_error()


def test_c_norm_refuses():
    lib = _lib.lib()

    def forward(dtype=1, rows=4, c=48, x=64, gate=None, kind=0, act=0, eps=1e-6, pdtype=0, weight=64, next_weight=None, y=64,
                z=None, stats=None):
        return lib.oss_gated_norm_forward(dtype, rows, c, x, c, x, c, gate, c, kind, act, 0, eps, pdtype, weight, None, None,
                                          next_weight, None, y, z, stats, None)

    for change, message in (
            (dict(dtype=3), "dtype"), (dict(pdtype=-1), "parameter dtype"), (dict(rows=-1), "rows"), (dict(c=0), "channels"),
            (dict(c=8193), "channels"), (dict(kind=3), "gate kind"), (dict(act=3), "activation"), (dict(eps=-1.0), "eps"),
            (dict(eps=math.nan), "eps"), (dict(x=None), "non-null"), (dict(kind=1), "non-null"), (dict(weight=None), "weight"),
            (dict(y=None), "y must be"), (dict(z=64), "next_weight"), (dict(stats=8), "aligned")):
        assert forward(**change) == 1 and message in last_error(), change
    assert forward(rows=0) == 0
    need = lib.oss_gated_norm_backward_scratch_bytes(4, 48)
    assert need > 0 and lib.oss_gated_norm_backward_scratch_bytes(0, 48) == 0
    rc = lib.oss_gated_norm_backward(1, 4, 48, 64, 48, 64, 48, None, 0, 0, 0, 0, 1e-6, 0, 64, None, None, None, None, 64, 64, 48,
                                     None, 0, 64, 64, None, 64, None, None, None, None, 64, need - 1, None)
    assert rc == 4 and "scratch" in last_error()
