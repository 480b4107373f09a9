"""The norms before and after a block, fused with its gate and residual scale.

A block of the canvas model ends in ``y = x + scale * act(gate) * norm(h)``
and the next one begins with ``norm(y)``; ``gated_residual_norm`` is both in
one kernel of liboss_b200.so, and their backward in two.
"""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from ._raster import stream_of
from .attention import DTYPES

KINDS = ("rms", "layer")
ACTS = {"none": 0, "sigmoid": 1, "silu": 2}
MAX_CHANNELS = 8192


def _rows(t: torch.Tensor, c: int) -> torch.Tensor:
    """t as (rows, c) with unit last stride: a view where its strides allow one."""
    t = t.reshape(-1, c)
    return t if t.stride(1) == 1 or c == 1 else t.contiguous()


def _ptr_stride(t):
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


def _gate_kind(gate, c):
    return 0 if gate is None else 2 if gate.size(1) == c and c > 1 else 1


class _GatedNorm(Function):
    @staticmethod
    def forward(ctx, x, h, gate, weight, bias, scale, next_weight, next_bias, layer, act, eps):
        lib = _lib.lib()
        rows, c = x.shape
        params = (weight, bias, scale, next_weight, next_bias)
        with torch.cuda.device(x.device):
            y = torch.empty((rows, c), device=x.device, dtype=x.dtype)
            z = torch.empty_like(y) if next_weight is not None else None
            stats = torch.empty((rows, 4), device=x.device, dtype=torch.float32) if any(ctx.needs_input_grad) else None
            _lib.check(
                lib.oss_gated_norm_forward(DTYPES[x.dtype], rows, c, *_ptr_stride(x), *_ptr_stride(h), *_ptr_stride(gate),
                                           _gate_kind(gate, c), act, layer, eps, DTYPES[weight.dtype],
                                           *(_lib.ptr(t) for t in params), y.data_ptr(), _lib.ptr(z), _lib.ptr(stats),
                                           stream_of(x)),
                "oss_gated_norm_forward",
            )
        ctx.save_for_backward(x, h, gate, *params, stats)
        ctx.meta = (layer, act, eps)
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz):
        if dy is None and dz is None:
            return (None,) * 11
        lib = _lib.lib()
        x, h, gate, *params, stats = ctx.saved_tensors
        layer, act, eps = ctx.meta
        rows, c = x.shape
        need = ctx.needs_input_grad
        with torch.cuda.device(x.device):
            dy, dz = (None if t is None else _rows(t, c) for t in (dy, dz))
            dx, dh = (torch.empty((rows, c), device=x.device, dtype=x.dtype) if n else None for n in need[:2])
            dgate = torch.empty(gate.shape, device=x.device, dtype=x.dtype) if need[2] else None
            dparams = [torch.empty_like(t) if n else None for t, n in zip(params, need[3:8])]
            # without dz the second norm takes no part
            zeros = [i for i in (3, 4) if dz is None and dparams[i] is not None]
            for i in zeros:
                dparams[i].zero_()
            nbytes = lib.oss_gated_norm_backward_scratch_bytes(rows, c)
            scratch = torch.empty((max(16, nbytes),), device=x.device, dtype=torch.uint8)
            _lib.check(
                lib.oss_gated_norm_backward(DTYPES[x.dtype], rows, c, *_ptr_stride(x), *_ptr_stride(h), *_ptr_stride(gate),
                                            _gate_kind(gate, c), act, layer, eps, DTYPES[params[0].dtype],
                                            *(_lib.ptr(t) for t in params), stats.data_ptr(), *_ptr_stride(dy),
                                            *_ptr_stride(dz), _lib.ptr(dx), _lib.ptr(dh), _lib.ptr(dgate),
                                            *(None if i in zeros else _lib.ptr(t) for i, t in enumerate(dparams)),
                                            scratch.data_ptr(), scratch.numel(), stream_of(x)),
                "oss_gated_norm_backward",
            )
        return dx, dh, dgate, *dparams, None, None, None


def gated_residual_norm(x, h, weight, next_weight=None, *, gate=None, gate_act="none", scale=None, bias=None, next_bias=None,
                        eps=1e-6, kind="rms"):
    """y = x + scale * act(gate) * norm(h; weight, bias), and z = norm(y; next_weight, next_bias).

    x, h         (..., C), one shape and type of fp32, bf16 and fp16, C <= 8192; any strides
    weight, bias, scale, next_weight, next_bias
                 (C,) parameters of one type, fp32 or x's; only weight is required (scale 1, no biases)
    gate         (..., C) of x's type, or (..., 1): one for each row; None: 1
    gate_act     "none", "sigmoid" or "silu" of the gate
    kind         "rms" (u / sqrt(mean(u^2) + eps)) or "layer" ((u - mean) / sqrt(var + eps)); biases are for "layer"

    Returns (y, z), or y alone without next_weight.  The arithmetic is fp32, each result rounded once (z is taken
    from y before it is rounded).  Differentiable once, in every tensor, with the same bits on every run."""
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {KINDS}, got {kind!r}")
    if gate_act not in ACTS:
        raise ValueError(f"gate_act must be one of {sorted(ACTS)}, got {gate_act!r}")
    if gate is None and gate_act != "none":
        raise ValueError("gate_act applies with gate only")
    eps = float(eps)
    if not 0.0 <= eps < 3.0e38:
        raise ValueError("eps must be non-negative and finite")
    if kind == "rms" and (bias is not None or next_bias is not None):
        raise ValueError("biases are for kind='layer'")
    if next_bias is not None and next_weight is None:
        raise ValueError("next_bias needs next_weight")
    for t, name in ((x, "x"), (h, "h"), (gate, "gate")):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be CUDA")
        if t.dtype not in DTYPES or t.dtype != x.dtype or t.device != x.device:
            raise RuntimeError("x, h and gate must be fp32, bf16 or fp16, of one type and device")
    if x.dim() < 1 or not 1 <= x.size(-1) <= MAX_CHANNELS:
        raise RuntimeError(f"x must be (..., C) with C in [1, {MAX_CHANNELS}]")
    if h.shape != x.shape:
        raise RuntimeError("h must have x's shape")
    c = x.size(-1)
    if gate is not None and (gate.dim() != x.dim() or gate.shape[:-1] != x.shape[:-1] or gate.size(-1) not in (1, c)):
        raise RuntimeError("gate must be (..., C) or (..., 1)")
    for t, name in ((weight, "weight"), (next_weight, "next_weight"), (scale, "scale"), (bias, "bias"),
                    (next_bias, "next_bias")):
        if t is None:
            if name == "weight":
                raise RuntimeError("weight must be given")
            continue
        if t.device != x.device or t.dim() != 1 or t.size(0) != c:
            raise RuntimeError(f"{name} must be (C,) on x's device")
        if t.dtype not in (torch.float32, x.dtype) or t.dtype != weight.dtype:
            raise RuntimeError("parameters must be of one type, fp32 or x's")
    g = None if gate is None else _rows(gate, gate.size(-1))
    params = [None if t is None else t.contiguous() for t in (weight, bias, scale, next_weight, next_bias)]
    y, z = _GatedNorm.apply(_rows(x, c), _rows(h, c), g, *params, int(kind == "layer"), ACTS[gate_act], eps)
    return (y.view(x.shape), z.view(x.shape)) if z is not None else y.view(x.shape)
