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
from ._raster import check_no_tangent, on_device_of, stream_of
from .attention import DTYPES

KINDS = ("rms", "layer")
ACTS = {"none": 0, "sigmoid": 1, "silu": 2}
MAX_CHANNELS = 8192


def _rows(t: torch.Tensor, c: int) -> torch.Tensor:
    """t as (rows, c) with unit last stride: a view where its strides allow one."""
    if t.dim() != 2:
        t = t.reshape(-1, c)
    return t if t.stride(1) == 1 or c == 1 else t.contiguous()


def _call_args(x, h, gate, params, layer, act, eps):
    """The arguments that the forward and the backward entry points begin with."""
    rows, c = x.shape
    ptr = _lib.ptr
    weight, bias, scale, next_weight, next_bias = params
    if gate is None:
        g = (None, 0, 0)
    else:
        g = (gate.data_ptr(), gate.stride(0), 2 if gate.size(1) == c and c > 1 else 1)
    return (DTYPES[x.dtype], rows, c, x.data_ptr(), x.stride(0), h.data_ptr(), h.stride(0), *g, act, layer, eps,
            DTYPES[weight.dtype], weight.data_ptr(), ptr(bias), ptr(scale), ptr(next_weight), ptr(next_bias))


def norm_forward(x, h, gate, params, layer, act, eps, want_stats):
    """(y, z or None, stats or None) of rows."""
    with on_device_of(x):
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        z = torch.empty(x.shape, device=x.device, dtype=x.dtype) if params[3] is not None else None
        stats = torch.empty((x.size(0), 4), device=x.device, dtype=torch.float32) if want_stats else None
        rc = _lib.lib().oss_gated_norm_forward(*_call_args(x, h, gate, params, layer, act, eps), y.data_ptr(), _lib.ptr(z),
                                               _lib.ptr(stats), stream_of(x))
        if rc:
            _lib.check(rc, "oss_gated_norm_forward")
    return y, z, stats


class _GatedNorm(Function):
    @staticmethod
    def forward(ctx, x, h, gate, weight, bias, scale, next_weight, next_bias, layer, act, eps):
        params = (weight, bias, scale, next_weight, next_bias)
        y, z, stats = norm_forward(x, h, gate, params, layer, act, eps, True)
        ctx.save_for_backward(x, h, gate, *params, stats)
        ctx.meta = (layer, act, eps)
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz):
        if dy is None and dz is None:
            return (None,) * 11
        lib, ptr = _lib.lib(), _lib.ptr
        x, h, gate, *params, stats = ctx.saved_tensors
        rows, c = x.shape
        need = ctx.needs_input_grad
        with on_device_of(x):
            dev, dtype = x.device, x.dtype
            dy, dz = (None if t is None else _rows(t, c) for t in (dy, dz))
            dx = torch.empty((rows, c), device=dev, dtype=dtype) if need[0] else None
            dh = torch.empty((rows, c), device=dev, dtype=dtype) if need[1] else None
            dgate = torch.empty(gate.shape, device=dev, dtype=dtype) if need[2] else None
            dparams = [torch.empty(c, device=dev, dtype=t.dtype) if n else None for t, n in zip(params, need[3:8])]
            wanted = [ptr(t) for t in dparams]
            if dz is None:  # the second norm takes no part
                for i in (3, 4):
                    if dparams[i] is not None:
                        dparams[i].zero_()
                        wanted[i] = None
            nbytes = lib.oss_gated_norm_backward_scratch_bytes(rows, c)
            scratch = torch.empty(max(16, nbytes), device=dev, dtype=torch.uint8)
            rc = lib.oss_gated_norm_backward(*_call_args(x, h, gate, params, *ctx.meta), stats.data_ptr(), ptr(dy),
                                             0 if dy is None else dy.stride(0), ptr(dz), 0 if dz is None else dz.stride(0),
                                             ptr(dx), ptr(dh), ptr(dgate), *wanted, scratch.data_ptr(), nbytes, stream_of(x))
            if rc:
                _lib.check(rc, "oss_gated_norm_backward")
        return dx, dh, dgate, *dparams, None, None, None


def gated_residual_norm(x, h, weight, next_weight=None, *, gate=None, gate_act="none", scale=None, bias=None, next_bias=None,
                        eps=1e-6, kind="rms"):
    """y = x + scale * act(gate) * norm(h; weight, bias), and z = norm(y; next_weight, next_bias).

    x, h         (..., C), one shape and type of fp32, bf16 and fp16, C <= 8192; any strides
    weight, bias, scale, next_weight, next_bias
                 (C,) parameters of one type, fp32 or x's; only weight is required (scale 1, no biases)
    gate         (..., C) of x's type, or (..., 1): one for each row; None: 1
    gate_act     "none", "sigmoid" or "silu" of the gate; without a gate it changes nothing
    kind         "rms" (u / sqrt(mean(u^2) + eps)) or "layer" ((u - mean) / sqrt(var + eps)); biases are for "layer"

    Returns (y, z), or y alone without next_weight.  The arithmetic is fp32, each result rounded once (z is taken
    from y before it is rounded).  Differentiable once, in every tensor, in reverse mode, with the same bits on every run."""
    if kind not in KINDS:
        raise ValueError(f"kind must be one of {KINDS}, got {kind!r}")
    if gate_act not in ACTS:
        raise ValueError(f"gate_act must be one of {sorted(ACTS)}, got {gate_act!r}")
    eps = float(eps)
    if not 0.0 <= eps < 3.0e38:
        raise ValueError("eps must be non-negative and finite")
    if kind == "rms" and (bias is not None or next_bias is not None):
        raise ValueError("biases are for kind='layer'")
    if next_bias is not None and next_weight is None:
        raise ValueError("next_bias needs next_weight")
    dtype, dev, shape = x.dtype, x.device, x.shape
    for t, name in ((x, "x"), (h, "h"), (gate, "gate")):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be CUDA")
        if t.dtype is not dtype or t.device != dev or dtype not in DTYPES:
            raise RuntimeError("x, h and gate must be fp32, bf16 or fp16, of one type and device")
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_CHANNELS:
        raise RuntimeError(f"x must be (..., C) with C in [1, {MAX_CHANNELS}]")
    if h.shape != shape:
        raise RuntimeError("h must have x's shape")
    c = shape[-1]
    if gate is not None and (gate.dim() != len(shape) or gate.shape[:-1] != shape[:-1] or gate.shape[-1] not in (1, c)):
        raise RuntimeError("gate must be (..., C) or (..., 1)")
    if weight is None:
        raise RuntimeError("weight must be given")
    wtype = weight.dtype
    if wtype is not torch.float32 and wtype is not dtype:
        raise RuntimeError("parameters must be of one type, fp32 or x's")
    grad = torch.is_grad_enabled() and (x.requires_grad or h.requires_grad or (gate is not None and gate.requires_grad))
    want_grad = torch.is_grad_enabled()
    params = []
    for t, name in ((weight, "weight"), (bias, "bias"), (scale, "scale"), (next_weight, "next_weight"), (next_bias, "next_bias")):
        if t is not None:
            if t.device != dev or t.dim() != 1 or t.size(0) != c:
                raise RuntimeError(f"{name} must be (C,) on x's device")
            if t.dtype is not wtype:
                raise RuntimeError("parameters must be of one type, fp32 or x's")
            grad = grad or (want_grad and t.requires_grad)
            t = t.contiguous()
        params.append(t)
    check_no_tangent("gated_residual_norm", x, h, gate, *params)
    x2, h2 = _rows(x, c), _rows(h, c)
    g2 = None if gate is None else _rows(gate, gate.shape[-1])
    layer, act = int(kind == "layer"), ACTS[gate_act] if gate is not None else 0
    if grad:
        y, z = _GatedNorm.apply(x2, h2, g2, *params, layer, act, eps)
    else:
        y, z, _ = norm_forward(x2, h2, g2, params, layer, act, eps, False)
    if len(shape) != 2:
        y, z = y.view(shape), None if z is None else z.view(shape)
    return y if z is None else (y, z)
