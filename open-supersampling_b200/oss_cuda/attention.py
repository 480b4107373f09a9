"""Window attention on the B200 kernels.

The reference exports ``fused_window_cross_attention`` as an unimplemented stub
(oss/cuda/oss_cuda/attention.py:7-11).  Here it is the attention of packed
windows: the queries of a tile over the Gaussians binned into it (the offsets
are what ``tile_bin_counting_sort`` returns), overlapping windows of an image,
a causal history of tokens, or one new token over its history, with grouped
heads and a learned relative position bias.  Forward, backward and the bias's
gradient run in liboss_b200.so; every gradient is the same bits on every run.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from ._raster import check_int_cuda, check_no_tangent, on_device_of, stream_of

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
LSE_PAIR = 16  # OSS_ATTENTION_LSE_PAIR
MAX_HEAD_DIM = 128
MAX_BIAS_ENTRIES = 4096
MAX_TOKENS = 2**30
MAX_SCALE = 2.0**127


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride along its last axis (the kernels take any other strides)."""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _bias_args(table, buckets, q_pos, k_pos):
    if table is None:
        return _NO_BIAS
    ny, nx = buckets.shape
    return (table.data_ptr(), DTYPES[table.dtype], table.size(0), buckets.data_ptr(), (ny - 1) // 2, (nx - 1) // 2,
            q_pos.data_ptr(), k_pos.data_ptr(), q_pos.dim())


_NO_BIAS = (None, 0, 0, None, 0, 0, None, None, 1)


def _call_args(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos, lse_pair=LSE_PAIR):
    """The arguments that the forward and the backward entry points begin with."""
    tq, h, d = q.shape
    tk, kv, _ = k.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    return (DTYPES[q.dtype] | lse_pair, tq, tk, q_offsets.size(0) - 1, h, kv, d, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1],
            v.data_ptr(), vs[0], vs[1], q_offsets.data_ptr(), k_offsets.data_ptr(), scale, causal,
            *_bias_args(table, buckets, q_pos, k_pos))


def attention_forward(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos, want_lse):
    """(out, and for the backward lse and what rounding took from out, or None); arguments as checked by fused_window_cross_attention."""
    lib = _lib.lib()
    with on_device_of(q):
        q, k, v = _rows(q), _rows(k), _rows(v)
        args = _call_args(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos)
        dev = q.device
        out = torch.empty(q.shape, device=dev, dtype=q.dtype)
        lse = torch.empty((2, q.size(1), q.size(0)), device=dev, dtype=torch.float32) if want_lse else None
        lo = torch.empty_like(out) if want_lse and q.dtype is not torch.float32 else None
        nbytes = lib.oss_window_attention_scratch_bytes(*args[:7], causal, 0 if table is None else buckets.numel())
        scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
        rc = lib.oss_window_attention_forward(*args, out.data_ptr(), _lib.ptr(lse), _lib.ptr(lo), _lib.ptr(scratch), nbytes,
                                               stream_of(q))
        if rc:
            _lib.check(rc, "oss_window_attention_forward")
    return out, lse, lo


def attention_backward(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos, out, lse, lo,
                       grad, want_table):
    """(d_q, d_k, d_v, d_table or None)."""
    lib = _lib.lib()
    with on_device_of(q):
        q, k, v, grad = _rows(q), _rows(k), _rows(v), _rows(grad)
        args = _call_args(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos)
        dev, dtype = q.device, q.dtype
        dq = torch.empty(q.shape, device=dev, dtype=dtype)
        dk = torch.empty(k.shape, device=dev, dtype=dtype)
        dv = torch.empty(k.shape, device=dev, dtype=dtype)
        dtable = torch.empty(table.shape, device=dev, dtype=table.dtype) if want_table else None
        nbytes = lib.oss_window_attention_backward_scratch_bytes(*args[:7], causal, 0 if table is None else buckets.numel(),
                                                                 table.size(0) if want_table else 0)
        scratch = torch.empty(max(1, nbytes), device=dev, dtype=torch.uint8)
        gs = grad.stride()
        rc = lib.oss_window_attention_backward(*args, out.data_ptr(), lse.data_ptr(), _lib.ptr(lo), grad.data_ptr(), gs[0], gs[1],
                                               dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(dtable),
                                               scratch.data_ptr(), nbytes, stream_of(q))
        if rc:
            _lib.check(rc, "oss_window_attention_backward")
    return dq, dk, dv, dtable


class _WindowAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos):
        out, lse, lo = attention_forward(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos,
                                         any(ctx.needs_input_grad))
        ctx.save_for_backward(q, k, v, q_offsets, k_offsets, table, buckets, q_pos, k_pos, out, lse, lo)
        ctx.meta = (scale, causal)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, q_offsets, k_offsets, table, buckets, q_pos, k_pos, out, lse, lo = ctx.saved_tensors
        scale, causal = ctx.meta
        need = ctx.needs_input_grad
        dq, dk, dv, dtable = attention_backward(q, k, v, q_offsets, k_offsets, scale, causal, table, buckets, q_pos, k_pos,
                                                out, lse, lo, grad, table is not None and need[7])
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None, dtable,
                None, None, None)


def _check_bias(q, k, bias_table, buckets, q_pos, k_pos):
    if bias_table is None:
        if buckets is not None or q_pos is not None or k_pos is not None:
            raise ValueError("buckets, q_pos and k_pos apply with bias_table only")
        return
    if buckets is None or q_pos is None or k_pos is None:
        raise ValueError("bias_table needs buckets, q_pos and k_pos")
    if not bias_table.is_cuda or bias_table.device != q.device:
        raise RuntimeError("bias_table must be on q's device")
    if bias_table.dtype not in (torch.float32, q.dtype):
        raise RuntimeError("bias_table must be fp32 or of q's type")
    if bias_table.dim() != 2 or bias_table.size(0) < 1 or bias_table.size(1) != q.size(1):
        raise RuntimeError("bias_table must be (num_buckets, H)")
    for t, name in ((buckets, "buckets"), (q_pos, "q_pos"), (k_pos, "k_pos")):
        check_int_cuda(t, name)
        if t.device != q.device:
            raise RuntimeError(f"{name} must be on q's device")
    if buckets.dim() != 2 or buckets.size(0) % 2 == 0 or buckets.size(1) % 2 == 0:
        raise RuntimeError("buckets must be (2 * reach_y + 1, 2 * reach_x + 1)")
    if buckets.numel() > MAX_BIAS_ENTRIES:
        raise RuntimeError(f"buckets must have at most {MAX_BIAS_ENTRIES} entries")
    for t, name, n in ((q_pos, "q_pos", q.size(0)), (k_pos, "k_pos", k.size(0))):
        if t.dim() not in (1, 2) or t.size(0) != n or (t.dim() == 2 and t.size(1) != 2):
            raise RuntimeError(f"{name} must be ({name[0].upper()},) or ({name[0].upper()}, 2)")
    if q_pos.dim() != k_pos.dim():
        raise RuntimeError("q_pos and k_pos must have the same number of axes")
    if q_pos.dim() == 1 and buckets.size(0) != 1:
        raise RuntimeError("positions of one axis need buckets of shape (1, 2 * reach + 1)")


def fused_window_cross_attention(q, k, v, q_offsets, k_offsets, *, scale=None, causal=False, bias_table=None, buckets=None,
                                 q_pos=None, k_pos=None):
    """Softmax attention inside packed windows: (Tq, H, D).

    q            (Tq, H, D); k, v (Tk, Hkv, D): one type of fp32, bf16 and fp16, D <= 128, any strides.
                 H is a multiple of Hkv; query head h reads key head h // (H // Hkv).
    q_offsets, k_offsets
                 (W + 1,) int32 on the device, non-decreasing: window w holds queries
                 [q_offsets[w], q_offsets[w + 1]) and keys [k_offsets[w], k_offsets[w + 1]).  They are not
                 read on the host, so nothing synchronises and the call can be captured in a CUDA graph
                 (values outside the tensors are clamped).  Windows may be empty on either side.
    scale        of the scores, positive, at most 2**127; default D ** -0.5
    causal       query i of a window sees key j where j <= i + (keys - queries): the last query sees all
    bias_table   (num_buckets, H), fp32 or of q's type: bias_table[buckets[clamp(k_pos[j] - q_pos[i])], h] is
                 added to the scaled score (minus infinity leaves a key no weight, the lowest finite value only
                 lowers it).  buckets is (2 ry + 1, 2 rx + 1) int32 of at most 4096 entries
                 (window_position_buckets, log_position_buckets; an entry outside the table adds no bias),
                 q_pos (Tq, 2) and k_pos (Tk, 2) int32 (y, x), or (Tq,) and (Tk,) with a (1, 2 r + 1) map.

    A query that sees no key (or only keys whose score is minus infinity), or lies outside every window, gives
    zeros.  Differentiable once, in q, k, v and bias_table, in reverse mode, with the same bits on every run.
    Scores, softmax and sums are held in fp32; with 16-bit inputs the weights are rounded to their type before
    they meet v.  Where a gradient is wanted, long windows of those types also multiply what that rounding took,
    so that out's last bit may differ from a call without.  A value that is not finite reaches only the rows
    whose window and causal mask show it.  To capture a backward into a graph, drop earlier eager graphs of the
    same leaves first."""
    dtype, dev, qs, ks = q.dtype, q.device, q.shape, k.shape
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be CUDA")
        if t.dim() != 3:
            raise RuntimeError(f"{name} must be (tokens, heads, head dim)")
        if t.dtype is not dtype or t.device != dev or dtype not in DTYPES:
            raise RuntimeError("q, k and v must be fp32, bf16 or fp16, of one type and device")
    if ks != v.shape or ks[2] != qs[2]:
        raise RuntimeError("k and v must have the same shape and q's head dim")
    if not 1 <= qs[2] <= MAX_HEAD_DIM:
        raise RuntimeError(f"head dim must be in [1, {MAX_HEAD_DIM}]")
    if ks[1] < 1 or qs[1] < 1 or qs[1] % ks[1] != 0:
        raise RuntimeError("the heads of q must be a multiple of those of k")
    if qs[0] >= MAX_TOKENS or ks[0] >= MAX_TOKENS:
        raise RuntimeError("at most 2**30 - 1 tokens")
    for t, name in ((q_offsets, "q_offsets"), (k_offsets, "k_offsets")):
        check_int_cuda(t, name)
        if t.dim() != 1 or t.size(0) < 1 or t.device != dev:
            raise RuntimeError(f"{name} must be (windows + 1,) on q's device")
    if q_offsets.size(0) != k_offsets.size(0):
        raise RuntimeError("q_offsets and k_offsets must have the same length")
    if bias_table is not None or buckets is not None or q_pos is not None or k_pos is not None:
        _check_bias(q, k, bias_table, buckets, q_pos, k_pos)
    scale = 1.0 / math.sqrt(qs[2]) if scale is None else float(scale)
    if not 0.0 < scale <= MAX_SCALE:
        raise ValueError("scale must be positive, at most 2**127")
    check_no_tangent("fused_window_cross_attention", q, k, v, bias_table)
    if bias_table is not None:
        bias_table = bias_table.contiguous()
    args = (q, k, v, q_offsets, k_offsets, scale, int(bool(causal)), bias_table, buckets, q_pos, k_pos)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (bias_table is not None and bias_table.requires_grad)):
        return _WindowAttention.apply(*args)
    return attention_forward(*args, False)[0]


def window_position_buckets(reach_y: int, reach_x: int, device=None) -> torch.Tensor:
    """One bucket for each offset (dy, dx) with |dy| <= reach_y and |dx| <= reach_x (offsets beyond share the
    nearest): the (2 reach_y + 1, 2 reach_x + 1) int32 map of a table of as many rows."""
    reach_y, reach_x = int(reach_y), int(reach_x)
    ny, nx = 2 * reach_y + 1, 2 * reach_x + 1
    if reach_y < 0 or reach_x < 0 or ny * nx > MAX_BIAS_ENTRIES:
        raise ValueError(f"reaches must be non-negative with at most {MAX_BIAS_ENTRIES} offsets")
    return torch.arange(ny * nx, device=device, dtype=torch.int32).view(ny, nx)


def log_position_buckets(num_buckets: int, max_distance: int, causal: bool = False, device=None) -> torch.Tensor:
    """Buckets of a distance along one axis, the (1, 2 max_distance + 1) int32 map: one for each of the nearest
    distances, then ever wider ones (in the logarithm of the distance) up to max_distance and beyond.  causal:
    all buckets are for keys at or before the query; otherwise half of them are for keys behind it."""
    num_buckets, max_distance = int(num_buckets), int(max_distance)
    side = num_buckets if causal else num_buckets // 2
    near = side // 2
    if near < 1 or max_distance <= near or 2 * max_distance + 1 > MAX_BIAS_ENTRIES:
        raise ValueError("needs at least 2 buckets a side, max_distance above half of them and at most 2047")
    wide = side - near
    r = torch.arange(max_distance + 1, dtype=torch.float64)
    steps = (r.clamp(min=1) / near).log() / math.log(max_distance / near) * wide
    # a distance beside a border is told by whole numbers: (max / near)^k <= (r / near)^wide
    for i in ((steps - steps.round()).abs() < 1e-9).nonzero().flatten().tolist():
        k = round(float(steps[i]))
        if i > near:
            steps[i] = k if max_distance**k * near ** (wide - k) <= i**wide else k - 1
    b = torch.where(r < near, r, (near + steps.floor()).clamp(max=side - 1)).to(torch.int32)
    after = torch.zeros_like(b) if causal else b + side
    return torch.cat([b.flip(0), after[1:]]).view(1, -1).to(device)
