"""Window attention and the gated residual norm in float64, with the error that arithmetic in
the kernels' types may leave at each value.

u is half a step of the inputs' type (torch.finfo(t).eps / 2), f = 2^-24 of fp32. First-order
bounds, in the order of the computation:

  score      a fp32 sum of dim exact products, times the scale, plus the bias: off by at most
             ds = (dim + 8) f (scale |q|.|k| + |bias|)
  weight     a relative (2 ds_max + 16 f): its own score and its row's sum; ex2.approx is 2 ulp.
             Rounded to the type before it meets v (u; fp16 below its normal range 2^-25 absolute)
  out        (u + a) sum p |v|, and u |out| for its own rounding
  delta      dout . out in fp32: the error of out, (dim + 8) f |dout|.|out|
  ds         a |ds| + p ((dim + 8) f |dout|.|v| + error of delta), u |ds| where it is rounded.
             fp16 keeps ds times a power of two that puts 2 dim max|dout| max|v| at most at 2^15,
             so its subnormal step is 2^-24 of that
  dq, dk, dv the errors of ds and p through |k|, |q|, |dout|, and the result's own rounding
  dtable     the sum of the unrounded ds errors, and the rounding to the table's type
Sums of n terms in fp32 add n f of the sum of magnitudes. SLACK covers the second order.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0**-24
SLACK = 1.05


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bias_of(table, buckets, q_pos, k_pos):
    """(Lq, Lk, H) float64 and the (Lq, Lk) rows of the table (-1: none)."""
    ry, rx = (buckets.shape[0] - 1) // 2, (buckets.shape[1] - 1) // 2
    qp, kp = q_pos.long(), k_pos.long()
    if qp.dim() == 1:
        qp, kp = torch.stack([torch.zeros_like(qp), qp], 1), torch.stack([torch.zeros_like(kp), kp], 1)
    d = kp[None] - qp[:, None]
    row = buckets.long()[d[..., 0].clamp(-ry, ry) + ry, d[..., 1].clamp(-rx, rx) + rx]
    ok = (row >= 0) & (row < table.shape[0])
    row = torch.where(ok, row, torch.full_like(row, -1))
    return torch.where(ok[..., None], table.double()[row.clamp(min=0)], torch.zeros((), dtype=torch.float64)), row


def window_attention(q, k, v, qo, ko, scale=None, causal=False, table=None, buckets=None, q_pos=None, k_pos=None, dout=None):
    """{name: (value, allowed error)} in float64 on the CPU; gradients where dout is given."""
    dtype = q.dtype
    u = half_step(dtype) if dtype != torch.float32 else F32
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    dout = None if dout is None else dout.detach().cpu().double()
    table_type = None if table is None else table.dtype
    table, buckets, q_pos, k_pos = (None if t is None else t.detach().cpu() for t in (table, buckets, q_pos, k_pos))
    tq, h, d = q.shape
    kv = k.shape[1]
    g = h // kv
    scale = d**-0.5 if scale is None else scale
    res = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in res.items()}
    if table is not None:
        res["dtable"], tol["dtable"] = torch.zeros(table.shape, dtype=torch.float64), torch.zeros(table.shape, dtype=torch.float64)
    if dout is not None:
        ds_step = 2 * d * float(dout.abs().amax()) * float(v.abs().amax()) * 2.0**-39 if tiny and min(tq, k.shape[0]) else 0.0
    for a, b, c, e in zip(qo[:-1], qo[1:], ko[:-1], ko[1:]):
        lq, lk = b - a, e - c
        if lq <= 0:
            continue
        kk, vv = k[c:e].repeat_interleave(g, 1), v[c:e].repeat_interleave(g, 1)  # (lk, h, d)
        qq = q[a:b]
        s = torch.einsum("ihd,jhd->hij", qq, kk) * scale
        size = torch.einsum("ihd,jhd->hij", qq.abs(), kk.abs()) * scale
        if table is not None:
            bias, row = bias_of(table, buckets, q_pos[a:b], k_pos[c:e])
            s = s + bias.permute(2, 0, 1)
            size = size + bias.permute(2, 0, 1).abs().nan_to_num(posinf=0.0)
        seen = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            seen = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
        s = s.masked_fill(~seen, -math.inf)
        size = torch.where(seen, size, torch.zeros_like(size))
        p = torch.softmax(s, -1).nan_to_num(nan=0.0) if lk else s
        dscore = (d + 8) * F32 * size.amax(-1, keepdim=True) if lk else size
        rel = 2 * dscore + (16 + lk) * F32
        pe = p * (rel + (u if dtype != torch.float32 else 0.0)) + torch.where(p > 0, tiny, 0.0)  # weight as it meets v
        o = torch.einsum("hij,jhd->ihd", p, vv)
        oe = torch.einsum("hij,jhd->ihd", pe, vv.abs())
        res["out"][a:b] = o
        tol["out"][a:b] = oe + u * o.abs() + tiny
        if dout is None or lk == 0:
            continue
        go = dout[a:b]
        dp = torch.einsum("ihd,jhd->hij", go, vv)
        dpe = (d + 8) * F32 * torch.einsum("ihd,jhd->hij", go.abs(), vv.abs())
        delta = (go * o).sum(-1).t()[..., None]
        deltae = ((go.abs() * (oe + u * o.abs() + tiny)).sum(-1) + (d + 8) * F32 * (go * o).abs().sum(-1)).t()[..., None]
        ds = p * (dp - delta)
        dse = rel * ds.abs() + p * (dpe + deltae + 4 * F32 * (dp.abs() + delta.abs()))
        if table is not None:
            flat, at = row.reshape(-1), row.reshape(-1) >= 0
            res["dtable"].index_add_(0, flat[at], ds.permute(1, 2, 0).reshape(-1, h)[at])
            tol["dtable"].index_add_(0, flat[at], dse.permute(1, 2, 0).reshape(-1, h)[at])
        dse = dse + (u * ds.abs() + torch.where(p > 0, ds_step, 0.0) if dtype != torch.float32 else 0.0)
        dse = dse + lk * F32 * ds.abs()
        res["dq"][a:b] = scale * torch.einsum("hij,jhd->ihd", ds, kk)
        tol["dq"][a:b] = scale * torch.einsum("hij,jhd->ihd", dse, kk.abs())
        many = g * lq * F32  # the sum over rows and heads
        grouped = lambda t: t.reshape(lk, kv, g, d).sum(2)  # noqa: E731
        res["dk"][c:e] = scale * grouped(torch.einsum("hij,ihd->jhd", ds, qq))
        tol["dk"][c:e] = scale * grouped(torch.einsum("hij,ihd->jhd", dse + many * ds.abs(), qq.abs()))
        res["dv"][c:e] = grouped(torch.einsum("hij,ihd->jhd", p, go))
        tol["dv"][c:e] = grouped(torch.einsum("hij,ihd->jhd", pe + many * p, go.abs()))
    for n in ("dq", "dk", "dv"):
        tol[n] = tol[n] + u * res[n].abs() + tiny
    if table is not None:
        tol["dtable"] = tol["dtable"] + half_step(table_type) * res["dtable"].abs() + (2.0**-25 if table_type == torch.float16 else 0.0)
    names = ["out"] + ([] if dout is None else ["dq", "dk", "dv"] + (["dtable"] if table is not None else []))
    return {n: (res[n], tol[n] * SLACK + 1e-35) for n in names}


def check(got, want, what=""):
    value, allowed = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN at other places"
    off = (got - value).abs()
    bad = (off > allowed) & ~torch.isnan(value) & ~((got == value))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float((off / allowed)[bad].max()):.3g} times the allowed error, {float(off[bad].max()):.3g}")


def gated_norm(x, h, weight, next_weight=None, gate=None, act="none", scale=None, bias=None, next_bias=None, eps=1e-6,
               kind="rms", dy=None, dz=None):
    """Values and gradients of the gated residual norm, by autograd in float64 on the CPU."""
    names = ["x", "h", "weight", "next_weight", "gate", "scale", "bias", "next_bias"]
    t = {n: None if a is None else a.detach().cpu().double().requires_grad_(True)
         for n, a in zip(names, (x, h, weight, next_weight, gate, scale, bias, next_bias))}

    def norm(v, w, b):
        m = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
        n = (v - m) / ((v - m).square().mean(-1, keepdim=True) + eps).sqrt() * w
        return n if b is None else n + b

    n = norm(t["h"], t["weight"], t["bias"])
    if t["scale"] is not None:
        n = n * t["scale"]
    if t["gate"] is not None:
        a = t["gate"]
        n = n * (a if act == "none" else torch.sigmoid(a) if act == "sigmoid" else a * torch.sigmoid(a))
    y = t["x"] + n
    res = {"y": y.detach()}
    outs, grads = [y], [torch.zeros_like(y) if dy is None else dy.detach().cpu().double()]
    if next_weight is not None:
        z = norm(y, t["next_weight"], t["next_bias"])
        res["z"] = z.detach()
        outs.append(z)
        grads.append(torch.zeros_like(z) if dz is None else dz.detach().cpu().double())
    if dy is not None or dz is not None:
        leaves = [k for k in names if t[k] is not None]
        for k, d in zip(leaves, torch.autograd.grad(outs, [t[k] for k in leaves], grads, allow_unused=True)):
            res["d" + k] = torch.zeros_like(t[k]) if d is None else d
    return res
