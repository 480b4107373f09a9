"""Cases of the window attention, its relative position bias and the gated residual norm.

Each case is one call (or one forward and backward) of an operator at a size that the canvas
model around the rasterizer meets: the 16-pixel tiles of 540p and 1080p frames with the
Gaussians binned into them, windows that overlap, histories of frames, single tokens.
"""
from __future__ import annotations

import math
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a whole 1080p frame served: every 16x16 tile's pixels attend to the Gaussians of that tile (200k of them)
        attention("1080p tiles, forward", "bf16", lengths="tiles", windows=8160, lq=256, lk=24, heads=4, kv_heads=2, dim=32),
        # training on a 540p frame: 2040 tiles, few Gaussians each, with a learned bias by their offset in pixels
        attention("540p tiles, training", "bf16", lengths="tiles", windows=2040, lq=256, lk=8, heads=4, kv_heads=4, dim=32,
                  bias="window", side=16, margin=0, train=True),
        # windows of 16x16 over keys of the 24x24 around them: head size 30 fills no vector
        attention("overlapping windows, training", "fp16", lengths="even", windows=135, lq=256, lk=576, heads=6, kv_heads=6,
                  dim=30, bias="window", side=16, margin=4, train=True),
        # packed token histories of very different lengths, causal, grouped heads, logarithmic buckets
        attention("packed histories, training", "bf16", lengths="histories", windows=7, lq=4095, lk=4095, heads=8, kv_heads=2,
                  dim=64, causal=True, bias="log", train=True),
        # one long history taken in at once: the tile tokens of eight 540p frames
        attention("long history, forward", "bf16", lengths="even", windows=1, lq=16320, lk=16320, heads=8, kv_heads=2, dim=128,
                  causal=True),
        # one new token for each of 68 streams over their histories
        attention("single tokens, forward", "bf16", lengths="ragged", windows=68, lq=1, lk=8160, heads=16, kv_heads=2, dim=128,
                  causal=True),
        # the least a call can do: latency
        attention("few windows, training", "fp32", lengths="ragged", windows=6, lq=40, lk=60, heads=2, kv_heads=2, dim=16,
                  bias="window", side=16, margin=0, train=True),
        # 32-bit training as the renderer trains: 8x8 queries over the 12x12 around them
        attention("32-bit windows, training", "fp32", lengths="even", windows=510, lq=64, lk=144, heads=4, kv_heads=4, dim=32,
                  train=True),
        # single tokens through a block's end: latency
        norm("few rows, forward", "bf16", rows=17, channels=256, gate="full", act="sigmoid"),
        # every pixel token of a 540p frame
        norm("540p pixels, forward", "bf16", rows=522240, channels=128, gate="full", act="none"),
        # training over the tile tokens of sixteen 540p frames
        norm("frame tokens, training", "bf16", rows=32640, channels=1024, gate="full", act="silu", train=True),
        # odd sizes in 32 bits, layer norms with biases, one gate a token
        norm("odd rows, training", "fp32", rows=4097, channels=181, gate="row", act="sigmoid", kind="layer", train=True),
    ]


def attention(name, dtype, lengths, windows, lq, lk, heads, kv_heads, dim, causal=False, bias="none", side=0, margin=0, train=False):
    return {"name": name, "op": "attention", "dtype": dtype, "lengths": lengths, "windows": windows, "lq": lq, "lk": lk,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal, "bias": bias, "side": side, "margin": margin,
            "train": train}


def norm(name, dtype, rows, channels, gate, act, kind="rms", train=False):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "channels": channels, "gate": gate, "act": act,
            "kind": kind, "train": train}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.3:
        train = rng.random() < 0.5
        channels = _spread(rng, 16, 4096)
        rows = _spread(rng, 1, min(522240, 20_000_000 // channels))
        c = norm("", rng.choice(["bf16", "fp16", "fp32"]), rows, channels, rng.choice(["full", "row", "none"]),
                 rng.choice(["none", "sigmoid", "silu"]), rng.choice(["rms", "layer"]), train)
    else:
        what = rng.choice(["tiles", "windows", "histories", "single"])
        dtype = rng.choice(["bf16", "fp16", "fp32"] if what != "histories" else ["bf16", "fp16"])
        kv_heads = rng.choice([1, 2, 3, 4])
        heads = kv_heads * rng.choice([1, 2, 4])
        dim = rng.choice([16, 20, 30, 32, 48, 64, 80, 128])
        train = rng.random() < 0.5
        if what == "tiles":
            c = attention("", dtype, "tiles", _spread(rng, 4, 1000), rng.choice([16, 64, 256]), _spread(rng, 4, 90), heads,
                          kv_heads, dim, bias=rng.choice(["none", "window"]), side=16, train=train)
        elif what == "windows":
            side, margin = rng.choice([4, 7, 8, 12, 16]), rng.choice([0, 2, 4])
            c = attention("", dtype, "even", _spread(rng, 1, 120), side * side, (side + 2 * margin) ** 2, heads, kv_heads, dim,
                          bias=rng.choice(["none", "window"]), side=side, margin=margin, train=train)
        elif what == "histories":
            n = _spread(rng, 33, 4000)
            c = attention("", dtype, "histories", rng.randrange(1, 7), n, n, heads, kv_heads, dim, causal=True,
                          bias=rng.choice(["none", "log"]), train=train)
        else:
            c = attention("", dtype, "ragged", _spread(rng, 1, 130), 1, _spread(rng, 2, 8160), heads, kv_heads, dim, causal=True,
                          bias=rng.choice(["none", "log"]))
    del c["name"]
    return c


# ------------------------------------------------------------------ sizes (from the case alone)
LOG_BUCKETS, LOG_DISTANCE = 32, 128


def _lengths(case):
    """Queries and keys of each window."""
    s, lq, lk = case["windows"], case["lq"], case["lk"]
    r = np.random.RandomState(1234567)
    if case["lengths"] == "even":
        return np.full(s, lq), np.full(s, lk)
    if case["lengths"] == "tiles":  # Gaussians fall into tiles unevenly, into some not at all
        density = r.gamma(2.0, 0.5, s)
        return np.full(s, lq), np.minimum(r.poisson(density * lk), 8 * lk)
    if case["lengths"] == "histories":  # the longest, then shorter and shorter ones, to a single token
        n = np.array([max(1, lq >> (2 * i if i > 2 else i)) for i in range(s)])
        return n, n
    q = np.ones(s, dtype=np.int64) if lq == 1 else r.randint(0, lq + 1, s)  # ragged
    k = r.randint(max(1, lk // 8), lk + 1, s)
    q[0], k[0] = lq, lk
    return q, k


def _pairs(case):
    q, k = (x.astype(np.float64) for x in _lengths(case))
    if not case["causal"]:
        return float((q * k).sum())
    # row i of a window sees k - q + 1 + i keys, none where that is negative
    first = k - q + 1
    hidden = np.minimum(np.maximum(1 - first, 0), q)
    return float(((q - hidden) * (np.maximum(first, 1) + k) / 2).sum())


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        t, c = case["rows"], case["channels"]
        g = {"full": t * c, "row": t, "none": 0}[case["gate"]]
        vectors = (3 if case["kind"] == "rms" else 5) * c * 4
        if not case["train"]:
            return {"bytes": e * (4.0 * t * c + g) + vectors, "flops": 12.0 * t * c}
        return {"bytes": e * (8.0 * t * c + 2.0 * g) + 2 * vectors, "flops": 40.0 * t * c}
    q, k = _lengths(case)
    tq, tk = int(q.sum()), int(k.sum())
    d, h, kv = case["dim"], case["heads"], case["kv_heads"]
    pos = 0 if case["bias"] == "none" else (tq + tk) * (8 if case["bias"] == "window" else 4)
    once = e * (2.0 * tq * h * d + 2.0 * tk * kv * d)
    return {"bytes": (2 if case["train"] else 1) * once + pos, "flops": (14.0 if case["train"] else 4.0) * d * h * _pairs(case)}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def randn(*shape, dtype=dtype, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    st = {"case": case}
    if case["op"] == "norm":
        t, c = case["rows"], case["channels"]
        st["x"], st["h"] = randn(t, c), randn(t, c, scale=2.0, shift=0.1)
        st["gate"] = None if case["gate"] == "none" else randn(t, c if case["gate"] == "full" else 1)
        st["weight"] = randn(c, dtype=torch.float32, scale=0.2, shift=1.0)
        st["next_weight"] = randn(c, dtype=torch.float32, scale=0.2, shift=1.0)
        st["scale"] = randn(c, dtype=torch.float32, scale=0.1, shift=0.3)
        layer = case["kind"] == "layer"
        st["bias"] = randn(c, dtype=torch.float32, scale=0.1) if layer else None
        st["next_bias"] = randn(c, dtype=torch.float32, scale=0.1) if layer else None
        names = ["x", "h", "gate", "weight", "next_weight", "scale", "bias", "next_bias"]
        if case["train"]:
            st["dy"], st["dz"] = randn(t, c), randn(t, c)
    else:
        ql, kl = _lengths(case)
        qo, ko = np.concatenate([[0], np.cumsum(ql)]), np.concatenate([[0], np.cumsum(kl)])
        tq, tk, d = int(qo[-1]), int(ko[-1]), case["dim"]
        # logits of a trained model spread by more than 1 where it has learned to look
        st["q"] = randn(tq, case["heads"], d, scale=1.5)
        st["k"], st["v"] = randn(tk, case["kv_heads"], d), randn(tk, case["kv_heads"], d)
        st["q_offsets"] = torch.tensor(qo, dtype=torch.int32, device="cuda")
        st["k_offsets"] = torch.tensor(ko, dtype=torch.int32, device="cuda")
        st["longest"] = (int(ql.max()), int(kl.max()))
        names = ["q", "k", "v"]
        st["bias_table"] = st["buckets"] = st["q_pos"] = st["k_pos"] = None
        if case["bias"] == "window":
            side, margin = case["side"], case["margin"]
            reach = side - 1 + margin
            n = 2 * reach + 1
            st["buckets"] = torch.arange(n * n, dtype=torch.int32, device="cuda").view(n, n)
            st["bias_table"] = randn(n * n, case["heads"], scale=0.5)
            st["q_pos"] = _grid(tq, st["q_offsets"], side, 0)
            if case["lengths"] == "even":
                st["k_pos"] = _grid(tk, st["k_offsets"], side + 2 * margin, -margin)
            else:  # Gaussians anywhere in their tile
                st["k_pos"] = torch.randint(0, side, (tk, 2), generator=gen, device="cuda", dtype=torch.int32)
            names.append("bias_table")
        elif case["bias"] == "log":
            st["buckets"] = _log_buckets().cuda()
            st["bias_table"] = randn(LOG_BUCKETS, case["heads"], scale=0.5)
            st["k_pos"] = _within(tk, st["k_offsets"]).int()
            # queries are the last tokens of their history
            behind = (st["k_offsets"].diff() - st["q_offsets"].diff())[_window_of(tq, st["q_offsets"])]
            st["q_pos"] = (_within(tq, st["q_offsets"]) + behind).int()
            names.append("bias_table")
        if case["train"]:
            st["dout"] = randn(tq, case["heads"], d)
    st["leaves"] = [n for n in names if st[n] is not None]
    if case["train"]:
        for n in st["leaves"]:
            st[n].requires_grad_(True)
    return st


def _window_of(t, offsets):
    return (torch.searchsorted(offsets, torch.arange(t, device=offsets.device, dtype=torch.int32), right=True) - 1).long()


def _within(t, offsets):
    return torch.arange(t, device=offsets.device) - offsets.long()[_window_of(t, offsets)]


def _grid(t, offsets, side, start):
    """(y, x) of each token in its window of `side` columns."""
    i = _within(t, offsets)
    return torch.stack([i // side + start, i % side + start], dim=1).int()


def _log_buckets():
    """One bucket for each of the nearest past distances, then ever wider ones up to the last; the future is never seen."""
    past = torch.arange(LOG_DISTANCE, -1, -1, dtype=torch.float64)
    near = LOG_BUCKETS // 2
    far = near + (past.clamp(min=1) / near).log() / math.log(LOG_DISTANCE / near) * (LOG_BUCKETS - near)
    b = torch.where(past < near, past, far.floor().clamp(max=LOG_BUCKETS - 1))
    return torch.cat([b, torch.zeros(LOG_DISTANCE, dtype=torch.float64)]).int().view(1, -1)


# ------------------------------------------------------------------ one pass
def run(st):
    return run_norm(st) if st["case"]["op"] == "norm" else run_attention(st)


def _package():
    if "open-supersampling_b200" not in sys.path:
        sys.path.insert(0, "open-supersampling_b200")
    import oss_cuda

    return oss_cuda


def run_attention(st):
    case = st["case"]
    if own:
        out = _package().fused_window_cross_attention(
            st["q"], st["k"], st["v"], st["q_offsets"], st["k_offsets"], causal=case["causal"], bias_table=st["bias_table"],
            buckets=st["buckets"], q_pos=st["q_pos"], k_pos=st["k_pos"])
        if not case["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, [st[n] for n in st["leaves"]], st["dout"])
        return {"out": out.detach(), **{"d_" + n: g for n, g in zip(st["leaves"], grads)}}
    with torch.no_grad():
        return plain_attention(st)


def run_norm(st):
    case = st["case"]
    if own:
        y, z = _package().gated_residual_norm(
            st["x"], st["h"], st["weight"], st["next_weight"], gate=st["gate"], gate_act=case["act"], scale=st["scale"],
            bias=st["bias"], next_bias=st["next_bias"], eps=1e-6, kind=case["kind"])
        if not case["train"]:
            return {"y": y, "z": z}
        grads = torch.autograd.grad([y, z], [st[n] for n in st["leaves"]], [st["dy"], st["dz"]])
        return {"y": y.detach(), "z": z.detach(), **{"d_" + n: g for n, g in zip(st["leaves"], grads)}}
    with torch.no_grad():
        return plain_norm(st)


# ------------------------------------------------------------------ plain forms: 32 bits, rounded at the end
def plain_attention(st):
    case = st["case"]
    q, k, v, qo, ko = st["q"], st["k"], st["v"], st["q_offsets"].long(), st["k_offsets"].long()
    (tq, h, d), kv, s = q.shape, k.shape[1], qo.numel() - 1
    nq, nk = max(1, st["longest"][0]), max(1, st["longest"][1])
    aq, ak = torch.arange(nq, device=q.device), torch.arange(nk, device=q.device)
    lq, lk = qo.diff(), ko.diff()
    iq = (qo[:-1, None] + aq).clamp(max=max(tq - 1, 0))
    ik = (ko[:-1, None] + ak).clamp(max=max(k.shape[0] - 1, 0))
    mine_q, mine_k = aq < lq[:, None], ak < lk[:, None]
    seen = mine_q[:, :, None] & mine_k[:, None, :]  # (s, nq, nk)
    if case["causal"]:
        seen = seen & (ak[None, None, :] <= aq[None, :, None] + (lk - lq)[:, None, None])
    # (s, kv, g, nq, d) against (s, kv, 1, nk, d)
    qf = (q[iq].float() * mine_q[:, :, None, None]).view(s, nq, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    kf = (k[ik].float() * mine_k[:, :, None, None]).permute(0, 2, 1, 3).unsqueeze(2)
    vf = (v[ik].float() * mine_k[:, :, None, None]).permute(0, 2, 1, 3).unsqueeze(2)
    scale = 1.0 / math.sqrt(d)
    logits = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    if st["bias_table"] is not None:
        bucket = plain_bucket(st["buckets"], st["q_pos"], st["k_pos"], iq, ik)  # (s, nq, nk)
        logits += st["bias_table"].float()[bucket].view(s, nq, nk, kv, h // kv).permute(0, 3, 4, 1, 2)
    logits.masked_fill_(~seen[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del logits
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    back_q = _window_of(tq, st["q_offsets"]) * nq + _within(tq, st["q_offsets"])
    back_k = _window_of(k.shape[0], st["k_offsets"]) * nk + _within(k.shape[0], st["k_offsets"])

    def rows(t, n, back):  # (s, kv, g, n, d) to packed rows of heads
        return t.permute(0, 3, 1, 2, 4).reshape(s * n, -1, d)[back]

    out = {"out": rows(torch.matmul(p, vf), nq, back_q).to(q.dtype)}
    if not case["train"]:
        return out
    gf = (st["dout"][iq].float() * mine_q[:, :, None, None]).view(s, nq, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), gf).sum(2, keepdim=True)
    dp = torch.matmul(gf, vf.transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del p, dp
    dq = torch.matmul(ds, kf) * scale
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(2, keepdim=True) * scale
    out["d_q"] = rows(dq, nq, back_q).to(q.dtype)
    out["d_k"], out["d_v"] = rows(dk, nk, back_k).to(q.dtype), rows(dv, nk, back_k).to(q.dtype)
    if st["bias_table"] is not None:
        dt = torch.zeros(st["bias_table"].shape, dtype=torch.float64, device=q.device)
        dt.index_add_(0, bucket.reshape(-1), ds.permute(0, 3, 4, 1, 2).reshape(-1, h).double())
        out["d_bias_table"] = dt.to(st["bias_table"].dtype)
    return out


def plain_bucket(buckets, q_pos, k_pos, iq, ik):
    reach = [(n - 1) // 2 for n in buckets.shape]
    if q_pos.dim() == 1:
        at = (k_pos[ik][:, None, :] - q_pos[iq][:, :, None]).clamp(-reach[1], reach[1]) + reach[1]
        return buckets[0][at.long()].long()
    dy = (k_pos[..., 0][ik][:, None, :] - q_pos[..., 0][iq][:, :, None]).clamp(-reach[0], reach[0]) + reach[0]
    dx = (k_pos[..., 1][ik][:, None, :] - q_pos[..., 1][iq][:, :, None]).clamp(-reach[1], reach[1]) + reach[1]
    return buckets[dy.long(), dx.long()].long()


def plain_standard(u, kind, eps=1e-6):
    """The normalised rows and the reciprocal of their deviation."""
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    r = torch.rsqrt((u * u).mean(-1, keepdim=True) + eps)
    return u * r, r


def plain_standard_back(g, n, r, kind):
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * r


def plain_norm(st):
    case, dtype = st["case"], st["x"].dtype
    kind, act = case["kind"], case["act"]
    x, h, scale = st["x"].float(), st["h"].float(), st["scale"].float()
    n1, r1 = plain_standard(h, kind)
    w1, w2 = st["weight"].float(), st["next_weight"].float()
    b1 = 0.0 if st["bias"] is None else st["bias"].float()
    b2 = 0.0 if st["next_bias"] is None else st["next_bias"].float()
    t = n1 * w1 + b1
    raw = torch.ones_like(x[:, :1]) if st["gate"] is None else st["gate"].float()
    sig = torch.sigmoid(raw)
    a = raw if act == "none" or st["gate"] is None else sig if act == "sigmoid" else raw * sig
    y = x + scale * a * t
    n2, r2 = plain_standard(y, kind)
    out = {"y": y.to(dtype), "z": (n2 * w2 + b2).to(dtype)}
    if not case["train"]:
        return out
    dz = st["dz"].float()
    g = st["dy"].float() + plain_standard_back(dz * w2, n2, r2, kind)
    dt = g * scale * a
    out["d_x"], out["d_h"] = g.to(dtype), plain_standard_back(dt * w1, n1, r1, kind).to(dtype)
    if st["gate"] is not None:
        da = g * scale * t
        slope = 1.0 if act == "none" else sig * (1 - sig) if act == "sigmoid" else sig * (1 + raw * (1 - sig))
        da = (da if case["gate"] == "full" else da.sum(-1, keepdim=True)) * slope
        out["d_gate"] = da.to(dtype)
    out["d_weight"] = (dt * n1).double().sum(0).float()
    out["d_next_weight"] = (dz * n2).double().sum(0).float()
    out["d_scale"] = (g * a * t).double().sum(0).float()
    if kind == "layer":
        out["d_bias"], out["d_next_bias"] = dt.double().sum(0).float(), dz.double().sum(0).float()
    return out


# ------------------------------------------------------------------ the definitions in 64 bits, window by window
def exact(case, seed):
    st = prepare(case, seed)
    wide = {n: st[n].detach().double() for n in st["leaves"]}
    if case["train"]:
        for t in wide.values():
            t.requires_grad_(True)
    with torch.set_grad_enabled(case["train"]):
        results = _exact_norm(case, wide) if case["op"] == "norm" else _exact_attention(case, st, wide)
    if not case["train"]:
        return results
    if case["op"] == "norm":
        grads = torch.autograd.grad([results["y"], results["z"]], list(wide.values()), [st["dy"].double(), st["dz"].double()])
        return {"y": results["y"].detach(), "z": results["z"].detach(), **{"d_" + n: g for n, g in zip(wide, grads)}}
    return results


def _exact_norm(case, w):
    c = case["channels"]

    def standard(u, weight, bias):
        if case["kind"] == "layer":
            return torch.nn.functional.layer_norm(u, (c,), weight, bias, 1e-6)
        return u / (u.square().sum(-1, keepdim=True) / c + 1e-6).sqrt() * weight

    t = standard(w["h"], w["weight"], w.get("bias"))
    if "gate" in w:
        t = t * {"none": lambda g: g, "sigmoid": torch.special.expit, "silu": torch.nn.functional.silu}[case["act"]](w["gate"])
    y = torch.addcmul(w["x"], w["scale"].expand_as(t), t)
    return {"y": y, "z": standard(y, w["next_weight"], w.get("next_bias"))}


def _exact_attention(case, st, w):
    """One window at a time, long ones in bands of rows; gradients by differentiating each band."""
    q, k, v = w["q"], w["k"], w["v"]
    table, buckets = w.get("bias_table"), st["buckets"]
    h, d, group = case["heads"], case["dim"], case["heads"] // case["kv_heads"]
    ql, kl = _lengths(case)
    if case["train"] and len(ql) > 4000:
        return None
    qo, ko = np.concatenate([[0], np.cumsum(ql)]), np.concatenate([[0], np.cumsum(kl)])
    out = torch.zeros_like(q, requires_grad=False)
    names = list(w)
    grads = [torch.zeros_like(t, requires_grad=False) for t in w.values()]
    for i in range(len(ql)):
        if ql[i] == 0 or kl[i] == 0:
            continue
        ks = slice(int(ko[i]), int(ko[i + 1]))
        kw, vw = k[ks].detach(), v[ks].detach()
        step = max(1, int(5e8 // (h * int(kl[i]))))
        for a in range(0, int(ql[i]), step):
            b = min(int(ql[i]), a + step)
            qs = slice(int(qo[i]) + a, int(qo[i]) + b)
            part = [t.detach().requires_grad_(case["train"]) for t in (q[qs], kw, vw)]
            if table is not None:
                part.append(table.detach().requires_grad_(case["train"]))
            logits = torch.einsum("ihd,jhd->hij", part[0], part[1].repeat_interleave(group, 1)) / d ** 0.5
            if table is not None:
                rel = st["k_pos"][ks][None].long() - st["q_pos"][qs][:, None].long()
                if rel.dim() == 2:
                    rel = torch.stack([torch.zeros_like(rel), rel], -1)
                n = torch.tensor([(s - 1) // 2 for s in buckets.shape], device=rel.device)
                rel = torch.minimum(torch.maximum(rel, -n), n) + n
                logits = logits + part[3][buckets[rel[..., 0], rel[..., 1]].long()].permute(2, 0, 1)
            if case["causal"]:
                row = torch.arange(a, b, device=q.device)[:, None] + int(kl[i] - ql[i])
                logits = logits.masked_fill(torch.arange(int(kl[i]), device=q.device) > row, -math.inf)
            o = torch.einsum("hij,jhd->ihd", torch.nan_to_num(torch.softmax(logits, -1), nan=0.0), part[2].repeat_interleave(group, 1))
            out[qs] = o.detach()
            if case["train"]:
                got = torch.autograd.grad(o, part, st["dout"][qs].double())
                for to, at, g in zip(grads, (qs, ks, ks, slice(None)), got):
                    to[at] += g
            del logits, o, part
    if not case["train"]:
        return {"out": out}
    return {"out": out, **{"d_" + n: g for n, g in zip(names, grads)}}
