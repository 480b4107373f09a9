"""Window attention and its bucketed position bias against float64 (tests/attention_reference.py
states the allowed errors)."""
from __future__ import annotations

import itertools
import math

import pytest
import torch

from attention_reference import check, window_attention

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def offsets(lengths, first=0):
    return [first] + [first + n for n in itertools.accumulate(lengths)]


def inputs(ql, kl, heads, kv, dim, dtype, seed=0, qfirst=0, kfirst=0, qtail=0, ktail=0):
    g = torch.Generator().manual_seed(seed)
    qo, ko = offsets(ql, qfirst), offsets(kl, kfirst)
    q = torch.randn(qo[-1] + qtail, heads, dim, generator=g) * 1.5
    k = torch.randn(ko[-1] + ktail, kv, dim, generator=g)
    v = torch.randn(ko[-1] + ktail, kv, dim, generator=g)
    do = torch.randn(qo[-1] + qtail, heads, dim, generator=g)
    return [t.to(dtype) for t in (q, k, v, do)], qo, ko, g


def run(dev, q, k, v, qo, ko, dout=None, table=None, **kw):
    """Outputs and gradients of the kernels on dev, as a dict."""
    from oss_cuda import fused_window_cross_attention

    leaves = [t.to(dev).requires_grad_(dout is not None) for t in (q, k, v)]
    if table is not None:
        leaves.append(table.to(dev).requires_grad_(dout is not None))
        kw["bias_table"] = leaves[3]
    kw = {n: t.to(dev) if torch.is_tensor(t) else t for n, t in kw.items()}
    i32 = dict(dtype=torch.int32, device=dev)
    out = fused_window_cross_attention(*leaves[:3], torch.tensor(qo, **i32), torch.tensor(ko, **i32), **kw)
    res = {"out": out.detach()}
    if dout is not None:
        res.update(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, dout.to(dev))))
    return res


def compare(got, want):
    for n in want:
        check(got[n], want[n], n)


def both(dev, q, k, v, qo, ko, dout=None, **kw):
    got = run(dev, q, k, v, qo, ko, dout, **kw)
    ref = {"table": kw.pop("table", None), **kw}
    compare(got, window_attention(q, k, v, qo, ko, dout=dout, **ref))
    return got


LENGTHS = [
    ([1], [1]),
    ([0, 5, 0, 3], [4, 0, 0, 7]),
    ([16, 64, 65, 1, 63], [63, 64, 65, 129, 1]),
    ([128, 127, 129], [128, 255, 257]),
    ([300], [513]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", range(len(LENGTHS)))
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(cuda_device, dtype, lengths, causal):
    ql, kl = LENGTHS[lengths]
    (q, k, v, do), qo, ko, _ = inputs(ql, kl, 4, 2, 32, TYPES[dtype], seed=lengths)
    both(cuda_device, q, k, v, qo, ko, do, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 16, 30, 40, 64, 72, 96, 100, 128])
def test_head_dims(cuda_device, dtype, dim):
    (q, k, v, do), qo, ko, _ = inputs([70, 9], [140, 33], 2, 1, dim, TYPES[dtype], seed=dim)
    both(cuda_device, q, k, v, qo, ko, do, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (6, 2), (5, 1), (8, 1), (16, 2)])
def test_grouped_heads(cuda_device, dtype, heads, kv):
    # few queries a window: the heads of a group share tiles
    (q, k, v, do), qo, ko, _ = inputs([1, 3, 12, 1], [40, 150, 2, 77], heads, kv, 32, TYPES[dtype], seed=heads)
    both(cuda_device, q, k, v, qo, ko, do, causal=True)
    (q, k, v, do), qo, ko, _ = inputs([130, 40], [150, 90], heads, kv, 32, TYPES[dtype], seed=heads)
    both(cuda_device, q, k, v, qo, ko, do)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [7, 16, 30, 32, 48, 64])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 2), (6, 3), (5, 5)])
@pytest.mark.parametrize("biased", [False, True])
def test_few_keys(cuda_device, dtype, dim, heads, kv, biased):
    """Tiles with few Gaussians, some with none, and one crowded: every kernel in one call."""
    from oss_cuda import window_position_buckets

    kl = [0, 1, 7, 8, 9, 16, 17, 31, 32, 33, 5, 0, 2, 12, 64, 3, 65, 140, 1, 20]
    ql = [16, 1, 33, 0, 256, 100, 15, 17, 64, 47, 64, 0, 130, 16, 70, 40, 80, 90, 31, 32]
    (q, k, v, do), qo, ko, g = inputs(ql, kl, heads, kv, dim, TYPES[dtype], seed=dim, qfirst=3, ktail=5)
    kw = {}
    if biased:
        kw = dict(table=torch.randn(81, heads, generator=g).to(TYPES[dtype]), buckets=window_position_buckets(4, 4),
                  q_pos=torch.randint(0, 5, (q.size(0), 2), generator=g).int(),
                  k_pos=torch.randint(0, 5 if dim % 3 else 12, (k.size(0), 2), generator=g).int())
    both(cuda_device, q, k, v, qo, ko, do, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lk", [20, 50, 100])
def test_many_queries_of_few_keys(cuda_device, dtype, lk):
    """One window's rows shared out over blocks, its key gradients joined."""
    from oss_cuda import window_position_buckets

    (q, k, v, do), qo, ko, g = inputs([6000, 4097], [lk, lk], 2, 1, 32, TYPES[dtype], seed=lk)
    kw = dict(table=torch.randn(25, 2, generator=g).to(TYPES[dtype]), buckets=window_position_buckets(2, 2),
              q_pos=torch.randint(0, 3, (q.size(0), 2), generator=g).int(), k_pos=torch.randint(0, 3, (k.size(0), 2), generator=g).int())
    both(cuda_device, q, k, v, qo, ko, do, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,kv", [(8, 4, 4), (20, 6, 3), (31, 2, 1), (32, 5, 5), (64, 4, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_windows_of_every_class(cuda_device, dtype, dim, heads, kv, biased):
    """Windows of every class of the few-keys kernels and beyond in one call, with pieces of rows around 64."""
    kl = [0, 1, 15, 16, 17, 32, 33, 48, 64, 65, 80, 96, 97, 127, 128, 129, 300] + [3] * 20
    ql = [7, 64, 65, 1, 130, 3, 63, 128, 5, 66, 17, 129, 2, 64, 33, 70, 9] + [0, 1, 40, 2] * 5
    (q, k, v, do), qo, ko, g = inputs(ql, kl, heads, kv, dim, TYPES[dtype], seed=dim, qfirst=2, ktail=3, qtail=70)
    kw = {}
    if biased:
        kw = {"buckets": torch.arange(35, dtype=torch.int32).view(5, 7), "table": torch.randn(35, heads, generator=g),
              "q_pos": torch.randint(0, 9, (q.shape[0], 2), generator=g).int(),
              "k_pos": torch.randint(0, 9, (k.shape[0], 2), generator=g).int()}
    both(cuda_device, q, k, v, qo, ko, do, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,lk,causal", [(1, 3000, True), (2, 5001, False), (17, 2100, True)])
def test_long_axis_is_split_and_joined(cuda_device, dtype, lq, lk, causal):
    from oss_cuda import _lib

    assert _lib.lib().oss_window_attention_scratch_bytes(0, 2 * lq, lk + 700, 2, 4, 2, 64, int(causal), 0) > 0
    (q, k, v, do), qo, ko, _ = inputs([lq, lq], [lk, 700], 4, 2, 64, TYPES[dtype], seed=lk)
    both(cuda_device, q, k, v, qo, ko, causal=causal)
    both(cuda_device, q, k, v, qo, ko, do, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_outside_the_windows_are_zero(cuda_device, dtype):
    (q, k, v, do), qo, ko, _ = inputs([20, 150], [30, 140], 2, 2, 32, TYPES[dtype], qfirst=140, kfirst=9, qtail=200, ktail=70)
    nan = float("nan")
    for t, o in ((q, qo), (k, ko), (v, ko)):  # nothing of these rows is used
        t[:o[0]] = nan
        t[o[-1]:] = nan
    zero = {"q": q.clone(), "k": k.clone(), "v": v.clone()}
    got = run(cuda_device, q, k, v, qo, ko, do)
    for t, o in ((zero["q"], qo), (zero["k"], ko), (zero["v"], ko)):
        t[:o[0]] = 0
        t[o[-1]:] = 0
    compare(got, window_attention(zero["q"], zero["k"], zero["v"], qo, ko, dout=do))
    for n, o in (("out", qo), ("dq", qo), ("dk", ko), ("dv", ko)):
        assert not got[n][:o[0]].any() and not got[n][o[-1]:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_neighbours_not_finite(cuda_device, dtype):
    """NaN and infinities in other windows, and behind the causal mask, stay where they are."""
    (q, k, v, do), qo, ko, _ = inputs([70, 60, 80], [70, 60, 80], 2, 2, 32, TYPES[dtype])
    want = window_attention(q, k, v, qo, ko, causal=True, dout=do)
    bad_k, bad_v, bad_q, bad_do = k.clone(), v.clone(), q.clone(), do.clone()
    bad_k[70:130] = float("inf")
    bad_v[70:130] = float("nan")
    bad_q[70:130] = float("nan")
    bad_do[70:130] = float("inf")
    got = run(cuda_device, bad_q, bad_k, bad_v, qo, ko, bad_do, causal=True)
    for n in ("out", "dq", "dk", "dv"):
        for rows in (slice(0, 70), slice(130, 210)):
            check(got[n][rows], tuple(t[rows] for t in want[n]), n)
    # the last window's keys from its 41st on: queries before it do not see them
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[170:] = float("nan")
    bad_v[170:] = float("inf")
    got = run(cuda_device, q, bad_k, bad_v, qo, ko, do, causal=True)
    for n in ("out", "dq"):
        check(got[n][:170], tuple(t[:170] for t in want[n]), n)
        assert torch.isnan(got[n][170:]).all()
    # and dk, dv of keys that no query with a NaN sees
    bad_q, bad_do = q.clone(), do.clone()
    bad_q[130:150] = float("nan")
    bad_do[130:150] = float("inf")
    got = run(cuda_device, bad_q, k, v, qo, ko, bad_do, causal=True)
    for n in ("dk", "dv"):
        check(got[n][150:], tuple(t[150:] for t in want[n]), n)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(cuda_device, dtype):
    """Scores far beyond exp's range, rising and falling along the keys."""
    (q, k, v, do), qo, ko, _ = inputs([40, 40], [400, 300], 2, 1, 64, TYPES[dtype])
    ramp = torch.linspace(0.1, 12, 400)[:, None, None]
    k[:400] = (k[:400].float() * ramp).to(k.dtype)
    k[400:] = (k[400:].float() * ramp[:300].flip(0)).to(k.dtype)
    both(cuda_device, q, k, v, qo, ko, do)


@pytest.mark.parametrize("dtype", TYPES)
def test_scale_argument(cuda_device, dtype):
    (q, k, v, do), qo, ko, _ = inputs([33], [70], 2, 2, 24, TYPES[dtype])
    both(cuda_device, q, k, v, qo, ko, do, scale=0.37)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(cuda_device, dtype):
    """Views of one packed projection, heads before tokens, and rows that no vector is aligned to."""
    dev, t = cuda_device, TYPES[dtype]
    (q, k, v, do), qo, ko, _ = inputs([90, 45], [90, 45], 4, 2, 32, t)
    want = window_attention(q, k, v, qo, ko, causal=True, dout=do)
    packed = torch.cat([q, k, v], 1).to(dev)
    from oss_cuda import fused_window_cross_attention

    off = torch.tensor(qo, dtype=torch.int32, device=dev)

    def go(a, b, c, d):
        leaves = [x.detach().requires_grad_(True) for x in (a, b, c)]
        out = fused_window_cross_attention(*leaves, off, off, causal=True)
        compare(dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, d)))), want)

    g = do.to(dev)
    go(packed[:, :4], packed[:, 4:6], packed[:, 6:], g)
    q2, k2, v2 = (x.to(dev).transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    go(q2, k2, v2, g.transpose(0, 1).contiguous().transpose(0, 1))
    odd = [torch.zeros(x.shape[0] * x.shape[1] * 33 + 1, dtype=t, device=dev)[1:].view(x.shape[0], x.shape[1], 33) for x in (q, k, v, do)]
    for o, x in zip(odd, (q, k, v, do)):
        o[..., :32] = x.to(dev)
    go(*(o[..., :32] for o in odd))
    go(q.to(dev), k.to(dev), v.to(dev).transpose(1, 2).contiguous().transpose(1, 2), g)
    # one key head broadcast to both, one gradient to all rows
    kb, vb = (x.to(dev)[:, :1].expand(-1, 2, -1) for x in (k, v))
    gb = g[:1].expand(g.shape[0], -1, -1)
    leaves = [x.detach().requires_grad_(True) for x in (q.to(dev), kb, vb)]
    out = fused_window_cross_attention(*leaves, off, off)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, gb))))
    compare(got, window_attention(q, kb.cpu(), vb.cpu(), qo, ko, dout=gb))


def grid(side, start=0):
    y, x = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
    return (torch.stack([y.reshape(-1), x.reshape(-1)], 1) + start).int()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("table_type", ["same", "fp32"])
@pytest.mark.parametrize("side,margin,reach", [(4, 0, 3), (8, 2, 9), (7, 1, 4), (8, 3, 0), (12, 2, 13)])
def test_window_bias(cuda_device, dtype, table_type, side, margin, reach):
    """Two-axis buckets: exactly as far as the window goes, and clamped."""
    from oss_cuda import window_position_buckets

    t = TYPES[dtype]
    n, m = side * side, (side + 2 * margin) ** 2
    (q, k, v, do), qo, ko, g = inputs([n, n], [m, m], 4, 2, 30, t, seed=side)
    buckets = window_position_buckets(reach, reach)
    table = torch.randn(buckets.numel(), 4, generator=g).to(torch.float32 if table_type == "fp32" else t)
    qp = torch.cat([grid(side)] * 2)
    kp = torch.cat([grid(side + 2 * margin, -margin)] * 2)
    both(cuda_device, q, k, v, qo, ko, do, table=table, buckets=buckets, q_pos=qp, k_pos=kp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[1, 33, 300], [515]])
def test_log_bias(cuda_device, dtype, causal, lengths):
    from oss_cuda import log_position_buckets

    (q, k, v, do), qo, ko, g = inputs(lengths, lengths, 4, 2, 64, TYPES[dtype])
    buckets = log_position_buckets(16, 60, causal=causal)
    table = torch.randn(16, 4, generator=g).to(TYPES[dtype])
    pos = torch.cat([torch.arange(n) for n in lengths]).int()
    both(cuda_device, q, k, v, qo, ko, do, causal=causal, table=table, buckets=buckets, q_pos=pos, k_pos=pos)


@pytest.mark.parametrize("dtype", TYPES)
def test_bias_for_single_tokens(cuda_device, dtype):
    from oss_cuda import log_position_buckets

    lk = [900, 31, 2048]
    (q, k, v, _), qo, ko, g = inputs([1, 1, 1], lk, 6, 2, 48, TYPES[dtype])
    buckets = log_position_buckets(32, 128, causal=True)
    table = torch.randn(32, 6, generator=g).to(TYPES[dtype])
    qp = torch.tensor([n - 1 for n in lk]).int()
    kp = torch.cat([torch.arange(n) for n in lk]).int()
    both(cuda_device, q, k, v, qo, ko, causal=True, table=table, buckets=buckets, q_pos=qp, k_pos=kp)


@pytest.mark.parametrize("dtype", TYPES)
def test_bias_odd_maps_and_positions(cuda_device, dtype):
    """Buckets that repeat, that no pair reaches, and outside the table; scattered and extreme positions."""
    (q, k, v, do), qo, ko, g = inputs([60, 31], [130, 64], 3, 1, 16, TYPES[dtype])
    buckets = torch.randint(-2, 14, (7, 11), generator=g).int()
    table = torch.randn(12, 3, generator=g).to(TYPES[dtype])
    qp = torch.randint(-6, 7, (91, 2), generator=g).int()
    kp = torch.randint(-6, 7, (194, 2), generator=g).int()
    kp[:5] = 2**31 - 1
    qp[:5] = -(2**31)
    got = both(cuda_device, q, k, v, qo, ko, do, table=table, buckets=buckets, q_pos=qp, k_pos=kp)
    unused = [b for b in range(12) if not (buckets == b).any()]
    assert not got["dtable"][unused].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_bias_that_hides_keys(cuda_device, dtype):
    """A bucket of minus infinity hides its keys, of some rows all of them; the lowest value of the type only
    lowers them."""
    (q, k, v, do), qo, ko, g = inputs([64], [64], 2, 2, 32, TYPES[dtype])
    buckets = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    qp = torch.zeros(64, dtype=torch.int32)
    qp[10:20] = 100  # every key lies behind these queries
    kp = torch.arange(64).int() - 20
    table = torch.zeros(3, 2)
    table[0] = -math.inf
    table[1] = 0.5
    got = both(cuda_device, q, k, v, qo, ko, do, table=table.to(TYPES[dtype]), buckets=buckets, q_pos=qp, k_pos=kp)
    assert not got["out"][10:20].any() and not got["dq"][10:20].any()
    table[0] = torch.finfo(TYPES[dtype]).min
    got = both(cuda_device, q, k, v, qo, ko, table=table.to(TYPES[dtype]), buckets=buckets, q_pos=qp, k_pos=kp)
    assert torch.isfinite(got["out"]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_bias_gradient_not_finite(cuda_device, dtype):
    """A gradient that is not finite makes the buckets it reaches NaN, and no others."""
    (q, k, v, do), qo, ko, g = inputs([8, 8], [8, 8], 2, 2, 16, TYPES[dtype])
    buckets = torch.tensor([[0, 1, 2, 3, 4]], dtype=torch.int32)
    table = torch.randn(5, 2, generator=g).to(TYPES[dtype])
    qp = torch.zeros(16, dtype=torch.int32)
    kp = torch.tensor([0, 1] * 4 + [-2, -1] * 4, dtype=torch.int32)
    do[3, 1, 2] = float("inf")
    got = run(cuda_device, q, k, v, qo, ko, do, table=table, buckets=buckets, q_pos=qp, k_pos=kp)
    bad = torch.isnan(got["dtable"]).cpu()
    assert bad[[2, 3], 1].all() and not bad[:, 0].any() and not bad[[0, 1, 4], 1].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [1e-6, 3e3])
def test_gradients_of_any_size(cuda_device, dtype, size):
    """Gradients far below and above what the weights' type holds on the way."""
    from oss_cuda import window_position_buckets

    (q, k, v, do), qo, ko, g = inputs([64], [100], 2, 2, 64, TYPES[dtype])
    table = torch.randn(25, 2, generator=g)
    pos = dict(buckets=window_position_buckets(2, 2), q_pos=torch.randint(0, 3, (64, 2), generator=g).int(),
               k_pos=torch.randint(0, 3, (100, 2), generator=g).int())
    both(cuda_device, q, k, v, qo, ko, (do.float() * size).to(do.dtype), table=table, **pos)


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_time(cuda_device, dtype):
    from oss_cuda import log_position_buckets

    lengths = [1200, 7, 333]
    (q, k, v, do), qo, ko, g = inputs(lengths, lengths, 4, 2, 64, TYPES[dtype])
    pos = torch.cat([torch.arange(n) for n in lengths]).int()
    kw = dict(causal=True, table=torch.randn(8, 4, generator=g).to(TYPES[dtype]), buckets=log_position_buckets(8, 20, causal=True),
              q_pos=pos, k_pos=pos)
    first = run(cuda_device, q, k, v, qo, ko, do, **kw)
    for _ in range(3):
        again = run(cuda_device, q, k, v, qo, ko, do, **kw)
        for n in first:
            assert torch.equal(first[n], again[n]), n


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_against_differences(cuda_device, dtype):
    """The directional derivative of a weighted sum of outputs, from outputs of fp32 inputs a step apart."""
    from oss_cuda import fused_window_cross_attention, log_position_buckets

    dev = cuda_device
    (q, k, v, do), qo, ko, g = inputs([20, 40], [30, 50], 4, 2, 32, TYPES[dtype])
    q, k, v, do = (t.to(dev).float() for t in (q, k, v, do))
    table = torch.randn(8, 4, generator=g).to(dev)
    off = [torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko)]
    kw = dict(buckets=log_position_buckets(8, 9).to(dev), q_pos=torch.randint(0, 20, (60,), generator=g).int().to(dev),
              k_pos=torch.randint(0, 20, (80,), generator=g).int().to(dev))
    leaves = [t.to(TYPES[dtype]).requires_grad_(True) for t in (q, k, v, table)]
    out = fused_window_cross_attention(*leaves[:3], *off, bias_table=leaves[3], **kw)
    grads = torch.autograd.grad(out, leaves, do.to(TYPES[dtype]))
    with torch.no_grad():
        for i, t in enumerate((q, k, v, table)):
            step = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(dev)
            e = 2.0**-8
            sides = []
            for sign in (1, -1):
                moved = [a.to(TYPES[dtype]).float() for a in (q, k, v, table)]
                moved[i] = moved[i] + sign * e * step
                o = fused_window_cross_attention(*moved[:3], *off, bias_table=moved[3], **kw)
                sides.append((o.double() * do.to(TYPES[dtype]).double()).sum())
            by_difference = float((sides[0] - sides[1]) / (2 * e))
            mine = float((grads[i].double() * step.double()).sum())
            size = float((grads[i].double() * step.double()).square().sum().sqrt())
            # the second differences leave e^2 of the third derivative, the type's rounding averages out over
            # the elements; both are small against the root of the sum of squares of the terms
            assert abs(mine - by_difference) <= (5e-3 if dtype == "fp32" else 5e-2) * size


def test_no_windows_and_no_tokens(cuda_device):
    (q, k, v, do), _, _, _ = inputs([5], [6], 2, 2, 16, torch.float32)
    got = run(cuda_device, q, k, v, [0], [0], do)
    assert not any(t.any() for t in got.values())
    got = run(cuda_device, q[:0], k, v, [0, 0], [0, 6], do[:0])
    assert got["out"].shape == (0, 2, 16) and not got["dk"].any() and not got["dv"].any()
    got = run(cuda_device, q, k[:0], v[:0], [0, 5], [0, 0], do)
    assert not got["out"].any() and not got["dq"].any()
    got = run(cuda_device, q[:0], k[:0], v[:0], [0, 0], [0, 0], do[:0])
    assert got["dk"].shape == (0, 2, 16)


def test_offsets_outside_the_tensors_are_clamped(cuda_device):
    (q, k, v, do), _, _, _ = inputs([50], [60], 2, 2, 16, torch.bfloat16)
    a = run(cuda_device, q, k, v, [0, 20, 50], [0, 30, 60], do)
    b = run(cuda_device, q, k, v, [-7, 20, 900], [-1, 30, 2**30], do)
    for n in a:
        assert torch.equal(a[n], b[n])


def test_many_windows(cuda_device):
    """More windows than one pass of the search over them tells apart."""
    g = torch.Generator().manual_seed(3)
    ql = torch.randint(0, 4, (5000,), generator=g).tolist()
    kl = torch.randint(0, 5, (5000,), generator=g).tolist()
    (q, k, v, do), qo, ko, _ = inputs(ql, kl, 2, 1, 16, torch.bfloat16)
    both(cuda_device, q, k, v, qo, ko, do)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("lk", [60, 70, 130, 190])
def test_blocks_that_walk_many_tiles(cuda_device, dim, lk):
    """Far more tiles than blocks, of one to three tiles of keys, and of both parities in turn."""
    g = torch.Generator().manual_seed(lk)
    kl = (lk + torch.randint(-6, 7, (700,), generator=g)).tolist()
    (q, k, v, do), qo, ko, _ = inputs([140] * 700, kl, 8, 4, dim, torch.bfloat16, seed=lk)
    got = run(cuda_device, q, k, v, qo, ko, do)
    again = run(cuda_device, q, k, v, qo, ko, do)
    for n in got:
        assert torch.equal(got[n], again[n])
    for w in (0, 1, 2, 3, 350, 351, 697, 698, 699):  # the windows that are compared with the formula
        a, b, c, e = qo[w], qo[w + 1], ko[w], ko[w + 1]
        want = window_attention(q[a:b], k[c:e], v[c:e], [0, b - a], [0, e - c], dout=do[a:b])
        for n, (lo, hi) in (("out", (a, b)), ("dq", (a, b)), ("dk", (c, e)), ("dv", (c, e))):
            check(got[n][lo:hi], want[n], f"{n} of window {w}")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_capture_and_replay(cuda_device, dtype):
    """Two graphs of a forward and backward each, replayed in turn with other inputs and offsets, on their own stream."""
    from oss_cuda import fused_window_cross_attention

    dev = cuda_device
    sets = []
    for seed, (ql, kl) in enumerate([([60, 4], [100, 28]), ([10, 54], [3, 125])]):
        (q, k, v, do), qo, ko, _ = inputs(ql, kl, 4, 2, 32, TYPES[dtype], seed=seed)
        sets.append(([t.to(dev) for t in (q, k, v, do)], *(torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko))))
    static = [t.clone() for t in sets[0][0]]
    off = [t.clone() for t in sets[0][1:]]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in static[:3]]
        out = fused_window_cross_attention(*leaves, *off, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, static[3]))

    want = []
    for tensors, qo, ko in sets:
        for a, b in zip(static + off, [*tensors, qo, ko]):
            a.copy_(b)
        want.append([t.clone() for t in step()])
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    for i in (0, 1, 1, 0):
        tensors, qo, ko = sets[i]
        for a, b in zip(static + off, [*tensors, qo, ko]):
            a.copy_(b)
        for graph, res in zip(graphs, results):
            graph.replay()
            torch.cuda.synchronize(dev)
            for a, b in zip(res, want[i]):
                assert torch.equal(a, b)


def test_two_streams_at_once(cuda_device):
    dev = cuda_device
    args = [inputs([200, 77], [150, 300], 4, 2, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    alone = [run(dev, q, k, v, qo, ko, do, causal=True) for (q, k, v, do), qo, ko, _ in args]
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in args]
    for _ in range(3):
        got = []
        for s, ((q, k, v, do), qo, ko, _) in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(run(dev, q, k, v, qo, ko, do, causal=True))
        torch.cuda.synchronize(dev)
        for a, b in zip(alone, got):
            for n in a:
                assert torch.equal(a[n], b[n])


def test_one_tensor_as_keys_and_values(cuda_device):
    from oss_cuda import fused_window_cross_attention

    (q, k, _, do), qo, ko, _ = inputs([40], [90], 2, 2, 32, torch.float32)
    off = [torch.tensor(o, dtype=torch.int32, device=cuda_device) for o in (qo, ko)]
    leaves = [t.to(cuda_device).requires_grad_(True) for t in (q, k)]
    out = fused_window_cross_attention(leaves[0], leaves[1], leaves[1], *off)
    dq, dk = torch.autograd.grad(out, leaves, do.to(cuda_device))
    want = window_attention(q, k, k, qo, ko, dout=do)
    check(dq, want["dq"])
    check(dk, tuple(a + b for a, b in zip(want["dk"], want["dv"])))


def test_no_wait_ran_out(cuda_device):
    """The waits inside the kernels are bounded; none of the calls above may have come to a bound."""
    import ctypes

    from oss_cuda import _lib

    count = ctypes.c_uint32(7)
    _lib.check(_lib.lib().oss_window_attention_timeouts(ctypes.addressof(count)), "oss_window_attention_timeouts")
    assert count.value == 0
