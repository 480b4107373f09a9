"""Window attention where single values, sizes or callers could go wrong, against float64
(tests/attention_reference.py states the allowed errors)."""
from __future__ import annotations

import math
import threading

import pytest
import torch

from attention_reference import bias_of, check, window_attention
from test_gpu_window_attention import TYPES, both, inputs, run

pytestmark = pytest.mark.gpu


def window_of(w, q, k, v, qo, ko, dout, **kw):
    """The formula for window w alone."""
    a, b, c, e = qo[w], qo[w + 1], ko[w], ko[w + 1]
    for n, (lo, hi) in (("q_pos", (a, b)), ("k_pos", (c, e))):
        if n in kw:
            kw[n] = kw[n][lo:hi]
    return window_attention(q[a:b], k[c:e], v[c:e], [0, b - a], [0, e - c], dout=dout[a:b], **kw)


def check_window(got, want, w, qo, ko, names=("out", "dq", "dk", "dv")):
    for n in names:
        o = qo if n in ("out", "dq") else ko
        check(got[n][o[w]:o[w + 1]], want[n], f"{n} of window {w}")


# one window of each of the backward's kernels, and one more that holds the large values
LARGE_Q, LARGE_K = [130, 60, 48, 70], [200, 50, 20, 140]


def large_case(dtype, dim):
    """Windows whose pairs reach rows of the table of their own: 25 rows each."""
    (q, k, v, do), qo, ko, g = inputs(LARGE_Q, LARGE_K, 4, 2, dim, dtype, seed=dim, qfirst=3, kfirst=5, qtail=9, ktail=7)
    pos = [torch.randint(0, 3, (t.shape[0], 2), generator=g).int() for t in (q, k)]
    for w in range(4):  # window w reaches columns 5 w .. 5 w + 4 of the map
        pos[1][ko[w]:ko[w + 1], 1] += 5 * w - 8
    kw = dict(table=torch.randn(100, 4, generator=g).to(dtype), buckets=torch.arange(100, dtype=torch.int32).view(5, 20)[:, :19].contiguous(),
              q_pos=pos[0], k_pos=pos[1])
    return q, k, v, do, qo, ko, kw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 72])
@pytest.mark.parametrize("where", ["padding", "neighbour"])
def test_large_values_elsewhere_change_nothing(cuda_device, dtype, dim, where):
    """Large finite values of rows that no window holds, or of another window, cost the others no precision."""
    q, k, v, do, qo, ko, kw = large_case(TYPES[dtype], dim)
    big = 6e4 if dtype == "fp16" else 1e16
    if where == "padding":
        for t, o in ((v, ko), (do, qo)):
            t[:o[0]] = big
            t[o[-1]:] = -big
    else:
        v[ko[3]:ko[4]] *= 2000 if dtype == "fp16" else big
        do[qo[3]:qo[4]] *= 2000 if dtype == "fp16" else big
    got = run(cuda_device, q, k, v, qo, ko, do, **kw)
    column = torch.arange(100) % 20
    for w in range(3 if where == "neighbour" else 4):
        want = window_of(w, q, k, v, qo, ko, do, **kw)
        check_window(got, want, w, qo, ko)
        mine = (column >= (5 * w - 1 if w else 0)) & (column <= 5 * w + 3)
        check(got["dtable"][mine.to(cuda_device)], tuple(t[mine] for t in want["dtable"]), f"dtable of window {w}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,heads,kv,dim", [([1024], 2, 2, 32), ([1024] * 4, 4, 2, 64), ([3000], 8, 1, 128)])
@pytest.mark.parametrize("biased", [False, True])
def test_no_keys_at_all(cuda_device, dtype, queries, heads, kv, dim, biased):
    """Enough queries that they are shared out over blocks, and nothing for them to see."""
    (q, k, v, do), qo, ko, g = inputs(queries, [0] * len(queries), heads, kv, dim, TYPES[dtype])
    kw = {}
    if biased:
        kw = dict(table=torch.randn(3, heads, generator=g).to(TYPES[dtype]), buckets=torch.tensor([[0, 1, 2]], dtype=torch.int32),
                  q_pos=torch.zeros(q.shape[0], dtype=torch.int32), k_pos=torch.zeros(0, dtype=torch.int32))
    got = run(cuda_device, q, k, v, qo, ko, do, **kw)
    assert got["dk"].shape == k.shape and got["dv"].shape == v.shape
    for n in got:
        assert not got[n].any(), n


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("keys", [7, 16, 30])
@pytest.mark.parametrize("size", [2.0**-8, 2.0**-14, 2.0**-20])
def test_bias_gradient_of_small_windows(cuda_device, dtype, keys, size):
    """Windows of ordinary gradients, then ones of far smaller gradients, each with rows of the table of their own; the
    same for the heads of a group."""
    windows = 1024  # more than the blocks' warps: each walks windows of both kinds
    (q, k, v, do), qo, ko, g = inputs([64] * windows, [keys] * windows, 4, 1, 16, TYPES[dtype], seed=keys)
    small = torch.arange(windows) >= windows // 2
    rows_q, rows_k = small.repeat_interleave(64), small.repeat_interleave(keys)
    scale = torch.where(rows_q, size, 1.0)[:, None, None].expand(-1, 4, 1).clone()
    scale[:, 2] *= size  # and one head
    do = (do.double() * scale).to(TYPES[dtype])
    qp, kp = torch.randint(0, 2, (q.shape[0],), generator=g).int(), torch.randint(0, 2, (k.shape[0],), generator=g).int()
    kp += torch.where(rows_k, 6, 0).int()
    table = torch.randn(17, 4, generator=g)
    buckets = torch.arange(17, dtype=torch.int32).view(1, 17)
    kw = dict(table=table, buckets=buckets, q_pos=qp, k_pos=kp)
    got = run(cuda_device, q, k, v, qo, ko, do, **kw)["dtable"]
    # the formula, all windows at once
    qd, kd, vd, dd = (t.double().view(windows, -1, t.shape[1], 16) for t in (q, k, v, do))
    row = (kp.view(windows, 1, -1) - qp.view(windows, -1, 1) + 8).long()
    s = torch.einsum("wihd,wjd->whij", qd, kd[:, :, 0]) / 4 + table.double()[row].permute(0, 3, 1, 2)
    p = torch.softmax(s, -1)
    dp = torch.einsum("wihd,wjd->whij", dd, vd[:, :, 0])
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    want, size_of = torch.zeros(17, 4, dtype=torch.float64), torch.zeros(17, 4, dtype=torch.float64)
    # a pair's term is off by its score's, dp's and delta's errors (as the formula's, 24 = dim + 8, without out's rounding:
    # these kernels take delta from p and dp), and by half a step of the sums, 2^-20 of the 16 rows' sum of magnitudes
    f = 2.0**-24
    score = 24 * f * (torch.einsum("wihd,wjd->whij", qd.abs(), kd[:, :, 0].abs()) / 4 + table.abs().max())
    dpe = 24 * f * torch.einsum("wihd,wjd->whij", dd.abs(), vd[:, :, 0].abs())
    rel = 2 * score.amax(-1, keepdim=True) + (16 + keys) * f
    off = rel * ds.abs() + p * (dpe + (p * (dpe + rel * dp.abs())).sum(-1, keepdim=True) + 4 * f * dp.abs())
    step = ds.abs().view(windows, 4, 4, 16 * keys).sum(-1)[..., None, None].expand(-1, -1, -1, 16, keys).reshape(ds.shape)
    off = off + 2.0**-21 * step
    flat = row.reshape(-1)
    want.index_add_(0, flat, ds.permute(0, 2, 3, 1).reshape(-1, 4))
    size_of.index_add_(0, flat, off.permute(0, 2, 3, 1).reshape(-1, 4))
    check(got, (want, 1.05 * size_of + f * want.abs() + 1e-35), "dtable")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keys", [20, 100])
def test_host_threads_with_other_maps(cuda_device, dtype, keys):
    """Threads that call at once with bias maps of very different size, and so shared memory: no launch fails, no result
    changes. The calls go to the C entry points, which hold no lock, so that many of them overlap."""
    from oss_cuda import _lib, attention, window_position_buckets

    dev, lib = cuda_device, _lib.lib()
    calls = []
    for reach in (0, 31, 2, 31):
        (q, k, v, do), qo, ko, g = inputs([40, 30], [keys, keys], 1, 1, 32, TYPES[dtype], seed=reach)
        i32 = dict(dtype=torch.int32, device=dev)
        buckets = window_position_buckets(reach, reach).to(dev)
        table = torch.randn(buckets.numel(), 1, generator=g).to(dev)
        pos = [torch.randint(-20, 20, (t.shape[0], 2), generator=g).int().to(dev) for t in (q, k)]
        q, k, v, do = (t.to(dev) for t in (q, k, v, do))
        keep = (q, k, v, torch.tensor(qo, **i32), torch.tensor(ko, **i32), 0.2, 0, table, buckets, *pos)
        args = attention._call_args(*keep, lse_pair=0)
        out, dq, dk, dv, dt = (torch.empty_like(t) for t in (q, q, k, v, table))
        lo, lse = torch.empty_like(q), torch.empty(1, q.shape[0], device=dev)
        sizes = (lib.oss_window_attention_scratch_bytes(*args[:7], 0, buckets.numel()),
                 lib.oss_window_attention_backward_scratch_bytes(*args[:7], 0, buckets.numel(), table.shape[0]))
        scratch = [torch.empty(n + 16, dtype=torch.uint8, device=dev) for n in sizes]
        stream = torch.cuda.Stream(dev)
        forward = (*args, out.data_ptr(), lse.data_ptr(), lo.data_ptr(), scratch[0].data_ptr(), sizes[0], stream.cuda_stream)
        backward = (*args, out.data_ptr(), lse.data_ptr(), lo.data_ptr(), do.data_ptr(), do.stride(0), do.stride(1), dq.data_ptr(),
                    dk.data_ptr(), dv.data_ptr(), dt.data_ptr(), scratch[1].data_ptr(), sizes[1], stream.cuda_stream)
        calls.append((forward, backward, (out, dq, dk, dv, dt), (keep, do, lo, lse, scratch, stream)))
    torch.cuda.synchronize(dev)

    def both_ways(i):
        return lib.oss_window_attention_forward(*calls[i][0]) or lib.oss_window_attention_backward(*calls[i][1])

    want = []
    for i, (_, _, results, _) in enumerate(calls):
        assert both_ways(i) == 0
        torch.cuda.synchronize(dev)
        want.append([t.clone() for t in results])
    refused = []

    def work(i):
        for _ in range(400):
            rc = both_ways(i)
            if rc:
                refused.append((i, rc, lib.oss_last_error().decode()))

    with torch.cuda.device(dev):
        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
        for x in threads:
            x.start()
        for x in threads:
            x.join()
    torch.cuda.synchronize(dev)
    assert not refused, (len(refused), refused[:2])
    for (_, _, results, _), w in zip(calls, want):
        assert all(torch.equal(a, b) for a, b in zip(results, w))


def test_forward_mode_level_without_a_tangent(cuda_device):
    """Inside a forward-mode level, calls without tangents give what they give outside."""
    import torch.autograd.forward_ad as forward_ad

    from oss_cuda import gated_residual_norm

    (q, k, v, do), qo, ko, _ = inputs([20], [30], 2, 2, 16, torch.float32)
    x, w = torch.randn(4, 8, device=cuda_device), torch.ones(8, device=cuda_device)
    want, norm = run(cuda_device, q, k, v, qo, ko, do), gated_residual_norm(x, x, w)
    with forward_ad.dual_level():
        got = run(cuda_device, q, k, v, qo, ko, do)
        assert torch.equal(gated_residual_norm(x, x, w), norm)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [50, 300])
def test_hidden_pairs_leave_the_table_alone(cuda_device, dtype, tokens):
    """A gradient that is not finite reaches the rows of the table that its query sees; hidden pairs reach none."""
    (q, k, v, do), qo, ko, g = inputs([tokens], [tokens], 2, 1, 32, TYPES[dtype], seed=tokens)
    pos = torch.arange(tokens).int()
    kw = dict(causal=True, table=torch.randn(7, 2, generator=g), buckets=torch.arange(7, dtype=torch.int32).view(1, 7),
              q_pos=pos, k_pos=pos)
    do[tokens // 2, 1, 3] = float("nan")
    got = run(cuda_device, q, k, v, qo, ko, do, **kw)["dtable"].cpu()
    assert torch.isnan(got[:4, 1]).all() and torch.isfinite(got[:, 0]).all()
    assert not got[4:].any()


def long_case(dtype, tokens, dim, seed=1):
    (q, k, v, do), qo, ko, _ = inputs([tokens], [tokens], 2, 1, dim, dtype, seed=seed)
    return {"q": q, "k": k, "v": v, "dout": do}, qo


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bad", ["first key", "first value", "every value", "every key infinite", "last gradient", "last query"])
def test_visible_values_that_are_not_finite_cost_little(cuda_device, dtype, bad):
    """A NaN that a row sees is left alone: a causal call with one takes no more than some times the call without."""
    dev = cuda_device
    t, off = long_case(TYPES[dtype], 4096, 64)
    clean = {n: x.to(dev) for n, x in t.items()}
    if bad == "first key":
        t["k"][0] = math.nan
    elif bad == "first value":
        t["v"][0, 0, 3] = math.inf
    elif bad == "every value":
        t["v"][:] = math.nan
    elif bad == "every key infinite":
        t["k"][:] = math.inf
    elif bad == "last gradient":
        t["dout"][-1] = math.inf
    else:
        t["q"][-1] = math.nan
    spoilt = {n: x.to(dev) for n, x in t.items()}

    def milliseconds(x):
        best = math.inf
        for _ in range(3):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            run(dev, x["q"], x["k"], x["v"], off, off, x["dout"], causal=True)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    without = milliseconds(clean)
    assert milliseconds(spoilt) < 8 * without + 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,at", [(700, 350), (1500, 1023), (60, 31)])
@pytest.mark.parametrize("dim", [32, 72])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_one_value_that_is_not_finite(cuda_device, dtype, tokens, at, dim, value):
    """It reaches the rows that see it, and no others: clean ones are right to the last bit that is theirs."""
    t, off = long_case(TYPES[dtype], tokens, dim)
    want = window_attention(t["q"], t["k"], t["v"], off, off, causal=True, dout=t["dout"])

    def go(name, index):
        x = {n: y.clone() for n, y in t.items()}
        x[name][index] = value
        return run(cuda_device, x["q"], x["k"], x["v"], off, off, x["dout"], causal=True)

    def clean(got, n, rows):
        check(got[n][rows], tuple(y[rows] for y in want[n]), n)

    before, after = slice(0, at), slice(at, tokens)
    got = go("v", (at, 0, 5))
    clean(got, "out", before)
    assert not torch.isfinite(got["out"][after, :, 5]).any()
    others = [c for c in range(dim) if c != 5]
    check(got["out"][:, :, others], tuple(y[:, :, others] for y in want["out"]), "other columns of out")
    clean(got, "dq", before)
    clean(got, "dv", slice(0, tokens))
    # delta of the rows that see it is NaN or an infinity, and so is every ds of theirs
    assert not torch.isfinite(got["dq"][after]).any() and not torch.isfinite(got["dk"]).any()
    got = go("k", (at, 0))
    clean(got, "out", before)
    clean(got, "dq", before)
    got = go("dout", (at, 1, 7))
    check(got["dv"][at + 1:], tuple(y[at + 1:] for y in want["dv"]), "dv")
    check(got["dk"][at + 1:], tuple(y[at + 1:] for y in want["dk"]), "dk")
    assert not torch.isfinite(got["dv"][:at + 1, :, 7]).any()
    check(got["dv"][:, :, [c for c in range(dim) if c != 7]], tuple(y[:, :, [c for c in range(dim) if c != 7]] for y in want["dv"]), "dv")
    got = go("q", (at, 1))
    clean(got, "dk", slice(at + 1, tokens))
    clean(got, "dv", slice(at + 1, tokens))
    clean(got, "out", before)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keys", [12, 50, 200])
@pytest.mark.parametrize("where", [2**29 - 40, -(2**29) + 40, 2**31 - 2])
@pytest.mark.parametrize("reach", [(2, 2), (9, 30)])
def test_far_positions(cuda_device, dtype, keys, where, reach):
    """Positions far from 0 along both axes, under maps of few and of many columns: only differences count (beyond 2^29
    a position counts as 2^29)."""
    (q, k, v, do), qo, ko, g = inputs([40, 70], [keys, keys], 4, 2, 32, TYPES[dtype], seed=keys)
    buckets = torch.arange((2 * reach[0] + 1) * (2 * reach[1] + 1), dtype=torch.int32).view(2 * reach[0] + 1, -1)
    table = torch.randn(buckets.numel(), 4, generator=g)
    near = [torch.randint(0, 3, (x.shape[0], 2), generator=g) for x in (q, k)]
    at = [(x + where).clamp(-(2**31), 2**31 - 1).int() for x in near]
    ref = [x.clamp(-(2**29), 2**29) for x in at]
    want = window_attention(q, k, v, qo, ko, dout=do, table=table, buckets=buckets, q_pos=ref[0], k_pos=ref[1])
    got = run(cuda_device, q, k, v, qo, ko, do, table=table, buckets=buckets, q_pos=at[0], k_pos=at[1])
    for n in want:
        check(got[n], want[n], n)


# value of the table, and its type where not fp32
ALIKE = {"-1e9": (-1e9, None), "-3e7 of q's type": (-3e7, "same"), "lowest": (-math.inf, None), "lowest of q's type": (-math.inf, "same"),
         "highest": (math.inf, None)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", ALIKE)
@pytest.mark.parametrize("keys", [13, 20, 50, 300])
def test_rows_whose_keys_are_all_equally_far(cuda_device, dtype, bias, keys):
    """A row all of whose keys stand at one very low (or high) finite bias weighs them as without it, and so do its gradients."""
    t = TYPES[dtype]
    value, table_type = ALIKE[bias]
    tt = t if table_type == "same" else torch.float32
    value = min(max(value, torch.finfo(tt).min), torch.finfo(tt).max)
    (q, k, v, do), qo, ko, _ = inputs([40, 9], [keys, keys], 4, 2, 32, t, seed=keys)
    q.zero_()  # equal scores: what rounding takes from a score of 0 beside the bias is nothing
    table = torch.zeros(3, 4, dtype=tt)
    kw = dict(buckets=torch.tensor([[0, 1, 2]], dtype=torch.int32), q_pos=torch.zeros(49, dtype=torch.int32),
              k_pos=torch.full((2 * keys,), 5, dtype=torch.int32))
    want = window_attention(q, k, v, qo, ko, dout=do, table=table, **kw)
    table[2] = value
    got = run(cuda_device, q, k, v, qo, ko, do, table=table, **kw)
    for n in want:
        check(got[n], want[n], n)
    if value < 0:  # and beside one key that is not low, they count for nothing
        kw["k_pos"][[3, keys + 3]] = 0
        got = run(cuda_device, q, k, v, qo, ko, do, table=table, **kw)
        # the weight of the one key is 1, dp less delta the difference of two fp32 sums of dim products
        want = window_attention(q, k[[3, keys + 3]], v[[3, keys + 3]], qo, [0, 1, 2], dout=do, table=torch.zeros(3, 4, dtype=tt),
                                **{**kw, "k_pos": kw["k_pos"][[3, keys + 3]]})
        for n in ("out", "dq"):
            check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
def test_split_row_whose_keys_are_all_equally_far(cuda_device, dtype):
    (q, k, v, do), qo, ko, _ = inputs([1, 1], [3000, 2100], 4, 2, 64, TYPES[dtype])
    q.zero_()
    kw = dict(buckets=torch.tensor([[0, 0, 0]], dtype=torch.int32), q_pos=torch.zeros(2, dtype=torch.int32),
              k_pos=torch.zeros(5100, dtype=torch.int32))
    want = window_attention(q, k, v, qo, ko, dout=do, causal=True, table=torch.zeros(1, 4), **kw)
    got = run(cuda_device, q, k, v, qo, ko, do, causal=True, table=torch.full((1, 4), -1e9), **kw)
    for n in want:
        check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_rounding_of_out_at_any_address(cuda_device, dtype, shift):
    """The C entry points take what rounding took from out wherever its type may lie."""
    from oss_cuda import _lib, attention

    dev, lib, t = cuda_device, _lib.lib(), TYPES[dtype]
    (q, k, v, do), qo, ko, _ = inputs([150, 20], [200, 90], 2, 2, 32, t)
    want = window_attention(q, k, v, qo, ko, dout=do)
    q, k, v, do = (x.to(dev) for x in (q, k, v, do))
    off = [torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko)]
    args = attention._call_args(q, k, v, *off, 32**-0.5, 0, None, None, None, None)
    out, dq, dk, dv = (torch.empty_like(x) for x in (q, q, k, v))
    lse = torch.empty(2, *q.shape[1::-1], device=dev)
    lo = torch.empty(q.numel() + 8, dtype=t, device=dev)[shift:]
    sizes = (lib.oss_window_attention_scratch_bytes(*args[:7], 0, 0), lib.oss_window_attention_backward_scratch_bytes(*args[:7], 0, 0, 0))
    scratch = [torch.empty(n + 16, dtype=torch.uint8, device=dev) for n in sizes]
    stream = torch.cuda.current_stream(dev).cuda_stream
    saved = (out.data_ptr(), lse.data_ptr(), lo.data_ptr())
    _lib.check(lib.oss_window_attention_forward(*args, *saved, scratch[0].data_ptr(), sizes[0], stream), "forward")
    _lib.check(lib.oss_window_attention_backward(*args, *saved, do.data_ptr(), do.stride(0), do.stride(1), dq.data_ptr(), dk.data_ptr(),
                                                 dv.data_ptr(), None, scratch[1].data_ptr(), sizes[1], stream), "backward")
    for n, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(got, want[n], n)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_map_without_its_gradient(cuda_device, dtype):
    """Few keys a window under a map too large for the kernels of short windows, the table taking no gradient."""
    from oss_cuda import fused_window_cross_attention

    (q, k, v, do), qo, ko, g = inputs([70, 33, 20], [20, 50, 7], 4, 2, 32, TYPES[dtype])
    kw = dict(table=torch.randn(4095, 4, generator=g), buckets=torch.arange(4095, dtype=torch.int32).view(63, 65),
              q_pos=torch.randint(0, 32, (q.shape[0], 2), generator=g).int(), k_pos=torch.randint(0, 32, (k.shape[0], 2), generator=g).int())
    want = window_attention(q, k, v, qo, ko, dout=do, **kw)
    dev = cuda_device
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    off = [torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko)]
    kw = {n: t.to(dev) for n, t in kw.items()}
    out = fused_window_cross_attention(*leaves, *off, bias_table=kw.pop("table"), **kw)
    for n, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do.to(dev)))):
        check(got, want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,kv", [(128, 1, 1), (128, 4, 2), (32, 2, 2), (64, 2, 1)])
@pytest.mark.parametrize("shape", [(63, 65), (1, 4095)])
def test_largest_maps(cuda_device, dtype, dim, heads, kv, shape):
    """As many entries as a map may have, under every kernel."""
    (q, k, v, do), qo, ko, g = inputs([130, 60, 33], [200, 50, 20], heads, kv, dim, TYPES[dtype], seed=dim)
    buckets = torch.arange(shape[0] * shape[1], dtype=torch.int32).view(shape)
    table = torch.randn(buckets.numel(), heads, generator=g)
    spread = [(n - 1) // 2 for n in shape]
    pos = [torch.stack([torch.randint(-s // 2, s // 2 + 2, (x.shape[0],), generator=g) for s in spread], 1).int() for x in (q, k)]
    kw = dict(table=table, buckets=buckets, q_pos=pos[0], k_pos=pos[1])
    want = window_attention(q, k, v, qo, ko, dout=do, **kw)
    # Most rows of the table have one pair, many of them with next to no gradient. A pair's term joins integers at
    # 2^-30 of the sum of magnitudes of its tile (2^-60 in fp32), of which rounding takes half a step at most; a tile
    # is no more than 128 queries by all keys of the window.
    for a, b, c, e in zip(qo[:-1], qo[1:], ko[:-1], ko[1:]):
        bias, row = bias_of(table, buckets, pos[0][a:b], pos[1][c:e])
        qq, kk, vv, gg = (t.double() for t in (q[a:b], k[c:e].repeat_interleave(heads // kv, 1), v[c:e].repeat_interleave(heads // kv, 1), do[a:b]))
        p = torch.softmax(torch.einsum("ihd,jhd->hij", qq, kk) / dim**0.5 + bias.permute(2, 0, 1), -1)
        dp = torch.einsum("ihd,jhd->hij", gg, vv)
        ds = (p * (dp - (p * dp).sum(-1, keepdim=True))).abs()
        for i in range(0, b - a, 128):
            step = ds[:, i:i + 128].sum((1, 2)) * 2.0 ** (-61 if dtype == "fp32" else -31)
            rows = row[i:i + 128].reshape(-1)
            want["dtable"][1].index_add_(0, rows, 1.05 * step.expand(rows.numel(), heads))
    got = run(cuda_device, q, k, v, qo, ko, do, **kw)
    for n in want:
        check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,kv", [(7, 4, 2), (30, 3, 3), (32, 8, 2)])
@pytest.mark.parametrize("reach", [2, 6])
def test_few_keys_on_average_with_a_bias_gradient(cuda_device, dtype, dim, heads, kv, reach):
    """Windows of either class of the few-keys backward, and some of more keys, where the average has few."""
    from oss_cuda import window_position_buckets

    kl = [32, 17, 0, 31, 20, 16, 9, 60, 8, 1, 70] + [2] * 25
    ql = [64, 130, 5, 33, 16, 70, 3, 40, 90, 1, 20] + [7, 0, 40, 1, 18] * 5
    (q, k, v, do), qo, ko, g = inputs(ql, kl, heads, kv, dim, TYPES[dtype], seed=dim, qfirst=2, ktail=3)
    buckets = window_position_buckets(reach, reach)
    both(cuda_device, q, k, v, qo, ko, do, table=torch.randn(buckets.numel(), heads, generator=g).to(TYPES[dtype]), buckets=buckets,
         q_pos=torch.randint(0, 5, (q.shape[0], 2), generator=g).int(), k_pos=torch.randint(0, 5, (k.shape[0], 2), generator=g).int())
