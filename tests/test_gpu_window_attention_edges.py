"""Window attention where single values, sizes or callers could go wrong, against float64
(tests/attention_reference.py states the allowed errors)."""
from __future__ import annotations

import pytest
import torch

from attention_reference import check, window_attention
from test_gpu_window_attention import TYPES, inputs, run

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
