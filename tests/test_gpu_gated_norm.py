"""The gated residual norm against float64."""
from __future__ import annotations

import pytest
import torch

from attention_reference import F32, gated_norm, half_step

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def tensors(rows, c, dtype, gate, kind, params=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)

    def randn(*s, scale=1.0, shift=0.0, t=dtype):
        return (torch.randn(*s, generator=g) * scale + shift).to(t)

    a = {"x": randn(rows, c), "h": randn(rows, c, scale=2.0, shift=0.3),
         "weight": randn(c, scale=0.2, shift=1.0, t=params), "next_weight": randn(c, scale=0.2, shift=1.0, t=params),
         "scale": randn(c, scale=0.2, shift=0.5, t=params),
         "gate": None if gate == "none" else randn(rows, c if gate == "full" else 1)}
    if kind == "layer":
        a["bias"], a["next_bias"] = randn(c, scale=0.1, t=params), randn(c, scale=0.1, t=params)
    return a, randn(rows, c), randn(rows, c)


def run(dev, a, act="none", kind="rms", eps=1e-6, dy=None, dz=None):
    from oss_cuda import gated_residual_norm

    train = dy is not None or dz is not None
    t = {n: None if v is None else v.to(dev).detach().requires_grad_(train) for n, v in a.items()}
    kw = {n: t.get(n) for n in ("gate", "scale", "bias", "next_bias")}
    out = gated_residual_norm(t["x"], t["h"], t["weight"], t.get("next_weight"), gate_act=act, kind=kind, eps=eps, **kw)
    y, z = out if isinstance(out, tuple) else (out, None)
    res = {"y": y.detach()}
    if z is not None:
        res["z"] = z.detach()
    if train:
        outs, grads = zip(*[(o, d.to(dev)) for o, d in ((y, dy), (z, dz)) if o is not None and d is not None])
        leaves = [n for n in t if t[n] is not None]
        got = torch.autograd.grad(outs, [t[n] for n in leaves], grads, allow_unused=True)
        res.update({"d" + n: g for n, g in zip(leaves, got)})
    return res


def check(got, want, a, kind):
    """Rounding of each result, half a step; and fp32 on the way: a row's sums of c terms (c f at worst; pairwise
    sums of 8 and a tree are far below), some forty roundings, sigmoid with __expf (2^-21). Every value is a sum of
    few products of factors of the size of a deviation, so they are taken against the largest value of its row
    (of the whole result for the parameters, whose sums over rows cancel)."""
    rows, c = a["x"].shape
    for n, w in want.items():
        u = half_step(a[n[1:]].dtype if n.startswith("d") else a["x"].dtype)
        g = got[n].detach().cpu().double()
        assert g.shape == w.shape, n
        f = (64 + 8 + c / 8) * F32
        if n in ("dweight", "dscale", "dnext_weight", "dbias", "dnext_bias"):
            size = w.abs().max() + rows**0.5 * 4
            f = f + rows * F32 / 4
        else:
            size = w.abs().amax(-1, keepdim=True) + 4.0
            if n == "dgate" and w.shape[-1] == 1:
                size = size + c**0.5 * 4
        tiny = 2.0**-25 if g.dtype == torch.float16 or a["x"].dtype == torch.float16 else 0.0
        off = (g - w).abs()
        allowed = u * w.abs() * 1.01 + f * size + tiny
        assert (off <= allowed).all(), f"{n}: {float((off / allowed).max()):.3g} times the allowed error"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 2), (17, 8), (5, 63), (33, 64), (9, 100), (130, 128), (7, 181), (40, 256), (3, 257),
                                    (4, 1000), (11, 1024), (3, 2048), (2, 2056), (5, 5003), (2, 8192), (3000, 24)])
def test_sizes(cuda_device, dtype, kind, rows, c):
    if c == 1 and kind == "layer":
        pytest.skip("one channel has no deviation")
    a, dy, dz = tensors(rows, c, TYPES[dtype], "full" if rows % 2 else "row", kind, seed=c)
    eps = 0.1 if c < 4 else 1e-6  # the norm of a channel or two is its sign where eps is small: nothing to compare
    want = gated_norm(**a, act="sigmoid", kind=kind, eps=eps, dy=dy, dz=dz)
    check(run(cuda_device, a, "sigmoid", kind, eps, dy, dz), want, a, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["none", "row", "full"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
def test_gates(cuda_device, dtype, gate, act):
    if gate == "none" and act != "none":
        pytest.skip("no gate, no activation")
    for c in (40, 300):
        a, dy, dz = tensors(50, c, TYPES[dtype], gate, "layer")
        want = gated_norm(**a, act=act, kind="layer", dy=dy, dz=dz)
        check(run(cuda_device, a, act, "layer", dy=dy, dz=dz), want, a, "layer")


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_activation_without_gate_changes_nothing(cuda_device, act):
    a, dy, dz = tensors(37, 72, torch.bfloat16, "none", "rms")
    want, got = (run(cuda_device, a, x, dy=dy, dz=dz) for x in ("none", act))
    assert all(torch.equal(got[n], want[n]) for n in want if want[n] is not None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("leave", [["scale"], ["gate"], ["next_weight"], ["scale", "gate", "next_weight"]])
def test_parts_left_out(cuda_device, dtype, leave):
    a, dy, dz = tensors(37, 72, TYPES[dtype], "full", "rms", params=TYPES[dtype])
    for n in leave:
        a[n] = None
    dz = None if "next_weight" in leave else dz
    want = gated_norm(**a, dy=dy, dz=dz)
    check(run(cuda_device, a, dy=dy, dz=dz), want, a, "rms")


@pytest.mark.parametrize("which", ["dy", "dz"])
def test_one_result_used(cuda_device, which):
    a, dy, dz = tensors(37, 72, torch.bfloat16, "full", "layer")
    kw = {"dy": dy} if which == "dy" else {"dz": dz}
    want = gated_norm(**a, kind="layer", **kw)
    got = run(cuda_device, a, "none", "layer", **kw)
    got = {n: torch.zeros_like(a[n[1:]]) if g is None else g for n, g in got.items()}
    check(got, want, a, "layer")


def test_some_gradients_wanted(cuda_device):
    from oss_cuda import gated_residual_norm

    a, dy, dz = tensors(20, 48, torch.float32, "full", "rms")
    t = {n: v.to(cuda_device) for n, v in a.items() if v is not None}
    want = gated_norm(**a, dy=dy, dz=dz)
    for n in t:
        leaf = t[n].detach().requires_grad_(True)
        args = {**t, n: leaf}
        y, z = gated_residual_norm(args["x"], args["h"], args["weight"], args["next_weight"], gate=args["gate"], scale=args["scale"])
        (g,) = torch.autograd.grad([y, z], [leaf], [dy.to(cuda_device), dz.to(cuda_device)])
        check({"d" + n: g}, {"d" + n: want["d" + n]}, a, "rms")


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(cuda_device, dtype):
    """Batches of rows, slices of wider rows, transposed tensors, rows no vector is aligned to."""
    from oss_cuda import gated_residual_norm

    a, dy, dz = tensors(24, 64, TYPES[dtype], "full", "rms")
    want = gated_norm(**a)
    dev = cuda_device
    w, w2, s = (a[n].to(dev) for n in ("weight", "next_weight", "scale"))
    x, h, g = (a[n].to(dev) for n in ("x", "h", "gate"))

    def go(x, h, g):
        y, z = gated_residual_norm(x, h, w, w2, gate=g, scale=s)
        assert y.shape == x.shape and y.is_contiguous()
        check({"y": y.reshape(24, 64), "z": z.reshape(24, 64)}, want, a, "rms")

    go(x.view(2, 3, 4, 64), h.view(2, 3, 4, 64), g.view(2, 3, 4, 64))
    wide = torch.cat([x, h, g], 1)
    go(wide[:, :64], wide[:, 64:128], wide[:, 128:])
    odd = torch.cat([wide[:, :1], wide], 1)
    go(odd[:, 1:65], odd[:, 65:129], odd[:, 129:])
    go(x.t().contiguous().t(), h.t().contiguous().t(), g.t().contiguous().t())


def test_expanded_gate_takes_its_gradient(cuda_device):
    """One gate for all rows, broadcast by the caller."""
    a, dy, dz = tensors(30, 40, torch.float32, "none", "rms")
    from oss_cuda import gated_residual_norm

    gate = torch.randn(40)
    a["gate"] = gate.expand(30, 40)
    want = gated_norm(**a, act="silu", dy=dy, dz=dz)
    leaf = gate.to(cuda_device).requires_grad_(True)
    t = {n: v.to(cuda_device) for n, v in a.items()}
    y, z = gated_residual_norm(t["x"], t["h"], t["weight"], t["next_weight"], gate=leaf.expand(30, 40), gate_act="silu", scale=t["scale"])
    (g,) = torch.autograd.grad([y, z], [leaf], [dy.to(cuda_device), dz.to(cuda_device)])
    off = (g.cpu().double() - want["dgate"].sum(0)).abs().max()
    assert off <= 30 * 200 * F32 * 4


def test_rows_not_finite_stay_alone(cuda_device):
    a, _, _ = tensors(40, 96, torch.bfloat16, "full", "layer")
    want = gated_norm(**a, kind="layer")
    a["h"][7] = float("nan")
    a["x"][21] = float("inf")
    got = run(cuda_device, a, "none", "layer")
    rows = [r for r in range(40) if r not in (7, 21)]
    check({n: got[n][rows] for n in want}, {n: w[rows] for n, w in want.items()}, a, "layer")
    assert torch.isnan(got["y"][7]).all() and torch.isinf(got["y"][21]).all()


def test_constant_rows(cuda_device):
    """A row without deviation: eps alone holds the quotient."""
    a, dy, dz = tensors(4, 64, torch.float32, "none", "layer")
    a["h"][1] = 3.0
    a["h"][2] = 0.0
    want = gated_norm(**a, kind="layer", eps=1e-2, dy=dy, dz=dz)
    check(run(cuda_device, a, "none", "layer", 1e-2, dy, dz), want, a, "layer")


def test_large_mean_is_taken_out_first(cuda_device):
    a, _, _ = tensors(8, 512, torch.float32, "none", "layer")
    a["h"] += 1000.0
    want = gated_norm(**a, kind="layer")
    got = run(cuda_device, a, "none", "layer")
    # h itself holds its deviations to 2^-24 of 1000; a mean that is off by as much moves all of them
    assert (got["y"].cpu().double() - want["y"]).abs().max() <= 1000 * 8 * F32


def test_no_rows(cuda_device):
    a, dy, dz = tensors(0, 32, torch.float32, "full", "layer")
    got = run(cuda_device, a, "none", "layer", dy=dy, dz=dz)
    assert got["y"].shape == (0, 32) and not got["dweight"].any() and not got["dnext_bias"].any()


def test_same_bits_every_time(cuda_device):
    a, dy, dz = tensors(5000, 128, torch.bfloat16, "row", "layer")
    first = run(cuda_device, a, "sigmoid", "layer", dy=dy, dz=dz)
    again = run(cuda_device, a, "sigmoid", "layer", dy=dy, dz=dz)
    for n in first:
        assert torch.equal(first[n], again[n])


def test_capture_and_replay(cuda_device):
    from oss_cuda import gated_residual_norm

    dev = cuda_device
    a, dy, dz = tensors(60, 96, torch.bfloat16, "full", "rms")
    t = {n: v.to(dev) for n, v in a.items()}
    dy, dz = dy.to(dev), dz.to(dev)

    def step():
        leaves = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        y, z = gated_residual_norm(leaves["x"], leaves["h"], leaves["weight"], leaves["next_weight"], gate=leaves["gate"],
                                   scale=leaves["scale"], gate_act="silu")
        return (y.detach(), z.detach(), *torch.autograd.grad([y, z], list(leaves.values()), [dy, dz]))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    t["x"].mul_(-0.5)
    t["gate"].add_(1.0)
    graph.replay()
    for x, y in zip(res, step()):
        assert torch.equal(x, y)
