"""The feature block of a canvas as it is used: Gaussians sorted into tiles, their features normed, attending
to the pixels of their tile with a learned position bias, gated back into the residual stream and rendered.

Each operator's values and gradients are checked in place, against float64 of what it was given there."""
from __future__ import annotations

import pytest
import torch

from attention_reference import check, gated_norm, window_attention
from test_gpu_gated_norm import check as check_norm

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
H, W, TILE, HEADS, KV, DIM = 40, 56, 16, 4, 2, 8
C = HEADS * DIM


def scene(dev, dtype, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    ty, tx = -(-H // TILE), -(-W // TILE)
    y, x = torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij")
    tile_of = (y // TILE * tx + x // TILE).flatten()
    order = torch.argsort(tile_of, stable=True)  # the pixels tile by tile; tiles at the rim are smaller
    k_off = torch.zeros(ty * tx + 1, dtype=torch.int32)
    k_off[1:] = torch.bincount(tile_of, minlength=ty * tx).cumsum(0)
    xy = torch.rand(n, 2, generator=g) * torch.tensor([W - 1.0, H - 17.0])  # the last row of tiles holds none
    s = {"xy": xy, "scale": torch.rand(n, 2, generator=g) * 3 + 1, "rot": torch.rand(n, generator=g),
         "tile": (xy[:, 1].long() // TILE * tx + xy[:, 0].long() // TILE).int(), "k_off": k_off,
         "k_pos": torch.stack([y.flatten(), x.flatten()], 1)[order].int(), "tiles": ty * tx}

    def randn(*shape, t=dtype, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g) * scale + shift).to(t)

    s["leaves"] = {"x": randn(n, C), "h": randn(n, C), "k": randn(H * W, KV, DIM), "v": randn(H * W, KV, DIM), "gate": randn(n, C),
                   "w1": randn(C, t=torch.float32, scale=0.2, shift=1.0), "w2": randn(C, t=torch.float32, scale=0.2, shift=1.0),
                   "w3": randn(C, t=torch.float32, scale=0.2, shift=1.0),
                   "table": randn(31 * 31, HEADS, t=torch.float32, scale=0.3)}
    move = lambda t: t.to(dev) if torch.is_tensor(t) else t  # noqa: E731
    return {a: {c: move(d) for c, d in b.items()} if isinstance(b, dict) else move(b) for a, b in s.items()}


def block(s, leaves):
    """The block's intermediate values, by name."""
    import oss_cuda

    gid, q_off = oss_cuda.tile_bin_counting_sort(s["tile"], torch.arange(s["tile"].numel(), device=s["tile"].device).int(),
                                                 s["tiles"])
    at = gid.long()
    xy = s["xy"][at]
    y1, z1 = oss_cuda.gated_residual_norm(leaves["x"], leaves["h"], leaves["w1"], leaves["w2"])
    q = z1.view(-1, HEADS, DIM)
    o = oss_cuda.fused_window_cross_attention(
        q, leaves["k"], leaves["v"], q_off, s["k_off"], bias_table=leaves["table"],
        buckets=oss_cuda.window_position_buckets(15, 15, device=q.device), q_pos=xy.flip(1).int().contiguous(), k_pos=s["k_pos"])
    y2 = oss_cuda.gated_residual_norm(y1, o.reshape(-1, C), leaves["w3"], gate=leaves["gate"], gate_act="sigmoid")
    return dict(q_off=q_off, at=at, q_pos=xy.flip(1).int(), y1=y1, z1=z1, o=o, y2=y2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 70, 900])
def test_block_and_its_gradients(cuda_device, dtype, n):
    import oss_cuda

    s = scene(cuda_device, TYPES[dtype], n)
    leaves = {a: t.requires_grad_(True) for a, t in s["leaves"].items()}
    m = block(s, leaves)
    for name in ("y1", "z1", "o", "y2"):
        m[name].retain_grad()
    at = m["at"]
    image = oss_cuda.rasterize_gaussians(s["xy"][at], s["scale"][at], s["rot"][at], m["y2"].float(), H, W)
    target = torch.randn(image.shape, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    (image * target).sum().backward()
    assert image.shape == (C, H, W) and torch.isfinite(image).all() and image.abs().max() > 0
    grad = {a: t.grad for a, t in leaves.items()}
    assert all(torch.isfinite(t).all() for t in grad.values())
    assert m["y2"].grad.abs().max() > 0

    a = {"x": leaves["x"], "h": leaves["h"], "weight": leaves["w1"], "next_weight": leaves["w2"]}
    want = gated_norm(**a, dy=m["y1"].grad, dz=m["z1"].grad)
    got = {"y": m["y1"], "z": m["z1"], "dx": grad["x"], "dh": grad["h"], "dweight": grad["w1"], "dnext_weight": grad["w2"]}
    check_scaled(got, want, a)

    want = window_attention(m["z1"].view(-1, HEADS, DIM), leaves["k"], leaves["v"], m["q_off"].tolist(), s["k_off"].tolist(),
                            dout=m["o"].grad, table=leaves["table"], buckets=oss_cuda.window_position_buckets(15, 15),
                            q_pos=m["q_pos"], k_pos=s["k_pos"])
    got = {"out": m["o"], "dq": m["z1"].grad.view(-1, HEADS, DIM), "dk": grad["k"], "dv": grad["v"], "dtable": grad["table"]}
    for name in want:
        check(got[name], want[name], name)

    a = {"x": m["y1"], "h": m["o"].reshape(-1, C), "weight": leaves["w3"], "gate": leaves["gate"]}
    want = gated_norm(**a, act="sigmoid", dy=m["y2"].grad)
    got = {"y": m["y2"], "dx": m["y1"].grad, "dh": m["o"].grad.view(-1, C), "dweight": grad["w3"], "dgate": grad["gate"]}
    check_scaled(got, want, a)


def check_scaled(got, want, a):
    """check_norm's errors are for gradients of the size of one: a power of two brings these there (exact), and the
    values of the rms norm take none."""
    dtype = a["x"].dtype
    if dtype == torch.float16:  # its subnormal step does not scale along: the values alone
        got, want = ({n: t for n, t in d.items() if not n.startswith("d")} for d in (got, want))
    for side in (False, True):
        names = [n for n in want if n.startswith("d") == side and n in got]
        if not names:
            continue
        top = max(float(want[n].abs().max()) for n in names)
        by = 2.0 ** -torch.tensor(max(top, 1e-30)).log2().floor().item() if side else 1.0
        check_norm({n: got[n].detach().cpu().double() * by for n in names}, {n: want[n] * by for n in names}, a, "rms")


@pytest.mark.parametrize("dtype", TYPES)
def test_block_captured_and_replayed(cuda_device, dtype):
    a, b = (scene(cuda_device, TYPES[dtype], 300, seed) for seed in (2, 3))
    with torch.no_grad():
        want = [block(s, s["leaves"]) for s in (a, b)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(a, a["leaves"])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = block(a, a["leaves"])
        for s, w in zip((a, b), want):
            for name, t in s.items():  # the other scene's values into the captured tensors
                if torch.is_tensor(t):
                    a[name].copy_(t)
            for name, t in s["leaves"].items():
                a["leaves"][name].copy_(t)
            graph.replay()
            for name in ("q_off", "at", "y1", "z1", "o", "y2"):
                assert torch.equal(got[name], w[name]), name
