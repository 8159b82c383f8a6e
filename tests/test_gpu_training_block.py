"""The training operators together, as the training step of a Swin block: bias
table -> window attention -> projections -> residual sum, drop path and norm2
-> MLP on 8-bit copies, against the same block in 64 bits."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import crumpet_amd
import training_reference as ref
from crumpet_amd import training
from helpers import seeded
from oracle import oracle

pytestmark = pytest.mark.gpu

VOLUME, WS, SHIFT, C, HEADS = (12, 6, 12), (6, 6, 6), (3, 3, 3), 48, 3


def _params():
    shapes = {"norm1_w": (C,), "norm1_b": (C,), "table": (11 ** 3, HEADS), "qkv_w": (3 * C, C), "qkv_b": (3 * C,),
              "proj_w": (C, C), "proj_b": (C,), "norm2_w": (C,), "norm2_b": (C,), "w1": (4 * C, C), "b1": (4 * C,),
              "w2": (C, 4 * C), "b2": (C,)}
    p = {n: 0.1 * seeded(s, torch.float32, 100 + i) for i, (n, s) in enumerate(shapes.items())}
    for n in ("norm1_w", "norm2_w"):
        p[n] += 1
    for n in ("qkv_w", "proj_w", "w1", "w2"):
        p[n] *= 10 * p[n].shape[1] ** -0.5
    return p


def _block(x, p, plan, drop, dtype):
    """A shifted block with the framework's operators; Linears in ``dtype``."""
    b = x.shape[0]
    h = F.layer_norm(x, (C,), p["norm1_w"], p["norm1_b"]).to(dtype)
    win = crumpet_amd.fused_shift_partition_3d(h, WS, SHIFT)
    c = {n: v.to(dtype) for n, v in p.items() if n not in ("norm1_w", "norm1_b", "norm2_w", "norm2_b", "table")}
    qkv = F.linear(win, c["qkv_w"], c["qkv_b"])
    bias = training.relative_position_bias(p["table"], plan)
    a = training.window_attention(qkv, bias, HEADS, volume=VOLUME, window_size=WS, shift_size=SHIFT)
    y = crumpet_amd.fused_unshift_unpartition_3d(F.linear(a, c["proj_w"], c["proj_b"]), b, *VOLUME, C, WS, SHIFT)
    x1, h = training.residual_norm(x, y, weight=p["norm2_w"], bias=p["norm2_b"], scale=drop)
    h = training.linear_8bit(h, c["w1"], c["b1"])
    return x1 + training.linear_8bit(h, c["w2"], c["b2"], "gelu")


def _plain(x, p, index, drop):
    n = WS[0] * WS[1] * WS[2]

    def windows(t):
        t = torch.roll(t, [-s for s in SHIFT], (1, 2, 3))
        g = [v // w for v, w in zip(VOLUME, WS)]
        t = t.view(-1, g[0], WS[0], g[1], WS[1], g[2], WS[2], t.shape[-1])
        return t.permute(0, 1, 3, 5, 2, 4, 6, 7).reshape(-1, n, t.shape[-1])

    def volume(t):
        g = [v // w for v, w in zip(VOLUME, WS)]
        t = t.view(-1, *g, *WS, t.shape[-1]).permute(0, 1, 4, 2, 5, 3, 6, 7).reshape(-1, *VOLUME, t.shape[-1])
        return torch.roll(t, SHIFT, (1, 2, 3))

    h = F.layer_norm(x, (C,), p["norm1_w"], p["norm1_b"])
    q, k, v = F.linear(windows(h), p["qkv_w"], p["qkv_b"]).view(-1, n, 3, HEADS, 16).permute(2, 0, 3, 1, 4)
    s = 0.25 * q @ k.transpose(2, 3) + p["table"][index.reshape(-1)].view(n, n, HEADS).permute(2, 0, 1)
    mask = ref.shift_mask(VOLUME, WS, SHIFT).double()
    s = s + mask.repeat(s.shape[0] // mask.shape[0], 1, 1)[:, None]
    a = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(-1, n, C)
    x1 = x + drop[:, None, None, None, None] * volume(F.linear(a, p["proj_w"], p["proj_b"]))
    h = F.layer_norm(x1, (C,), p["norm2_w"], p["norm2_b"])
    return x1 + F.linear(F.gelu(F.linear(h, p["w1"], p["b1"])), p["w2"], p["b2"])


@pytest.mark.parametrize("dtype,tol", [(torch.float16, 2.0 ** -6), (torch.bfloat16, 2.0 ** -5)], ids=str)
def test_training_step(dev, dtype, tol):
    """Norm-wise: the gradients take the 8-bit copies, half a step of which is
    up to 2^-7 of a group's largest value (2^-9 to 2^-8 of the norm of normal
    values, in two layers), and about ten roundings of half a step of the
    16-bit type; bf16's 2^-9 each add up to as much again."""
    p, x, g = _params(), seeded((2, *VOLUME, C), torch.float32, 1), seeded((2, *VOLUME, C), torch.float32, 2)
    index = torch.from_numpy(oracle.relative_position_index(WS))
    drop = torch.tensor([1.25, 1.0])
    leaves = {n: v.to(dev).requires_grad_() for n, v in p.items()}
    xd = x.to(dev).requires_grad_()
    plan = training.BiasBuckets(index.to(dev), 11 ** 3)
    out = _block(xd, leaves, plan, drop.to(dev), dtype)
    found = torch.autograd.grad(out, [xd, *leaves.values()], g.to(dev))
    p64 = {n: v.double().requires_grad_() for n, v in p.items()}
    x64 = x.double().requires_grad_()
    out64 = _plain(x64, p64, index, drop.double())
    expected = torch.autograd.grad(out64, [x64, *p64.values()], g.double())
    assert float((out.cpu() - out64).norm() / out64.norm()) < tol
    for name, a, b in zip(["x", *p], found, expected):
        assert a.dtype == torch.float32
        assert float((a.cpu().double() - b).norm() / b.norm()) < tol, name


def test_training_step_captured(dev):
    p, index = _params(), torch.from_numpy(oracle.relative_position_index(WS))
    leaves = {n: v.to(dev).requires_grad_() for n, v in p.items()}
    x = seeded((1, *VOLUME, C), torch.float32, 1).to(dev).requires_grad_()
    g = seeded((1, *VOLUME, C), torch.float32, 2).to(dev)
    drop = torch.ones(1, device=dev)
    plan = training.BiasBuckets(index.to(dev), 11 ** 3)

    def step():
        out = _block(x, leaves, plan, drop, torch.float16)
        return (out, *torch.autograd.grad(out, [x, *leaves.values()], g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    names = ["out", "x", *p]
    # torch's own Linear and LayerNorm gradients are left out of the bitwise comparison
    ours = ("out", "table", "norm2_w", "norm2_b", "w1", "b1", "w2", "b2")
    for s in range(3):
        with torch.no_grad():
            x.copy_(seeded((1, *VOLUME, C), torch.float32, 10 + s))
            g.copy_(seeded((1, *VOLUME, C), torch.float32, 20 + s))
        graph.replay()
        expected = step()
        torch.cuda.synchronize()
        for n, a, b in zip(names, outs, expected):
            if n in ours:
                assert torch.equal(a, b), (s, n)
            else:
                torch.testing.assert_close(a, b, rtol=2.0 ** -9, atol=2.0 ** -9 * float(b.abs().max()))
