"""training.residual_norm and its gradients against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import training_reference as ref
from crumpet_amd import training
from helpers import seeded

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
         (torch.float32, torch.float16), (torch.float32, torch.bfloat16)]


def _params(C, S, kind="layer", post=True, gate="sample", scale=True, dtype=torch.float32):
    p = {"weight": 1 + 0.1 * seeded((C,), torch.float32, 1), "post_weight": None, "post_bias": None, "gate": None,
         "scale": None, "bias": 0.1 * seeded((C,), torch.float32, 2) if kind == "layer" else None}
    if post:
        p["post_weight"] = 1 + 0.1 * seeded((C,), torch.float32, 3)
        p["post_bias"] = 0.1 * seeded((C,), torch.float32, 4) if kind == "layer" else None
    if gate:
        p["gate"] = 0.5 * seeded((S, C) if gate == "sample" else (C,), torch.float32, 5)
    p = {k: None if v is None else v.to(dtype) for k, v in p.items()}
    if scale:
        p["scale"] = torch.tensor([1.25, 0.0, 1.0, 0.5][:S] + [1.25] * max(0, S - 4))
    return p


def _run(dev, x, y, gs, go, kind, post, params, e=1e-5):
    t = {k: v.to(dev) for k, v in params.items() if v is not None}
    leaves = {"x": x.to(dev).requires_grad_(), "y": y.to(dev).requires_grad_()}
    leaves.update({k: v.requires_grad_() for k, v in t.items() if k != "scale"})
    args = {k: leaves.get(k, t.get(k)) for k in params}
    x1, h = training.residual_norm(leaves["x"], leaves["y"], norm=kind, post=post, eps=e, **args)
    outs = [(o, g.to(dev)) for o, g in ((x1, gs), (h, go)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    found = {"sum": x1, "out": h}
    found.update({"grad_" + k: g for k, g in zip(leaves, grads) if g is not None})
    return found


def _check(dev, shape, types, kind="layer", post=True, gate="sample", scale=True, seed=0, param_dtype=torch.float32):
    x, y = seeded(shape, types[0], seed + 10), seeded(shape, types[1], seed + 11)
    gs, go = seeded(shape, types[0], seed + 12), seeded(shape, types[1], seed + 13)
    p = _params(shape[-1], shape[0], kind, post, gate, scale, param_dtype)
    ref.check(_run(dev, x, y, gs, go, kind, post, p), ref.residual_norm(x, y, gs, go, kind, post, **p))


# a row in 8 to 64 lanes or the workgroup, whole and partly filled; channels one by one
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("C", [8, 48, 64, 96, 200, 384, 768, 1032, 2056, 4104, 1, 3, 65, 100, 257, 1025])
def test_channels(dev, types, C):
    _check(dev, (2, 5, C), types)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "sample"])
@pytest.mark.parametrize("scale", [False, True])
def test_forms(dev, kind, post, gate, scale):
    _check(dev, (4, 37, 48), (torch.float32, torch.float16), kind, post, gate, scale)
    _check(dev, (3, 9, 50), (torch.bfloat16, torch.bfloat16), kind, post, gate, scale)


@pytest.mark.parametrize("shape", [(1, 1, 48), (1, 70001, 48), (5, 3, 4, 5, 2, 96), (1000, 2, 16)], ids=str)
def test_rows(dev, shape):
    _check(dev, shape, (torch.float32, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_parameters_of_16_bits(dev, dtype):
    _check(dev, (3, 20, 64), (dtype, dtype), param_dtype=dtype)


def test_without_parameters(dev):
    x, y, gs, go = (seeded((40, 32), torch.float32, i) for i in range(4))
    none = dict.fromkeys(("weight", "bias", "post_weight", "post_bias", "gate", "scale"))
    for post in (False, True):
        ref.check(_run(dev, x, y, gs, go, "layer", post, none), ref.residual_norm(x, y, gs, go, "layer", post))


def test_one_row_vector(dev):
    x, y, gs, go = (seeded((32,), torch.float32, i) for i in range(4))
    none = dict.fromkeys(("weight", "bias", "post_weight", "post_bias", "gate", "scale"))
    expected = ref.residual_norm(*(t[None] for t in (x, y, gs, go)))
    found = _run(dev, x, y, gs, go, "layer", False, none)
    ref.check({k: v[None] for k, v in found.items()}, expected)


@pytest.mark.parametrize("which", ["sum", "out"])
def test_one_result_used(dev, which):
    shape = (2, 9, 48)
    x, y = seeded(shape, torch.float32, 0), seeded(shape, torch.float16, 1)
    gs, go = (seeded(shape, torch.float32, 2), None) if which == "sum" else (None, seeded(shape, torch.float16, 3))
    p = _params(48, 2)
    ref.check(_run(dev, x, y, gs, go, "layer", True, p), ref.residual_norm(x, y, gs, go, "layer", True, **p))


def test_constant_rows_and_dropped_samples(dev):
    """A row of equal values has no deviation: eps alone; a dropped sample's
    branch gets no gradient, even where it holds infinities."""
    x, y = torch.full((2, 3, 48), 2.0), torch.full((2, 3, 48), -1.0)
    gs, go = seeded((2, 3, 48), torch.float32, 2), seeded((2, 3, 48), torch.float32, 3)
    p = _params(48, 2, post=False, gate=None, scale=False)
    ref.check(_run(dev, x, y, gs, go, "layer", False, p, 1e-2), ref.residual_norm(x, y, gs, go, "layer", False, 1e-2, **p))
    p = _params(48, 2, post=False, gate=None)
    found = _run(dev, x, y, gs, go, "layer", False, p)
    assert torch.equal(found["grad_y"][1], torch.zeros_like(found["grad_y"][1]))
    assert torch.equal(found["sum"][1].cpu(), x[1])


def test_large_offsets_cancel(dev):
    """Rows far from zero: two passes over the row keep the deviation."""
    shape = (2, 8, 96)
    x, y = seeded(shape, torch.float32, 0) + 1000, seeded(shape, torch.float32, 1)
    gs, go = seeded(shape, torch.float32, 2), seeded(shape, torch.float32, 3)
    p = _params(96, 2, post=False, gate=None, scale=False)
    ref.check(_run(dev, x, y, gs, go, "layer", False, p), ref.residual_norm(x, y, gs, go, "layer", False, **p))


def test_strides(dev):
    shape = (3, 10, 48)
    x, y = seeded(shape, torch.float32, 0), seeded(shape, torch.float16, 1)
    gs, go = seeded(shape, torch.float32, 2), seeded(shape, torch.float16, 3)
    p = {k: None if v is None else v for k, v in _params(48, 3).items()}
    expected = ref.residual_norm(x, y, gs, go, "layer", True, **p)

    def turned(t):
        return t.to(dev).transpose(0, 2).contiguous().transpose(0, 2)

    def shifted(t):  # storage that starts at no multiple of 16 bytes
        return torch.cat([t.new_zeros(1), t.flatten()]).to(dev)[1:].view_as(t)

    for f in (turned, shifted):
        a, b = f(x).requires_grad_(), f(y).requires_grad_()
        q = {k: None if v is None else shifted(v) for k, v in p.items()}
        x1, h = training.residual_norm(a, b, post=True, **q)
        dx, dy = torch.autograd.grad((x1, h), (a, b), (f(gs), f(go)))
        ref.check({"sum": x1, "out": h, "grad_x": dx, "grad_y": dy}, expected)


def test_nothing_to_norm(dev):
    p = {k: None if v is None else v.to(dev).requires_grad_(k != "scale") for k, v in _params(48, 2).items()}
    x = torch.zeros((2, 0, 48), device=dev, requires_grad=True)
    x1, h = training.residual_norm(x, x, post=True, **p)
    assert x1.shape == h.shape == (2, 0, 48)
    grads = torch.autograd.grad(x1.sum() + h.sum(), [p["weight"], p["gate"]])
    assert all(torch.equal(g, torch.zeros_like(g)) for g in grads)


def test_repeats_captured_and_on_another_stream(dev):
    shape = (4, 500, 96)
    data = [[seeded(shape, t, 10 * s + i) for i, t in enumerate((torch.float32, torch.float16) * 2)] for s in range(4)]
    p = {k: None if v is None else v.to(dev) for k, v in _params(96, 4).items()}
    leaves = [v.requires_grad_() for k, v in p.items() if k != "scale"]

    def run(x, y, gs, go):
        x1, h = training.residual_norm(x, y, post=True, **p)
        return (x1, h, *torch.autograd.grad((x1, h), [x, y, *leaves], (gs, go)))

    ins = [t.to(dev) for t in data[0]]
    ins[0].requires_grad_()
    ins[1].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = run(*ins)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, run(*ins)))
    del first  # no eager graph of the leaves lives during the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(*ins)
    for s in (1, 2, 3):
        with torch.no_grad():
            for t, v in zip(ins, data[s]):
                t.copy_(v)
        graph.replay()
        expected = run(*ins)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expected))


def test_compiled(dev):
    x, y = (seeded((2, 9, 48), torch.float32, i).to(dev).requires_grad_() for i in range(2))
    w = torch.ones(48, device=dev, requires_grad=True)

    def f(x, y, w):
        a, b = training.residual_norm(x, y, weight=w)
        return a * 2 + b

    out = torch.compile(f, backend="aot_eager", fullgraph=True)(x, y, w)
    found = torch.autograd.grad(out.sum(), (x, y, w))
    expected = torch.autograd.grad(f(x, y, w).sum(), (x, y, w))
    assert all(torch.equal(a, b) for a, b in zip(found, expected))


def test_refusals(dev):
    x = torch.zeros((2, 4, 48), device=dev)

    def refused(match, *args, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            training.residual_norm(*args, **kw)

    refused("one shape", x, x[:, :3])
    refused("norm must be one of", x, x, norm="batch")
    refused("need post", x, x, post_weight=torch.ones(48, device=dev))
    refused("weight must have shape", x, x, weight=torch.ones(47, device=dev))
    refused("gate must have shape", x, x, gate=torch.ones((3, 48), device=dev))
    refused("scale must have shape", x, x, scale=torch.ones(3, device=dev))
    refused("scale has no gradient", x.requires_grad_(), x, scale=torch.ones(2, device=dev, requires_grad=True))
    refused("float32 or of y's type", x.half(), x)
    refused("float32, float16 or bfloat16", x.double(), x.double())
    refused("must be on", x, x.cpu())
    refused("8192", torch.zeros((1, 8200), device=dev), torch.zeros((1, 8200), device=dev))
    refused("4096", torch.zeros((1, 4097), device=dev), torch.zeros((1, 4097), device=dev))
    a, b = training.residual_norm(x, x)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(b.sum(), x, create_graph=True)


def test_infinities_are_not_hidden(dev):
    x = torch.zeros((1, 2, 48), device=dev)
    x[0, 0, 3] = math.inf
    _, h = training.residual_norm(x, torch.zeros_like(x))
    assert h[0, 0].isnan().any() and not h[0, 1].isnan().any()
