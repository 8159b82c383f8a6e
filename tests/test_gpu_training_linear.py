"""training.linear_8bit and its gradients against 64 bits; the 8-bit copy itself, exactly."""

from __future__ import annotations

import math

import pytest
import torch

import training_reference as ref
from crumpet_amd import training
from helpers import seeded

pytestmark = pytest.mark.gpu

HALF = (torch.float16, torch.bfloat16)


def _inputs(rows, K, n_out, dtype, seed=0):
    return (seeded((rows, K), dtype, seed), (seeded((n_out, K), torch.float32, seed + 1) * K ** -0.5).to(dtype),
            seeded((n_out,), dtype, seed + 2), seeded((rows, n_out), dtype, seed + 3))


def _run(dev, x, w, b, g, activation="none"):
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b) if t is not None]
    y = training.linear_8bit(leaves[0], leaves[1], leaves[2] if b is not None else None, activation)
    grads = torch.autograd.grad(y, leaves, g.to(dev))
    return {"out": y, **dict(zip(("grad_x", "grad_weight", "grad_bias"), grads))}


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("activation", ["none", "gelu"])
@pytest.mark.parametrize("rows,K,n_out", [(1, 16, 16), (5, 48, 32), (63, 32, 48), (64, 96, 16), (65, 192, 48),
                                          (129, 80, 144), (257, 48, 192), (300, 272, 272), (1000, 64, 128),
                                          (2, 1536, 384)])
def test_sizes(dev, dtype, activation, rows, K, n_out):
    x, w, b, g = _inputs(rows, K, n_out, dtype, seed=rows)
    ref.check(_run(dev, x, w, b, g, activation), ref.linear_8bit(x, w, b, g, activation))


@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_many_rows(dev, activation):
    x, w, b, g = _inputs(40007, 96, 48, torch.bfloat16)
    ref.check(_run(dev, x, w, b, g, activation), ref.linear_8bit(x, w, b, g, activation))


def _copy(dev, x):
    K = x.shape[1]
    w = torch.zeros((16, K), dtype=x.dtype, device=dev)
    _, codes, exps = torch.ops.crumpet_ops.linear_8bit_forward(x.to(dev), w, None, 0)
    assert codes.shape == x.shape and exps.shape == (x.shape[0], (K + 31) // 32)
    e = exps.cpu().double().repeat_interleave(32, 1)[:, :K]
    step = torch.where(e == -128, math.nan, 2.0 ** e)
    return codes.cpu().double() * step, codes.cpu()


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("K", [16, 32, 48, 208])
def test_the_copy_is_exact(dev, dtype, K):
    x = seeded((300, K), dtype, K)
    x *= 2.0 ** torch.randint(-14, 8, (300, 1), generator=torch.Generator().manual_seed(1)).to(dtype)
    kept, codes = _copy(dev, x)
    assert torch.equal(kept, ref.eight_bits(x)) and int(codes.min()) >= -127


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_the_copy_at_its_limits(dev, dtype):
    info = torch.finfo(dtype)
    tiny = info.tiny * info.eps  # the smallest subnormal
    rows = [[0.0], [info.max], [-info.max, 1.0], [tiny], [-tiny, tiny], [info.tiny], [127.0, 0.5, 1.5, 2.5, -0.5],
            [127.5, 1.0], [128.0, 64.0], [126.5], [254.0, 1.0, 3.0], [-0.0, 0.0], [1.0] * 32]
    x = torch.zeros((len(rows), 32), dtype=dtype)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r, dtype=torch.float64).to(dtype)
    kept, _ = _copy(dev, x)
    assert torch.equal(kept, ref.eight_bits(x))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(dev, bad):
    x, w, b, g = _inputs(70, 96, 32, torch.float16)
    x[3, 40] = bad
    kept, _ = _copy(dev, x)
    assert kept[3, 32:64].isnan().all() and int(kept.isnan().sum()) == 32
    found = _run(dev, x, w, b, g, "gelu")
    assert not found["out"][[0, 4]].isnan().any() and not found["out"][3].isfinite().any()
    dx = found["grad_x"].isnan()
    assert dx[3, 32:64].all() and int(dx.sum()) == 32
    dw = found["grad_weight"].isnan()
    assert dw[:, 32:64].all() and int(dw.sum()) == 32 * 32
    assert not found["grad_bias"].isnan().any()


@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_large_and_small_inputs(dev, activation):
    """The GELU's both tails, and gradients near the end of fp16's range."""
    x, w, b, g = _inputs(200, 64, 32, torch.float16)
    x = torch.cat([x * 20, x * 1e-4, x * 3])[:, :]
    g = torch.cat([g, g * 100, g * 1e-3])
    ref.check(_run(dev, x, w, b, g, activation), ref.linear_8bit(x, w, b, g, activation))


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_shapes_strides_and_no_bias(dev, dtype):
    x, w, _, g = _inputs(2 * 3 * 4 * 5, 48, 32, dtype)
    expected = ref.linear_8bit(x, w, None, g, "gelu")
    a = x.view(2, 3, 4, 5, 48).to(dev).permute(3, 2, 1, 0, 4).contiguous().permute(3, 2, 1, 0, 4).requires_grad_()
    ww = torch.cat([w.new_zeros(1), w.flatten()]).to(dev)[1:].view(32, 48).requires_grad_()
    y = training.linear_8bit(a, ww, None, "gelu")
    assert y.shape == (2, 3, 4, 5, 32)
    go = g.view(2, 3, 4, 5, 32).to(dev).transpose(0, 4).contiguous().transpose(0, 4)
    dx, dw = torch.autograd.grad(y, (a, ww), go)
    ref.check({"out": y.reshape(-1, 32), "grad_x": dx.reshape(-1, 48), "grad_weight": dw}, expected)
    wt = w.t().contiguous().to(dev).t().requires_grad_()
    y = training.linear_8bit(x.to(dev), wt, None, "gelu")
    (dw,) = torch.autograd.grad(y, wt, g.to(dev))
    ref.check({"out": y, "grad_weight": dw}, expected)


def test_each_gradient_alone(dev):
    x, w, b, g = _inputs(100, 64, 48, torch.float16)
    both = _run(dev, x, w, b, g, "gelu")
    for name in ("x", "weight", "bias"):
        t = {"x": x.to(dev), "weight": w.to(dev), "bias": b.to(dev)}
        t[name] = t[name].requires_grad_()
        (d,) = torch.autograd.grad(training.linear_8bit(t["x"], t["weight"], t["bias"], "gelu"), t[name], g.to(dev))
        assert torch.equal(d, both["grad_" + name])
    with torch.no_grad():
        assert torch.equal(training.linear_8bit(x.to(dev), w.to(dev), b.to(dev), "gelu"), both["out"])


def test_what_is_kept(dev):
    """33/32 bytes a value and the weight: neither x nor act(x)."""
    x, w, b, _ = (t.to(dev) for t in _inputs(1000, 64, 48, torch.float16))
    w.requires_grad_()
    before = torch.cuda.memory_allocated()
    y = training.linear_8bit(x, w, b, "gelu")
    assert torch.cuda.memory_allocated() - before - 1000 * 48 * 2 <= 1000 * 66 + 4 * 512  # the allocator's granules
    held = torch.cuda.memory_allocated()
    del x
    assert held - torch.cuda.memory_allocated() >= 1000 * 64 * 2
    assert y.requires_grad


def test_autocast(dev):
    x, w, b, g = _inputs(100, 64, 48, torch.bfloat16)
    expected = ref.linear_8bit(x, w, b, g, "gelu")
    leaves = [t.float().to(dev).requires_grad_() for t in (x, w, b)]
    with torch.autocast("cuda", torch.bfloat16):
        y = training.linear_8bit(*leaves, activation="gelu")
    assert y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, leaves, g.to(dev))
    assert all(d.dtype == torch.float32 for d in grads)
    ref.check({"out": y, **dict(zip(("grad_x", "grad_weight", "grad_bias"), grads))}, expected)


def test_no_rows(dev):
    x = torch.zeros((0, 32), dtype=torch.float16, device=dev, requires_grad=True)
    w = torch.ones((16, 32), dtype=torch.float16, device=dev, requires_grad=True)
    b = torch.ones(16, dtype=torch.float16, device=dev, requires_grad=True)
    y = training.linear_8bit(x, w, b)
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == (0, 32) and not dw.any() and not db.any()


def test_repeats_captured_and_on_another_stream(dev):
    sets = [_inputs(3000, 96, 48, torch.float16, seed=10 * s) for s in range(4)]
    ins = [t.to(dev) for t in sets[0]]
    for t in ins[:3]:
        t.requires_grad_()

    def run():
        y = training.linear_8bit(*ins[:3], "gelu")
        return (y, *torch.autograd.grad(y, ins[:3], ins[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    del first  # no eager graph of the leaves lives during the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for s in (1, 2, 3):
        with torch.no_grad():
            for t, v in zip(ins, sets[s]):
                t.copy_(v)
        graph.replay()
        expected = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expected))


def test_compiled(dev):
    x, w, b, g = (t.to(dev) for t in _inputs(50, 48, 32, torch.float16))
    for t in (x, w, b):
        t.requires_grad_()
    y = torch.compile(lambda *a: training.linear_8bit(*a, "gelu"), backend="aot_eager", fullgraph=True)(x, w, b)
    found = torch.autograd.grad(y, (x, w, b), g)
    e = training.linear_8bit(x, w, b, "gelu")
    expected = torch.autograd.grad(e, (x, w, b), g)
    assert torch.equal(y, e) and all(torch.equal(p, q) for p, q in zip(found, expected))


def test_refusals(dev):
    x, w, b, _ = (t.to(dev) for t in _inputs(4, 32, 16, torch.float16))

    def refused(match, *args):
        with pytest.raises((RuntimeError, ValueError), match=match):
            training.linear_8bit(*args)

    refused("activation must be one of", x, w, b, "relu")
    refused("weight must have shape", x, w[:, :16], b)
    refused("x's type", x, w.float(), b)
    refused("bias must have shape", x, w, b[:8])
    refused("bias must have shape", x, w, b.float())
    refused("float16 or bfloat16", x.float(), w.float(), b.float())
    refused("multiples of 16", x[:, :24].contiguous(), w[:, :24].contiguous(), b)
    refused("multiples of 16", x, w[:8], b[:8])
    refused("must be on", x, w.cpu(), b)
    w.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(training.linear_8bit(x, w, b).sum(), w, create_graph=True)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("rows,K", [(5, 16), (70, 48), (300, 80), (70000, 112)])
def test_an_infinite_weight_stays_infinite(dev, dtype, rows, K):
    """Short last steps read weights of other columns beside zeros of x."""
    x = seeded((rows, K), dtype, 1).abs() + 0.5
    for k in (0, K // 2, K - 1):
        w = torch.zeros(32, K, dtype=dtype)
        w[3, k], w[20, k] = math.inf, -math.inf
        y = training.linear_8bit(x.to(dev), w.to(dev)).cpu()
        assert (y[:, 3] == math.inf).all() and (y[:, 20] == -math.inf).all()
        y[:, 3] = y[:, 20] = 0
        assert (y == 0).all()


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_the_largest_numbers_stay_finite(dev, dtype, activation):
    """The copy of the type's largest numbers is rounded up to what the type does
    not hold (64 steps of the last exponent); as an operand it is the largest."""
    top = torch.finfo(dtype).max
    x = torch.zeros(8, 64, dtype=dtype)
    x[0, 0], x[1, 1], x[2, 40] = top, -top, top / 2
    x[3, :4] = torch.tensor([top / 4, -top / 3, top / 5, 1.0], dtype=torch.float64).to(dtype)
    x[4, 32:36] = torch.tensor([top, -top * 0.99, top * 0.3, -top], dtype=torch.float64).to(dtype)
    kept = ref.eight_bits(x).clamp(-top, top)
    w = torch.zeros(16, 64, dtype=dtype, device=dev)
    _, codes, exps = torch.ops.crumpet_ops.linear_8bit_forward(x.to(dev), w, None, int(activation == "gelu"))
    # a gradient of one row at a time hands the copy back, times 2^-4; of its
    # GELU the far sides, which are the number itself and 0
    for r in range(5):
        g = torch.zeros(8, 16, dtype=dtype, device=dev)
        g[r, 2] = 2.0 ** -4
        _, dw, _ = torch.ops.crumpet_ops.linear_8bit_backward(g, codes, exps, w, int(activation == "gelu"), False, True,
                                                              False)
        want = kept[r].clamp(min=0) if activation == "gelu" else kept[r]
        want = torch.where(kept[r].abs() > 100, want, dw[2].cpu().double() * 16) / 16
        assert torch.equal(dw[2].cpu().double(), want.to(dtype).double())


@pytest.mark.parametrize("rows", [64, 700])
@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2), (1, 2)], ids=str)
def test_some_of_the_gradients(dev, rows, wanted):
    """One chunk of rows, whose sums are the results, and several."""
    leaves = [t.to(dev) for t in _inputs(rows, 48, 80, torch.float16)]
    g = leaves.pop()

    def run(which):
        x, w, b = (t.clone().requires_grad_(i in which) for i, t in enumerate(leaves))
        y = training.linear_8bit(x, w, b, activation="gelu")
        return torch.autograd.grad(y, [t for i, t in enumerate((x, w, b)) if i in which], g)

    whole = run((0, 1, 2))
    for i, d in zip(wanted, run(wanted), strict=True):
        assert torch.equal(d, whole[i])
