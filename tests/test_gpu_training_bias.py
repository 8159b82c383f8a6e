"""training.relative_position_bias and the table's gradient against 64 bits."""

from __future__ import annotations

import pytest
import torch

import training_reference as ref
from crumpet_amd import training
from helpers import seeded

pytestmark = pytest.mark.gpu

ALL = (torch.float32, torch.float16, torch.bfloat16)


def _window_index(ws):
    from oracle import oracle

    index = torch.from_numpy(oracle.relative_position_index(ws))
    return index, (2 * ws[0] - 1) * (2 * ws[1] - 1) * (2 * ws[2] - 1)


def _run(dev, table, index, buckets, grad):
    t = table.to(dev).requires_grad_()
    plan = training.BiasBuckets(index.to(dev), buckets)
    out = training.relative_position_bias(t, plan)
    (dtable,) = torch.autograd.grad(out, t, grad.to(dev))
    return {"bias": out, "grad_table": dtable}


def _check(dev, index, buckets, heads, dtype, seed=0):
    table, grad = seeded((buckets, heads), dtype, seed), seeded((heads, *index.shape), dtype, seed + 1)
    ref.check(_run(dev, table, index, buckets, grad), ref.position_bias(table, index, grad))


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("ws,heads", [((7, 7, 7), 3), ((6, 6, 6), 24), ((2, 3, 5), 1), ((1, 1, 1), 2)], ids=str)
def test_windows(dev, dtype, ws, heads):
    index, buckets = _window_index(ws)
    _check(dev, index, buckets, heads, dtype)
    # part of a window, as smaller volumes use, in place
    n = max(1, index.shape[0] * 2 // 3)
    _check(dev, index[:n, :n], buckets, heads, dtype)


# few buckets, so that each has more pairs than a segment, and more than 64 segments
@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("nq,nk,buckets,heads", [(1, 1, 1, 1), (100, 333, 3, 5), (700, 901, 4, 2), (513, 257, 32, 7)])
def test_long_buckets(dev, dtype, nq, nk, buckets, heads):
    g = torch.Generator().manual_seed(nq)
    index = (torch.rand((nq, nk), generator=g) ** 3 * buckets).long()
    _check(dev, index, buckets, heads, dtype)


@pytest.mark.parametrize("pairs", [2047, 2048, 2049, 4096])
def test_segment_limits(dev, pairs):
    """All pairs in one bucket of five, the others empty."""
    index = torch.full((1, pairs), 3)
    _check(dev, index, 5, 2, torch.float32)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8])
def test_index_types_are_copied(dev, dtype):
    index, buckets = _window_index((2, 2, 3))
    table, grad = seeded((buckets, 2), torch.float32, 0), seeded((2, 12, 12), torch.float32, 1)
    mine = index.to(dev, dtype)
    plan = training.BiasBuckets(mine, buckets)
    mine.zero_()
    t = table.to(dev).requires_grad_()
    out = training.relative_position_bias(t, plan)
    (d,) = torch.autograd.grad(out, t, grad.to(dev))
    ref.check({"bias": out, "grad_table": d}, ref.position_bias(table, index, grad))


def test_strides_of_table_and_gradient(dev):
    index, buckets = _window_index((3, 3, 3))
    table, grad = seeded((buckets, 4), torch.float32, 0), seeded((4, 27, 27), torch.float32, 1)
    t = table.t().contiguous().to(dev).t().requires_grad_()
    out = training.relative_position_bias(t, training.BiasBuckets(index.to(dev), buckets))
    (d,) = torch.autograd.grad(out, t, grad.transpose(0, 2).contiguous().to(dev).transpose(0, 2))
    ref.check({"bias": out, "grad_table": d}, ref.position_bias(table, index, grad))
    (d,) = torch.autograd.grad(training.relative_position_bias(t, training.BiasBuckets(index.to(dev), buckets)).sum(), t)
    ref.check({"grad_table": d}, ref.position_bias(table, index, torch.ones_like(grad)))


def test_empty_index(dev):
    t = torch.ones((4, 2), device=dev, requires_grad=True)
    out = training.relative_position_bias(t, training.BiasBuckets(torch.zeros((0, 3), dtype=torch.int64, device=dev), 4))
    assert out.shape == (2, 0, 3)
    (d,) = torch.autograd.grad(out.sum(), t)
    assert torch.equal(d, torch.zeros_like(t))


def test_repeats_captured_and_on_another_stream(dev):
    index, buckets = _window_index((5, 5, 5))
    for few in (False, True):
        i = index % 7 if few else index
        n = 7 if few else buckets
        plan = training.BiasBuckets(i.to(dev), n)
        t = seeded((n, 6), torch.float32, 0).to(dev).requires_grad_()
        g = seeded((6, 125, 125), torch.float32, 1).to(dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(training.relative_position_bias(t, plan), t, g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = training.relative_position_bias(t, plan)
            (d,) = torch.autograd.grad(out, t, g)
        for seed in range(3):
            with torch.no_grad():
                t.copy_(seeded((n, 6), torch.float32, 10 + seed))
                g.copy_(seeded((6, 125, 125), torch.float32, 20 + seed))
            graph.replay()
            e = training.relative_position_bias(t, plan)
            (de,) = torch.autograd.grad(e, t, g)
            torch.cuda.synchronize()
            assert torch.equal(out, e) and torch.equal(d, de)


def test_compiled(dev):
    index, buckets = _window_index((3, 3, 3))
    plan = training.BiasBuckets(index.to(dev), buckets)
    t = seeded((buckets, 2), torch.float32, 0).to(dev).requires_grad_()
    g = seeded((2, 27, 27), torch.float32, 1).to(dev)
    out = torch.compile(lambda t: training.relative_position_bias(t, plan), backend="aot_eager", fullgraph=True)(t)
    (d,) = torch.autograd.grad(out, t, g)
    e = training.relative_position_bias(t, plan)
    (de,) = torch.autograd.grad(e, t, g)
    assert torch.equal(out, e) and torch.equal(d, de)


def test_refusals(dev):
    index = torch.tensor([[0, 1], [2, 3]], device=dev)
    plan = training.BiasBuckets(index, 4)
    for bad in (torch.tensor([[0, 4]], device=dev), torch.tensor([[-1, 0]], device=dev)):
        with pytest.raises(ValueError, match="0 .. 3"):
            training.BiasBuckets(bad, 4)
    with pytest.raises(ValueError, match="queries, keys"):
        training.BiasBuckets(index[0], 4)
    with pytest.raises(ValueError, match="integers"):
        training.BiasBuckets(index.float(), 4)
    with pytest.raises(ValueError, match=r"\[4, heads\]"):
        training.relative_position_bias(torch.zeros((5, 2), device=dev), plan)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        training.relative_position_bias(torch.zeros((4, 2), device=dev, dtype=torch.float64), plan)
    with pytest.raises(TypeError, match="BiasBuckets"):
        training.relative_position_bias(torch.zeros((4, 2), device=dev), index)
    t = torch.zeros((4, 2), device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(training.relative_position_bias(t, plan).sum(), t, create_graph=True)


def test_the_ops_own_bounds(dev):
    """The dispatcher op takes any index; one outside the table reads as 0,
    and sorted pairs outside the gradient add nothing."""
    table = torch.ones((3, 2), device=dev)
    index = torch.tensor([[0, 7], [-5, 2]], dtype=torch.int32, device=dev)
    empty = torch.zeros((0, 2), dtype=torch.int32, device=dev)
    out = torch.ops.crumpet_ops.bucket_bias(table, index, index.flatten(), empty, None)
    assert out[0].tolist() == [[1.0, 0.0], [0.0, 1.0]]
    grad = torch.ones((2, 2, 2), device=dev)
    order = torch.tensor([0, 9, -1, 3], dtype=torch.int32, device=dev)
    segments = torch.tensor([[-3, 2], [2, 9], [4, 4]], dtype=torch.int32, device=dev)
    d = torch.ops.crumpet_ops.bucket_bias_backward(grad, order, segments, None, 3)
    assert d.tolist() == [[1.0, 1.0], [1.0, 1.0], [0.0, 0.0]]
