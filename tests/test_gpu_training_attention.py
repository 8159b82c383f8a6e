"""training.window_attention and its gradients against 64 bits, within bounds
derived from the operator's roundings (training_reference)."""

from __future__ import annotations

import math

import pytest
import torch

import training_reference as ref
from crumpet_amd import training
from helpers import seeded

pytestmark = pytest.mark.gpu

HALF = (torch.float16, torch.bfloat16)
ALL = (torch.float32, *HALF)


def _inputs(B, N, H, D, dtype, seed=0, bias_dtype=torch.float32):
    return (seeded((B, N, 3 * H * D), dtype, seed), seeded((H, N, N), bias_dtype, seed + 1),
            seeded((B, N, H * D), dtype, seed + 2))


def _run(dev, qkv, bias, heads, grad, **kw):
    x, b = qkv.to(dev).requires_grad_(), bias.to(dev).requires_grad_()
    kw = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in kw.items()}
    out = training.window_attention(x, b, heads, **kw)
    dqkv, dbias = torch.autograd.grad(out, (x, b), grad.to(dev))
    return {"out": out, "grad_qkv": dqkv, "grad_bias": dbias}


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("N", [1, 2, 16, 17, 63, 65, 130])
def test_sizes(dev, dtype, D, N):
    qkv, bias, g = _inputs(3, N, 2, D, dtype, seed=N)
    ref.check(_run(dev, qkv, bias, 2, g), ref.window_attention(qkv, bias, 2, g))


# a window's tiles of 16 keys and the limits between kernel forms
@pytest.mark.parametrize("dtype,D", [(torch.float16, 16), (torch.bfloat16, 32), (torch.bfloat16, 64)], ids=str)
@pytest.mark.parametrize("N", [64, 112, 113, 216, 224, 225, 343, 352, 353, 512, 513, 600])
def test_window_sizes(dev, dtype, D, N):
    qkv, bias, g = _inputs(2, N, 3, D, dtype, seed=N)
    ref.check(_run(dev, qkv, bias, 3, g), ref.window_attention(qkv, bias, 3, g))


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_many_windows_in_uneven_groups(dev, dtype):
    qkv, bias, g = _inputs(301, 27, 3, 16, dtype)
    ref.check(_run(dev, qkv, bias, 3, g), ref.window_attention(qkv, bias, 3, g))


REGIONS = [((6, 6, 6), (3, 3, 3), (1, 1, 1)), ((4, 8, 6), (4, 4, 3), (0, 2, 1)), ((8, 8, 8), (8, 8, 8), (3, 0, 4)),
           ((14, 7, 7), (7, 7, 7), (3, 3, 3)), ((10, 5, 12), (5, 5, 6), (0, 0, 0)), ((18, 6, 12), (6, 6, 6), (3, 3, 3))]


@pytest.mark.parametrize("dtype,D", [(torch.float16, 16), (torch.bfloat16, 32), (torch.float32, 16),
                                     (torch.float16, 64)], ids=str)
@pytest.mark.parametrize("volume,ws,shift", REGIONS, ids=str)
def test_shifted_windows(dev, dtype, D, volume, ws, shift):
    nW = math.prod(v // w for v, w in zip(volume, ws))
    N = math.prod(ws)
    qkv, bias, g = _inputs(2 * nW, N, 2, D, dtype, seed=N)
    found = _run(dev, qkv, bias, 2, g, volume=volume, window_size=ws, shift_size=shift)
    mask = ref.shift_mask(volume, ws, shift)
    ref.check(found, ref.window_attention(qkv, bias, 2, g, mask))


def _mask(M, N, kind, dtype):
    g = torch.Generator().manual_seed(N + M)
    off = torch.rand((M, N, N), generator=g) < 0.3
    off[0, N // 2] = True  # a query without keys
    off[-1, 0] = True
    low = {"inf": -math.inf, "lowest": torch.finfo(dtype).min, "hundred": -100.0}[kind]
    m = (0.5 * torch.randn((M, N, N), generator=g)).to(dtype)
    return m.masked_fill(off, low)


@pytest.mark.parametrize("dtype,D,mask_dtype", [(torch.float16, 16, torch.float16), (torch.bfloat16, 32, torch.bfloat16),
                                                (torch.bfloat16, 16, torch.float32), (torch.float32, 16, torch.float32),
                                                (torch.float16, 64, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("kind", ["inf", "lowest", "hundred"])
@pytest.mark.parametrize("M,N", [(1, 17), (2, 64), (4, 113), (2, 343)])
def test_mask_tensors(dev, dtype, D, mask_dtype, kind, M, N):
    mask = _mask(M, N, kind, mask_dtype)
    qkv, bias, g = _inputs(4, N, 2, D, dtype, seed=N)
    found = _run(dev, qkv, bias, 2, g, mask=mask)
    ref.check(found, ref.window_attention(qkv, bias, 2, g, mask))
    if kind == "inf":
        rows = found["out"].view(4, N, -1)[0, N // 2]
        assert torch.equal(rows, torch.zeros_like(rows))
        dq = found["grad_qkv"].view(4, N, 3, -1)[0, N // 2, 0]
        assert torch.equal(dq, torch.zeros_like(dq))
        assert torch.isfinite(found["grad_bias"]).all()


@pytest.mark.parametrize("dtype,D,mask_dtype", [(torch.float16, 16, torch.float16), (torch.bfloat16, 32, torch.bfloat16),
                                                (torch.float16, 32, torch.float32)], ids=str)
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 15, 16, 18, 47, 48, 65, 127, 226, 349, 350, 352, 511, 512])
def test_mask_rows_read_four_at_a_time(dev, dtype, D, mask_dtype, N):
    """Rows of odd and even lengths, ends inside and at the end of a group of
    four, the last row's at the end of the mask's and the bias' memory."""
    mask = _mask(2, N, "hundred", mask_dtype)
    qkv, bias, g = _inputs(4, N, 2, D, dtype, seed=N)
    ref.check(_run(dev, qkv, bias, 2, g, mask=mask), ref.window_attention(qkv, bias, 2, g, mask))


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_a_nan_stays_in_its_window_and_head(dev, dtype):
    qkv, bias, g = _inputs(3, 40, 2, 16, dtype)
    qkv[1, 7, 16 + 3] = math.nan  # head 1's q
    found = _run(dev, qkv, bias, 2, g)
    out = found["out"].view(3, 40, 2, 16)
    assert out[1, 7, 1].isnan().all() and int(out.isnan().sum()) == 16
    d = found["grad_qkv"].view(3, 40, 3, 2, 16)
    assert not d[[0, 2]].isnan().any() and not d[1, :, :, 0].isnan().any()
    assert not found["grad_bias"][0].isnan().any()


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_sharp_and_flat_scores(dev, dtype):
    """q = k = 4 v: the diagonal dominates by tens of octaves; and all equal."""
    x = seeded((4, 216, 2, 16), dtype, 5)
    qkv = torch.stack([4 * x, 4 * x, x], 2).reshape(4, 216, -1)
    _, bias, g = _inputs(4, 216, 2, 16, dtype)
    ref.check(_run(dev, qkv, bias, 2, g), ref.window_attention(qkv, bias, 2, g))
    flat = torch.zeros_like(qkv)
    ref.check(_run(dev, flat, 0 * bias, 2, g), ref.window_attention(flat, 0 * bias, 2, g))


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("N,D", [(80, 16), (80, 32), (80, 64), (600, 16)])
def test_the_kept_rest_belongs_to_the_output(dev, dtype, N, D):
    """With equal scores every weight is exactly 1 and out + rest the mean of v:
    the sum is off by at most (N + 1) 2^-23 of the mean magnitude, its product
    with 1/N by 2^-22 of itself (reciprocal and product), the rest by half a
    step of fp16 (or a step of fp32's, which bf16 keeps as bits).  The sums of many windows hold means near a tie of the
    output's rounding, where a rest that belongs to the other neighbour is a
    whole step off."""
    qkv = seeded((90, N, 3 * D), dtype, 7)
    qkv[..., :2 * D] = 0
    bias = torch.zeros(1, N, N, device=dev)
    out, rest, _, _ = torch.ops.crumpet_ops.window_attention_forward(qkv.to(dev), bias, 1, None, [], D ** -0.5)
    v = qkv[..., 2 * D:].double()
    mean, size = v.mean(1, keepdim=True), v.abs().mean(1, keepdim=True)
    out, rest = out.cpu(), rest.cpu()
    if dtype == torch.bfloat16:
        bits = (out.view(torch.int16).int() << 16) + rest.view(torch.int16).int()
        both, kept = bits.view(torch.float32).double(), 2.0 ** -23
    else:
        both, kept = out.double() + rest.double(), 2.0 ** -22
    bound = (N + 1) * 2.0 ** -23 * size + (2.0 ** -22 + kept) * mean.abs() + 2.0 ** -25
    assert ((both - mean).abs() <= bound).all()


@pytest.mark.parametrize("scale", [0.0, -0.5, 2.0 ** -30, 3.0])
def test_scales(dev, scale):
    qkv, bias, g = _inputs(2, 70, 2, 16, torch.bfloat16)
    ref.check(_run(dev, qkv, bias, 2, g, scale=scale), ref.window_attention(qkv, bias, 2, g, scale=scale))


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("how", ["token_slice", "window_slice", "channel_major", "offset", "overlap"])
def test_strides(dev, dtype, how):
    qkv, bias, g = _inputs(4, 50, 2, 16, dtype)
    x = qkv.to(dev)
    if how == "token_slice":
        big = torch.empty((4, 50, 200), dtype=dtype, device=dev)
        big[..., 8:104] = x
        x = big[..., 8:104]
    elif how == "window_slice":
        big = torch.empty((8, 60, 96), dtype=dtype, device=dev)
        big[::2, 5:55] = x
        x = big[::2, 5:55]
    elif how == "channel_major":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    elif how == "offset":  # rows that start at no multiple of 16 bytes
        big = torch.empty(x.numel() + 3, dtype=dtype, device=dev)
        big[3:] = x.flatten()
        x = big[3:].view_as(x)
    else:  # every window the same memory
        x, qkv = x[:1].expand(4, -1, -1), qkv[:1].expand(4, -1, -1)
    x = x.detach().requires_grad_()
    b = bias.to(dev).requires_grad_()
    out = training.window_attention(x, b, 2)
    # the gradient arrives expanded or transposed, as sums and permutes make them
    go = g.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    dqkv, dbias = torch.autograd.grad(out, (x, b), go)
    ref.check({"out": out, "grad_qkv": dqkv, "grad_bias": dbias}, ref.window_attention(qkv.contiguous(), bias, 2, g))


@pytest.mark.parametrize("bias_dtype", ALL, ids=str)
def test_bias_types_and_strides(dev, bias_dtype):
    qkv, bias, g = _inputs(5, 33, 3, 16, torch.float16, bias_dtype=bias_dtype)
    b = bias.permute(2, 1, 0).contiguous().to(dev).permute(2, 1, 0).requires_grad_()
    x = qkv.to(dev).requires_grad_()
    out = training.window_attention(x, b, 3)
    dqkv, dbias = torch.autograd.grad(out, (x, b), g.to(dev))
    assert dbias.dtype == bias_dtype
    ref.check({"out": out, "grad_qkv": dqkv, "grad_bias": dbias}, ref.window_attention(qkv, bias, 3, g))


@pytest.mark.parametrize("dtype,D", [(torch.float16, 16), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.float32, 16)],
                         ids=str)
@pytest.mark.parametrize("N,shifted", [(40, False), (27, True), (343, True)])
def test_a_bias_of_the_lowest_value(dev, dtype, D, N, shifted):
    """fp32's lowest value absorbs a score: a query with nothing else weighs its
    keys equally, one with a few such keys leaves them out."""
    qkv, bias, g = _inputs(8, N, 2, D, dtype, seed=N)
    low = torch.finfo(torch.float32).min
    bias[0, 1], bias[1, N - 1] = low, low
    bias[1, 3, ::2] = low
    where = {}
    mask = None
    if shifted:
        w = round(N ** (1 / 3))
        where = dict(volume=(2 * w,) * 3, window_size=(w,) * 3, shift_size=(w // 2,) * 3)
        mask = ref.shift_mask(*where.values())
    found = _run(dev, qkv, bias, 2, g, **where)
    ref.check(found, ref.window_attention(qkv, bias, 2, g, torch.zeros(1, N, N) if mask is None else mask))


@pytest.mark.parametrize("N", [33, 343])
def test_mask_views(dev, N):
    qkv, bias, g = _inputs(4, N, 1, 32, torch.bfloat16)
    mask = _mask(2, N, "hundred", torch.bfloat16)
    expected = ref.window_attention(qkv, bias, 1, g, mask)
    big = torch.zeros((4, N, N), dtype=torch.bfloat16, device=dev)
    big[::2] = mask.to(dev)
    ref.check(_run(dev, qkv, bias, 1, g, mask=big[::2]), expected)
    turned = mask.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    ref.check(_run(dev, qkv, bias, 1, g, mask=turned), expected)
    one = mask[:1].to(dev).expand(4, -1, -1)
    ref.check(_run(dev, qkv, bias, 1, g, mask=one), ref.window_attention(qkv, bias, 1, g, mask[:1]))


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("N", [40, 343])
def test_without_gradients(dev, dtype, N):
    qkv, bias, g = _inputs(3, N, 2, 16, dtype)
    out = training.window_attention(qkv.to(dev), bias.to(dev), 2)
    assert not out.requires_grad
    ref.check({"out": out}, ref.window_attention(qkv, bias, 2, g, keep=False))


def test_one_gradient_of_two(dev):
    qkv, bias, g = (t.to(dev) for t in _inputs(3, 40, 2, 16, torch.float16))
    both = _run(dev, qkv, bias, 2, g)
    x = qkv.clone().requires_grad_()
    (dqkv,) = torch.autograd.grad(training.window_attention(x, bias, 2), x, g)
    assert torch.equal(dqkv, both["grad_qkv"])
    b = bias.clone().requires_grad_()
    (dbias,) = torch.autograd.grad(training.window_attention(qkv, b, 2), b, g)
    assert torch.equal(dbias, both["grad_bias"])


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_results_repeat_bit_for_bit(dev, dtype):
    qkv, bias, g = _inputs(150, 64, 3, 16, dtype)
    first = _run(dev, qkv, bias, 3, g)
    for _ in range(3):
        again = _run(dev, qkv, bias, 3, g)
        assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("shape", [(0, 16, 96), (3, 0, 96)])
def test_nothing_to_attend(dev, shape):
    x = torch.zeros(shape, dtype=torch.float16, device=dev, requires_grad=True)
    b = torch.ones((2, shape[1], shape[1]), device=dev, requires_grad=True)
    out = training.window_attention(x, b, 2)
    assert out.shape == (shape[0], shape[1], 32)
    dqkv, dbias = torch.autograd.grad(out.sum(), (x, b))
    assert dqkv.shape == shape and torch.equal(dbias, torch.zeros_like(b))


@pytest.mark.parametrize("dtype,D", [(torch.float16, 16), (torch.float32, 32)], ids=str)
def test_on_another_stream(dev, dtype, D):
    qkv, bias, g = _inputs(40, 343, 2, D, dtype)
    expected = _run(dev, qkv, bias, 2, g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        found = _run(dev, qkv, bias, 2, g)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(found[k], expected[k]) for k in found)


@pytest.mark.parametrize("dtype,N", [(torch.float16, 343), (torch.bfloat16, 64), (torch.float32, 40)], ids=str)
def test_captured_with_its_backward_pass(dev, dtype, N):
    """Two graphs of the same sizes, replayed in turn with eager work between."""
    sets = [_inputs(30, N, 2, 16, dtype, seed=s) for s in (0, 10, 20, 30)]
    graphs = []
    for first in sets[:2]:
        x, b, g = (t.to(dev) for t in first)
        x.requires_grad_()
        b.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(training.window_attention(x, b, 2), (x, b), g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = training.window_attention(x, b, 2)
            grads = torch.autograd.grad(out, (x, b), g)
        graphs.append((graph, (x, b, g), (out, *grads)))
    for k in range(4):
        for i, (graph, ins, outs) in enumerate(graphs):
            new = sets[(k + i) % 4]
            with torch.no_grad():
                for t, v in zip(ins, new):
                    t.copy_(v)
            graph.replay()
            expected = _run(dev, new[0], new[1], 2, new[2])
            torch.cuda.synchronize()
            for got, name in zip(outs, ("out", "grad_qkv", "grad_bias")):
                assert torch.equal(got, expected[name]), (k, i, name)


def test_compiled(dev):
    qkv, bias, g = (t.to(dev) for t in _inputs(8, 27, 2, 16, torch.float16))
    eager = _run(dev, qkv, bias, 2, g, volume=(6, 6, 6), window_size=(3, 3, 3), shift_size=(1, 1, 1))
    x, b = qkv.clone().requires_grad_(), bias.clone().requires_grad_()

    def f(x, b):
        return training.window_attention(x, b, 2, volume=(6, 6, 6), window_size=(3, 3, 3), shift_size=(1, 1, 1))

    out = torch.compile(f, backend="aot_eager", fullgraph=True)(x, b)
    dqkv, dbias = torch.autograd.grad(out, (x, b), g)
    assert torch.equal(out, eager["out"]) and torch.equal(dqkv, eager["grad_qkv"]) and torch.equal(dbias, eager["grad_bias"])


def test_refusals(dev):
    qkv, bias, _ = (t.to(dev) for t in _inputs(2, 8, 2, 16, torch.float16))

    def refused(match, *args, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            training.window_attention(*args, **kw)

    refused("last axis", qkv, bias, 5)
    refused("bias must have shape", qkv, bias[:1], 2)
    refused("head_dim 8", qkv, bias.repeat(2, 1, 1), 4)
    refused("float32, float16 or bfloat16", qkv.double(), bias, 2)
    refused("mask must have shape", qkv, bias, 2, mask=torch.zeros(2, 8, 7, device=dev))
    refused("multiple of the masks", qkv, bias, 2, mask=torch.zeros(3, 8, 8, device=dev))
    refused("mask holds no window", qkv, bias, 2, mask=torch.zeros(0, 8, 8, device=dev))
    refused("no gradient", qkv, bias, 2, mask=torch.zeros(2, 8, 8, device=dev, requires_grad=True))
    refused("belong together", qkv, bias, 2, volume=(2, 2, 2))
    refused("exclude each other", qkv, bias, 2, mask=torch.zeros(2, 8, 8, device=dev), volume=(2, 2, 2),
            window_size=(2, 2, 2), shift_size=(1, 1, 1))
    refused("window volume", qkv, bias, 2, volume=(3, 3, 3), window_size=(3, 3, 3), shift_size=(1, 1, 1))
    refused("multiple of the volume", qkv, bias, 2, volume=(6, 2, 2), window_size=(2, 2, 2), shift_size=(1, 1, 1))
    refused("must be on", qkv, bias.cpu(), 2)
    x = qkv.clone().requires_grad_()
    out = training.window_attention(x, bias, 2)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out.sum(), x, create_graph=True)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)
