"""The training operators on tensors of more than 2^32 elements: the last rows against a call on them alone."""

from __future__ import annotations

import pytest
import torch

from crumpet_amd import training

pytestmark = pytest.mark.gpu

MORE = 1 << 32


@pytest.fixture(autouse=True)
def _memory(dev):
    if torch.cuda.get_device_properties(dev).total_memory < 200 << 30:
        pytest.skip("needs 200 GB of device memory")
    yield
    torch.cuda.empty_cache()


def _tail(dev, shape, dtype, rows, seed):
    """Zeros but for the last rows, and those rows."""
    g = torch.Generator(device=dev).manual_seed(seed)
    last = torch.randn((rows, *shape[1:]), generator=g, device=dev).to(dtype)
    whole = torch.zeros(shape, dtype=dtype, device=dev)
    whole[-rows:] = last
    return whole, last


def _same(found, expected):
    for f, e in zip(found, expected, strict=True):
        assert torch.equal(f[-e.shape[0]:] if f.shape != e.shape else f, e)


@pytest.mark.parametrize("dtype,D", [(torch.float16, 16), (torch.bfloat16, 64)], ids=str)
def test_attention(dev, dtype, D):
    N, H = 64, 2
    B = MORE // (N * 3 * H * D) + 5
    qkv, last = _tail(dev, (B, N, 3 * H * D), dtype, 5, 1)
    grad, last_grad = _tail(dev, (B, N, H * D), dtype, 5, 2)
    bias = torch.randn(H, N, N, generator=torch.Generator().manual_seed(3)).to(dev)

    def run(x, g):
        x, b = x.requires_grad_(), bias.clone().requires_grad_()
        out = training.window_attention(x, b, H)
        dx, db = torch.autograd.grad(out, (x, b), g)
        return out.detach(), dx, db

    *found, found_bias = run(qkv, grad)
    *expected, expected_bias = run(last, last_grad)
    _same(found, expected)
    # the other windows add zeros; the five are summed in one range or two
    torch.testing.assert_close(found_bias, expected_bias, rtol=0, atol=5 * 2.0 ** -23 * float(expected_bias.abs().max()))


def test_norm(dev):
    C, dtype = 512, torch.float16
    T = MORE // C + 5
    (x, xl), (y, yl), (gs, gsl), (gh, ghl) = (_tail(dev, (T, C), dtype, 5, s) for s in range(4))
    found = training.residual_norm(x.requires_grad_(), y.requires_grad_(), norm="rms")
    found = [*(t.detach() for t in found), *torch.autograd.grad(found, (x, y), (gs, gh))]
    expected = training.residual_norm(xl.requires_grad_(), yl.requires_grad_(), norm="rms")
    expected = [*(t.detach() for t in expected), *torch.autograd.grad(expected, (xl, yl), (gsl, ghl))]
    _same(found, expected)


def test_linear(dev):
    K, n_out, dtype = 272, 16, torch.bfloat16
    rows = MORE // K + 5
    x, xl = _tail(dev, (rows, K), dtype, 5, 1)
    g, gl = _tail(dev, (rows, n_out), dtype, 5, 2)
    w = torch.randn(n_out, K, generator=torch.Generator().manual_seed(3)).to(dev, dtype).requires_grad_()

    def run(x, g):
        x = x.requires_grad_()
        y = training.linear_8bit(x, w, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))

    _same(run(x, g), run(xl, gl))


def test_bias(dev):
    n, H, dtype = 16384, 17, torch.float16
    index = torch.zeros(n, n, dtype=torch.int32, device=dev)
    index[-1, -7:] = torch.tensor([1, 2, 3, 1, 2, 3, 4], dtype=torch.int32)
    table = torch.randn(6, H, generator=torch.Generator().manual_seed(0)).to(dev, dtype).requires_grad_()
    out = training.relative_position_bias(table, training.BiasBuckets(index, 6))
    assert out.numel() > MORE
    assert torch.equal(out[:, -1, -7:], table.detach()[index[-1, -7:].long()].t())
    assert torch.equal(out[:, 5, :9], table.detach()[0][:, None].expand(-1, 9))
    grad = torch.zeros_like(out)
    grad[:, -1, -7:] = torch.arange(1, 8, dtype=dtype, device=dev)
    grad[:, 9, 9] = 0.5
    (d,) = torch.autograd.grad(out, table, grad)
    want = torch.tensor([0.5, 1 + 4, 2 + 5, 3 + 6, 7, 0], dtype=dtype, device=dev)
    assert torch.equal(d, want[:, None].expand(-1, H))
