"""The 64-bit forms that the training operators are tested against: their
written-out gradients agree with autograd of the plain formula, and with
differences."""

from __future__ import annotations

import torch

import training_reference as ref


def _rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def _differences(f, x, d, h=1e-5):
    return float((f(x + h * d) - f(x - h * d)) / (2 * h))


def test_attention_gradients():
    B, N, H, D = 2, 5, 2, 16
    qkv, bias, g = _rand(B, N, 3 * H * D).requires_grad_(), _rand(H, N, N, seed=1).requires_grad_(), _rand(B, N, H * D)
    mask = torch.zeros(1, N, N, dtype=torch.float64)
    mask[0, 1, 2:] = -torch.inf

    def plain(x, b):
        q, k, v = x.view(B, N, 3, H, D).permute(2, 0, 3, 1, 4)
        s = D ** -0.5 * q @ k.transpose(2, 3) + b + mask
        return (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, N, -1)

    out = plain(qkv, bias)
    dqkv, dbias = torch.autograd.grad(out, (qkv, bias), g)
    ref.TINY[torch.float64] = 0.0
    found = ref.window_attention(qkv, bias, H, g, mask)
    for name, value in (("out", out), ("grad_qkv", dqkv), ("grad_bias", dbias)):
        torch.testing.assert_close(found[name][0], value.detach(), rtol=1e-10, atol=1e-12)
    d = _rand(B, N, 3 * H * D, seed=5)
    diff = _differences(lambda x: (plain(x, bias.detach()) * g).sum(), qkv.detach(), d)
    assert abs(diff - float((found["grad_qkv"][0] * d).sum())) < 1e-6


def test_norm_gradients():
    ref.TINY[torch.float64] = 0.0
    S, T, C = 3, 4, 10
    t = {n: _rand(*s, seed=i).requires_grad_() for i, (n, s) in enumerate(
        {"x": (S, T, C), "y": (S, T, C), "weight": (C,), "bias": (C,), "post_weight": (C,), "post_bias": (C,),
         "gate": (S, C)}.items())}
    scale = torch.tensor([0.0, 1.25, 1.0], dtype=torch.float64)
    gs, go = _rand(S, T, C, seed=20), _rand(S, T, C, seed=21)
    for kind in ("layer", "rms"):
        for post in (False, True):
            def norm(v):
                v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
                return v / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()

            u = norm(t["y"]) * t["post_weight"] + t["post_bias"] if post else t["y"]
            x1 = t["x"] + scale[:, None, None] * t["gate"][:, None] * u
            h = norm(x1) * t["weight"] + t["bias"]
            names = [n for n in t if post or not n.startswith("post")]
            grads = torch.autograd.grad((x1, h), [t[n] for n in names], (gs, go))
            found = ref.residual_norm(t["x"], t["y"], gs, go, kind, post, scale=scale,
                                      **{n: t[n] for n in names if n not in "xy"})
            for n, g in zip(names, grads):
                torch.testing.assert_close(found["grad_" + n][0], g, rtol=1e-9, atol=1e-11)
            torch.testing.assert_close(found["out"][0], h.detach(), rtol=1e-9, atol=1e-11)


def test_linear_gradients_at_the_copy():
    """x is already a multiple of its step, so the copy is x and the gradients are the layer's."""
    ref.TINY[torch.float64] = 0.0
    x = torch.randint(-127, 128, (6, 48), generator=torch.Generator().manual_seed(3)).double() / 32
    x[:, ::32] = 127 / 32
    assert torch.equal(ref.eight_bits(x), x)
    w, b, g = _rand(16, 48, seed=1).requires_grad_(), _rand(16, seed=2).requires_grad_(), _rand(6, 16, seed=4)
    x.requires_grad_()
    for activation in ("none", "gelu"):
        a = torch.nn.functional.gelu(x) if activation == "gelu" else x
        out = torch.nn.functional.linear(a, w, b)
        grads = torch.autograd.grad(out, (x, w, b), g)
        found = ref.linear_8bit(x, w, b, g, activation)
        for n, v in zip(("grad_x", "grad_weight", "grad_bias"), grads):
            torch.testing.assert_close(found[n][0], v, rtol=1e-9, atol=1e-11)
    d = _rand(16, 48, seed=9)
    act = torch.nn.functional.gelu(x.detach())
    diff = _differences(lambda v: (torch.nn.functional.linear(act, v, b.detach()) * g).sum(), w.detach(), d)
    assert abs(diff - float((found["grad_weight"][0] * d).sum())) < 1e-6


def test_the_copys_steps():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5] + [0.0] * 28, [127.5] + [1.0] * 31, [0.0] * 32,
                      [float("inf")] + [1.0] * 31], dtype=torch.float64)
    kept = ref.eight_bits(x)
    assert kept[0, :4].tolist() == [127.0, 0.0, 2.0, -2.0]  # step 1, ties to even
    assert kept[1, :2].tolist() == [128.0, 0.0]  # step 2: 127.5 / 2 rounds to 64, 1 / 2 to 0
    assert kept[2].abs().max() == 0
    assert kept[3].isnan().all()
    y = torch.randn(64, 96, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    top = y.reshape(64, 3, 32).abs().amax(-1, keepdim=True)
    # half a step; the step is at most twice the largest value over 127
    assert ((ref.eight_bits(y) - y).reshape(64, 3, 32).abs() <= top / 127).all()


def test_position_bias_gradient():
    ref.TINY[torch.float64] = 0.0
    index = torch.tensor([[0, 1, 1], [2, 0, 4]])
    table = _rand(6, 2).requires_grad_()
    g = _rand(2, 2, 3, seed=1)
    out = table[index.reshape(-1)].t().reshape(2, 2, 3)
    (grad,) = torch.autograd.grad(out, table, g)
    found = ref.position_bias(table, index, g)
    torch.testing.assert_close(found["grad_table"][0], grad)
    assert found["grad_table"][0][[3, 5]].abs().max() == 0


def test_shift_mask_is_the_oracles(oracle):
    import numpy as np

    for volume, ws, ss in (((6, 4, 4), (3, 2, 2), (1, 0, 1)), ((4, 4, 4), (2, 4, 2), (1, 3, 0))):
        bits = oracle.attn_mask_bits(*volume, ws, ss, "float32")
        expected = torch.from_numpy(np.ascontiguousarray(bits).view(np.float32).copy())
        assert torch.equal(ref.shift_mask(volume, ws, ss).reshape(-1), expected.reshape(-1))
