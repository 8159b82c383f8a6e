"""What the training operators refuse before any HIP call, and their meta forms (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from crumpet_amd import _native, training

i64, i32, f32, vp = ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_void_p
FAKE = vp(256)


def _fn(name, *types, result=ctypes.c_int):
    f = getattr(_native.hip_library(), name)
    f.restype, f.argtypes = result, types
    return f


def _error():
    f = _native.hip_library().crumpet_last_error
    f.restype = ctypes.c_char_p
    return f().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 8, 96))
    for call in (lambda: training.window_attention(x, torch.zeros((2, 8, 8)), 2),
                 lambda: training.residual_norm(x, x),
                 lambda: training.linear_8bit(x.half(), torch.zeros((16, 96)).half()),
                 lambda: training.BiasBuckets(torch.zeros((2, 2), dtype=torch.int64), 4)):
        with pytest.raises(RuntimeError, match="runs only on HIP"):
            call()


def test_meta_tensors_give_shapes():
    qkv = torch.zeros((4, 27, 96), device="meta", dtype=torch.float16)
    bias = torch.zeros((2, 27, 27), device="meta")
    out = training.window_attention(qkv, bias, 2, volume=(6, 6, 3), window_size=(3, 3, 3), shift_size=(1, 1, 0))
    assert out.shape == (4, 27, 32) and out.dtype == torch.float16
    x1, h = training.residual_norm(torch.zeros((2, 3, 8), device="meta"), torch.zeros((2, 3, 8), device="meta").half())
    assert x1.dtype == torch.float32 and h.dtype == torch.float16 and x1.shape == h.shape == (2, 3, 8)
    y = training.linear_8bit(torch.zeros((2, 3, 32), device="meta").half(), torch.zeros((48, 32), device="meta").half())
    assert y.shape == (2, 3, 48)


def test_attention_checks():
    f = _fn("crumpet_window_attention", vp, vp, vp, vp, vp, ctypes.POINTER(i64), i32, i64, i64, i64, i64, vp, vp, i32,
            i64, i64, ctypes.POINTER(i64), f32, vp)

    def call(dtype=1, B=8, H=3, N=27, D=16, bias=FAKE, mask=None, M=1, region=None, strides=None, out=FAKE, top=FAKE,
             inv=FAKE):
        st = (i64 * 2)(*(strides or (N * 3 * H * D, 3 * H * D)))
        reg = None if region is None else (i64 * 9)(*region)
        return f(out, FAKE, top, inv, FAKE, st, dtype, B, H, N, D, bias, mask, 0, M, N * N, reg, 0.25, None)

    assert call(B=0) == 0 and call(N=0) == 0 and call(H=0) == 0
    assert call(dtype=7) == 1 and call(B=-1) == 1
    assert call(D=24) == 2 and "head_dim 24" in _error()
    assert call(N=16385) == 2 and call(H=5000) == 2 and call(B=1 << 31) == 2
    assert call(B=(1 << 31) - 1) == 2 and "one launch" in _error()
    assert call(bias=None) == 1 and call(out=None) == 1 and call(top=None) == 1
    assert call(strides=(27 * 144, 145)) == 2 and "16-byte" in _error()
    assert call(out=vp(8)) == 2 and "aligned" in _error()
    assert call(mask=FAKE, M=3) == 1 and "multiple of the masks" in _error()
    assert call(mask=FAKE, M=0) == 1
    good = (6, 6, 6, 3, 3, 3, 1, 1, 1)
    assert call(mask=FAKE, region=good) == 1 and "exclude" in _error()
    assert call(region=(7, 6, 6, 3, 3, 3, 1, 1, 1)) == 1 and "divisible" in _error()
    assert call(region=(6, 6, 6, 3, 3, 3, 3, 1, 1)) == 1 and "shift_size" in _error()
    assert call(region=(6, 6, 6, 3, 3, 3, -1, 1, 1)) == 1
    assert call(region=(6, 6, 6, 3, 3, 2, 1, 1, 1)) == 1 and "window volume" in _error()
    assert call(region=(9, 6, 6, 3, 3, 3, 1, 1, 1)) == 1 and "multiple of the volume" in _error()
    # products that would pass 64 bits
    big = 1 << 40
    assert call(region=(big, big, big, big, big, big, 0, 0, 0)) == 1
    assert call(region=(big, big, big, 1, 1, 1, 0, 0, 0), N=1) == 1

    w = _fn("crumpet_window_attention_workspace", i64, i64, i64, result=i64)
    assert w(0, 3, 27) == 0 and w(-1, 3, 27) == -1 and w(8, 3, 16385) == -1
    assert w(8, 3, 27) >= 8 * 3 * 27 * 4 + 3 * 27 * 27 * 4


def test_bias_checks():
    f = _fn("crumpet_bucket_bias", vp, vp, i32, vp, i64, i64, i64, vp)
    assert f(None, None, 0, None, 4, 0, 4, None) == 0 and f(None, None, 0, None, 4, 2, 0, None) == 0
    assert f(None, FAKE, 0, FAKE, 4, 2, 4, None) == 1
    assert f(FAKE, FAKE, 5, FAKE, 4, 2, 4, None) == 1
    assert f(FAKE, FAKE, 0, FAKE, 4, 70000, 4, None) == 2
    assert f(FAKE, FAKE, 0, FAKE, 4, 2, 1 << 31, None) == 2
    g = _fn("crumpet_bucket_bias_backward", vp, vp, i32, i64, i64, i64, vp, vp, i64, vp, vp, vp)
    assert g(None, None, 0, 4, 0, 4, None, None, 0, None, None, None) == 0
    assert g(FAKE, FAKE, 0, 4, 2, 4, FAKE, FAKE, 3, None, None, None) == 1 and "do not match" in _error()
    assert g(FAKE, FAKE, 0, 4, 2, 4, FAKE, FAKE, 3, FAKE, None, None) == 1 and "workspace" in _error()
    assert g(FAKE, None, 0, 4, 2, 4, FAKE, FAKE, 4, None, None, None) == 1


def test_norm_checks():
    f = _fn("crumpet_residual_norm", vp, vp, vp, i32, vp, i32, i64, i64, i64, i32, i32, vp, vp, vp, i32, vp, vp, vp,
            f32, vp)

    def call(x_dtype=0, dtype=1, S=2, T=5, C=48, norm=0, x=FAKE, w=None):
        return f(FAKE, FAKE, x, x_dtype, FAKE, dtype, S, T, C, norm, 0, None, None, None, 0, None, w, None, 1e-5, None)

    assert call(S=0) == 0 and call(T=0) == 0
    assert call(norm=2) == 1 and call(S=-1) == 1 and call(dtype=4) == 1 and call(x=None) == 1
    assert call(x_dtype=1, dtype=2) == 2 and call(x_dtype=1, dtype=0) == 2
    assert call(C=0) == 2 and call(C=8200) == 2 and call(C=4097) == 2
    assert call(S=1 << 20) == 2 and call(T=1 << 31) == 2
    assert call(x=vp(8)) == 2 and call(w=vp(4)) == 2 and "aligned" in _error()
    w = _fn("crumpet_residual_norm_workspace", i64, i64, i64, result=i64)
    assert w(0, 5, 48) == 0 and w(2, 5, 0) == -1 and w(2, 5, 48) % (5 * 48 * 4) == 0
    g = _fn("crumpet_residual_norm_backward", vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, vp, i32, i64, i64, i64, i32,
            i32, vp, vp, vp, i32, vp, vp, f32, vp, vp)

    def back(gate_grad=None, gate=None, per=0, S=2, weight_grad=None, post_grad=None, ws=None):
        return g(FAKE, FAKE, weight_grad, None, gate_grad, post_grad, None, FAKE, FAKE, FAKE, 0, FAKE, 1, S, 5, 48, 0, 0,
                 None, None, gate, per, None, None, 1e-5, ws, None)

    assert back(S=0) == 0
    assert back(gate_grad=FAKE) == 1 and back(post_grad=FAKE) == 1 and "not there" in _error()
    assert back(weight_grad=FAKE) == 1 and "workspace" in _error()
    assert back(gate_grad=FAKE, gate=FAKE, per=1, S=70000, ws=FAKE) == 2


def test_linear_checks():
    f = _fn("crumpet_linear_8bit", vp, vp, vp, vp, i32, i64, i64, vp, vp, i64, i32, vp)

    def call(dtype=1, rows=4, K=32, n_out=16, act=0, x=FAKE, codes=None, exps=None):
        return f(FAKE, codes, exps, x, dtype, rows, K, FAKE, None, n_out, act, None)

    assert call(rows=0) == 0
    assert call(dtype=0) == 2 and call(dtype=9) == 1 and call(act=2) == 1 and call(rows=-1) == 1
    assert call(K=24) == 2 and call(n_out=8) == 2 and call(K=0) == 2 and call(K=65552) == 2
    assert call(x=None) == 1 and call(codes=FAKE) == 1 and call(x=vp(8)) == 2
    assert call(rows=1 << 40) == 2 and "one launch" in _error()
    w = _fn("crumpet_linear_8bit_workspace", i64, i64, i64, result=i64)
    assert w(0, 32, 16) == 0 and w(4, 24, 16) == -1 and w(4, 32, 16) >= 32 * 16 * 2 + (32 * 16 + 16) * 4
    g = _fn("crumpet_linear_8bit_backward", vp, vp, vp, vp, i32, vp, vp, i64, i64, vp, i64, i32, vp, vp)
    assert g(FAKE, FAKE, FAKE, FAKE, 1, FAKE, FAKE, 0, 32, FAKE, 16, 0, FAKE, None) == 0
    assert g(FAKE, FAKE, FAKE, FAKE, 1, None, FAKE, 4, 32, FAKE, 16, 0, FAKE, None) == 1
    assert g(FAKE, FAKE, FAKE, FAKE, 1, FAKE, FAKE, 4, 32, FAKE, 16, 0, None, None) == 1
    assert g(FAKE, FAKE, FAKE, FAKE, 1, FAKE, FAKE, 4, 32, FAKE, 16, 0, vp(264), None) == 2
