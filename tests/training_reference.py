"""The training operators in 64 bits on the CPU, with error bounds.

Each function returns ``{name: (value, bound)}``: what the operator returns,
and how far a kernel may be off that computes in fp32 and rounds where the
operator's documentation says so.  u = 2^-24 is half a step of fp32, ``eps(t)``
half a step of type t relative to a value; a sum of n fp32 terms is off by at
most about n u times the sum of their magnitudes.  Gradients are written out
and compared with autograd and with differences in test_training_reference.py.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half a subnormal step


def eps(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def rounded(value, error, t):
    """(value, bound) of a result rounded to t behind an error."""
    return value, error + eps(t) * (value.abs() + error) + TINY[t]


def window_attention(qkv, bias, heads, grad, mask=None, scale=None, keep=True):
    dt, bias_dt = qkv.dtype, bias.dtype
    f = [t.detach().cpu().double() for t in (qkv, bias, grad)]
    B, N, C3 = f[0].shape
    D = C3 // (3 * heads)
    scale = D ** -0.5 if scale is None else scale
    q, k, v = f[0].view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4)
    do = f[2].view(B, N, heads, D).transpose(1, 2)
    terms = f[1][None].expand(B, -1, -1, -1)
    if mask is not None:
        m = mask.detach().cpu().double()
        # a mask of the type's lowest value absorbs the score in fp32
        terms = terms + m.repeat(B // m.shape[0], 1, 1)[:, None]
    s = scale * q @ k.transpose(2, 3) + terms
    if mask is not None:
        s = torch.where(s < -1e30, torch.where(s == -math.inf, s, torch.full_like(s, -3e38)), s)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = p @ v
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq, dk, dv = scale * ds @ k, scale * ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do
    # scores are off by (D + 8) u of their terms' magnitudes, weights by twice that and the exponential's 2^-22
    finite = torch.where((terms > -1e30) & (terms < 1e30), terms.abs(), 0.0)
    off_s = (D + 8) * U * float((abs(scale) * q.abs() @ k.abs().transpose(2, 3) + finite).max()) if s.numel() else 0.0
    off_p = 2 * off_s + 2.0 ** -22 + (N + 4) * U
    # a weight below the smallest normal number may come out as 0
    least = 2.0 ** -126
    r = eps(dt) if dt != torch.float32 else 0.0
    pv = p @ v.abs()
    off_out = (off_p + (N + 4) * U + (r * r if keep else r)) * pv + least * v.abs().sum(-2, keepdim=True)
    off_dp = (D + 2) * U * do.abs() @ v.abs().transpose(2, 3)
    off_delta = (do.abs() * (off_out + r * r * out.abs() + (D + 4) * U * out.abs())).sum(-1, keepdim=True)
    off_ds = off_p * ds.abs() + p * (off_dp + off_delta) + 4 * U * p * dp.abs() + least * (1 + 2 * dp.abs().amax())
    tiny = TINY[dt]
    off_q = abs(scale) * ((r + N * U) * ds.abs() + off_ds + tiny) @ k.abs()
    off_k = abs(scale) * ((r + N * U) * ds.abs() + off_ds + tiny).transpose(2, 3) @ q.abs()
    off_v = ((r + N * U + off_p) * p + tiny + least).transpose(2, 3) @ do.abs()

    def rows(*parts):
        return torch.stack(parts).permute(1, 3, 0, 2, 4).reshape(B, N, -1)

    dbias, off_bias = ds.sum(0), off_ds.sum(0) + B * U * ds.abs().sum(0)
    return {"out": rounded(out.transpose(1, 2).reshape(B, N, -1), off_out.transpose(1, 2).reshape(B, N, -1), dt),
            "grad_qkv": rounded(rows(dq, dk, dv), rows(off_q, off_k, off_v), dt),
            "grad_bias": rounded(dbias, off_bias, bias_dt)}


def shift_mask(volume, ws, shift):
    """[windows, N, N]: -100 between tokens on two sides of a cyclic seam."""
    label = torch.zeros(volume)
    for a in range(3):
        at = torch.arange(volume[a])
        part = (at >= volume[a] - ws[a]).float() + (at >= volume[a] - shift[a]).float()
        label = label * 3 + (part if shift[a] else 0 * part).reshape([-1 if b == a else 1 for b in range(3)])
    n = [v // w for v, w in zip(volume, ws)]
    label = label.reshape(n[0], ws[0], n[1], ws[1], n[2], ws[2]).permute(0, 2, 4, 1, 3, 5)
    label = label.reshape(-1, ws[0] * ws[1] * ws[2])
    return (label[:, :, None] != label[:, None, :]).float() * -100.0


def position_bias(table, index, grad):
    t, g = table.detach().cpu().double(), grad.detach().cpu().double()
    index = index.cpu().long()
    nq, nk = index.shape
    out = t[index.reshape(-1)].t().reshape(-1, nq, nk)
    flat = g.reshape(g.shape[0], -1).t()
    dtable = torch.zeros_like(t).index_add_(0, index.reshape(-1), flat)
    size = torch.zeros_like(t).index_add_(0, index.reshape(-1), flat.abs())
    n = int(torch.bincount(index.reshape(-1), minlength=1).max()) if index.numel() else 0
    return {"bias": (out, torch.zeros_like(out)), "grad_table": rounded(dtable, n * U * size, table.dtype)}


def _norm(x, kind, e):
    d = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    r = (d.square().mean(-1, keepdim=True) + e).rsqrt()
    return d * r, r


def _norm_grad(g, n, r, kind):
    a = g.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return r * (g - a - n * (g * n).mean(-1, keepdim=True))


def residual_norm(x, y, grad_sum, grad_out, kind="layer", post=False, e=1e-5, **params):
    """params: weight, bias, post_weight, post_bias, gate, scale (or None)."""
    p = {k: v.detach().cpu().double() for k, v in params.items() if v is not None}
    xd, yd = x.detach().cpu().double(), y.detach().cpu().double()
    S, C = x.shape[0], x.shape[-1]
    xd, yd = xd.reshape(S, -1, C), yd.reshape(S, -1, C)
    T = xd.shape[1]
    gs = 0.0 * xd if grad_sum is None else grad_sum.detach().cpu().double().reshape(S, -1, C)
    go = 0.0 * xd if grad_out is None else grad_out.detach().cpu().double().reshape(S, -1, C)
    one = torch.ones(1, 1, 1, dtype=torch.float64)
    k = p["scale"].reshape(S, 1, 1) if "scale" in p else one
    gate = p["gate"].reshape(-1, 1, C) if "gate" in p else one
    w, pw = p.get("weight", one), p.get("post_weight", one)
    yn, yr = _norm(yd, kind, e) if post else (yd, None)
    u = yn * pw + p.get("post_bias", 0.0)
    x1 = xd + k * gate * u
    n, r = _norm(x1, kind, e)
    h = n * w + p.get("bias", 0.0)
    t = go * w
    dx = gs + _norm_grad(t, n, r, kind)
    du = dx * k * gate
    v = du * pw
    dy = _norm_grad(v, yn, yr, kind) if post else du

    # A norm of values that are off by o and at most m: the mean and the
    # differences are off by o + (C + 4) u m, which the deviation's inverse r
    # scales, and r itself by a relative (C + 8) u and what the values' error
    # moves it.
    def big(a):
        return a.abs().amax(-1, keepdim=True)

    def off_norm(values, off, nn, rr):
        o = big(off) + (C + 4) * U * big(values)
        return rr * 2 * o * (1 + nn.abs() * big(nn)) + (C + 8) * U * nn.abs()

    def off_norm_grad(g, off_g, nn, off_n, rr):
        # the sums' errors and those of their factors, times r; r's own relative error
        m = big(g)
        first = big(off_g) * (2 + big(nn) * nn.abs()) + m * (big(off_n) * (big(nn) + nn.abs()))
        sums = (C + 8) * U * m * (2 + big(nn) * nn.abs())
        rel_r = (C + 8) * U + 2 * big(off_n)
        return rr * (first + sums + rel_r * m * (2 + big(nn) * nn.abs()))

    off_yn = off_norm(yd, torch.zeros_like(yd), yn, yr) if post else torch.zeros_like(yd)
    off_u = off_yn * pw.abs() + 2 * U * (u.abs() + (yn * pw).abs())
    off_x1 = (k * gate).abs() * off_u + 4 * U * (xd.abs() + (k * gate * u).abs())
    off_n = off_norm(x1, off_x1, n, r)
    off_h = off_n * w.abs() + 2 * U * ((n * w).abs() + h.abs())
    off_t = 2 * U * t.abs()
    off_dx = off_norm_grad(t, off_t, n, off_n, r) + 4 * U * (gs.abs() + dx.abs())
    off_du = (k * gate).abs() * off_dx + 4 * U * du.abs()
    off_v = off_du * pw.abs() + 2 * U * v.abs()
    off_dy = off_norm_grad(v, off_v, yn, off_yn, yr) if post else off_du

    def total(a, off, over):
        count = S * T if 0 in over else T
        return a.sum(over), off.sum(over) + (count + 4) * U * a.abs().sum(over)

    res = {"sum": rounded(x1.reshape(x.shape), off_x1.reshape(x.shape), x.dtype),
           "out": rounded(h.reshape(x.shape), off_h.reshape(x.shape), y.dtype),
           "grad_x": rounded(dx.reshape(x.shape), off_dx.reshape(x.shape), x.dtype),
           "grad_y": rounded(dy.reshape(x.shape), off_dy.reshape(x.shape), y.dtype)}
    sums = {"weight": (go * n, go.abs() * off_n + 2 * U * (go * n).abs()), "bias": (go, 0 * go),
            "post_weight": (du * yn, off_du * yn.abs() + du.abs() * off_yn + 2 * U * (du * yn).abs()),
            "post_bias": (du, off_du),
            "gate": (dx * k * u, k.abs() * (off_dx * u.abs() + dx.abs() * off_u) + 4 * U * (dx * k * u).abs())}
    for name, (a, off) in sums.items():
        if name in p:
            over = (1,) if name == "gate" and p["gate"].dim() == 2 else (0, 1)
            res["grad_" + name] = rounded(*total(a, off, over), params[name].dtype)
    return res


def eight_bits(x):
    """The 8-bit copy: for every row and 32 columns whole numbers times 2^e, e
    the least integer >= -126 with 127 2^e >= the largest magnitude; groups
    that are not finite are NaN."""
    v = x.detach().cpu().double()
    kept = torch.empty_like(v)
    for a in range(0, v.shape[1], 32):
        g = v[:, a:a + 32]
        top = g.abs().amax(1, keepdim=True)
        step = torch.full_like(top, 2.0 ** -126)
        for e in range(-126, 128):
            step = torch.where(127 * step < top, torch.full_like(top, 2.0 ** e), step)
        kept[:, a:a + 32] = torch.where(torch.isfinite(top), torch.round(g / step) * step, math.nan)
    return kept


GELU_OFF = 3e-7  # the error function's published 1.5e-7, doubled, and a few steps of fp32


def linear_8bit(x, weight, bias, grad, activation="none"):
    dt = x.dtype
    xd, w, g = (t.detach().cpu().double() for t in (x, weight, grad))
    xd, g = xd.reshape(-1, w.shape[1]), g.reshape(-1, w.shape[0])
    rows, K, n_out = xd.shape[0], w.shape[1], w.shape[0]
    kept = eight_bits(xd)

    def cdf(t):
        return 0.5 * torch.special.erfc(-t / 2 ** 0.5)

    r = off = 0.0
    a, a_kept, slope = xd, kept, torch.ones_like(xd)
    if activation == "gelu":
        a, a_kept = xd * cdf(xd), kept * cdf(kept)
        slope = cdf(kept) + kept * torch.exp(-kept * kept / 2) / (2 * math.pi) ** 0.5
        r, off = eps(dt), GELU_OFF
    tiny = TINY[dt]
    out = a @ w.t()
    b = 0.0
    if bias is not None:
        b = bias.detach().cpu().double()
        out = out + b
    off_out = ((r + (K + 4) * U) * a.abs() + off * xd.abs() + tiny * (r > 0)) @ w.abs().t() + 2 * U * out.abs()
    da = g @ w
    size = g.abs() @ w.abs()
    dx = da * slope
    off_x = ((n_out + 4) * U * slope.abs() + (2 * off if activation == "gelu" else 0)) * size
    dw = g.t() @ a_kept
    off_w = g.abs().t() @ ((r + (rows + 4) * U) * a_kept.abs() + off * kept.abs() + tiny * (r > 0))
    db = g.sum(0)
    res = {"out": rounded(out.reshape(*x.shape[:-1], n_out), off_out.reshape(*x.shape[:-1], n_out), dt),
           "grad_x": rounded(dx.reshape(x.shape), off_x.reshape(x.shape), dt), "grad_weight": rounded(dw, off_w, dt)}
    if bias is not None:
        res["grad_bias"] = rounded(db, (rows + 4) * U * g.abs().sum(0), dt)
    return res


def check(found, expected):
    """found {name: tensor} within the bounds of expected; NaN where NaN is expected."""
    for name, got in found.items():
        value, bound = expected[name]
        got = got.detach().cpu().double()
        assert got.shape == value.shape, (name, got.shape, value.shape)
        assert torch.equal(got.isnan(), value.isnan()), name
        off = (got - value).abs()
        worst = torch.where(value.isnan(), torch.zeros_like(off), off - bound)
        assert off.numel() == 0 or float(worst.max()) <= 0, (name, float(worst.max()), float(off.nan_to_num().max()))
