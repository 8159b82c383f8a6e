"""The operators that train a Swin block, as cases that can be timed.

Each case is one forward and backward pass of one operator of
``crumpet_amd.training``: the learned relative-position bias, the window
attention that adds it, the norms around the residual sum, and the linear
layer that keeps its input in 8 bits for the backward pass.  With ``own``
false the same results come from elementary torch operations in 32 bits.
Sizes are the Swin UNETR stages at feature sizes 48 and 96 (windows of 7, 6
and 8, heads of 16 and 32), with ragged rows and other bucket rules between;
``draw`` gives more cases of the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32  # columns that share one exponent of the 8-bit copy


# ---- cases ---------------------------------------------------------------------------


def _bias(name, rule, nq, nk, heads, dtype, ws=(0, 0, 0)):
    """``rule`` "window": the offsets of a window's tokens (``ws``); "log": the
    distance of two positions in buckets that widen with it."""
    case = {"kind": "bias", "rule": rule, "nq": nq, "nk": nk, "heads": heads, "dtype": dtype}
    case.update(zip(("ws_d", "ws_h", "ws_w"), ws))
    return {"name": name, **case} if name else case


def _attention(name, outer, grid, ws, heads, hd, dtype, mode):
    """``outer`` volumes of ``grid`` windows.  mode: "none", "shifted" (the
    mask of the cyclic shift, from the geometry) or "mask" (a mask tensor with
    masked keys, among them rows where nothing is left)."""
    case = {"kind": "attention", "outer": outer, "heads": heads, "hd": hd, "dtype": dtype, "mode": mode}
    for a, n, w in zip("dhw", grid, ws):
        case.update({f"n{a}": n, f"ws_{a}": w})
    return {"name": name, **case} if name else case


def _norm(name, samples, tokens, C, x_dtype, dtype, norm, post, gate, drop):
    """``x`` (the residual stream) in x_dtype, the branch and the normed result
    in dtype.  gate: "none", "channel" ([C]) or "sample" ([samples, C])."""
    case = {"kind": "norm", "samples": samples, "tokens": tokens, "C": C, "x_dtype": x_dtype, "dtype": dtype,
            "norm": norm, "post": post, "gate": gate, "drop": drop}
    return {"name": name, **case} if name else case


def _linear(name, rows, K, n_out, dtype, activation):
    case = {"kind": "linear", "rows": rows, "K": K, "n_out": n_out, "dtype": dtype, "activation": activation}
    return {"name": name, **case} if name else case


def listed():
    return [
        # stage 0 of Swin UNETR: 7^3 windows, three heads; a few microseconds, the launches count
        _bias("bias_7x7x7_fp32", "window", 343, 343, 3, "fp32", (7, 7, 7)),
        # 8^3 windows with the heads of the deepest stage
        _bias("bias_8x8x8_fp32", "window", 512, 512, 24, "fp32", (8, 8, 8)),
        # distance buckets over longer sequences, ragged: few buckets, each with many members
        _bias("bias_log_bf16", "log", 1000, 1501, 12, "bf16"),
        # stage 3 of four 96^3 crops: one 6^3 window each, 24 heads
        _attention("attn_stage3_bf16", 4, (1, 1, 1), (6, 6, 6), 24, 16, "bf16", "none"),
        # stage 0 of four 96^3 crops, shifted block: the largest attention of the model
        _attention("attn_stage0_fp16", 4, (7, 7, 7), (7, 7, 7), 3, 16, "fp16", "shifted"),
        # feature size 96 (heads of 32), a mask tensor of the program's own
        _attention("attn_mask_hd32_bf16", 2, (4, 4, 4), (7, 7, 7), 6, 32, "bf16", "mask"),
        # stage 1 of one crop without autocast
        _attention("attn_stage1_fp32", 1, (4, 4, 4), (7, 7, 7), 6, 16, "fp32", "shifted"),
        # stage 3: residual sum and norm2 of four crops, a small call
        _norm("norm_stage3_fp16", 4, 216, 384, "fp16", "fp16", "layer", False, "none", False),
        # stage 0 under autocast: fp32 stream, fp16 branch, drop path
        _norm("norm_stage0_fp16", 4, 48 * 48 * 48, 48, "fp32", "fp16", "layer", False, "none", True),
        # sandwich norms with a gate for each sample, ragged token count
        _norm("norm_gated_bf16", 3, 4001, 768, "bf16", "bf16", "rms", True, "sample", False),
        # second linear of the stage-0 MLP behind its GELU, four crops
        _linear("linear8_mlp_stage0_fp16", 4 * 48 * 48 * 48, 192, 48, "fp16", "gelu"),
        # first linear of the stage-2 MLP, four crops, ragged token count
        _linear("linear8_stage2_bf16", 6911, 192, 768, "bf16", "none"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["bias", "attention", "attention", "norm", "linear"])
    if kind == "bias":
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        if rng.random() < 0.6:
            ws = tuple(rng.randint(2, 8) for _ in range(3))
            n = ws[0] * ws[1] * ws[2]
            return _bias(None, "window", n, n, rng.randint(1, 24), dtype, ws)
        return _bias(None, "log", _log_int(rng, 1, 1500), _log_int(rng, 1, 1500), rng.randint(1, 16), dtype)
    if kind == "attention":
        ws = tuple(rng.randint(2, 8) for _ in range(3))
        n = ws[0] * ws[1] * ws[2]
        hd = rng.choice([16, 16, 32, 32, 64])
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        heads = rng.choice([1, 2, 3, 6, 12])
        # scores within those of the largest listed case, fewer in fp32
        most = (2e8 if dtype == "fp32" else 4e8) * 16 / hd
        windows = _log_int(rng, 1, max(1, min(1400, int(most / (heads * n * n)))))
        grid = (rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 4))
        outer = max(1, windows // (grid[0] * grid[1] * grid[2]))
        return _attention(None, outer, grid, ws, heads, hd, dtype, rng.choice(["none", "shifted", "shifted", "mask"]))
    if kind == "norm":
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        x_dtype = rng.choice(["fp32", dtype])
        C = rng.choice([8 * rng.randint(1, 128), 16 * rng.randint(1, 64), _log_int(rng, 8, 1024)])
        samples = rng.randint(1, 6)
        tokens = _log_int(rng, 1, max(1, int(16e6 / (C * samples))))
        return _norm(None, samples, tokens, C, x_dtype, dtype, rng.choice(["layer", "rms"]), rng.random() < 0.5,
                     rng.choice(["none", "channel", "sample"]), rng.random() < 0.5)
    K, n_out = 16 * _log_int(rng, 1, 96), 16 * _log_int(rng, 1, 48)
    rows = _log_int(rng, 1, max(1, int(60e6 / (K + n_out))))
    rows = min(rows, max(1, int(4e9 / (K * n_out))))
    return _linear(None, rows, K, n_out, rng.choice(["fp16", "bf16"]), rng.choice(["none", "gelu"]))


# ---- inputs --------------------------------------------------------------------------


class _Random:
    """Seeded normal and uniform values on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, dtype, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, shape):
        return torch.rand(shape, generator=self.g, device="cuda")


def _window_index(ws):
    """[N, N] bucket of each pair of a window's tokens: its offset along the
    three axes, each moved to 0 .. 2 ws - 2."""
    axes = [torch.arange(w, device="cuda") for w in ws]
    at = torch.stack(torch.meshgrid(*axes, indexing="ij")).reshape(3, -1)
    off = at[:, :, None] - at[:, None, :]
    index = torch.zeros_like(off[0])
    for a in range(3):
        index = index * (2 * ws[a] - 1) + off[a] + ws[a] - 1
    return index, (2 * ws[0] - 1) * (2 * ws[1] - 1) * (2 * ws[2] - 1)


def _log_index(nq, nk):
    """[nq, nk] buckets of the distance key - query: 16 to each side, exact
    below 8, then widening up to a distance of 128."""
    d = torch.arange(nk, device="cuda")[None, :] - torch.arange(nq, device="cuda")[:, None]
    a = d.abs()
    far = 8 + (torch.log(a.clamp(min=1).double() / 8) / math.log(16.0) * 8).long()
    return torch.where(a < 8, a, far.clamp(max=15)) + 16 * (d > 0), 32


def _geometry(c):
    ws = (c["ws_d"], c["ws_h"], c["ws_w"])
    volume = tuple(n * w for n, w in zip((c["nd"], c["nh"], c["nw"]), ws))
    shift = tuple(w // 2 if v > w else 0 for v, w in zip(volume, ws))
    return volume, ws, shift


def _inputs(c, seed):
    r = _Random(seed)
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "bias":
        index, buckets = (_window_index((c["ws_d"], c["ws_h"], c["ws_w"])) if c["rule"] == "window"
                          else _log_index(c["nq"], c["nk"]))
        return {"index": index, "buckets": buckets, "table": r.normal((buckets, c["heads"]), dt, 0.5),
                "grad": r.normal((c["heads"], c["nq"], c["nk"]), dt)}
    if c["kind"] == "attention":
        volume, ws, shift = _geometry(c)
        n, windows = ws[0] * ws[1] * ws[2], c["nd"] * c["nh"] * c["nw"]
        B, C = c["outer"] * windows, c["heads"] * c["hd"]
        s = {"qkv": r.normal((B, n, 3 * C), dt), "bias": r.normal((c["heads"], n, n), torch.float32, 0.5),
             "grad": r.normal((B, n, C), dt), "mask": None}
        if c["mode"] == "mask":
            # a tenth of the keys masked, a few queries left with none
            off = r.uniform((windows, n, n)) < 0.1
            off |= r.uniform((windows, n, 1)) < 0.01
            s["mask"] = torch.zeros((windows, n, n), device="cuda", dtype=dt).masked_fill_(off, -math.inf)
        return s
    if c["kind"] == "norm":
        xt, S, C = DTYPES[c["x_dtype"]], c["samples"], c["C"]
        shape = (S, c["tokens"], C)
        s = {"x": r.normal(shape, xt), "y": r.normal(shape, dt), "grad_sum": r.normal(shape, xt),
             "grad_norm": r.normal(shape, dt), "weight": 1 + r.normal((C,), torch.float32, 0.1),
             "bias": r.normal((C,), torch.float32, 0.1) if c["norm"] == "layer" else None,
             "post_weight": None, "post_bias": None, "gate": None, "scale": None}
        if c["post"]:
            s["post_weight"] = 1 + r.normal((C,), torch.float32, 0.1)
            s["post_bias"] = r.normal((C,), torch.float32, 0.1) if c["norm"] == "layer" else None
        if c["gate"] != "none":
            s["gate"] = r.normal((S, C) if c["gate"] == "sample" else (C,), torch.float32, 0.5)
        if c["drop"]:  # drop path: whole samples without their branch, the others scaled up
            s["scale"] = (r.uniform((S,)) < 0.8).float() / 0.8
        return s
    K, n_out = c["K"], c["n_out"]
    return {"x": r.normal((c["rows"], K), dt), "weight": r.normal((n_out, K), dt, K ** -0.5),
            "bias": r.normal((n_out,), dt, 0.1), "grad": r.normal((c["rows"], n_out), dt)}


# what the passes differentiate for
_LEAVES = {"bias": ("table",), "attention": ("qkv", "bias"),
           "norm": ("x", "y", "post_weight", "post_bias", "gate", "weight", "bias"),
           "linear": ("x", "weight", "bias")}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own:
        from crumpet_amd import training

        s["training"] = training
        if case["kind"] == "bias":
            # kept with the module, as the index itself is
            s["plan"] = training.BiasBuckets(s["index"], s["buckets"])
        for name in _LEAVES[case["kind"]]:
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ---- the framework's calls -----------------------------------------------------------


def _own_pass(s):
    c, t = s["case"], s["training"]
    if c["kind"] == "bias":
        outs, grads = (t.relative_position_bias(s["table"], s["plan"]),), (s["grad"],)
        names = ("bias",)
    elif c["kind"] == "attention":
        geometry = {}
        if c["mode"] == "shifted":
            geometry = dict(zip(("volume", "window_size", "shift_size"), _geometry(c)))
        outs = (t.window_attention(s["qkv"], s["bias"], c["heads"], mask=s["mask"], **geometry),)
        names, grads = ("out",), (s["grad"],)
    elif c["kind"] == "norm":
        outs = t.residual_norm(s["x"], s["y"], norm=c["norm"], post=c["post"], post_weight=s["post_weight"],
                               post_bias=s["post_bias"], gate=s["gate"], scale=s["scale"], weight=s["weight"],
                               bias=s["bias"])
        names, grads = ("sum", "norm"), (s["grad_sum"], s["grad_norm"])
    else:
        outs = (t.linear_8bit(s["x"], s["weight"], s["bias"], activation=c["activation"]),)
        names, grads = ("out",), (s["grad"],)
    leaves = [n for n in _LEAVES[c["kind"]] if s[n] is not None]
    found = torch.autograd.grad(outs, [s[n] for n in leaves], grads)
    result = dict(zip(names, (o.detach() for o in outs)))
    result.update({"grad_" + n: g for n, g in zip(leaves, found)})
    return result


# ---- the plain form: elementary operations in 32 bits ---------------------------------


def _plain_bias(s):
    table, index = s["table"], s["index"]
    nq, nk = index.shape
    flat = index.reshape(-1)
    bias = table[flat].t().reshape(-1, nq, nk).contiguous()
    rows = s["grad"].float().reshape(-1, nq * nk).t()
    grad = torch.zeros(table.shape, device="cuda").index_add_(0, flat, rows)
    return {"bias": bias, "grad_table": grad.to(table.dtype)}


def _shift_mask(c):
    """[windows, N, N] of 0 where two tokens of a window stay neighbours under
    the cyclic shift, -100 elsewhere."""
    volume, ws, shift = _geometry(c)
    label = torch.zeros(volume, device="cuda")
    for a in range(3):
        at = torch.arange(volume[a], device="cuda")
        part = (at >= volume[a] - ws[a]).float() + (at >= volume[a] - shift[a]).float()
        label = label * 3 + (part if shift[a] else part * 0).reshape([-1 if b == a else 1 for b in range(3)])
    label = label.reshape(c["nd"], ws[0], c["nh"], ws[1], c["nw"], ws[2]).permute(0, 2, 4, 1, 3, 5)
    label = label.reshape(-1, ws[0] * ws[1] * ws[2])
    return (label[:, :, None] != label[:, None, :]).float() * -100.0


def _plain_attention(s):
    c, H, D = s["case"], s["case"]["heads"], s["case"]["hd"]
    B, n, _ = s["qkv"].shape
    q, k, v = s["qkv"].float().reshape(B, n, 3, H, D).permute(2, 0, 3, 1, 4).contiguous()
    scale = D ** -0.5
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale + s["bias"]
    mask = _shift_mask(c) if c["mode"] == "shifted" else s["mask"]
    if mask is not None:
        score = (score.reshape(-1, mask.shape[0], H, n, n) + mask.float()[:, None]).reshape(B, H, n, n)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)  # a row without keys gives zeros
    out = torch.matmul(p, v)
    do = s["grad"].float().reshape(B, n, H, D).transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    dqkv = torch.stack([dq, dk, dv]).permute(1, 3, 0, 2, 4).reshape(B, n, -1)
    return {"out": out.transpose(1, 2).reshape(B, n, -1).to(s["qkv"].dtype), "grad_qkv": dqkv.to(s["qkv"].dtype),
            "grad_bias": ds.sum(0)}


def _normed(x, kind):
    """(normed rows, 1 / their deviation)"""
    d = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-5)
    return d * r, r


def _normed_grad(g, n, r, kind):
    """Gradient of the rows from that of the normed ones."""
    g = g - n * (g * n).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return g * r


def _plain_norm(s):
    c, kind = s["case"], s["case"]["norm"]
    x, y = s["x"].float(), s["y"].float()
    yn, yr = _normed(y, kind) if c["post"] else (y, None)
    u = yn * s["post_weight"] if c["post"] else yn
    if s["post_bias"] is not None:
        u = u + s["post_bias"]
    k = torch.ones((c["samples"], 1, 1), device="cuda") if s["scale"] is None else s["scale"].reshape(-1, 1, 1)
    gate = 1.0 if s["gate"] is None else s["gate"].reshape(-1, 1, c["C"])
    x1 = x + k * gate * u
    n1, r1 = _normed(x1, kind)
    h = n1 * s["weight"]
    if s["bias"] is not None:
        h = h + s["bias"]
    gh = s["grad_norm"].float()
    result = {"sum": x1.to(s["x"].dtype), "norm": h.to(s["y"].dtype), "grad_weight": (gh * n1).sum((0, 1))}
    if s["bias"] is not None:
        result["grad_bias"] = gh.sum((0, 1))
    dx = s["grad_sum"].float() + _normed_grad(gh * s["weight"], n1, r1, kind)
    result["grad_x"] = dx.to(s["x"].dtype)
    du = dx * k * gate
    if s["gate"] is not None:
        dg = (dx * k * u).sum(1)
        result["grad_gate"] = dg if c["gate"] == "sample" else dg.sum(0)
    if c["post"]:
        result["grad_post_weight"] = (du * yn).sum((0, 1))
        if s["post_bias"] is not None:
            result["grad_post_bias"] = du.sum((0, 1))
        du = _normed_grad(du * s["post_weight"], yn, yr, kind)
    result["grad_y"] = du.to(s["y"].dtype)
    return result


def _eight_bits(x):
    """The 8-bit copy's values: whole multiples, up to 127, of a power of two
    for every 32 columns, the smallest one that reaches the largest of them."""
    rows, K = x.shape
    pad = -K % GROUP
    g = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, GROUP)
    m, e = torch.frexp(g.abs().amax(-1, keepdim=True))  # m 2^e with m in [1/2, 1)
    e = torch.where(m > 127 / 128, e - 6, e - 7).clamp(min=-126)
    step = torch.ldexp(torch.ones_like(m), e)
    return (torch.round(g / step) * step).reshape(rows, -1)[:, :K]


def _plain_linear(s):
    x, w, g = s["x"].float(), s["weight"].float(), s["grad"].float()
    kept = _eight_bits(x)
    da = torch.matmul(g, w)
    if s["case"]["activation"] == "gelu":
        out = 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
        phi = 0.5 * (1 + torch.erf(kept * 0.5 ** 0.5))
        dx = da * (phi + kept * torch.exp(-0.5 * kept * kept) * (2 * math.pi) ** -0.5)
        kept = kept * phi
    else:
        out, dx = x, da
    out = torch.matmul(out, w.t()) + s["bias"].float()
    dt = s["x"].dtype
    return {"out": out.to(dt), "grad_x": dx.to(dt), "grad_weight": torch.matmul(g.t(), kept).to(dt),
            "grad_bias": g.sum(0).to(dt)}


_PLAIN = {"bias": _plain_bias, "attention": _plain_attention, "norm": _plain_norm, "linear": _plain_linear}


def run(state):
    if own:
        return _own_pass(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------


def work(case):
    c = case
    e = DTYPES[c["dtype"]].itemsize
    if c["kind"] == "bias":
        pairs = c["nq"] * c["nk"]
        buckets = 32 if c["rule"] == "log" else math.prod(2 * c["ws_" + a] - 1 for a in "dhw")
        # bias written, its gradient read, the index read as the 32-bit number it needs, once
        return {"bytes": 2 * c["heads"] * pairs * e + 4 * pairs + 2 * buckets * c["heads"] * e,
                "flops": c["heads"] * pairs}
    if c["kind"] == "attention":
        volume, ws, _ = _geometry(c)
        n, windows = math.prod(ws), c["nd"] * c["nh"] * c["nw"]
        B, C = c["outer"] * windows, c["heads"] * c["hd"]
        mask = windows * n * n * e if c["mode"] == "mask" else 0
        # qkv and the output's gradient read, output and qkv's gradient written; bias and its gradient;
        # two products forward, five backward
        return {"bytes": 8 * B * n * C * e + 2 * c["heads"] * n * n * 4 + mask,
                "flops": 14 * B * c["heads"] * n * n * c["hd"]}
    if c["kind"] == "norm":
        ex = DTYPES[c["x_dtype"]].itemsize
        elements = c["samples"] * c["tokens"] * c["C"]
        return {"bytes": 4 * elements * (ex + e), "flops": 30 * elements}
    rows, K, n = c["rows"], c["K"], c["n_out"]
    return {"bytes": 2 * rows * (K + n) * e + 2 * n * (K + 1) * e, "flops": 6 * rows * K * n}


# ---- the definitions in 64 bits ----------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    f = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    c = case
    if c["kind"] == "bias":
        one = torch.nn.functional.one_hot
        nq, nk = s["index"].shape
        # row by row: the members of each bucket as a 0/1 matrix
        bias = f["table"].t()[:, s["index"]]
        grad = torch.zeros_like(f["table"])
        for i in range(nq):
            grad += torch.matmul(one(s["index"][i], s["buckets"]).double().t(), f["grad"][:, i].t().contiguous())
        return {"bias": bias, "grad_table": grad}
    if c["kind"] == "attention":
        return _exact_attention(c, f)
    if c["kind"] == "norm":
        return _exact_norm(c, f)
    return _exact_linear(c, s, f)


def _exact_attention(c, f):
    H, D = c["heads"], c["hd"]
    B, n, C3 = f["qkv"].shape
    mask = f["mask"]
    if c["mode"] == "shifted":
        mask = _shift_mask(c).double()
    out = torch.zeros((B, n, C3 // 3), dtype=torch.float64, device="cuda")
    dqkv, dbias = torch.zeros_like(f["qkv"]), torch.zeros_like(f["bias"])
    for h in range(H):  # one head at a time: the scores of a large case are several GB
        q, k, v = (f["qkv"][:, :, i * C3 // 3 + h * D:i * C3 // 3 + (h + 1) * D].contiguous() for i in range(3))
        g = f["grad"][:, :, h * D:(h + 1) * D].contiguous()
        a = torch.bmm(q, k.transpose(1, 2).contiguous()) / D ** 0.5 + f["bias"][h]
        if mask is not None:
            a += mask.repeat(B // mask.shape[0], 1, 1)
        a = torch.nan_to_num(torch.softmax(a, -1), nan=0.0)
        out[:, :, h * D:(h + 1) * D] = torch.bmm(a, v)
        da = torch.bmm(g, v.transpose(1, 2).contiguous())
        ds = a * da - a * torch.sum(a * da, -1, keepdim=True)
        dbias[h] = ds.sum(0)
        parts = (torch.bmm(ds, k) / D ** 0.5, torch.bmm(ds.transpose(1, 2).contiguous(), q) / D ** 0.5,
                 torch.bmm(a.transpose(1, 2).contiguous(), g))
        for i, d in enumerate(parts):
            dqkv[:, :, i * C3 // 3 + h * D:i * C3 // 3 + (h + 1) * D] = d
    return {"out": out, "grad_qkv": dqkv, "grad_bias": dbias}


def _exact_norm(c, f):
    leaves = {k: f[k].clone().requires_grad_() for k in _LEAVES["norm"] if f[k] is not None}

    def norm(t):
        if c["norm"] == "layer":
            t = t - t.mean(-1, keepdim=True)
        return t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt()

    with torch.enable_grad():
        u = leaves["y"]
        if c["post"]:
            u = norm(u) * leaves["post_weight"] + leaves.get("post_bias", 0.0)
        if "gate" in leaves:
            u = u * (leaves["gate"][:, None] if c["gate"] == "sample" else leaves["gate"])
        if f["scale"] is not None:
            u = u * f["scale"][:, None, None]
        total = leaves["x"] + u
        h = norm(total) * leaves["weight"] + leaves.get("bias", 0.0)
        grads = torch.autograd.grad((total, h), list(leaves.values()), (f["grad_sum"], f["grad_norm"]))
    return {"sum": total.detach(), "norm": h.detach(), **{"grad_" + k: g for k, g in zip(leaves, grads)}}


def _exact_linear(c, s, f):
    rows, K = s["x"].shape
    kept = torch.empty_like(f["x"])
    for a in range(0, K, GROUP):  # whole numbers of 2^e, e the least with 127 2^e >= the largest value
        part = f["x"][:, a:a + GROUP]
        top = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 127))
        e = torch.where(127 * 2.0 ** (e - 1) >= top, e - 1, e)
        e = torch.where(127 * 2.0 ** e < top, e + 1, e).clamp(min=-126)
        kept[:, a:a + GROUP] = torch.round(part * 2.0 ** -e) * 2.0 ** e
    dx = torch.matmul(f["grad"], f["weight"])
    act, act_kept = f["x"], kept
    if c["activation"] == "gelu":
        cdf = lambda t: 0.5 * torch.special.erfc(-t / 2 ** 0.5)  # noqa: E731
        act, act_kept = f["x"] * cdf(f["x"]), kept * cdf(kept)
        dx = dx * (cdf(kept) + kept * torch.exp(-kept * kept / 2) / (2 * math.pi) ** 0.5)
    return {"out": torch.matmul(act, f["weight"].t().contiguous()) + f["bias"], "grad_x": dx,
            "grad_weight": torch.matmul(f["grad"].t().contiguous(), act_kept), "grad_bias": f["grad"].sum(0)}
