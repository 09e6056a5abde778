# SPDX-License-Identifier: Apache-2.0
"""The 8-bit path of a layer, as measurable cases: e4m3 codes with one fp32 scale for each 128 columns of
an activation's row and for each 128 x 128 block of a weight.

Five kinds, each one call through the public device entry points:

  norm     v = x + residual, the new residual, RMSNorm of v in 8 bits and, where a router wants it, in
           bf16 or fp32 (k3d_add_norm)
  quant    act(gate) * up, or a plain row, in 8 bits (k3d_quant_f8)
  linear   y = act(x W^T + bias) + residual (k3d_linear_f8)
  grouped  rows sorted by expert times their experts' weights, ragged counts (k3d_grouped_f8)
  moe      the experts' layer for a routing: gate and up, gated activation in 8 bits, down, weighted sum
           (k3d_moe_f8)

Values: activations ~ N(0, 1) (quantised rows of them for the products), weights ~ N(0, 1/in) in codes
and block scales, norm weights ~ N(1, 0.1), biases ~ N(0, 0.1). Routings: distinct experts of a token,
with a popularity that falls as 1/rank (skewed) or none.
"""
import math
import os
import sys

import torch

own = False         # False: the plain forms below; True: the library's entry points

F8, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32
TYPES = {"f32": F32, "bf16": BF16}
CODE = {"f32": 0, "bf16": 1}
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
BLOCK, LEAST = 128, 2.0 ** -100
B1, B2 = 4.0, 25.0          # the two limits of the situ activation


def _norm(tokens, n, x, res, both):
    return dict(kind="norm", tokens=tokens, n=n, x=x, res=res, both=both)


def _quant(tokens, n, x, act):
    return dict(kind="quant", tokens=tokens, n=n, x=x, act=act)


def _linear(tokens, inn, out, y, bias, act, res):
    return dict(kind="linear", tokens=tokens, inn=inn, out=out, y=y, bias=bias, act=act, res=res)


def _grouped(tokens, topk, experts, inn, out, y, skew):
    return dict(kind="grouped", tokens=tokens, topk=topk, experts=experts, inn=inn, out=out, y=y, skew=skew)


def _moe(tokens, topk, experts, hidden, inter, act, skew):
    return dict(kind="moe", tokens=tokens, topk=topk, experts=experts, hidden=hidden, inter=inter, act=act, skew=skew)


def listed():
    return [
        # one decoded token: launch latency; its router reads the norm in bf16
        dict(_norm(1, 7168, "f32", "bf16", "bf16"), name="norm_1"),
        # a long prompt between two layers
        dict(_norm(4096, 7168, "bf16", "bf16", "none"), name="norm_4096"),
        # a decode batch's gated activation before the down product
        dict(_quant(64, 2048, "f32", "silu"), name="quant_64_gated"),
        # the same of a long prompt's eight experts a token
        dict(_quant(32768, 2048, "bf16", "silu"), name="quant_32768_gated"),
        # the fused projection of one decoded token: the weights' bytes are all there is
        dict(_linear(1, 7168, 12288, "bf16", True, "none", False), name="linear_1"),
        # the projection back onto an fp32 residual stream for a ragged decode batch
        dict(_linear(37, 12288, 7168, "f32", False, "none", True), name="linear_37_residual"),
        # no size a multiple of a block
        dict(_linear(333, 1001, 2047, "bf16", True, "gelu", True), name="linear_ragged_333"),
        # a long prompt through a wide projection: the matrix units' rate
        dict(_linear(4096, 7168, 12288, "bf16", True, "silu", False), name="linear_4096"),
        # a decode batch of 64 tokens: one or two rows an expert, most experts read
        dict(_grouped(64, 8, 384, 7168, 2048, "f32", False), name="grouped_64"),
        # a long prompt with popular experts: from a few rows to thousands
        dict(_grouped(4096, 8, 64, 7168, 2048, "bf16", True), name="grouped_4096_skewed"),
        # one decoded token through its eight experts
        dict(_moe(1, 8, 64, 7168, 2048, "silu", False), name="moe_1"),
        # a prompt's chunk through the experts' layer
        dict(_moe(2048, 8, 64, 7168, 2048, "situ", False), name="moe_2048"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm",) * 2 + ("quant",) * 2 + ("linear",) * 4 + ("grouped",) * 3 + ("moe",) * 2)
    if kind in ("norm", "quant"):
        step = rng.choice((128, 128, 8, 1))
        n = max(step, _log(rng, 64, 12288) // step * step)
    if kind == "norm":
        x, res = rng.choice(("f32", "bf16")), rng.choice(("f32", "bf16", "none"))
        return _norm(min(_log(rng, 1, 8192), max(1, 2048 * 7168 // n)), n, x, res, rng.choice(("none", "none", "bf16", "f32")))
    if kind == "quant":
        return _quant(min(_log(rng, 1, 32768), max(1, 16384 * 2048 // n)), n, rng.choice(("f32", "bf16", "bf16")),
                      rng.choice(("silu", "silu", "situ", "none")))
    if kind == "linear":
        step = rng.choice((128, 128, 128, 16, 1))
        inn = max(step, _log(rng, 256, 12288) // step * step)
        step = rng.choice((128, 32, 1))
        out = max(step, _log(rng, 64, 16384) // step * step)
        most = 4096 * 7168 * 12288 // (inn * out)
        return _linear(max(1, min(_log(rng, 1, 4096), most)), inn, out, rng.choice(("bf16", "f32")), rng.random() < 0.4,
                       rng.choice(ACTS), rng.random() < 0.4)
    experts = rng.choice((8, 16, 32, 64, rng.randint(3, 64)))
    topk = min(experts, rng.choice((1, 2, 4, 6, 8, 8)))
    tokens, skew = _log(rng, 1, 2048), rng.random() < 0.4
    step = rng.choice((128, 128, 64, 16))
    a, b = max(step, _log(rng, 512, 7168) // step * step), max(step, _log(rng, 256, 2048) // step * step)
    if kind == "grouped":
        if rng.random() < 0.5:
            a, b = b, a
        return _grouped(tokens, topk, experts, a, b, rng.choice(("bf16", "f32")), skew)
    return _moe(tokens, topk, experts, a, b, rng.choice(("silu", "situ")), skew)


# ------------------------------------------------------------------ inputs ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, sigma=1.0, mean=0.0, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).mul_(sigma).add_(mean).to(dtype)


def _up(n):
    return -(-n // BLOCK)


def _rows8(g, T, n):
    """Quantised rows of N(0, 1): codes [T][n up to a whole block, zeros behind n], scales [T][blocks]."""
    nb = _up(n)
    v = torch.zeros(T, nb * BLOCK, device="cuda")
    v[:, :n] = torch.randn(T, n, device="cuda", generator=g)
    v = v.view(T, nb, BLOCK)
    s = v.abs().amax(2).clamp_(min=LEAST) / 448
    return (v / s.unsqueeze(2)).to(F8).view(T, nb * BLOCK), s


def _weights8(g, mats, out, inn):
    """Codes [mats][out][in] and block scales [mats][out blocks][in blocks] of weights ~ N(0, 1/in): the largest of a
    block's 16384 is some 4.2 standard deviations."""
    q = torch.empty(mats, out, inn, device="cuda", dtype=F8)
    for i in range(mats):
        q[i] = torch.randn(out, inn, device="cuda", generator=g).mul_(448 / 4.2).clamp_(-448, 448)
    s = torch.rand(mats, _up(out), _up(inn), device="cuda", generator=g).mul_(0.3).add_(0.85)
    return q, s.mul_(4.2 / 448 * inn ** -0.5)


def _routing(g, T, k, experts, skew):
    """idx [T][k]: distinct experts of a token, drawn without return; wt: weights that sum to 1."""
    rank = torch.arange(experts, device="cuda", dtype=F32)
    lean = -torch.log(rank + 1) if skew else torch.zeros_like(rank)
    lean = lean[torch.randperm(experts, device="cuda", generator=g)]
    u = torch.rand(T, experts, device="cuda", generator=g).clamp_(1e-7, 1 - 1e-7)
    idx = torch.topk(lean - torch.log(-torch.log(u)), k, dim=1).indices
    wt = torch.rand(T, k, device="cuda", generator=g).add_(0.1)
    return idx.to(torch.int32), wt / wt.sum(1, keepdim=True)


def _sorted(idx, experts):
    """offsets [experts + 1] and perm: the assignments t k + j by expert, in their order within one."""
    flat = idx.flatten().long()
    perm = torch.sort(flat, stable=True).indices
    count = torch.bincount(flat, minlength=experts)
    offsets = torch.zeros(experts + 1, device="cuda", dtype=torch.int32)
    offsets[1:] = torch.cumsum(count, 0)
    return offsets, perm.to(torch.int32), int(count.max())


def _inputs(c, seed):
    g, T = _gen(seed), c["tokens"]
    if c["kind"] == "norm":
        d = {"xx": _normal(g, T, c["n"], dtype=TYPES[c["x"]]), "w": _normal(g, c["n"], sigma=0.1, mean=1.0)}
        d["r"] = _normal(g, T, c["n"], sigma=3.0, dtype=TYPES[c["res"]]) if c["res"] != "none" else None
        return d
    if c["kind"] == "quant":
        return {"xx": _normal(g, T, c["n"] * (1 if c["act"] == "none" else 2), dtype=TYPES[c["x"]])}
    if c["kind"] == "linear":
        d = {}
        d["q"], d["s"] = _rows8(g, T, c["inn"])
        w, d["ws"] = _weights8(g, 1, c["out"], c["inn"])
        d["w"] = w[0]
        d["bias_"] = _normal(g, c["out"], sigma=0.1) if c["bias"] else None
        d["r"] = _normal(g, T, c["out"], dtype=TYPES[c["y"]]) if c["res"] else None
        return d
    d = {}
    d["idx"], d["wt"] = _routing(g, T, c["topk"], c["experts"], c["skew"])
    d["offsets"], d["perm"], d["most"] = _sorted(d["idx"], c["experts"])
    if c["kind"] == "grouped":
        d["q"], d["s"] = _rows8(g, T, c["inn"])
        d["w"], d["ws"] = _weights8(g, c["experts"], c["out"], c["inn"])
        return d
    d["q"], d["s"] = _rows8(g, T, c["hidden"])
    for m, (o, i) in {"1": (c["inter"], c["hidden"]), "3": (c["inter"], c["hidden"]), "2": (c["hidden"], c["inter"])}.items():
        d["w" + m], d["ws" + m] = _weights8(g, c["experts"], o, i)
    return d


def _lib():
    path = os.path.join(os.getcwd(), "kimi-k3-in-c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import k3amd
    return k3amd


def _tiled(k3, w):
    """The weights as a program keeps them: laid out once, [mats] one after another."""
    mats, out, inn = w.shape
    size = k3.lib().k3d_f8_tiled_bytes(out, inn)
    t = torch.empty(mats * size, device="cuda", dtype=torch.uint8)
    k3.check(k3.lib().k3d_f8_tile(t.data_ptr(), w.data_ptr(), inn, out, inn, mats, _stream()), "k3d_f8_tile")
    return t


def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    T = s["tokens"]
    new = lambda *shape, dtype=F32: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
    if s["kind"] in ("norm", "quant"):
        s["q"], s["qs"] = new(T, _up(s["n"]) * BLOCK, dtype=F8), new(T, _up(s["n"]))
        if s["kind"] == "norm":
            s["sum"] = torch.empty_like(s["r"]) if s["r"] is not None else None
            s["yy"] = new(T, s["n"], dtype=TYPES[s["both"]]) if s["both"] != "none" else None
    elif s["kind"] == "linear":
        s["yy"] = new(T, s["out"], dtype=TYPES[s["y"]])
    elif s["kind"] == "grouped":
        s["yy"] = new(T * s["topk"], s["out"], dtype=TYPES[s["y"]])
    else:
        s["yy"] = new(T, s["hidden"], dtype=BF16)
    if own:
        k3 = _lib()
        L = k3.lib()
        k3.check(L.k3d_init(), "k3d_init")
        if s["kind"] == "linear":
            s["w"] = _tiled(k3, s["w"].unsqueeze(0))
            s["work"] = new(max(1, L.k3d_linear_f8_ws(T, s["inn"], s["out"])), dtype=torch.uint8)
        elif s["kind"] == "grouped":
            s["w"] = _tiled(k3, s["w"])
        elif s["kind"] == "moe":
            for m in "132":
                s["w" + m] = _tiled(k3, s["w" + m])
            size = L.k3d_moe_f8_ws(T, s["hidden"], s["inter"], s["experts"], s["topk"])
            s["work"] = new(max(1, size), dtype=torch.uint8)
    return s


# ------------------------------------------------------------------- calls ----
def _addr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own(s):
    k3 = _lib()
    L, T = k3.lib(), s["tokens"]
    if s["kind"] == "norm":
        n, nb, r, y = s["n"], _up(s["n"]), s["r"], s["yy"]
        k3.check(L.k3d_add_norm(
            _addr(y), 0 if s["both"] == "none" else CODE[s["both"]], n, s["q"].data_ptr(), nb * BLOCK, s["qs"].data_ptr(), nb,
            _addr(s["sum"]), n, s["xx"].data_ptr(), CODE[s["x"]], n, _addr(r), 0 if r is None else CODE[s["res"]], n, T, n,
            s["w"].data_ptr(), 1e-6, _stream()), "k3d_add_norm")
        return {"q": s["q"], "scale": s["qs"], "sum": s["sum"], "y": y}
    if s["kind"] == "quant":
        n, nb = s["n"], _up(s["n"])
        k3.check(L.k3d_quant_f8(
            s["q"].data_ptr(), nb * BLOCK, s["qs"].data_ptr(), nb, s["xx"].data_ptr(), CODE[s["x"]], s["xx"].shape[1], T, n,
            ("situ", "silu").index(s["act"]) if s["act"] != "none" else -1, B1, B2, _stream()), "k3d_quant_f8")
        return {"q": s["q"], "scale": s["qs"]}
    nb = s["s"].shape[1]
    x = (s["q"].data_ptr(), nb * BLOCK, s["s"].data_ptr(), nb)
    if s["kind"] == "linear":
        n = s["out"]
        k3.check(L.k3d_linear_f8(
            s["yy"].data_ptr(), CODE[s["y"]], n, *x, T, s["w"].data_ptr(), s["ws"].data_ptr(), nb, s["inn"], n, _addr(s["bias_"]),
            ACTS.index(s["act"]), _addr(s["r"]), n, s["work"].data_ptr(), s["work"].numel(), _stream()), "k3d_linear_f8")
    elif s["kind"] == "grouped":
        rows = T * s["topk"]
        k3.check(L.k3d_grouped_f8(
            s["yy"].data_ptr(), CODE[s["y"]], s["out"], None, rows, *x, s["perm"].data_ptr(), s["topk"], T, s["offsets"].data_ptr(),
            rows, s["experts"], s["w"].data_ptr(), s["ws"].data_ptr(), s["inn"], s["out"], _stream()), "k3d_grouped_f8")
    else:
        k3.check(L.k3d_moe_f8(
            s["yy"].data_ptr(), 1, s["hidden"], s["idx"].data_ptr(), s["wt"].data_ptr(), *x, T, s["w1"].data_ptr(),
            s["ws1"].data_ptr(), s["w3"].data_ptr(), s["ws3"].data_ptr(), s["w2"].data_ptr(), s["ws2"].data_ptr(), s["hidden"],
            s["inter"], s["experts"], s["topk"], ("situ", "silu").index(s["act"]), B1, B2, s["work"].data_ptr(),
            s["work"].numel(), _stream()), "k3d_moe_f8")
    return s["yy"]


def _quantise(u):
    """Codes and scales of fp32 rows, zeros behind a row's end."""
    T, n = u.shape
    nb = _up(n)
    v = torch.cat((u, u.new_zeros(T, nb * BLOCK - n)), 1).view(T, nb, BLOCK)
    s = torch.clamp(torch.amax(torch.abs(v), 2), min=LEAST) / 448
    return (v / s.unsqueeze(2)).to(F8).view(T, nb * BLOCK), s


def _values(q, s, n):
    """What codes and scales of rows stand for, n columns."""
    return (q.float().view(q.shape[0], -1, BLOCK) * s.unsqueeze(2)).flatten(1)[:, :n]


def _weights(q, s):
    """What weights' codes and block scales stand for."""
    out, inn = q.shape[-2:]
    s = s.repeat_interleave(BLOCK, -2)[..., :out, :].repeat_interleave(BLOCK, -1)[..., :inn]
    return q.float() * s


def _gated(g, u, act):
    if act == "silu":
        return g / (1 + torch.exp(-g)) * u
    return B1 * torch.tanh(g / B1) / (1 + torch.exp(-g)) * (B2 * torch.tanh(u / B2))


def _plain_norm(s):
    v = s["xx"].float()
    if s["r"] is not None:
        v = v + s["r"].float()
    u = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * s["w"]
    q, scale = _quantise(u)
    return {"q": q, "scale": scale, "sum": v.to(s["r"].dtype) if s["r"] is not None else None,
            "y": u.to(TYPES[s["both"]]) if s["both"] != "none" else None}


def _plain_quant(s):
    u = s["xx"].float()
    if s["act"] != "none":
        u = _gated(u[:, :s["n"]], u[:, s["n"]:], s["act"])
    q, scale = _quantise(u)
    return {"q": q, "scale": scale}


def _activate(v, act):
    if act == "relu":
        return torch.clamp(v, min=0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3)))
    return v


def _plain_linear(s):
    w = _weights(s["w"], s["ws"][0])
    v = _values(s["q"], s["s"], s["inn"]) @ w.T
    if s["bias_"] is not None:
        v = v + s["bias_"]
    v = _activate(v, s["act"])
    if s["r"] is not None:
        v = v + s["r"].float()
    return v.to(s["yy"].dtype)


def _place(s):
    """Each sorted row's expert, its place among the expert's rows, and its assignment."""
    perm = s["perm"].long()
    e = s["idx"].flatten().long()[perm]
    return e, torch.arange(perm.numel(), device="cuda") - s["offsets"].long()[e], perm


def _products(x, e, at, most, w, ws):
    """Row r of x times the weights of its expert: the experts' rows side by side, as one batch of products."""
    by = x.new_zeros(w.shape[0], most, x.shape[1])
    by[e, at] = x
    return torch.bmm(by, _weights(w, ws).transpose(1, 2).contiguous())[e, at]


def _plain_grouped(s):
    e, at, perm = _place(s)
    x = _values(s["q"], s["s"], s["inn"])[perm // s["topk"]]
    return _products(x, e, at, s["most"], s["w"], s["ws"]).to(s["yy"].dtype)


def _plain_moe(s):
    e, at, perm = _place(s)
    x = _values(s["q"], s["s"], s["hidden"])[perm // s["topk"]]
    g = _products(x, e, at, s["most"], s["w1"], s["ws1"])
    u = _products(x, e, at, s["most"], s["w3"], s["ws3"])
    h = _values(*_quantise(_gated(g, u, s["act"])), s["inter"])
    y = torch.empty(perm.numel(), s["hidden"], device="cuda")
    y[perm] = _products(h, e, at, s["most"], s["w2"], s["ws2"])
    return (y.view(s["tokens"], s["topk"], -1) * s["wt"].unsqueeze(2)).sum(1).to(BF16)


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear, "grouped": _plain_grouped,
            "moe": _plain_moe}[state["kind"]](state)


# ------------------------------------------------------ the same in 64 bits ----
def _exact_codes(u):
    """Codes (as the values that they round to) and scales, in 64 bits: a code is a multiple of 2^(e - 3), e its
    value's exponent and no less than -6."""
    T, n = u.shape
    nb = _up(n)
    v = torch.zeros(T, nb, BLOCK, dtype=torch.float64, device="cuda")
    v.view(T, -1)[:, :n] = u
    s = v.abs().amax(2).clamp(min=LEAST) / 448
    v = v / s[:, :, None]
    step = torch.exp2(torch.frexp(v)[1].clamp(min=-5).double() - 4)
    return (torch.round(v / step) * step).reshape(T, -1), s


def _exact_rows(q, s):
    return q.double() * s.double().repeat_interleave(BLOCK, 1)


def _exact_product(x, w, ws):
    """x [rows][whole blocks] times weights [out][in], a block of columns after another."""
    y = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    rows = torch.arange(w.shape[0], device="cuda") // BLOCK
    inn = w.shape[1]
    wide = 8 * BLOCK
    for k in range(0, inn, wide):
        b = w[:, k:k + wide].double()
        col = torch.arange(k, k + b.shape[1], device="cuda") // BLOCK
        b = b * ws.double()[rows][:, col]
        y += x[:, k:k + b.shape[1]] @ b.t()
    return y


def _exact_gated(g, u, act):
    a = g * torch.sigmoid(g) if act == "silu" else B1 * torch.tanh(g / B1) * torch.sigmoid(g)
    return a * (u if act == "silu" else B2 * torch.tanh(u / B2))


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "norm":
        v = d["xx"].double()
        if d["r"] is not None:
            v = v + d["r"].double()
        u = d["w"].double() * v * torch.rsqrt((v ** 2).sum(1, keepdim=True) / c["n"] + 1e-6)
        q, s = _exact_codes(u)
        return {"q": q, "scale": s, "sum": v if d["r"] is not None else None, "y": u if c["both"] != "none" else None}
    if c["kind"] == "quant":
        u, n = d["xx"].double(), c["n"]
        q, s = _exact_codes(u if c["act"] == "none" else _exact_gated(u[:, :n], u[:, n:], c["act"]))
        return {"q": q, "scale": s}
    x = _exact_rows(d["q"], d["s"])
    if c["kind"] == "linear":
        v = _exact_product(x, d["w"], d["ws"][0])
        if d["bias_"] is not None:
            v += d["bias_"].double()
        if c["act"] == "relu":
            v = torch.where(v > 0, v, torch.zeros_like(v))
        elif c["act"] == "silu":
            v = v * torch.sigmoid(v)
        elif c["act"] == "gelu":
            v = v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
        elif c["act"] == "gelu_tanh":       # (1 + tanh z) / 2 = sigmoid(2 z)
            v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * v * (1 + 0.044715 * v * v))
        return v if d["r"] is None else v + d["r"].double()
    off, perm, k = d["offsets"].tolist(), d["perm"].long(), c["topk"]
    y = torch.zeros(c["tokens"] * k, c["out"] if c["kind"] == "grouped" else c["hidden"], dtype=torch.float64, device="cuda")
    for e in range(c["experts"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        z = x[perm[a:b] // k]
        if c["kind"] == "grouped":
            y[a:b] = _exact_product(z, d["w"][e], d["ws"][e])
            continue
        h = _exact_gated(_exact_product(z, d["w1"][e], d["ws1"][e]), _exact_product(z, d["w3"][e], d["ws3"][e]), c["act"])
        y[perm[a:b]] = _exact_product(_exact_rows(*_exact_codes(h)), d["w2"][e], d["ws2"][e])
    if c["kind"] == "grouped":
        return y
    return torch.bmm(d["wt"].double()[:, None], y.view(c["tokens"], k, -1))[:, 0]


# ------------------------------------------------------------ what it takes ----
def _used(rows, experts):
    """Experts that a routing of so many rows meets, on average."""
    return experts * (1 - (1 - 1 / experts) ** rows)


def work(case):
    c, T = case, case["tokens"]
    size = {"f32": 4, "bf16": 2, "none": 0}
    if c["kind"] == "norm":
        n = T * c["n"]
        return {"bytes": n * (size[c["x"]] + 2 * size[c["res"]] + size[c["both"]] + 1) + 4 * T * _up(c["n"]) + 4 * c["n"],
                "flops": 6 * n}
    if c["kind"] == "quant":
        n = T * c["n"]
        return {"bytes": n * (size[c["x"]] * (1 if c["act"] == "none" else 2) + 1) + 4 * T * _up(c["n"]), "flops": 8 * n}
    if c["kind"] == "linear":
        b = T * c["inn"] + c["inn"] * c["out"] + T * c["out"] * size[c["y"]] * (2 if c["res"] else 1)
        return {"bytes": b, "flops": 2 * T * c["inn"] * c["out"]}
    rows = T * c["topk"]
    if c["kind"] == "grouped":
        return {"bytes": _used(rows, c["experts"]) * c["inn"] * c["out"] + T * c["inn"] + rows * c["out"] * size[c["y"]],
                "flops": 2 * rows * c["inn"] * c["out"]}
    return {"bytes": 3 * _used(rows, c["experts"]) * c["hidden"] * c["inter"] + T * c["hidden"] * 3,
            "flops": 6 * rows * c["hidden"] * c["inter"]}
