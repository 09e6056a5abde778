# SPDX-License-Identifier: Apache-2.0
"""The operators around the routed experts, as measurable cases.

Three kinds, each one call through the public device entry points:

  linear   y = act(x W^T + bias) + residual (k3d_linear): bf16 weights, x bf16 or fp32, y bf16 or
           fp32; the projections of a layer, and the logits of its router
  route    logits -> experts and weights (k3d_route): sigmoid or softmax scores, a selection bias,
           groups, top-k, renormalised weights
  qknorm   RMSNorm of every query and key head with the position rotation behind it
           (k3d_qk_norm_rope), out of the rows that a fused q/k/v projection wrote

Values: activations and residuals ~ N(0, 1), weights ~ N(0, 1/in), biases ~ N(0, 0.1), router
logits ~ N(0, 1.5), selection biases ~ N(0, 0.05), head rows ~ N(0, 1), norm weights ~ N(1, 0.1),
rotation frequencies base^(-2i/rot), positions of a batch of sequences.
"""
import math
import os
import sys

import torch

own = False         # False: the plain forms below; True: the library's entry points

ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _linear(tokens, inn, out, x, y, bias, act, res):
    return dict(kind="linear", tokens=tokens, inn=inn, out=out, x=x, y=y, bias=bias, act=act, res=res)


def _route(tokens, experts, topk, score, bias, groups=1, top_groups=1, group_top=1, dtype="f32", renorm=True, scale=1.0):
    return dict(kind="route", tokens=tokens, experts=experts, topk=topk, score=score, bias=bias, groups=groups,
                top_groups=top_groups, group_top=group_top, dtype=dtype, renorm=renorm, scale=scale)


def _qknorm(tokens, hq, hk, dim, rot, off, pairs, dtype, far):
    return dict(kind="qknorm", tokens=tokens, hq=hq, hk=hk, dim=dim, rot=rot, off=off, pairs=pairs, dtype=dtype, far=far)


def listed():
    return [
        # the fused projection of one decoded token: the weights' bytes are all there is
        dict(_linear(1, 7168, 12288, "bf16", "bf16", True, "none", False), name="linear_decode_1"),
        # the projection back onto the residual stream for a ragged decode batch
        dict(_linear(37, 12288, 7168, "bf16", "f32", False, "none", True), name="linear_decode_37_residual"),
        # the logits of a small prompt's router: few rows, fp32 activations kept whole
        dict(_linear(300, 7168, 384, "f32", "f32", False, "none", False), name="linear_logits_300"),
        # rows at any alignment, no size a multiple of a tile
        dict(_linear(333, 1001, 2047, "bf16", "bf16", True, "gelu", True), name="linear_ragged_333"),
        # a long prompt through a wide projection: the matrix units' rate
        dict(_linear(4096, 7168, 12288, "bf16", "bf16", True, "silu", False), name="linear_prompt_4096"),
        # one token over grouped experts: launch latency
        dict(_route(1, 384, 8, "sigmoid", True, 8, 4, 2, scale=2.5), name="route_1_grouped"),
        # a decode batch with softmax scores, no groups
        dict(_route(64, 128, 8, "softmax", False), name="route_64_softmax"),
        # an odd number of experts, logits in bf16: equal ones occur
        dict(_route(777, 823, 6, "softmax", True, dtype="bf16", renorm=False), name="route_777_bf16"),
        # a long prompt over the large expert count
        dict(_route(8192, 896, 16, "sigmoid", True, 8, 4, 2), name="route_8192_grouped"),
        # one decoded token at a far position
        dict(_qknorm(1, 64, 8, 128, 128, 0, "halves", "bf16", True), name="qknorm_1"),
        # heads with an unrotated part in front, pairs side by side, one shared key head, fp32
        dict(_qknorm(777, 12, 1, 192, 64, 128, "interleaved", "f32", False), name="qknorm_777_partial"),
        # a long prompt
        dict(_qknorm(4096, 64, 8, 128, 128, 0, "halves", "bf16", False), name="qknorm_4096"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("linear",) * 5 + ("route",) * 4 + ("qknorm",) * 3)
    if kind == "linear":
        step = rng.choice((64, 64, 64, 8, 1))
        inn = max(step, _log(rng, 256, 12288) // step * step)
        step = rng.choice((32, 32, 1))
        out = _log(rng, 64, 16384) // step * step
        x = rng.choice(("bf16", "bf16", "bf16", "f32"))
        most = 4096 * 7168 * 12288 // (1 if x == "bf16" else 4)
        return _linear(min(_log(rng, 1, 4096), max(1, most // (inn * out))), inn, out, x, rng.choice(("bf16", "f32")),
                       rng.random() < 0.5, rng.choice(ACTS), rng.random() < 0.5)
    if kind == "route":
        e, k, g = rng.choice(((384, 8, 8), (896, 16, 8), (256, 8, 8), (128, 8, 1), (64, 6, 1), (160, 6, 8), (0, 0, 0)))
        if e == 0:
            g = rng.choice((1, 1, rng.randint(2, 16)))
            e = g * max(1, _log(rng, 16, 1500) // g)
            k = rng.randint(1, min(24, e))
        elif rng.random() < 0.3:
            g = 1
        least = -(-k // (e // g))                       # groups that hold topk experts
        tg = g if g == 1 else rng.randint(least, g)
        return _route(_log(rng, 1, 8192), e, k, rng.choice(("sigmoid", "softmax")), rng.random() < 0.6, g, tg,
                      rng.choice((1, 2)) if e // g > 1 else 1, rng.choice(("f32", "f32", "bf16")), rng.random() < 0.75,
                      rng.choice((1.0, 2.5, 16.0)))
    dim = rng.choice((64, 128, 128, 128, 192, 256, 2 * rng.randint(16, 160)))
    rot = rng.choice((dim, dim, 2 * rng.randint(1, dim // 2), dim // 4 * 2))
    hq, hk = rng.choice(((64, 8), (96, 96), (32, 4), (12, 1), (rng.randint(1, 64), rng.randint(1, 16))))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    most = 4096 * 72 * 128 * 2 // ((hq + hk) * dim * (2 if dtype == "bf16" else 4))
    return _qknorm(min(_log(rng, 1, 8192), max(1, most)), hq, hk, dim, rot, rng.choice((0, dim - rot)),
                   rng.choice(("halves", "halves", "interleaved")), dtype, rng.random() < 0.3)


# ------------------------------------------------------------------ inputs ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, sigma=1.0, mean=0.0, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).mul_(sigma).add_(mean).to(dtype)


def _inputs(c, seed):
    g, T = _gen(seed), c["tokens"]
    if c["kind"] == "linear":
        d = {"x": _normal(g, T, c["inn"], dtype=TYPES[c["x"]]),
             "w": _normal(g, c["out"], c["inn"], sigma=c["inn"] ** -0.5, dtype=torch.bfloat16)}
        d["bias"] = _normal(g, c["out"], sigma=0.1) if c["bias"] else None
        d["res"] = _normal(g, T, c["out"], dtype=TYPES[c["y"]]) if c["res"] else None
        return d
    if c["kind"] == "route":
        return {"logits": _normal(g, T, c["experts"], sigma=1.5, dtype=TYPES[c["dtype"]]),
                "bias": _normal(g, c["experts"], sigma=0.05) if c["bias"] else None}
    hq, hk, dim = c["hq"], c["hk"], c["dim"]
    d = {"qkv": _normal(g, T, (hq + 2 * hk) * dim, dtype=TYPES[c["dtype"]]),
         "qw": _normal(g, dim, sigma=0.1, mean=1.0), "kw": _normal(g, dim, sigma=0.1, mean=1.0)}
    # a batch of sequences one after another, each at positions of its own
    n = int(torch.randint(1, 9, (1,), device="cuda", generator=g))
    start = torch.randint(0, 1000000 if c["far"] else 4096, (n,), device="cuda", generator=g)
    t = torch.arange(T, device="cuda")
    per = -(-T // n)
    d["pos"] = (start[t // per] + t % per).to(torch.int32)
    i = torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64)
    d["freq"] = torch.pow(torch.tensor(1e6, device="cuda", dtype=torch.float64), -2.0 * i / c["rot"])
    return d


def _lib():
    path = os.path.join(os.getcwd(), "kimi-k3-in-c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import k3amd
    return k3amd


def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    T = s["tokens"]
    if s["kind"] == "linear":
        s["y_out"] = torch.empty(T, s["out"], device="cuda", dtype=TYPES[s["y"]])
    elif s["kind"] == "route":
        s["idx"] = torch.empty(T, s["topk"], device="cuda", dtype=torch.int32)
        s["wt"] = torch.empty(T, s["topk"], device="cuda", dtype=torch.float32)
    else:
        s["q_out"] = torch.empty(T, s["hq"], s["dim"], device="cuda", dtype=TYPES[s["dtype"]])
        s["k_out"] = torch.empty(T, s["hk"], s["dim"], device="cuda", dtype=TYPES[s["dtype"]])
    if own:
        k3 = _lib()
        k3.check(k3.lib().k3d_init(), "k3d_init")
        if s["kind"] == "linear":
            size = k3.lib().k3d_linear_ws(T, s["inn"], s["out"], 1 if s["x"] == "bf16" else 0)
            s["ws"] = torch.empty(max(1, size), device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------------- calls ----
def _addr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own(s):
    k3 = _lib()
    L, T = k3.lib(), s["tokens"]
    if s["kind"] == "linear":
        y, n = s["y_out"], s["out"]
        k3.check(L.k3d_linear(
            y.data_ptr(), 1 if s["y"] == "bf16" else 0, n, s["x"].data_ptr(), 1 if s["x"].dtype == torch.bfloat16 else 0,
            s["inn"], T, s["w"].data_ptr(), s["inn"], s["inn"], n, _addr(s["bias"]), ACTS.index(s["act"]), _addr(s["res"]),
            n, s["ws"].data_ptr(), s["ws"].numel(), _stream()), "k3d_linear")
        return y
    if s["kind"] == "route":
        k3.check(L.k3d_route(
            s["idx"].data_ptr(), s["wt"].data_ptr(), s["logits"].data_ptr(), 1 if s["dtype"] == "bf16" else 0, s["experts"],
            T, s["experts"], _addr(s["bias"]), 0 if s["score"] == "sigmoid" else 1, s["groups"], s["top_groups"],
            s["group_top"], s["topk"], int(s["renorm"]), s["scale"], _stream()), "k3d_route")
        return {"idx": s["idx"], "wt": s["wt"]}
    hq, hk, dim, row = s["hq"], s["hk"], s["dim"], (s["hq"] + 2 * s["hk"]) * s["dim"]
    q = s["qkv"].data_ptr()
    k = q + hq * dim * s["qkv"].element_size()
    k3.check(L.k3d_qk_norm_rope(
        s["q_out"].data_ptr(), hq * dim, dim, s["k_out"].data_ptr(), hk * dim, dim, q, row, dim, k, row, dim,
        1 if s["dtype"] == "bf16" else 0, T, hq, hk, dim, s["qw"].data_ptr(), s["kw"].data_ptr(), 1e-6, s["pos"].data_ptr(),
        s["freq"].data_ptr(), s["rot"], s["off"], 0 if s["pairs"] == "halves" else 1, 1.0, _stream()), "k3d_qk_norm_rope")
    return {"q": s["q_out"], "k": s["k_out"]}


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
    v = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        v = v + s["bias"]
    v = _activate(v, s["act"])
    if s["res"] is not None:
        v = v + s["res"].float()
    return v.to(s["y_out"].dtype)


def _plain_route(s):
    # scores next to each other decide: 64 bits
    lg = s["logits"].double()
    if s["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-lg))
    else:
        e = torch.exp(lg - lg.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    pick = score if s["bias"] is None else score + s["bias"].double()
    if s["top_groups"] < s["groups"]:
        by = pick.view(pick.shape[0], s["groups"], -1)
        best = torch.sort(by, dim=2, descending=True).values[:, :, :s["group_top"]].sum(2)
        order = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        pick = torch.where(keep.unsqueeze(2), by, -math.inf).view(pick.shape)
    idx = torch.sort(pick, dim=1, descending=True, stable=True).indices[:, :s["topk"]]
    wt = torch.gather(score, 1, idx)
    if s["renorm"] and s["topk"] > 1:
        wt = wt / wt.sum(1, keepdim=True)
    return {"idx": idx.to(torch.int32), "wt": (wt * s["scale"]).float()}


def _plain_heads(v, w, s):
    u = v.float()
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + 1e-6) * w
    ang = s["pos"].double().unsqueeze(1) * s["freq"]            # far positions: 64 bits
    cos, sin = torch.cos(ang).float().unsqueeze(1), torch.sin(ang).float().unsqueeze(1)
    o, h = s["off"], s["rot"] // 2
    r = u[..., o:o + s["rot"]]
    a, b = (r[..., :h], r[..., h:]) if s["pairs"] == "halves" else (r[..., 0::2], r[..., 1::2])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.cat((a, b), -1) if s["pairs"] == "halves" else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((u[..., :o], r, u[..., o + s["rot"]:]), -1).to(v.dtype)


def _plain_qknorm(s):
    T, hq, hk, dim = s["tokens"], s["hq"], s["hk"], s["dim"]
    q = s["qkv"][:, :hq * dim].view(T, hq, dim)
    k = s["qkv"][:, hq * dim:(hq + hk) * dim].view(T, hk, dim)
    return {"q": _plain_heads(q, s["qw"], s), "k": _plain_heads(k, s["kw"], s)}


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "route": _plain_route, "qknorm": _plain_qknorm}[state["kind"]](state)


# ------------------------------------------------------ the same in 64 bits ----
def _exact_linear(c, d):
    T, out = c["tokens"], c["out"]
    y = torch.empty(T, out, dtype=torch.float64, device="cuda")
    x = d["x"].double()
    for o in range(0, out, 1024):
        v = torch.matmul(x, d["w"][o:o + 1024].double().t())
        if d["bias"] is not None:
            v += d["bias"][o:o + 1024].double()
        if c["act"] == "relu":
            v = torch.where(v > 0, v, torch.zeros_like(v))
        elif c["act"] == "silu":
            v = v * torch.sigmoid(v)
        elif c["act"] == "gelu":
            v = v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
        elif c["act"] == "gelu_tanh":       # (1 + tanh z) / 2 = sigmoid(2 z)
            v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * v * (1 + 0.044715 * v * v))
        if d["res"] is not None:
            v += d["res"][:, o:o + 1024].double()
        y[:, o:o + 1024] = v
    return y


def _exact_route(c, d):
    lg = d["logits"].double()
    score = torch.sigmoid(lg) if c["score"] == "sigmoid" else torch.softmax(lg, 1)
    pick = score.clone()
    if d["bias"] is not None:
        pick += d["bias"].double()
    T, n, g = c["tokens"], c["experts"], c["groups"]
    if c["top_groups"] < g:
        by = pick.view(T, g, n // g)
        value = by.amax(2)
        if c["group_top"] == 2:
            first = by.argmax(2, keepdim=True)
            value = value + by.scatter(2, first, -math.inf).amax(2)
        for _ in range(g - c["top_groups"]):            # drop the least, the later one of equals
            least = g - 1 - value.flip(1).argmin(1)
            value[torch.arange(T, device="cuda"), least] = math.inf
        pick = torch.where((value == math.inf).unsqueeze(2), -math.inf, by).reshape(T, n)
    idx = torch.empty(T, c["topk"], dtype=torch.int64, device="cuda")
    place = torch.arange(n, device="cuda")
    for j in range(c["topk"]):                          # the largest left, the first of equals
        top = pick.amax(1, keepdim=True)
        idx[:, j] = torch.where(pick == top, place, n).amin(1)
        pick.scatter_(1, idx[:, j:j + 1], -math.inf)
    wt = torch.gather(score, 1, idx) * c["scale"]
    if c["renorm"] and c["topk"] > 1:
        wt = wt * (c["scale"] / wt.sum(1, keepdim=True))
    return {"idx": idx.to(torch.int32), "wt": wt}


def _exact_heads(v, w, c, d):
    u = v.double()
    u = w.double() * u / torch.sqrt((u ** 2).sum(-1, keepdim=True) / c["dim"] + 1e-6)
    h, o = c["rot"] // 2, c["off"]
    i = torch.arange(h, device="cuda")
    first, second = (o + i, o + h + i) if c["pairs"] == "halves" else (o + 2 * i, o + 2 * i + 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), d["pos"].double()[:, None] * d["freq"][None])
    z = torch.complex(u[..., first], u[..., second]) * turn[:, None]
    u[..., first], u[..., second] = z.real, z.imag
    return u


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "linear":
        return _exact_linear(c, d)
    if c["kind"] == "route":
        return _exact_route(c, d)
    rows = d["qkv"].view(c["tokens"], -1, c["dim"])
    return {"q": _exact_heads(rows[:, :c["hq"]], d["qw"], c, d),
            "k": _exact_heads(rows[:, c["hq"]:c["hq"] + c["hk"]], d["kw"], c, d)}


# ------------------------------------------------------------ what it takes ----
def work(case):
    c, T = case, case["tokens"]
    size = {"f32": 4, "bf16": 2}
    if c["kind"] == "linear":
        b = T * c["inn"] * size[c["x"]] + 2 * c["inn"] * c["out"] + T * c["out"] * size[c["y"]] * (2 if c["res"] else 1)
        return {"bytes": b + (4 * c["out"] if c["bias"] else 0), "flops": 2 * T * c["inn"] * c["out"]}
    if c["kind"] == "route":
        n = c["experts"]
        return {"bytes": T * n * size[c["dtype"]] + (4 * n if c["bias"] else 0) + 8 * T * c["topk"], "flops": 5 * T * n}
    n = T * (c["hq"] + c["hk"]) * c["dim"]
    return {"bytes": 2 * n * size[c["dtype"]] + 4 * T + 8 * c["dim"] + 4 * c["rot"], "flops": 6 * n}
