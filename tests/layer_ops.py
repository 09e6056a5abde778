# SPDX-License-Identifier: Apache-2.0
"""64-bit restatements of the operators around the routed experts (k3d_linear, k3d_route,
k3d_qk_norm_rope), and their calls on torch tensors."""
import math

import numpy as np
import torch

F32, BF16 = torch.float32, torch.bfloat16
TYPE = {F32: 0, BF16: 1}
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}              # half a step, relative to the value
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def addr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------- linear ----
def linear(k3, x, w, bias=None, act="none", res=None, y=None, y_type=None, st=None, ws=None):
    """k3d_linear on 2-d views (their row strides)."""
    L, (T, inn), out = k3.lib(), x.shape, w.shape[0]
    y_type = y_type or (res.dtype if res is not None else F32)
    y = torch.empty(T, out, device="cuda", dtype=y_type) if y is None else y
    assert res is None or res.dtype == y.dtype
    need = L.k3d_linear_ws(T, inn, out, TYPE[x.dtype])
    ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8) if ws is None else ws
    k3.check(L.k3d_linear(addr(y), TYPE[y.dtype], y.stride(0), addr(x), TYPE[x.dtype], x.stride(0), T, addr(w), w.stride(0),
                          inn, out, addr(bias), ACTS.index(act), addr(res), res.stride(0) if res is not None else 0, addr(ws),
                          ws.numel(), stream() if st is None else st), "k3d_linear")
    return y


def act64(v, act):
    if act == "relu":
        return np.maximum(v, 0.0)
    if act == "silu":
        return v / (1.0 + np.exp(-v))
    if act == "gelu":
        return v * 0.5 * np.array([math.erfc(-a / math.sqrt(2.0)) for a in v.ravel()]).reshape(v.shape)
    if act == "gelu_tanh":
        return v / (1.0 + np.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))    # (1 + tanh z) / 2 without its cancellation
    return v


def f64(t):
    return t.detach().double().cpu().numpy()


def linear64(x, w, bias, act, res, y_type):
    """The result in 64 bits and how far off a kernel may be: `inn` fp32 additions of products, each off
    by at most a unit in the last place (2^-23) of a sum no larger than S = sum |x| |w| + |bias|,
    through an activation of slope at most 1.13; the activation's and the additions' own roundings,
    within 4 units of their values; half a step of y's type."""
    X, W = f64(x), f64(w)
    v, S = X @ W.T, np.abs(X) @ np.abs(W).T
    if bias is not None:
        b = f64(bias)
        v, S = v + b, S + np.abs(b)
    a = act64(v, act)
    y, r = a, 0.0
    if res is not None:
        r = f64(res)
        y = a + r
    tol = 1.13 * 2.0 ** -23 * (x.shape[1] + 1) * S + 2.0 ** -21 * (np.abs(v) + np.abs(a) + np.abs(r))
    return y, tol + (np.abs(y) + tol) * HALF[y_type]


# -------------------------------------------------------------------- route ----
def route(k3, logits, bias=None, score=0, groups=1, top_groups=1, group_top=1, topk=8, renorm=1, scale=1.0, st=None,
          idx=None, wt=None):
    L, (T, n) = k3.lib(), logits.shape
    idx = torch.empty(T, topk, device="cuda", dtype=torch.int32) if idx is None else idx
    wt = torch.empty(T, topk, device="cuda", dtype=F32) if wt is None else wt
    k3.check(L.k3d_route(addr(idx), addr(wt), addr(logits), TYPE[logits.dtype], logits.stride(0), T, n, addr(bias), score,
                         groups, top_groups, group_top, topk, renorm, scale, stream() if st is None else st), "k3d_route")
    return idx, wt


def route64(logits, bias, score, groups, top_groups, group_top, topk, renorm, scale):
    lg = f64(logits)
    T, n = lg.shape
    idx = np.full((T, topk), -1, np.int32)
    wt = np.zeros((T, topk))
    b = np.zeros(n) if bias is None else f64(bias)
    with np.errstate(all="ignore"):
        for t in range(T):
            l = lg[t]
            there = l > -np.inf                                    # (False for NaN)
            s = np.zeros(n)
            if score == 0:
                s[there] = 1.0 / (1.0 + np.exp(-l[there]))
            elif there.any():
                m = l[there].max()
                e = np.zeros(n)
                e[there] = np.where(l[there] == m, 1.0, np.exp(l[there] - m))
                s = e / e.sum()
            c = np.where(there, s + b, -np.inf)
            c[~(c > -np.inf)] = -np.inf
            if top_groups < groups:
                gs = n // groups
                val = np.full(groups, -np.inf)
                for g in range(groups):
                    best = np.sort(c[g * gs:(g + 1) * gs])[::-1]
                    best = best[best > -np.inf][:group_top]
                    if len(best):
                        val[g] = best.sum()
                order = np.argsort(-val, kind="stable")[:top_groups]
                keep = np.zeros(groups, bool)
                keep[order] = True
                c[~np.repeat(keep, gs)] = -np.inf
            order = np.argsort(-c, kind="stable")[:topk]
            order = order[c[order] > -np.inf]
            idx[t, :len(order)] = order
            w = s[order]
            if renorm and topk > 1:
                w = w / w.sum() if w.sum() > 0 else w * 0
            wt[t, :len(order)] = w * np.float64(np.float32(scale))
    return idx, wt


def check_route(got, want):
    idx, wt = got
    assert np.array_equal(idx.cpu().numpy(), want[0])
    w = f64(wt)
    # one rounding to fp32, behind fp64 arithmetic
    assert (np.abs(w - want[1]) <= 2.0 ** -24 * 1.0001 * np.abs(want[1]) + 2.0 ** -149).all()


# -------------------------------------------------------------------- heads ----
def heads(k3, q, k, qw, kw, pos, freq, rot, off=0, pairs=0, eps=1e-6, scale=1.0, qo=None, ko=None, st=None):
    """k3d_qk_norm_rope on views [T][heads][dim] (their strides)."""
    T, hq, dim = q.shape
    qo = torch.empty(T, hq, dim, device="cuda", dtype=q.dtype) if qo is None else qo
    ko = torch.empty(T, k.shape[1], dim, device="cuda", dtype=k.dtype) if ko is None else ko
    k3.check(k3.lib().k3d_qk_norm_rope(
        addr(qo), qo.stride(0), qo.stride(1), addr(ko), ko.stride(0), ko.stride(1), addr(q), q.stride(0), q.stride(1),
        addr(k), k.stride(0), k.stride(1), TYPE[q.dtype], T, hq, k.shape[1], dim, addr(qw), addr(kw), eps, addr(pos),
        addr(freq), rot, off, pairs, scale, stream() if st is None else st), "k3d_qk_norm_rope")
    return qo, ko


def heads64(v, w, pos, freq, rot, off, pairs, eps, scale):
    """The result in 64 bits and how far off: the mean of dim squares and the products up to the rotation in
    fp32 (dim + 12 roundings, one more for each of a pair's two terms), half a step of the type."""
    x = f64(v)
    dim = x.shape[-1]
    with np.errstate(all="ignore"):
        u = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if w is not None:
            u = u * f64(w)
        y, mag = u.copy(), np.abs(u)
        if rot:
            h = rot // 2
            a = f64(pos)[:, None] * f64(freq)[None]
            sc = np.float64(np.float32(scale))
            c, s = (sc * np.cos(a))[:, None], (sc * np.sin(a))[:, None]
            i = np.arange(h)
            one, two = (off + i, off + h + i) if pairs == 0 else (off + 2 * i, off + 2 * i + 1)
            p, q = u[..., one], u[..., two]
            y[..., one], y[..., two] = p * c - q * s, q * c + p * s
            mag[..., one] = mag[..., two] = abs(sc) * (np.abs(p) + np.abs(q))
    tol = (dim + 16) * 2.0 ** -24 * mag
    return y, tol + (np.abs(y) + tol) * HALF[v.dtype]


def within(got, want):
    y, tol = want
    d = np.abs(f64(got) - y)
    assert (d <= tol + 2.0 ** -133).all(), float((d / np.maximum(tol, 1e-300)).max())
