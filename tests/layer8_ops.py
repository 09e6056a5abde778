# SPDX-License-Identifier: Apache-2.0
"""64-bit restatements of a layer's 8-bit path (k3d_add_norm, k3d_quant_f8, k3d_linear_f8, k3d_group, k3d_grouped_f8,
k3d_moe_f8), and their calls on torch tensors."""
import numpy as np
import torch

from layer_ops import ACTS, BF16, F32, HALF, TYPE, act64, addr, f64, stream

F8 = torch.float8_e4m3fn
LEAST = 2.0 ** -100
NONE, SITU, SILU = -1, 0, 1


def nb(n):
    return -(-n // 128)


def rows_for(T, n, ldq=None, lds=None):
    """Uninitialised codes [T][ldq] and scales [T][lds], every byte a NaN."""
    q = torch.full((T, ldq or nb(n) * 128), 0x7f, device="cuda", dtype=torch.uint8)
    return q, torch.full((T, lds or nb(n)), float("nan"), device="cuda")


# -------------------------------------------------------------------- rows ----
def add_norm(k3, x, res=None, w=None, eps=1e-6, y=None, q=None, qs=None, sum_=None, r_type=None, n=None, st=None):
    T, n = x.shape[0], n or x.shape[1]
    r_type = res.dtype if res is not None else sum_.dtype if sum_ is not None else r_type or F32
    ld = lambda t: 0 if t is None else t.stride(0)      # noqa: E731
    k3.check(k3.lib().k3d_add_norm(
        addr(y), TYPE[y.dtype] if y is not None else 0, ld(y), addr(q), ld(q), addr(qs), ld(qs), addr(sum_), ld(sum_), addr(x),
        TYPE[x.dtype], ld(x), addr(res), TYPE[r_type], ld(res), T, n, addr(w), eps, stream() if st is None else st), "k3d_add_norm")


def norm64(x, res, w, eps):
    """v, u, and how far off u in fp32: the sum of n squares (n + 2 roundings, halved by the root), the root, the quotient, three
    products, v itself."""
    v = f64(x)
    mag = np.abs(v)
    if res is not None:
        r = f64(res)
        mag = mag + np.abs(r)
        v = v + r
    n = v.shape[1]
    with np.errstate(all="ignore"):
        rms = np.sqrt((v * v).mean(1, keepdims=True) + np.float64(np.float32(eps)))
        W = 1.0 if w is None else f64(w)
        u = v / rms * W
        # an element's own rounding is relative to it (a sum of two fp32 values: half a unit of itself)
        tol = (n / 2 + 16) * 2.0 ** -24 * np.abs(u)
    return v, u, tol


def quant(k3, x, n=None, act=NONE, b1=4.0, b2=25.0, q=None, qs=None, st=None):
    T = x.shape[0]
    n = n or (x.shape[1] if act == NONE else x.shape[1] // 2)
    if q is None:
        q, qs = rows_for(T, n)
    k3.check(k3.lib().k3d_quant_f8(addr(q), q.stride(0), addr(qs), qs.stride(0), addr(x), TYPE[x.dtype], x.stride(0), T, n, act, b1,
                                   b2, stream() if st is None else st), "k3d_quant_f8")
    return q, qs


def glu64(g, u, act, b1, b2):
    with np.errstate(all="ignore"):
        sg = np.where(g >= 0, 1.0 / (1.0 + np.exp(-np.abs(g))), np.exp(-np.abs(g)) / (1.0 + np.exp(-np.abs(g))))
        if act == SILU:
            return g * sg * u
        b1, b2 = np.float64(np.float32(b1)), np.float64(np.float32(b2))
        return b1 * np.tanh(g / b1) * sg * (b2 * np.tanh(u / b2))


def codes_of(q):
    return f64(q.view(F8).float())


def check_codes(q, qs, u, tol, n):
    """Codes and scales of rows that are u within tol (64 bits): the scale is the largest |u| / 448 within its own
    roundings, each code within half a step of u / scale (2^-4 of the value, 2^-10 below 2^-6), zeros behind n."""
    T = u.shape[0]
    blocks = nb(n)
    pad = np.zeros((T, blocks * 128))
    pad[:, :n] = u
    ptol = np.zeros_like(pad)
    ptol[:, :n] = tol
    pad, ptol = pad.reshape(T, blocks, 128), ptol.reshape(T, blocks, 128)
    s = f64(qs[:, :blocks])
    amax, at = np.abs(pad).max(2), ptol.max(2)
    want = np.maximum(amax, LEAST) / 448
    assert (np.abs(s - want) <= want * 2.0 ** -22 + at / 448).all()
    c = codes_of(q[:, :blocks * 128]).reshape(T, blocks, 128)
    v = pad / s[:, :, None]
    half = np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10)
    off = np.abs(c - v)
    slack = ptol / s[:, :, None] + np.abs(v) * 2.0 ** -21
    assert (off <= half + slack).all(), float((off - half - slack).max())
    assert (c.reshape(T, -1)[:, n:] == 0).all()


# ---------------------------------------------------------------- products ----
def weights(g, mats, out, inn, integers=False):
    """Codes [mats][out][in] (as uint8) and scales [mats][out blocks][in blocks]."""
    if integers:
        q = torch.randint(-3, 4, (mats, out, inn), device="cuda", generator=g).to(F32).to(F8)
        s = torch.pow(2.0, torch.randint(-2, 3, (mats, nb(out), nb(inn)), device="cuda", generator=g).to(F32))
        return q.view(torch.uint8), s
    q = (torch.randn(mats, out, inn, device="cuda", generator=g) * 100).clamp(-448, 448).to(F8)
    return q.view(torch.uint8), torch.rand(mats, nb(out), nb(inn), device="cuda", generator=g) * 1e-3 + 1e-4


def acts(g, T, inn, integers=False, ldq=None, lds=None):
    q, s = rows_for(T, inn, ldq, lds)
    q[:, :nb(inn) * 128] = 0
    if integers:
        q[:, :inn] = torch.randint(-3, 4, (T, inn), device="cuda", generator=g).to(F32).to(F8).view(torch.uint8)
        s[:, :nb(inn)] = torch.pow(2.0, torch.randint(-2, 3, (T, nb(inn)), device="cuda", generator=g).to(F32))
    else:
        q[:, :inn] = (torch.randn(T, inn, device="cuda", generator=g) * 100).clamp(-448, 448).to(F8).view(torch.uint8)
        s[:, :nb(inn)] = torch.rand(T, nb(inn), device="cuda", generator=g) * 0.02 + 1e-3
    return q, s


def tile(k3, q, ldw=None, st=None):
    mats, out, inn = q.shape
    size = k3.lib().k3d_f8_tiled_bytes(out, inn)
    t = torch.full((mats * size,), 0x7f, device="cuda", dtype=torch.uint8)
    k3.check(k3.lib().k3d_f8_tile(addr(t), addr(q), ldw or inn, out, inn, mats, stream() if st is None else st), "k3d_f8_tile")
    return t


def rows64(q, s, n):
    return codes_of(q)[:, :n] * np.repeat(f64(s), 128, 1)[:, :n]


def weights64(q, s):
    out, inn = q.shape
    return codes_of(q) * np.repeat(np.repeat(f64(s), 128, 0)[:out], 128, 1)[:, :inn]


def linear8(k3, x, xs, wt, ws, inn, out, bias=None, act="none", res=None, y=None, y_type=F32, st=None, ws_=None):
    L, T = k3.lib(), x.shape[0]
    y = torch.empty(T, out, device="cuda", dtype=res.dtype if res is not None else y_type) if y is None else y
    need = L.k3d_linear_f8_ws(T, inn, out)
    ws_ = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8) if ws_ is None else ws_
    k3.check(L.k3d_linear_f8(addr(y), TYPE[y.dtype], y.stride(0), addr(x), x.stride(0), addr(xs), xs.stride(0), T, addr(wt), addr(ws),
                             ws.stride(-2), inn, out, addr(bias), ACTS.index(act), addr(res), res.stride(0) if res is not None else 0,
                             addr(ws_), ws_.numel(), stream() if st is None else st), "k3d_linear_f8")
    return y


def largest8(X, W):
    """sum over each 8 columns of the largest |x| |w| among them"""
    n = X.shape[1]
    x = torch.zeros(X.shape[0], -(-n // 8) * 8, device="cuda")
    w = torch.zeros(W.shape[0], x.shape[1], device="cuda")
    x[:, :n], w[:, :n] = torch.from_numpy(np.abs(X)).cuda(), torch.from_numpy(np.abs(W)).cuda()
    s = torch.zeros(X.shape[0], W.shape[0], device="cuda")
    for k in range(0, x.shape[1], 8):
        m = torch.zeros_like(s)
        for i in range(k, k + 8):
            m = torch.maximum(m, x[:, i, None] * w[None, :, i])
        s += m
    return s.double().cpu().numpy() * (1 + 2.0 ** -12)


def product64(X, W, eight=False):
    """X W^T and how far off in fp32: `in` additions and the scales' products, each off by at most a unit in the last
    place (2^-23) of a sum no larger than S = sum |x| |w|. In 8-bit instructions (eight) each 8 products are aligned to the largest's
    exponent e and cut off 13 bits below it: each loses under 2^(e - 13), which is at most 2^-13 of the largest of them, so the
    8 lose under 2^-10 of it."""
    S = np.abs(X) @ np.abs(W).T
    tol = 2.0 ** -23 * (X.shape[1] + 8) * S
    return X @ W.T, tol + 2.0 ** -10 * largest8(X, W) if eight else tol


def linear8_64(X, W, bias, act, res, y_type):
    v, tol = product64(X, W, y_type == BF16)
    if bias is not None:
        b = f64(bias)
        v, tol = v + b, tol + 2.0 ** -23 * np.abs(b)
    a = act64(v, act)
    r = f64(res) if res is not None else 0.0
    y = a + r
    tol = 1.13 * tol + 2.0 ** -21 * (np.abs(v) + np.abs(a) + np.abs(r))
    return y, tol + (np.abs(y) + tol) * HALF[y_type]


def group(k3, idx, experts, st=None, offsets=None, perm=None):
    L, (T, k) = k3.lib(), idx.shape
    offsets = torch.full((experts + 1,), -7, device="cuda", dtype=torch.int32) if offsets is None else offsets
    perm = torch.full((T * k,), -7, device="cuda", dtype=torch.int32) if perm is None else perm
    need = L.k3d_group_ws(T, k, experts)
    ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
    k3.check(L.k3d_group(addr(offsets), addr(perm), addr(idx), T, k, experts, addr(ws), need, stream() if st is None else st), "k3d_group")
    return offsets, perm


def group64(idx, experts):
    flat = idx.cpu().numpy().reshape(-1)
    there = (flat >= 0) & (flat < experts)
    order = np.argsort(np.where(there, flat, experts), kind="stable")[:there.sum()]
    return np.concatenate(([0], np.cumsum(np.bincount(flat[there], minlength=experts)))), order


def grouped(k3, y, x, xs, offsets, rows, wt, ws, inn, out, x_rows=None, x_div=1, y_rows=None, st=None):
    experts = offsets.numel() - 1
    k3.check(k3.lib().k3d_grouped_f8(addr(y), TYPE[y.dtype], y.stride(0), addr(y_rows), y.shape[0], addr(x), x.stride(0), addr(xs),
                                     xs.stride(0), addr(x_rows), x_div, x.shape[0], addr(offsets), rows, experts, addr(wt), addr(ws),
                                     inn, out, stream() if st is None else st), "k3d_grouped_f8")
    return y


def moe8(k3, x, xs, idx, wt, bank, hidden, inter, act=SILU, b1=4.0, b2=25.0, out=None, out_type=F32, st=None, ws=None):
    """bank: (tiled, scales) of W1, W3, W2"""
    L, (T, k) = k3.lib(), idx.shape
    experts = bank[0][1].shape[0]
    out = torch.full((T, hidden), float("nan"), device="cuda", dtype=out_type) if out is None else out
    need = L.k3d_moe_f8_ws(T, hidden, inter, experts, k)
    ws = torch.full((need,), 0xff, device="cuda", dtype=torch.uint8) if ws is None else ws
    k3.check(L.k3d_moe_f8(addr(out), TYPE[out.dtype], out.stride(0), addr(idx), addr(wt), addr(x), x.stride(0), addr(xs), xs.stride(0), T,
                          *(addr(t) for pair in bank for t in pair), hidden, inter, experts, k, act, b1, b2, addr(ws), ws.numel(),
                          stream() if st is None else st), "k3d_moe_f8")
    return out


def moe64(X, idx, wt, W1, W3, W2, act, b1, b2, out_type):
    """The layer in 64 bits with the gated activation left unrounded, and how far off the kernel may be: h is off by g's and
    u's own errors and by its codes' half steps (2^-4 of it, and 2^-10 of the block's scale), through |W2|."""
    idx, wt = idx.cpu().numpy(), f64(wt)
    T, k = idx.shape
    y, tol = np.zeros((T, W2.shape[1])), np.zeros((T, W2.shape[1]))
    for t in range(T):
        for j in range(k):
            e = idx[t, j]
            if not 0 <= e < W1.shape[0]:
                continue
            (g, gt), (u, ut) = product64(X[t:t + 1], W1[e], True), product64(X[t:t + 1], W3[e], True)
            h = glu64(g, u, act, b1, b2)
            # |d act| <= 1.13 |dg| times |u|, |act(g)| times |du|
            ht = 1.13 * gt * (np.abs(u) + ut) + (np.abs(g) + gt) * ut + 2.0 ** -20 * np.abs(h)
            blocks = nb(h.shape[1])
            pad = np.zeros((1, blocks * 128))
            pad[:, :h.shape[1]] = np.abs(h) + ht
            s = np.repeat(np.maximum(pad.reshape(blocks, 128).max(1), LEAST) / 448, 128)[:h.shape[1]]
            ht = ht + np.abs(h) * 2.0 ** -4 * 1.001 + s * 2.0 ** -10
            v, vt = product64(h, W2[e], out_type == BF16)
            vt = vt * 1.1 + ht @ np.abs(W2[e]).T
            y[t] += wt[t, j] * v[0]
            tol[t] += abs(wt[t, j]) * (vt[0] + np.abs(v[0]) * k * 2.0 ** -22)
            if out_type == BF16:        # a slot's row as 16-bit integers: a step of its 64 columns' largest / 32767, and the scale's own roundings
                m = np.zeros(-(-v.shape[1] // 64) * 64)
                m[:v.shape[1]] = np.abs(v[0]) + vt[0]
                tol[t] += abs(wt[t, j]) * (np.repeat(np.maximum(m.reshape(-1, 64).max(1), LEAST), 64)[:v.shape[1]] * 2.0 ** -15 * 1.001)
    return y, tol
