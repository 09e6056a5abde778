# SPDX-License-Identifier: Apache-2.0
"""The 8-bit path of a layer as a layer uses it: k3d_add_norm, k3d_linear_f8, k3d_quant_f8, k3d_group, k3d_grouped_f8 and k3d_moe_f8 around
k3d_qk_norm_rope, k3d_linear and k3d_route. Every step against 64 bits of what it was given; the run eager, captured and
replayed, and beside itself on other streams."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import layer8_ops as l8
import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu

HID, HQ, HK, DIM, ROT, N, INTER = 1160, 12, 3, 64, 32, 12, 328
WIDE = (HQ + 2 * HK) * DIM
EPS = 1e-6
STEPS = 14


def say(msg):
    print(msg, flush=True)


class Layer8:
    """The weights of one layer, its tensors and workspaces for T tokens."""

    def __init__(self, k3, T, topk, seed):
        g, L = lo.gen(seed), k3.lib()
        self.k3, self.T, self.topk = k3, T, topk

        def w(mats, out, inn):
            q, s = l8.weights(g, mats, out, inn)
            s.mul_(inn ** -0.5 / (100 * 6e-4))
            return q, s, l8.tile(k3, q)
        self.wqkv, self.wo = w(1, WIDE, HID), w(1, HID, HQ * DIM)
        self.w1, self.w3, self.w2 = w(N, INTER, HID), w(N, INTER, HID), w(N, HID, INTER)
        self.w13, self.wd = w(N, 2 * INTER, HID), w(N, HID, INTER)
        self.wr = (torch.randn(N, HID, device="cuda", generator=g) * HID ** -0.5).to(BF16)
        self.bqkv, self.bias = torch.randn(WIDE, device="cuda", generator=g), torch.randn(N, device="cuda", generator=g) * 0.1
        self.n1, self.n2 = (torch.rand(HID, device="cuda", generator=g) + 0.5 for _ in range(2))
        self.qw, self.kw = (torch.rand(DIM, device="cuda", generator=g) + 0.5 for _ in range(2))
        self.freq = 10000.0 ** (-torch.arange(ROT // 2, device="cuda", dtype=torch.float64) / (ROT // 2))
        self.pos = torch.arange(T, device="cuda", dtype=torch.int32) + 70000
        self.pos[T // 2:T // 2 + T // 5] = -1                     # (padding in the batch)
        new = lambda *s, dtype=F32: torch.zeros(*s, device="cuda", dtype=dtype)       # noqa: E731
        self.x, self.res = new(T, HID, dtype=BF16), new(T, HID)
        self.sum, self.h, self.out, self.out2 = new(T, HID), new(T, HID), new(T, HID, dtype=BF16), new(T * topk, HID)
        self.q1, self.s1 = l8.rows_for(T, HID)
        self.q2, self.s2 = l8.rows_for(T, HQ * DIM)
        self.q3, self.s3 = l8.rows_for(T, HID)
        self.q4, self.s4 = l8.rows_for(T * topk, INTER)
        self.qkv, self.nr, self.gu = new(T, WIDE, dtype=BF16), new(T, HID, dtype=BF16), new(T * topk, 2 * INTER, dtype=BF16)
        self.logits, self.idx, self.wt = new(T, N), new(T, topk, dtype=torch.int32), new(T, topk)
        self.off, self.perm = new(N + 1, dtype=torch.int32), new(T * topk, dtype=torch.int32)
        byte = lambda n: torch.full((max(n, 1),), 0xff, device="cuda", dtype=torch.uint8)   # noqa: E731
        self.ws = byte(max(L.k3d_linear_f8_ws(T, i, o) for i, o in ((HID, WIDE), (HQ * DIM, HID))))
        self.wsr = byte(L.k3d_linear_ws(T, HID, N, 1))
        self.wsm = byte(L.k3d_moe_f8_ws(T, HID, INTER, N, topk))
        self.wsg = byte(L.k3d_group_ws(T, topk, N))

    def inputs(self, seed):
        g = lo.gen(seed)
        self.x.copy_(torch.randn(self.T, HID, device="cuda", generator=g))
        self.res.copy_(torch.randn(self.T, HID, device="cuda", generator=g))

    def heads(self):
        q = self.qkv[:, :HQ * DIM].unflatten(1, (HQ, DIM))
        return q, self.qkv[:, HQ * DIM:(HQ + HK) * DIM].unflatten(1, (HK, DIM))

    def one(self, i, st=None):
        k3, st = self.k3, lo.stream() if st is None else st
        L, T = k3.lib(), self.T
        if i == 0:
            l8.add_norm(k3, self.x, self.res, self.n1, EPS, q=self.q1, qs=self.s1, sum_=self.sum, st=st)
        elif i == 1:
            l8.linear8(k3, self.q1, self.s1, self.wqkv[2], self.wqkv[1], HID, WIDE, self.bqkv, y=self.qkv, ws_=self.ws, st=st)
        elif i == 2:
            q, k = self.heads()
            lo.heads(k3, q, k, self.qw, self.kw, self.pos, self.freq, ROT, eps=EPS, qo=q, ko=k, st=st)
        elif i == 3:                                              # (the heads' values stand for what attention gives)
            l8.quant(k3, self.qkv, HQ * DIM, q=self.q2, qs=self.s2, st=st)
        elif i == 4:
            l8.linear8(k3, self.q2, self.s2, self.wo[2], self.wo[1], HQ * DIM, HID, res=self.sum, y=self.h, ws_=self.ws, st=st)
        elif i == 5:
            l8.add_norm(k3, self.h, None, self.n2, EPS, y=self.nr, q=self.q3, qs=self.s3, st=st)
        elif i == 6:
            lo.linear(k3, self.nr, self.wr, y=self.logits, ws=self.wsr, st=st)
        elif i == 7:
            lo.route(k3, self.logits, self.bias, 0, 4, 2, 2, self.topk, 1, 2.5, idx=self.idx, wt=self.wt, st=st)
        elif i == 8:
            l8.moe8(k3, self.q3, self.s3, self.idx, self.wt, [(w[2], w[1]) for w in (self.w1, self.w3, self.w2)], HID, INTER,
                    out=self.out, ws=self.wsm, st=st)
        elif i == 9:
            k3.check(L.k3d_group(lo.addr(self.off), lo.addr(self.perm), lo.addr(self.idx), T, self.topk, N, lo.addr(self.wsg),
                                 self.wsg.numel(), st), "k3d_group")
        elif i == 10:
            l8.grouped(k3, self.gu, self.q3, self.s3, self.off, T * self.topk, self.w13[2], self.w13[1], HID, 2 * INTER,
                       x_rows=self.perm, x_div=self.topk, st=st)
        elif i == 11:
            l8.quant(k3, self.gu, INTER, l8.SITU, q=self.q4, qs=self.s4, st=st)
        elif i == 12:
            l8.grouped(k3, self.out2, self.q4, self.s4, self.off, T * self.topk, self.wd[2], self.wd[1], INTER, HID,
                       y_rows=self.perm, st=st)
        else:                                                     # the next layer's norm, the residual in its own place
            l8.add_norm(k3, self.out, self.h, self.n1, EPS, q=self.q1, qs=self.s1, sum_=self.h, st=st)

    def tensors(self):
        return [self.sum, self.qkv, self.q2, self.s2, self.nr, self.q3, self.s3, self.logits, self.idx, self.wt, self.out, self.off,
                self.perm, self.gu, self.q4, self.s4, self.out2, self.h, self.q1, self.s1]

    def clear(self):
        """Sentinels in every output and workspace (the fill kernels of the current stream)."""
        for t in self.tensors():
            t.fill_(float("nan") if t.dtype.is_floating_point else -9 if t.dtype == torch.int32 else 0x7f)
        for t in (self.ws, self.wsr, self.wsm, self.wsg):
            t.fill_(0xff)


def same(got, want):
    return torch.equal(got, want) and not (got.dtype.is_floating_point and bool(torch.isnan(got).any()))


@pytest.mark.parametrize("T,topk", [(1, 4), (5, 6), (23, 4), (150, 4), (700, 2)])
def test_layer(gpu, k3, T, topk):
    """The steps in a row, each against what 64 bits make of its actual inputs."""
    say(f"case: {T} tokens, top {topk}")
    m = Layer8(k3, T, topk, 900 + T)
    m.inputs(1)
    m.clear()
    m.one(0)
    v, u, tol = l8.norm64(m.x, m.res, m.n1, EPS)
    lo.within(m.sum, (v, 2.0 ** -24 * np.abs(v)))
    l8.check_codes(m.q1, m.s1, u, tol, HID)
    m.one(1)
    lo.within(m.qkv, l8.linear8_64(l8.rows64(m.q1, m.s1, HID), l8.weights64(m.wqkv[0][0], m.wqkv[1][0]), m.bqkv, "none", None, BF16))
    q, k = (h.clone() for h in m.heads())
    m.one(2)
    on = m.pos >= 0
    for got, was, w in zip(m.heads(), (q, k), (m.qw, m.kw)):
        y, tol = lo.heads64(was, w, m.pos.clamp(min=0), m.freq, ROT, 0, 0, EPS, 1.0)
        lo.within(got[on], (y[on.cpu().numpy()], tol[on.cpu().numpy()]))
        assert torch.equal(got[~on], was[~on])
    m.one(3)
    l8.check_codes(m.q2, m.s2, lo.f64(m.qkv[:, :HQ * DIM]), 0 * lo.f64(m.qkv[:, :HQ * DIM]), HQ * DIM)
    m.one(4)
    lo.within(m.h, l8.linear8_64(l8.rows64(m.q2, m.s2, HQ * DIM), l8.weights64(m.wo[0][0], m.wo[1][0]), None, "none", m.sum, F32))
    m.one(5)
    _, u, tol = l8.norm64(m.h, None, m.n2, EPS)
    lo.within(m.nr, (u, tol + (np.abs(u) + tol) * lo.HALF[BF16]))
    l8.check_codes(m.q3, m.s3, u, tol, HID)
    m.one(6)
    lo.within(m.logits, lo.linear64(m.nr, m.wr, None, "none", None, F32))
    m.one(7)
    lo.check_route((m.idx, m.wt), lo.route64(m.logits, m.bias, 0, 4, 2, 2, topk, 1, 2.5))
    m.one(8)
    X = l8.rows64(m.q3, m.s3, HID)
    some = sorted({0, T // 3, T // 2, T - 1})
    Ws = [[l8.weights64(w[0][e], w[1][e]) for e in range(N)] for w in (m.w1, m.w3, m.w2)]
    W1, W3, W2 = (np.stack(w) for w in Ws)
    y, tol = l8.moe64(X[some], m.idx[some], m.wt[some], W1, W3, W2, l8.SILU, 4.0, 25.0, BF16)
    lo.within(m.out[some], (y, tol + (np.abs(y) + tol) * lo.HALF[BF16]))
    m.one(9)
    off, perm = l8.group64(m.idx, N)
    assert (m.off.cpu().numpy() == off).all() and (m.perm.cpu().numpy()[:off[-1]] == perm).all()
    m.one(10)
    rows = T * topk
    for r in sorted({0, rows // 2, rows - 1}):
        e = int(np.searchsorted(off, r, "right")) - 1
        lo.within(m.gu[r:r + 1], l8.linear8_64(X[perm[r] // topk][None], l8.weights64(m.w13[0][e], m.w13[1][e]), None, "none", None, BF16))
    m.one(11)
    gate, up = lo.f64(m.gu[:, :INTER]), lo.f64(m.gu[:, INTER:])
    u = l8.glu64(gate, up, l8.SITU, 4.0, 25.0)
    l8.check_codes(m.q4, m.s4, u, 2.0 ** -20 * np.abs(u), INTER)
    m.one(12)
    for r in sorted({0, rows // 2, rows - 1}):
        e = int(np.searchsorted(off, r, "right")) - 1
        lo.within(m.out2[perm[r]][None], l8.linear8_64(l8.rows64(m.q4[r:r + 1], m.s4[r:r + 1], INTER),
                                                       l8.weights64(m.wd[0][e], m.wd[1][e]), None, "none", None, F32))
    assert not torch.isnan(m.out2).any()
    h = m.h.clone()
    m.one(13)
    v, u, tol = l8.norm64(m.out, h, m.n1, EPS)
    lo.within(m.h, (v, 2.0 ** -24 * np.abs(v)))
    l8.check_codes(m.q1, m.s1, u, tol, HID)
    torch.cuda.synchronize()


@pytest.mark.parametrize("T,topk", [(1, 4), (23, 4), (200, 4), (1100, 4)])
def test_layer_graph(gpu, k3, T, topk):
    """The whole run captured once and replayed on new inputs, with eager calls between the replays."""
    say(f"case: graph of {T} tokens")
    L, m, ex = k3.lib(), Layer8(k3, T, topk, 950), C.c_void_p()
    torch.cuda.synchronize()
    st = L.k3d_stream_create()
    try:
        k3.check(L.k3d_graph_begin(st))
        for i in range(STEPS):
            m.one(i, st)
        k3.check(L.k3d_graph_end(st, C.byref(ex)))
        last = None
        for r in range(4):
            m.inputs(10 + r)
            m.clear()
            for i in range(STEPS):
                m.one(i)
            want = [t.clone() for t in m.tensors()]
            assert last is None or not torch.equal(want[10], last)
            last = want[10]
            m.clear()
            torch.cuda.synchronize()
            k3.check(L.k3d_graph_launch(ex, st))
            k3.check(L.k3d_sync(st))
            for n, (got, w) in enumerate(zip(m.tensors(), want)):
                assert same(got, w), (r, n)
    finally:
        torch.cuda.synchronize()
        if ex:
            L.k3d_graph_destroy(ex)
        L.k3d_stream_destroy(st)


@pytest.mark.parametrize("T", [3, 130, 700])
def test_two_threads(gpu, k3, T):
    """Two host threads, a stream, tensors and workspaces each, inputs that change and sentinels before each pass."""
    say(f"case: two threads, {T} tokens")
    passes, ms = 5, [Layer8(k3, T, 4, 980 + i) for i in range(2)]
    sts, wrong, want, xs = [torch.cuda.Stream() for _ in ms], [], [], []
    for i, m in enumerate(ms):
        want.append([])
        xs.append([])
        for r in range(passes):
            m.inputs(50 + 10 * i + r)
            xs[i].append((m.x.clone(), m.res.clone()))
            m.clear()
            for s in range(STEPS):
                m.one(s)
            want[i].append([t.clone() for t in m.tensors()])
    torch.cuda.synchronize()
    start = threading.Barrier(len(ms))

    def work(i, m, st):
        try:
            got = []
            start.wait(30)
            with torch.cuda.stream(st):
                for r in range(passes):
                    m.x.copy_(xs[i][r][0])
                    m.res.copy_(xs[i][r][1])
                    m.clear()
                    for s in range(STEPS):
                        m.one(s, st.cuda_stream)
                    got.append([t.clone() for t in m.tensors()])
            st.synchronize()
            for r in range(passes):
                for n, (a, w) in enumerate(zip(got[r], want[i][r])):
                    assert same(a, w), (i, r, n)
        except BaseException as e:
            wrong.append(e)
    th = [threading.Thread(target=work, args=(i, m, st)) for i, (m, st) in enumerate(zip(ms, sts))]
    for t in th:
        t.start()
    for t in th:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong


@pytest.mark.parametrize("T", [9, 260])
def test_two_graphs(gpu, k3, T):
    """Two captured runs with workspaces of their own, replayed at the same time on two streams."""
    say(f"case: two graphs, {T} tokens")
    L, ms = k3.lib(), [Layer8(k3, T, 4, 990 + i) for i in range(2)]
    torch.cuda.synchronize()
    sts, exs = [L.k3d_stream_create() for _ in ms], [C.c_void_p() for _ in ms]
    try:
        for m, st, ex in zip(ms, sts, exs):
            k3.check(L.k3d_graph_begin(st))
            for i in range(STEPS):
                m.one(i, st)
            k3.check(L.k3d_graph_end(st, C.byref(ex)))
        for r in range(4):
            want = []
            for i, m in enumerate(ms):
                m.inputs(70 + 10 * i + r)
                m.clear()
                for s in range(STEPS):
                    m.one(s)
                want.append([t.clone() for t in m.tensors()])
                m.clear()
            torch.cuda.synchronize()
            for st, ex in zip(sts, exs):
                k3.check(L.k3d_graph_launch(ex, st))
            for st in sts:
                k3.check(L.k3d_sync(st))
            for m, w in zip(ms, want):
                for n, (a, b) in enumerate(zip(m.tensors(), w)):
                    assert same(a, b), (r, n)
    finally:
        torch.cuda.synchronize()
        for st, ex in zip(sts, exs):
            if ex:
                L.k3d_graph_destroy(ex)
            L.k3d_stream_destroy(st)


def test_past_32_bits(gpu, k3):
    """Rows, results and weights that lie more than 2^32 bytes from the first."""
    g = lo.gen(3)
    T, n = 530000, 4160
    say("case: rows past 2^32 bytes")
    x = torch.zeros(T, n, device="cuda", dtype=BF16)
    some = [0, T // 2, T - 1]
    x[some] = torch.randn(3, n, device="cuda", generator=g).to(BF16)
    q, qs = torch.empty(T, l8.nb(n) * 128, device="cuda", dtype=torch.uint8), torch.empty(T, l8.nb(n), device="cuda")
    s = torch.empty_like(x)
    l8.add_norm(k3, x, None, None, EPS, y=None, q=q, qs=qs, sum_=s)
    _, u, tol = l8.norm64(x[some], None, None, EPS)
    l8.check_codes(q[some], qs[some], u, tol, n)
    assert torch.equal(s, x)
    q.zero_()
    l8.quant(k3, x, q=q, qs=qs)
    l8.check_codes(q[some], qs[some], lo.f64(x[some]), 0 * u, n)
    del x, s, q, qs
    say("case: weights and results past 2^32 bytes")
    experts, inn, out, rows = 300, 2048, 8192, 150000
    w = torch.randint(0, 0x70, (1, out, inn), device="cuda", generator=g, dtype=torch.uint8)
    size = k3.lib().k3d_f8_tiled_bytes(out, inn)
    W = torch.zeros(experts * size, device="cuda", dtype=torch.uint8)
    W[-size:] = l8.tile(k3, w)
    ws = torch.rand(experts, l8.nb(out), l8.nb(inn), device="cuda", generator=g) * 1e-3
    assert W.numel() > 1 << 32 and rows * out * 4 > 1 << 32
    xq, xs = l8.acts(g, rows, inn)
    for last in (5, 140):                       # rows of the last expert
        off = torch.full((experts + 1,), rows - last, device="cuda", dtype=torch.int32)
        off[0], off[-1] = rows - last, rows
        for n_rows in (rows, 299 * 3):          # (what is chosen by: many rows an expert, or few)
            y = torch.full((rows, out), 7.0, device="cuda")
            o = off if n_rows == rows else off - (rows - last) + n_rows - last
            sl = slice(rows - n_rows, rows)     # (x from its start on, so that row numbers fit)
            yr = torch.arange(rows - n_rows, rows, device="cuda", dtype=torch.int32)
            l8.grouped(k3, y, xq[sl], xs[sl], o, n_rows, W, ws, inn, out, y_rows=yr)
            X = l8.rows64(xq[rows - last:], xs[rows - last:], inn)
            v, tol = l8.product64(X[[0, last - 1]], l8.weights64(w[0], ws[-1]))
            lo.within(y[[rows - last, rows - 1]], (v, tol + np.abs(v) * lo.HALF[F32]))
            assert (y[:rows - last] == 7).all()
    torch.cuda.synchronize()
