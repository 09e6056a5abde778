# SPDX-License-Identifier: Apache-2.0
"""k3d_linear, k3d_route and k3d_qk_norm_rope as a layer uses them, with k3d_moe_experts behind the routing: every step
against 64 bits of what it was given, eager, captured and replayed, and beside each other on two streams."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import layer_ops as lo
from conftest import max_err_rel_inf
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu

HID, HQ, HK, DIM, ROT, N, INTER = 1024, 12, 3, 64, 32, 12, 512
EPS = 1e-6
TOL = 1e-4              # of k3d_moe_experts, of the largest value


def say(msg):
    print(msg, flush=True)


class Layer:
    """The weights of one layer, and its tensors for T tokens."""

    def __init__(self, k3, T, topk, seed):
        g = lo.gen(seed)
        L = k3.lib()
        self.k3, self.T, self.topk = k3, T, topk
        wide = (HQ + 2 * HK) * DIM

        def w(out, inn):
            return (torch.randn(out, inn, device="cuda", generator=g) * inn ** -0.5).to(BF16)
        self.wqkv, self.bqkv = w(wide, HID), torch.randn(wide, device="cuda", generator=g)
        self.wo, self.wr = w(HID, HQ * DIM), w(N, HID)
        self.qw, self.kw = (torch.rand(DIM, device="cuda", generator=g) + 0.5 for _ in range(2))
        self.bias = torch.randn(N, device="cuda", generator=g) * 0.1
        self.freq = 10000.0 ** (-torch.arange(ROT // 2, device="cuda", dtype=torch.float64) / (ROT // 2))
        self.pos = torch.arange(T, device="cuda", dtype=torch.int32) + 70000
        self.pos[T // 2:T // 2 + T // 5] = -1                     # (padding in the batch)
        new = lambda *s, dtype: torch.zeros(*s, device="cuda", dtype=dtype)
        self.x = new(T, HID, dtype=BF16)
        self.qkv, self.h = new(T, wide, dtype=BF16), new(T, HID, dtype=F32)
        self.xr = new(T, HID, dtype=F32)
        self.logits, self.out = new(T, N, dtype=F32), new(T, HID, dtype=F32)
        self.idx, self.wt = new(T, topk, dtype=torch.int32), new(T, topk, dtype=F32)
        self.drops = new(1, dtype=torch.int32)
        need = max(L.k3d_linear_ws(T, i, o, t) for i, o, t in ((HID, wide, 1), (HQ * DIM, HID, 1), (HID, N, 0)))
        self.ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
        self.wsm = torch.empty(L.k3d_moe_ws(T, HID, INTER, N, topk, 0), device="cuda", dtype=torch.uint8)
        self.perm, self.off = new(T * topk, dtype=torch.int32), new(N + 1, dtype=torch.int32)
        self.experts = [k3.gen_expert(HID, INTER, seed, e) for e in range(N)]
        self.bank = k3.DevBank(self.experts, HID, INTER, k3.K3D_LAYOUT_TILED)

    def inputs(self, seed):
        self.x.copy_(torch.randn(self.T, HID, device="cuda", generator=lo.gen(seed)))
        self.xr.copy_(self.x)

    def heads(self):
        q = self.qkv[:, :HQ * DIM].unflatten(1, (HQ, DIM))
        return q, self.qkv[:, HQ * DIM:(HQ + HK) * DIM].unflatten(1, (HK, DIM))

    def one(self, i, st=None):
        """Step i of the layer."""
        k3, st = self.k3, lo.stream() if st is None else st
        if i == 0:
            lo.linear(k3, self.x, self.wqkv, self.bqkv, y=self.qkv, ws=self.ws, st=st)
        elif i == 1:
            q, k = self.heads()
            lo.heads(k3, q, k, self.qw, self.kw, self.pos, self.freq, ROT, eps=EPS, qo=q, ko=k, st=st)
        elif i == 2:                                              # (the heads' values stand for what attention gives)
            lo.linear(k3, self.qkv[:, :HQ * DIM], self.wo, None, "none", self.xr, y=self.h, ws=self.ws, st=st)
        elif i == 3:
            lo.linear(k3, self.h, self.wr, y=self.logits, ws=self.ws, st=st)
        elif i == 4:
            lo.route(k3, self.logits, self.bias, 0, 4, 2, 2, self.topk, 1, 2.5, idx=self.idx, wt=self.wt, st=st)
        else:
            L = k3.lib()
            k3.check(L.k3d_moe_experts(lo.addr(self.out), lo.addr(self.idx), lo.addr(self.wt), lo.addr(self.h), self.T,
                                       self.bank.table.ptr, self.bank.layout, HID, INTER, N, self.topk, k3.K3_ACT_SILU, 4.0, 25.0,
                                       0, lo.addr(self.wsm), self.wsm.numel(), lo.addr(self.perm), lo.addr(self.off),
                                       lo.addr(self.drops), st), "k3d_moe_experts")

    def tensors(self):
        return [self.qkv, self.h, self.logits, self.idx, self.wt, self.out]


@pytest.mark.parametrize("T,topk", [(1, 4), (5, 6), (23, 4), (150, 4), (600, 2)])
def test_layer(gpu, k3, orc, T, topk):
    """The steps in a row, each against what 64 bits make of its actual inputs."""
    say(f"case: {T} tokens, top {topk}")
    m = Layer(k3, T, topk, 900 + T)
    try:
        m.inputs(1)
        m.one(0)
        lo.within(m.qkv, lo.linear64(m.x, m.wqkv, m.bqkv, "none", None, BF16))
        before = m.qkv.clone()
        q, k = (h.clone() for h in m.heads())
        m.one(1)
        on = (m.pos >= 0).cpu().numpy()
        for got, was, w in zip(m.heads(), (q, k), (m.qw, m.kw)):
            y, tol = lo.heads64(was, w, m.pos.clamp(min=0), m.freq, ROT, 0, 0, EPS, 1.0)
            lo.within(got[on], (y[on], tol[on]))
            assert torch.equal(got[~torch.from_numpy(on).cuda()], was[~torch.from_numpy(on).cuda()])
        assert torch.equal(m.qkv[:, (HQ + HK) * DIM:], before[:, (HQ + HK) * DIM:])     # the values' part
        m.one(2)
        lo.within(m.h, lo.linear64(m.qkv[:, :HQ * DIM], m.wo, None, "none", m.xr, F32))
        m.one(3)
        lo.within(m.logits, lo.linear64(m.h, m.wr, None, "none", None, F32))
        m.one(4)
        lo.check_route((m.idx, m.wt), lo.route64(m.logits, m.bias, 0, 4, 2, 2, topk, 1, 2.5))
        m.one(5)
        torch.cuda.synchronize()
        out, idx, wt, h = (t.cpu().numpy() for t in (m.out, m.idx, m.wt, m.h))
        assert int(m.drops) == 0
        for t in sorted({0, T // 2, T - 1}):
            acc = np.zeros(HID, np.float32)
            for e, v in zip(idx[t], wt[t]):
                acc = acc + v * orc.expert_ffn(h[t], m.experts[int(e)], HID, INTER, act=1, wt=1.0)
            assert max_err_rel_inf(out[t], acc) <= TOL, t
    finally:
        torch.cuda.synchronize()
        m.bank.free()


@pytest.mark.parametrize("T,topk", [(1, 4), (23, 4), (200, 4)])
def test_layer_graph(gpu, k3, T, topk):
    """The whole run captured once and replayed on new inputs, with eager calls between the replays."""
    say(f"case: graph of {T} tokens")
    L, m, ex = k3.lib(), Layer(k3, T, topk, 950), C.c_void_p()
    torch.cuda.synchronize()
    st = L.k3d_stream_create()
    try:
        k3.check(L.k3d_graph_begin(st))
        for i in range(6):
            m.one(i, st)
        k3.check(L.k3d_graph_end(st, C.byref(ex)))
        for r in range(4):
            m.inputs(10 + r)
            for i in range(6):
                m.one(i)
            want = [t.clone() for t in m.tensors()]
            for t in m.tensors():
                t.zero_()
            torch.cuda.synchronize()
            k3.check(L.k3d_graph_launch(ex, st))
            k3.check(L.k3d_sync(st))
            for got, w in zip(m.tensors()[:-1], want[:-1]):
                assert torch.equal(got, w)
            assert max_err_rel_inf(m.out.cpu().numpy(), want[-1].cpu().numpy()) <= TOL
    finally:
        torch.cuda.synchronize()
        if ex:
            L.k3d_graph_destroy(ex)
        L.k3d_stream_destroy(st)
        m.bank.free()


@pytest.mark.parametrize("T", [3, 130])
def test_two_streams(gpu, k3, T):
    """Two host threads, a stream and a workspace each, the first five steps over and over: the same bits as alone."""
    say(f"case: two threads, {T} tokens")
    L = k3.lib()
    ms = [Layer(k3, T, 4, 970 + i) for i in range(2)]
    sts = [L.k3d_stream_create() for _ in ms]
    wrong = []
    try:
        want = []
        for i, m in enumerate(ms):
            m.inputs(30 + i)
            for s in range(5):
                m.one(s)
            want.append([t.clone() for t in m.tensors()[:5]])
        torch.cuda.synchronize()

        def work(m, st, w):
            try:
                for _ in range(20):
                    for s in range(5):
                        m.one(s, st)
                k3.check(L.k3d_sync(st))
            except Exception as e:
                wrong.append(e)
        th = [threading.Thread(target=work, args=a) for a in zip(ms, sts, want)]
        for t in th:
            t.start()
        for t in th:
            t.join()
        assert not wrong
        for m, w in zip(ms, want):
            for got, v in zip(m.tensors(), w):
                assert torch.equal(got, v)
    finally:
        torch.cuda.synchronize()
        for st in sts:
            L.k3d_stream_destroy(st)
        for m in ms:
            m.bank.free()
