# SPDX-License-Identifier: Apache-2.0
"""k3d_moe_f8 held closely: its gated activation is k3d_quant_f8's of k3d_grouped_f8's fp32 products, code for code, and behind it only
the down products' and the result's own roundings are left."""
import ctypes as C

import numpy as np
import pytest
import torch

from layer8_ops import (BF16, F32, F8, HALF, LEAST, SILU, SITU, acts, codes_of, f64, group, grouped, moe8, nb, quant, tile, weights)
from layer_ops import gen

pytestmark = pytest.mark.gpu


def sparse_down(g, experts, hidden, inter, size):
    """Codes and scales of W2 with one column in eight of a row: an 8-bit instruction, which aligns eight neighbouring products, then
    cuts nothing. size [hidden]: how large the codes of an output are."""
    v = torch.randn(experts, hidden, inter, device="cuda", generator=g) * size[None, :, None]
    k = torch.arange(inter, device="cuda") % 8 == torch.arange(hidden, device="cuda")[:, None] % 8
    q = torch.where(k, v.clamp(-448, 448), 0.0).to(F8).view(torch.uint8)
    return q, torch.rand(experts, nb(hidden), nb(inter), device="cuda", generator=g) * 1e-3 + 1e-4


def sizes(hidden):
    """Each group of 64 outputs with a size of its own, and an output 2^8 to 2^11 larger in each."""
    o = torch.arange(hidden, device="cuda")
    s = torch.tensor([0.25, 2.0, 0.5, 1.0, 0.125], device="cuda")[o // 64 % 5]
    return torch.where(o % 64 == 11, 300.0, s)


class Case:
    def __init__(self, gpu, T, k, experts, hidden, inter, act, integers, idx=None):
        g = gen(T + hidden)
        self.gpu, self.k, self.hidden, self.inter, self.act = gpu, k, hidden, inter, act
        self.x, self.xs = acts(g, T, hidden, integers)
        self.w = [weights(g, experts, inter, hidden, integers) for _ in range(2)] + [sparse_down(g, experts, hidden, inter, sizes(hidden))]
        if idx is None:
            idx = torch.stack([torch.randperm(experts, device="cuda", generator=g)[:k] for _ in range(T)])
        self.idx = idx.to(torch.int32)
        self.wt = torch.rand(T, k, device="cuda", generator=g) + 0.1
        self.bank = [(tile(gpu, q), s) for q, s in self.w]

    def layer(self, out_type):
        return moe8(self.gpu, self.x, self.xs, self.idx, self.wt, self.bank, self.hidden, self.inter, self.act, out_type=out_type)

    def slots(self):
        """The slots' rows in 64 bits from the gated activation's codes, and the sums of magnitudes behind them."""
        T, k, (q, s) = self.idx.shape[0], self.k, self.w[2]
        off, perm = group(self.gpu, self.idx, q.shape[0])
        gu = torch.empty(T * k, 2 * self.inter, device="cuda")
        for part, bank in ((gu[:, :self.inter], self.bank[0]), (gu[:, self.inter:], self.bank[1])):
            grouped(self.gpu, part, self.x, self.xs, off, T * k, *bank, self.hidden, self.inter, perm, k)
        hq, hs = quant(self.gpu, gu, act=self.act)
        h = torch.from_numpy(codes_of(hq) * np.repeat(f64(hs), 128, 1)).cuda()[:, :self.inter]
        y = torch.zeros(T * k, self.hidden, dtype=torch.float64, device="cuda")
        S = torch.zeros_like(y)
        o = off.tolist()
        for e in range(q.shape[0]):
            W = q[e].view(F8).double() * s[e].double().repeat_interleave(128, 0)[:self.hidden].repeat_interleave(128, 1)[:, :self.inter]
            r = slice(o[e], o[e + 1])
            y[perm[r].long()] = h[r] @ W.T
            S[perm[r].long()] = h[r].abs() @ W.abs().T
        return y.view(T, k, -1).cpu().numpy(), S.view(T, k, -1).cpu().numpy()


def check(c, out, out_type, sixteen):
    """A slot's row: inter + 8 roundings of S; where it waits in 16 bits (sixteen), half a step of its own, 2^-11 of it, and 2^-39 of the largest of
    its 64. The weighted sum: k products and k sums; the result's half step."""
    y, S = c.slots()
    tol = 2.0 ** -23 * (c.inter + 8) * S
    if sixteen:
        m = np.zeros(y.shape[:2] + (-(-c.hidden // 64) * 64,))
        m[..., :c.hidden] = np.abs(y)
        m = np.maximum(m.reshape(*y.shape[:2], -1, 64).max(-1), LEAST)
        tol = tol + np.abs(y) * 2.0 ** -11 + np.repeat(m, 64, 2)[..., :c.hidden] * 2.0 ** -39
    w = f64(c.wt)[:, :, None]
    tol = (w * tol).sum(1) + (w * np.abs(y)).sum(1) * 2.0 ** -23 * (c.k + 1)
    want = (w * y).sum(1)
    tol = 1.001 * (tol + (np.abs(want) + tol) * HALF[out_type])
    off = np.abs(f64(out) - want)
    assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), int((off > tol).sum()), off.size)


FEW = [(1, 4, 6, 1024, 256), (1, 8, 64, 584, 384), (3, 4, 6, 1024, 256), (12, 4, 6, 1001, 200), (20, 4, 6, 4224, 256)]
MANY = [(70, 4, 6, 584, 384), (400, 4, 6, 1160, 328), (300, 2, 3, 256, 129)]


@pytest.mark.parametrize("T,k,experts,hidden,inter", FEW + MANY)
@pytest.mark.parametrize("act", [SILU, SITU])
def test_fp32(gpu, T, k, experts, hidden, inter, act):
    """An fp32 result: every product as exact as fp32, at any number of rows."""
    c = Case(gpu, T, k, experts, hidden, inter, act, False)
    check(c, c.layer(F32), F32, False)


@pytest.mark.parametrize("T,k,experts,hidden,inter", FEW)
@pytest.mark.parametrize("act", [SILU, SITU])
def test_bf16_few_rows(gpu, T, k, experts, hidden, inter, act):
    """A bf16 result of few rows an expert: gate and up as exact as fp32."""
    c = Case(gpu, T, k, experts, hidden, inter, act, False)
    check(c, c.layer(BF16), BF16, T * k > 10 * experts)


def counted(counts, k, g):
    """A routing of sum(counts) slots whose experts have so many each, k to a token."""
    idx = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    return idx[torch.randperm(idx.numel(), device="cuda", generator=g)].view(-1, k)


@pytest.mark.parametrize("counts,k,hidden,inter", [
    ([47, 40, 60, 50, 43, 40], 4, 584, 384), ([400, 100, 128, 129, 3, 256, 257, 327], 2, 1160, 328), ([300, 0, 600, 1, 99], 1, 200, 129),
    ([100, 129, 300, 0, 71], 2, 8443, 200), ([513, 127], 1, 16700, 64)])
@pytest.mark.parametrize("act", [SILU, SITU])
def test_bf16_many_rows(gpu, counts, k, hidden, inter, act):
    """A bf16 result of many rows an expert: gate and up on integers (exact in every instruction), outputs of many sizes."""
    c = Case(gpu, sum(counts) // k, k, len(counts), hidden, inter, act, True, counted(counts, k, gen(hidden)))
    check(c, c.layer(BF16), BF16, True)


def test_outputs_apart(gpu):
    """An output that is no number leaves its neighbours' bits as they were, and one 2^11 larger their precision."""
    c = Case(gpu, 90, 4, 6, 584, 384, SILU, True)
    clean = c.layer(BF16)
    check(c, clean, BF16, True)
    q = c.w[2][0]
    for code in (0x7f, 0x7e):                  # NaN; the largest, whose scale makes it infinite
        w, s = q.clone(), c.w[2][1].clone()
        w[:, 70] = code
        if code == 0x7e:
            s[:, 0] = 3e38                      # (outputs 0 to 127)
        c.bank[2] = (tile(gpu, w), s)
        y = c.layer(BF16)
        if code == 0x7f:
            assert torch.isnan(y[:, 70]).all()
            y[:, 70] = clean[:, 70]
            assert torch.equal(y, clean)
        else:
            assert not torch.isfinite(y[:, 70]).any()
            assert torch.equal(y[:, 128:], clean[:, 128:])


@pytest.mark.parametrize("T,k,experts,hidden,inter", [(1, 4, 6, 584, 384), (7, 4, 6, 100, 500), (300, 2, 5, 200, 129), (700, 8, 9, 129, 200)])
@pytest.mark.parametrize("out_type", [F32, BF16])
def test_workspace(gpu, T, k, experts, hidden, inter, out_type):
    """The layer stays within its workspace, and takes nothing of what lay there."""
    c = Case(gpu, T, k, experts, hidden, inter, SILU, False)
    need = gpu.lib().k3d_moe_f8_ws(T, hidden, inter, experts, k)
    want = c.layer(out_type)
    for fill in (0x00, 0xff, 0x7f):
        ws = torch.full((need + 4096,), fill, device="cuda", dtype=torch.uint8)
        assert torch.equal(moe8(gpu, c.x, c.xs, c.idx, c.wt, c.bank, hidden, inter, SILU, out_type=out_type, ws=ws[:need]), want)
        assert (ws[need:] == fill).all()


@pytest.mark.parametrize("T", [5, 300])
@pytest.mark.parametrize("out_type", [F32, BF16])
def test_captured(gpu, k3, T, out_type):
    """Captured once, replayed on other inputs and over other tensors' old values, beside eager calls."""
    L, k, experts, hidden, inter = k3.lib(), 4, 6, 584, 384
    c = Case(gpu, T, k, experts, hidden, inter, SITU, False)
    others = [Case(gpu, T, k, experts, hidden, inter, SITU, True), c]
    keep = [(o.x.clone(), o.xs.clone(), o.idx.clone(), o.wt.clone()) for o in others]
    ws = torch.full((L.k3d_moe_f8_ws(T, hidden, inter, experts, k),), 0xff, device="cuda", dtype=torch.uint8)
    out = torch.full((T, hidden), float("nan"), device="cuda", dtype=out_type)
    run = lambda st=None: moe8(gpu, c.x, c.xs, c.idx, c.wt, c.bank, hidden, inter, SITU, out=out, st=st, ws=ws)    # noqa: E731
    ex = C.c_void_p()
    torch.cuda.synchronize()
    st = L.k3d_stream_create()
    try:
        k3.check(L.k3d_graph_begin(st))
        run(st)
        k3.check(L.k3d_graph_end(st, C.byref(ex)))
        for r in range(5):
            for t, v in zip((c.x, c.xs, c.idx, c.wt), keep[r % 2]):
                t.copy_(v)
            want = run().clone()
            ws.fill_(0xff)
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            k3.check(L.k3d_graph_launch(ex, st))
            k3.check(L.k3d_sync(st))
            assert torch.equal(out, want), r
    finally:
        torch.cuda.synchronize()
        if ex:
            L.k3d_graph_destroy(ex)
        L.k3d_stream_destroy(st)


@pytest.mark.parametrize("out_type", [F32, BF16])
def test_past_32_bits(gpu, out_type):
    """Slots' rows that lie more than 2^32 bytes from the first: copies of 64 tokens, whose results are one another's."""
    c, copies = Case(gpu, 64, 8, 16, 8192, 128, SILU, True), 520
    big = [t.repeat(copies, 1) for t in (c.x, c.xs, c.idx, c.wt)]
    assert 64 * copies * 8 * 8192 * 2 > 1 << 32
    out = moe8(gpu, *big, c.bank, 8192, 128, SILU, out_type=out_type).view(copies, 64, 8192)
    check(c, out[0], out_type, out_type == BF16)
    assert torch.equal(out, out[:1].expand_as(out))
