# SPDX-License-Identifier: Apache-2.0
"""k3d_qk_norm_rope against the norm and the rotation in 64 bits (layer_ops.heads64)."""
import ctypes as C

import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)


def freqs(rot, base=1e6):
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    return torch.pow(torch.tensor(base, device="cuda", dtype=torch.float64), -2.0 * i / max(rot, 1))


def inputs(T, hq, hk, dim, dtype, seed, far=False):
    """Views of q and k in a fused buffer with values behind them, norm weights, positions."""
    g = lo.gen(seed)
    qkv = torch.randn(T, (hq + 2 * hk) * dim, device="cuda", generator=g).to(dtype)
    q = qkv[:, :hq * dim].view(T, hq, dim)
    k = qkv[:, hq * dim:(hq + hk) * dim].view(T, hk, dim)
    qw, kw = (1 + 0.1 * torch.randn(dim, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, 2 ** 31 - 1 if far else 8192, (T,), device="cuda", generator=g).int()
    return qkv, q, k, qw, kw, pos


def check(k3, q, k, qw, kw, pos, freq, rot, off=0, pairs=0, eps=1e-6, scale=1.0):
    qo, ko = lo.heads(k3, q, k, qw, kw, pos, freq, rot, off, pairs, eps, scale)
    lo.within(qo, lo.heads64(q, qw, pos, freq, rot, off, pairs, eps, scale))
    lo.within(ko, lo.heads64(k, kw, pos, freq, rot, off, pairs, eps, scale))
    return qo, ko


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("T,hq,hk,dim,rot,off", [
    (1, 64, 8, 128, 128, 0), (1, 1, 1, 1, 0, 0), (2, 3, 1, 2, 2, 0), (3, 5, 2, 7, 4, 1), (5, 4, 4, 64, 64, 0), (7, 2, 1, 33, 32, 1),
    (9, 12, 1, 192, 64, 128), (4, 12, 1, 192, 64, 0), (6, 8, 2, 80, 20, 60), (10, 6, 6, 96, 48, 24), (3, 2, 2, 256, 256, 0),
    (2, 3, 1, 320, 100, 220), (5, 1, 2, 512, 64, 448), (2, 2, 2, 576, 64, 512), (3, 1, 1, 1024, 1024, 0), (2, 1, 1, 1023, 1022, 1),
    (4, 2, 1, 770, 770, 0), (33, 1, 0, 128, 64, 0), (33, 0, 3, 128, 64, 64), (300, 16, 2, 128, 128, 0), (700, 1, 1, 64, 32, 0),
    (2, 300, 100, 64, 64, 0), (1, 7, 1, 514, 2, 512), (6, 3, 2, 128, 0, 0)])
def test_shapes(gpu, k3, T, hq, hk, dim, rot, off, pairs, dtype):
    say(f"case: {T} {hq} {hk} {dim} {rot} {off} {pairs} {dtype}")
    _, q, k, qw, kw, pos = inputs(T, hq, hk, dim, dtype, T + dim)
    check(k3, q, k, qw, kw, pos, freqs(rot), rot, off, pairs)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_positions(gpu, k3, dtype):
    """Positions to 2^31 - 1 at frequency 1 (an fp32 angle is off by 128 there); other bases, no weights, a scale."""
    say(f"case: {dtype}")
    _, q, k, qw, kw, pos = inputs(50, 4, 2, 64, dtype, 3, far=True)
    pos[0], pos[1] = 2 ** 31 - 1, 0
    for base in (1e6, 1e4, 2.0, 1.0):
        check(k3, q, k, None, None, pos, freqs(64, base), 64, 0, 0, 1e-5, 1.3)
        check(k3, q, k, qw, None, pos, -freqs(64, base), 64, 0, 1, 0.0, -0.5)


@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,rot,off", [(128, 128, 0), (128, 64, 64), (66, 34, 3), (1000, 500, 500)])
def test_in_place_and_head_major(gpu, k3, dim, rot, off, pairs, dtype):
    """Over the input itself, with the values behind left alone; heads outermost; out of odd starts."""
    say(f"case: {dim} {pairs} {dtype}")
    qkv, q, k, qw, kw, pos = inputs(40, 5, 2, dim, dtype, 5)
    f = freqs(rot)
    want = lo.heads(k3, q, k, qw, kw, pos, f, rot, off, pairs)
    behind = qkv[:, 7 * dim:].clone()
    q2, k2 = q.permute(1, 0, 2).contiguous().permute(1, 0, 2), k.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    odd = torch.zeros(40 * 5 * (dim + 1) + 1, device="cuda", dtype=dtype)[1:].view(40, 5, dim + 1)[:, :, :dim]
    odd.copy_(q)
    got = lo.heads(k3, q2, k2, qw, kw, pos, f, rot, off, pairs, qo=q2, ko=k2)
    lo.within(got[0], lo.heads64(q, qw, pos, f, rot, off, pairs, 1e-6, 1.0))
    lo.within(got[1], lo.heads64(k, kw, pos, f, rot, off, pairs, 1e-6, 1.0))
    lo.within(lo.heads(k3, odd, k, qw, kw, pos, f, rot, off, pairs, qo=odd)[0], lo.heads64(q, qw, pos, f, rot, off, pairs, 1e-6, 1.0))
    lo.heads(k3, q, k, qw, kw, pos, f, rot, off, pairs, qo=q, ko=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 7 * dim:], behind)


def test_padding(gpu, k3):
    """Tokens of negative position: their rows stay as they were, NaN among them; also without a rotation."""
    say("case: padding")
    for rot in (128, 0):
        _, q, k, qw, kw, pos = inputs(37, 8, 1, 128, BF16, 6)
        pos[5], pos[20:] = -1, -(2 ** 31)
        q[30] = float("nan")
        qo, ko = torch.full_like(q, 3.0).contiguous(), torch.full_like(k, 4.0).contiguous()
        lo.heads(k3, q, k, qw, kw, pos, freqs(rot), rot, qo=qo, ko=ko)
        live = pos >= 0
        y, tol = lo.heads64(q, qw, pos, freqs(rot), rot, 0, 0, 1e-6, 1.0)
        m = live.cpu().numpy()
        lo.within(qo[live], (y[m], tol[m]))
        assert (qo[~live] == 3).all() and (ko[~live] == 4).all()
    _, q, k, qw, kw, pos = inputs(9, 2, 1, 64, F32, 7)
    qo, ko = lo.heads(k3, q, k, qw, kw, None, None, 0)             # no positions: no padding
    lo.within(qo, lo.heads64(q, qw, None, None, 0, 0, 0, 1e-6, 1.0))


def test_values(gpu, k3):
    """Rows of zeros (with and without eps), infinities and NaN stay in their head; the largest and smallest bf16."""
    say("case: values")
    _, q, k, qw, kw, pos = inputs(4, 4, 1, 128, F32, 8)
    clean = lo.heads(k3, q, k, qw, kw, pos, freqs(128), 128)[0]
    q[0, 1] = 0
    q[1, 2, 5], q[2, 0, 7] = float("nan"), float("inf")
    got = lo.heads(k3, q, k, qw, kw, pos, freqs(128), 128)[0]
    assert (got[0, 1] == 0).all() and torch.isnan(got[1, 2]).all() and torch.isnan(got[2, 0]).any()
    for t, h in ((0, 0), (0, 2), (1, 1), (1, 3), (2, 1), (3, 3)):
        assert torch.equal(got[t, h], clean[t, h])
    assert torch.isnan(lo.heads(k3, q, k, qw, kw, pos, freqs(128), 128, eps=0.0)[0][0, 1]).all()
    q[3] = 1e-18                                                   # (squares under the smallest normal fp32 number but for eps)
    lo.within(lo.heads(k3, q, k, qw, kw, pos, freqs(128), 128)[0][3:], tuple(v[3:] for v in lo.heads64(q, qw, pos, freqs(128), 128, 0, 0, 1e-6, 1.0)))


def test_far_token(gpu, k3):
    """Rows past 2^32 bytes from their start."""
    say("case: far token")
    q = torch.zeros(3, 1 << 30, device="cuda", dtype=BF16)[:, :512].view(3, 4, 128)
    q.copy_(torch.randn(3, 4, 128, device="cuda", generator=lo.gen(1)))
    _, _, k, qw, kw, pos = inputs(3, 1, 1, 128, BF16, 9)
    check(k3, q, k, qw, kw, pos, freqs(128), 128)


@pytest.mark.parametrize("T", [1, 500])
def test_graph(gpu, k3, T):
    say(f"case: {T}")
    L = k3.lib()
    _, q, k, qw, kw, pos = inputs(T, 8, 2, 128, BF16, 10)
    f = freqs(128)
    qo, ko = torch.zeros(T, 8, 128, device="cuda", dtype=BF16), torch.zeros(T, 2, 128, device="cuda", dtype=BF16)
    torch.cuda.synchronize()
    st, ex = L.k3d_stream_create(), C.c_void_p()
    try:
        k3.check(L.k3d_graph_begin(st))
        lo.heads(k3, q, k, qw, kw, pos, f, 128, qo=qo, ko=ko, st=st)
        k3.check(L.k3d_graph_end(st, C.byref(ex)))
        for i in range(4):
            pos.add_(1)
            q.copy_(torch.randn(T, 8, 128, device="cuda", generator=lo.gen(40 + i)))
            want = lo.heads(k3, q, k, qw, kw, pos, f, 128)
            torch.cuda.synchronize()
            k3.check(L.k3d_graph_launch(ex, st))
            k3.check(L.k3d_sync(st))
            assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    finally:
        if ex:
            L.k3d_graph_destroy(ex)
        L.k3d_stream_destroy(st)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("dim", [4, 5, 7, 8, 9, 11, 15, 16, 17, 23, 31, 63, 65, 129, 255, 257, 519, 1021])
def test_any_borders(gpu, k3, dim, pairs, dtype):
    """Rotated ranges that begin, halve and end anywhere, at odd strides and starts, out of place and in place; what lies between the heads
    stays as it is."""
    for n, (rot, off) in enumerate([(dim // 2 * 2, dim % 2), (2, dim - 2), (dim // 4 * 2, 1), (dim // 6 * 2, dim // 3), (0, 0)]):
        say(f"case: {dim} {rot} {off} {pairs} {dtype}")
        T, hq, hk, hs = 6, 5, 2, dim + 1 + n
        ld = (hq + hk) * hs + 3
        g = lo.gen(dim + n)
        buf = torch.randn(T * ld + 5, device="cuda", generator=g).to(dtype)
        def views(b):
            rows = b[1 + n % 2:1 + n % 2 + T * ld].view(T, ld)[:, :(hq + hk) * hs].unflatten(1, (hq + hk, hs))
            return rows[:, :hq, :dim], rows[:, hq:, :dim]
        q, k = views(buf)
        qw = torch.rand(dim, device="cuda", generator=g) + 0.5
        pos = torch.randint(0, 5000, (T,), device="cuda", generator=g).int()
        pos[2] = -1
        on = torch.arange(T, device="cuda") != 2
        freq = freqs(rot) if rot else torch.ones(1, device="cuda", dtype=torch.float64)
        want = [lo.heads64(v[on], w, pos[on], freq, rot, off, pairs, 1e-6, 1.0) for v, w in ((q, qw), (k, None))]
        out = torch.full_like(buf, 7.0)
        qo, ko = views(out)
        was = buf.clone()
        lo.heads(k3, q, k, qw, None, pos, freq, rot, off, pairs, qo=qo, ko=ko)
        assert torch.equal(buf, was)
        for v, w in zip((qo, ko), want):
            lo.within(v[on], w)
            v[on] = 7.0
        assert (out == 7).all()                                    # the padding token and all between the heads
        lo.heads(k3, q, k, qw, None, pos, freq, rot, off, pairs, qo=q, ko=k)
        for v, u, w in zip((q, k), views(was), want):
            lo.within(v[on], w)
            v[on] = u[on]
        assert torch.equal(buf, was)
