# SPDX-License-Identifier: Apache-2.0
"""k3d_route against its definition in 64 bits: experts exactly, weights within their one rounding."""
import ctypes as C
import itertools

import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def say(msg):
    print(msg, flush=True)


def both(k3, lg, bias=None, score=0, groups=1, top_groups=1, group_top=1, topk=8, renorm=1, scale=1.0):
    got = lo.route(k3, lg, bias, score, groups, top_groups, group_top, topk, renorm, scale)
    lo.check_route(got, lo.route64(lg, bias, score, groups, top_groups, group_top, topk, renorm, scale))
    return got


def logits(T, n, seed, dtype=F32, sigma=1.5):
    return (torch.randn(T, n, device="cuda", generator=lo.gen(seed)) * sigma).to(dtype)


def biases(n, seed, sigma=0.05):
    return torch.randn(n, device="cuda", generator=lo.gen(seed)) * sigma


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("n,groups,top_groups,topk", [
    (1, 1, 1, 1), (2, 2, 1, 1), (16, 1, 1, 16), (60, 1, 1, 4), (64, 8, 3, 6), (64, 64, 9, 9), (65, 5, 2, 7), (128, 1, 1, 8),
    (130, 10, 10, 64), (160, 8, 3, 6), (192, 3, 1, 64), (256, 8, 4, 8), (257, 1, 1, 12), (384, 8, 4, 8), (500, 20, 6, 10), (513, 27, 4, 9),
    (823, 1, 1, 6), (896, 8, 4, 16), (896, 1, 1, 64), (1024, 32, 5, 24), (1025, 41, 2, 3), (1500, 1, 1, 24), (2047, 1, 1, 33),
    (2048, 64, 7, 64), (2048, 1, 1, 1)])
def test_shapes(gpu, k3, n, groups, top_groups, topk, score):
    say(f"case: {n} {groups} {top_groups} {topk} {score}")
    for T, dtype, use in ((1, F32, True), (3, BF16, False), (130, F32, False), (67, BF16, True)):
        b = biases(n, n) if use else None
        for group_top in (1, 2):
            both(k3, logits(T, n, n + T, dtype), b, score, groups, top_groups, group_top, topk, 1, 2.5)
    both(k3, logits(5, n, 3), None, score, groups, top_groups, 1, topk, 0, 1.0)


@pytest.mark.parametrize("T", [1023, 1024, 4099])
@pytest.mark.parametrize("score,groups,dtype", [(0, 8, F32), (1, 1, BF16), (1, 8, F32), (0, 1, BF16)])
def test_many_tokens(gpu, k3, T, score, groups, dtype):
    say(f"case: {T} {score} {groups}")
    both(k3, logits(T, 384, T, dtype), biases(384, 1), score, groups, max(1, groups // 2), 2, 8, 1, 1.0)


@pytest.mark.parametrize("score,groups", itertools.product([0, 1], [1, 8]))
@pytest.mark.parametrize("n", [64, 384, 896, 2048])
def test_ties(gpu, k3, score, groups, n):
    """Equal choices go to the lower expert, equal groups to the lower group: a few distinct values, all
    equal, all zero (a padded token's logits), equal pairs far apart."""
    say(f"case: {n} {score} {groups}")
    g = lo.gen(n)
    few = torch.randint(0, 3, (20, n), device="cuda", generator=g).float()
    far = logits(4, n, 5)
    far[:, n - 7:] = far[:, :7]
    lg = torch.cat([few, torch.zeros(2, n, device="cuda"), torch.full((1, n), 2.5, device="cuda"), far,
                    torch.arange(n, device="cuda").float()[None] / 64, -torch.arange(n, device="cuda").float()[None] / 64])
    for b in (None, torch.zeros(n, device="cuda"), (torch.arange(n, device="cuda") % 5).float()):
        for topk in (1, 8, min(64, n // groups * max(1, groups // 2))):
            both(k3, lg, b, score, groups, max(1, groups // 2), 2, topk)
            both(k3, lg.to(BF16), b, score, groups, max(1, groups // 2), 1, topk)


@pytest.mark.parametrize("score", [0, 1])
def test_close(gpu, k3, score):
    """Choices a few units of fp32 apart, and closer: 64 bits tell them, in experts and in groups."""
    say(f"case: {score}")
    n = 256
    base = torch.full((40, n), 0.75, device="cuda")
    ulps = torch.randint(-3, 4, (40, n), device="cuda", generator=lo.gen(1))
    lg = (base.view(torch.int32) + ulps.int()).view(F32)
    b = torch.randint(-4, 5, (n,), device="cuda", generator=lo.gen(2)).float() * 2.0 ** -27
    for bias in (None, b):
        for groups in (1, 8):
            both(k3, lg, bias, score, groups, max(1, groups // 2), 2, 16)


@pytest.mark.parametrize("score,groups", itertools.product([0, 1], [1, 8]))
def test_masked(gpu, k3, score, groups):
    """Experts that cannot be taken: some, all but a few, all; as logits of -inf or NaN and as biases."""
    say(f"case: {score} {groups}")
    n, k = 128, 8
    lg = logits(12, n, 7)
    lg[0] = -INF
    lg[1] = NAN
    lg[2, 3:] = -INF
    lg[3, ::2] = -INF
    lg[4, 5] = NAN
    lg[5, 9:20] = INF
    lg[6, :60] = -INF
    lg[7] = torch.finfo(F32).min
    lg[8, :] = -INF
    lg[8, 100] = 0.5
    lg[9, 64:] = NAN
    lg[10] = INF
    lg[11] *= 60                                              # saturated both ways
    for bias in (None, biases(n, 1), torch.where(torch.arange(n, device="cuda") % 3 == 0, -INF, 0.1),
                 torch.where(torch.arange(n, device="cuda") < 30, NAN, -0.3), torch.full((n,), -INF, device="cuda"),
                 torch.where(torch.arange(n, device="cuda") == 77, INF, 0.0)):
        for group_top in (1, 2):
            for renorm in (0, 1):
                both(k3, lg, bias, score, groups, max(1, groups // 4), group_top, k, renorm)
    if score == 0:                                            # (a token whose weights sum to nothing)
        idx, wt = lo.route(k3, torch.full((1, n), -2000.0, device="cuda"), topk=4)
        assert idx.tolist() == [[0, 1, 2, 3]] and wt.tolist() == [[0, 0, 0, 0]]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_neighbours(gpu, k3, dtype):
    """Rows inside a wider buffer at any alignment; nothing beside idx and wt is written."""
    say(f"case: {dtype}")
    for n, ld, off in ((60, 61, 1), (384, 400, 3), (896, 1793, 8)):
        buf = torch.full((70 * ld + off,), 50.0, device="cuda", dtype=dtype)
        lg = buf[off:].view(70, ld)[:, :n]
        lg.copy_(logits(70, n, n))
        idx = torch.full((71, 6), -9, device="cuda", dtype=torch.int32)
        wt = torch.full((71, 6), -9.0, device="cuda")
        lo.route(k3, lg, topk=6, idx=idx[:70], wt=wt[:70])
        lo.check_route((idx[:70], wt[:70]), lo.route64(lg, None, 0, 1, 1, 1, 6, 1, 1.0))
        assert (idx[70] == -9).all() and (wt[70] == -9).all()


def test_far_row(gpu, k3):
    """A row past 2^32 bytes from the start."""
    say("case: far row")
    lg = torch.zeros(3, 1 << 30, device="cuda", dtype=F32)[:, :200]
    lg.copy_(logits(3, 200, 1))
    both(k3, lg, topk=5)


@pytest.mark.parametrize("T,n,groups", [(1, 384, 8), (100, 896, 1), (2000, 256, 8)])
def test_graph(gpu, k3, T, n, groups):
    say(f"case: {T}")
    L = k3.lib()
    lg, b = logits(T, n, 1), biases(n, 2)
    idx = torch.zeros(T, 8, device="cuda", dtype=torch.int32)
    wt = torch.zeros(T, 8, device="cuda")
    torch.cuda.synchronize()
    st, ex = L.k3d_stream_create(), C.c_void_p()
    try:
        k3.check(L.k3d_graph_begin(st))
        lo.route(k3, lg, b, 1, groups, max(1, groups // 2), 2, 8, idx=idx, wt=wt, st=st)
        k3.check(L.k3d_graph_end(st, C.byref(ex)))
        for i in range(4):
            lg.copy_(logits(T, n, 30 + i))
            want = lo.route(k3, lg, b, 1, groups, max(1, groups // 2), 2, 8)
            torch.cuda.synchronize()
            k3.check(L.k3d_graph_launch(ex, st))
            k3.check(L.k3d_sync(st))
            assert torch.equal(idx, want[0]) and torch.equal(wt, want[1])
    finally:
        if ex:
            L.k3d_graph_destroy(ex)
        L.k3d_stream_destroy(st)
