# SPDX-License-Identifier: Apache-2.0
"""k3d_f8_tile, k3d_linear_f8, k3d_group, k3d_grouped_f8 and k3d_moe_f8 against 64 bits."""
import numpy as np
import pytest
import torch

from layer8_ops import (ACTS, BF16, F32, HALF, SILU, SITU, acts, codes_of, f64, group, group64, grouped, linear8, linear8_64, moe64, moe8,
                        nb, product64, rows64, tile, weights, weights64)
from layer_ops import gen, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out,inn", [(1, 1), (16, 128), (17, 129), (128, 128), (129, 1000), (300, 16), (257, 511)])
def test_tile(gpu, out, inn):
    """Every code in its place, zeros around; a stride and an odd address."""
    g = gen(out)
    w = torch.randint(0, 256, (2 * out * (inn + 5) + 1,), device="cuda", generator=g, dtype=torch.uint8)
    W = w[1:].view(2, out, inn + 5)
    t = tile(gpu, W[:, :, :inn], inn + 5).view(2, nb(out), nb(inn), 8, 2, 4, 16, 16)
    # [mat][row block][column block][row tile][half][piece of four][row][byte]
    full = torch.zeros(2, nb(out) * 128, nb(inn) * 128, device="cuda", dtype=torch.uint8)
    full[:, :out, :inn] = W[:, :, :inn]
    want = full.view(2, nb(out), 8, 16, nb(inn), 2, 4, 16).permute(0, 1, 4, 2, 5, 6, 3, 7)
    assert torch.equal(t, want)


LIN = [(1, 128, 16), (1, 1, 1), (2, 130, 17), (3, 7168, 300), (8, 256, 128), (9, 1000, 100), (16, 4096, 512), (17, 1001, 300),
       (31, 7168, 40), (33, 640, 129), (48, 2304, 777), (64, 8320, 256), (64, 128, 64), (65, 128, 64), (100, 1001, 300), (128, 2048, 128),
       (129, 512, 4096), (200, 7168, 384), (300, 129, 2047), (513, 1280, 257), (1000, 640, 1000), (2048, 512, 8192), (4097, 256, 4095), (7, 33000, 130), (70, 9000, 300)]


@pytest.mark.parametrize("T,inn,out", LIN)
def test_linear_exact(gpu, T, inn, out):
    """Integers with scales of powers of two: every sum is exact in fp32, in any order."""
    g = gen(T + inn)
    x, xs = acts(g, T, inn, True, nb(inn) * 128 + 32, nb(inn) + 3)
    w, ws = weights(g, 1, out, inn, True)
    y = torch.full((T, out + 3), 7.0, device="cuda")
    linear8(gpu, x, xs, tile(gpu, w), ws, inn, out, y=y[:, 1:out + 1])
    want = rows64(x[:, :nb(inn) * 128], xs[:, :nb(inn)], inn) @ weights64(w[0], ws[0]).T
    assert np.array_equal(f64(y[:, 1:out + 1]), want)
    assert (y[:, 0] == 7).all() and (y[:, out + 1:] == 7).all()


@pytest.mark.parametrize("T,inn,out", LIN)
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_linear(gpu, T, inn, out, y_type):
    g = gen(T * 7 + inn)
    x, xs = acts(g, T, inn)
    w, ws = weights(g, 1, out, inn)
    wt = tile(gpu, w)
    bias = torch.randn(out + 1, device="cuda", generator=g)[1:]
    res = torch.randn(T, out + 1, device="cuda", generator=g).to(y_type)[:, 1:]
    X, W = rows64(x, xs, inn), weights64(w[0], ws[0])
    i = (T + inn) % 5
    within(linear8(gpu, x, xs, wt, ws, inn, out, y_type=y_type), linear8_64(X, W, None, "none", None, y_type))
    got = linear8(gpu, x, xs, wt, ws, inn, out, bias, ACTS[i], res)
    if T * out <= 1 << 20:
        within(got, linear8_64(X, W, bias, ACTS[i], res, y_type))
    # the residual in y's place, and the same bits again
    place = res.clone()
    assert torch.equal(linear8(gpu, x, xs, wt, ws, inn, out, bias, ACTS[i], place, y=place), got)


@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("out", [4090, 8187, 12281])
def test_linear_few_rows_wide(gpu, out, y_type):
    """One to three tiles of W a workgroup, each number of pieces of x: exact integers (a bf16 result is their rounding)."""
    g = gen(out)
    inn = 700
    w, ws = weights(g, 1, out, inn, True)
    wt = tile(gpu, w)
    W = torch.from_numpy(weights64(w[0], ws[0])).cuda()
    for T in (1, 16, 17, 32, 33, 48, 49, 64):
        x, xs = acts(g, T, inn, True)
        want = torch.from_numpy(rows64(x, xs, inn)).cuda() @ W.T
        y = torch.full((T + 1, out), 7.0, device="cuda", dtype=y_type)
        linear8(gpu, x, xs, wt, ws, inn, out, y=y[:T])
        assert torch.equal(y[:T], want.to(y_type)) and (y[T:] == 7).all(), T


def test_linear_values(gpu):
    """A NaN code or scale stays with its row; rows and outputs that end inside a block take nothing of their neighbours."""
    for T in (5, 40, 300):
        g = gen(T)
        x, xs = acts(g, T, 300)
        w, ws = weights(g, 1, 200, 300)
        clean = linear8(gpu, x, xs, tile(gpu, w), ws, 300, 200)
        x[3, 17] = 0x7f
        xs[1, 2] = float("inf")
        w[0, 150, 299] = 0xff
        y = linear8(gpu, x, xs, tile(gpu, w), ws, 300, 200)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[3] = True
        bad[:, 150] = True
        assert torch.isnan(y[bad]).all()
        bad[1] = True
        assert not torch.isfinite(y[1]).any()
        assert torch.equal(y[~bad], clean[~bad])


# ----------------------------------------------------------------- experts ----
@pytest.mark.parametrize("T,k,experts", [(1, 1, 1), (1, 8, 384), (5, 3, 4), (64, 8, 384), (100, 64, 2048), (512, 8, 64), (513, 8, 64),
                                         (4096, 8, 384), (4096, 2, 2048), (20000, 1, 3)])
def test_group(gpu, T, k, experts):
    g = gen(T + k)
    idx = torch.randint(-2, experts + 2, (T, k), device="cuda", generator=g, dtype=torch.int32)
    off, perm = group(gpu, idx, experts)
    o, p = group64(idx, experts)
    assert np.array_equal(off.cpu().numpy(), o)
    assert np.array_equal(perm.cpu().numpy()[:len(p)], p) and (perm[len(p):] == -7).all()


def test_group_one_expert_and_none(gpu):
    for v in (2, -1, 5):
        idx = torch.full((700, 8), v, device="cuda", dtype=torch.int32)
        off, perm = group(gpu, idx, 5)
        o, p = group64(idx, 5)
        assert np.array_equal(off.cpu().numpy(), o) and np.array_equal(perm.cpu().numpy()[:len(p)], p)


def counts_to_offsets(n):
    return torch.tensor(np.concatenate(([0], np.cumsum(n))), device="cuda", dtype=torch.int32)


GROUPED = [([0, 1, 0], 128, 16), ([3], 130, 17), ([1, 0, 2, 7, 8, 9, 0, 0, 15], 256, 130), ([16, 17, 31, 0, 33, 1], 1001, 300),
           ([64, 65, 0, 1, 30], 640, 128), ([100, 0, 127, 128, 129, 5, 300], 384, 257), ([256, 257, 600, 0, 1], 512, 520),
           ([0] * 70 + [4] + [0] * 60 + [2, 3], 200, 40), ([1] * 384, 128, 33), ([2000, 0, 0, 1], 256, 128), ([0, 0], 128, 128), ([2] * 64, 128, 2040), ([12, 30, 1, 0, 17], 4200, 2040)]


@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_grouped_exact(gpu, case):
    """Exact integers; rows through a map of x and into a map of y; what no row has is left as it was."""
    counts, inn, out = GROUPED[case]
    g = gen(case)
    rows, e = sum(counts), len(counts)
    off = counts_to_offsets(counts)
    w, ws = weights(g, e, out, inn, True)
    wt = tile(gpu, w)
    tokens = max(1, rows // 2)
    x, xs = acts(g, tokens, inn, True, nb(inn) * 128 + 16, nb(inn) + 1)
    x_rows = torch.randint(0, tokens * 3, (rows + 1,), device="cuda", generator=g, dtype=torch.int32)
    y_rows = torch.randperm(rows + 5, device="cuda", generator=g).to(torch.int32)
    X = rows64(x[:, :nb(inn) * 128], xs[:, :nb(inn)], inn)
    want = np.full((rows + 5, out), 7.0)
    at = np.repeat(np.arange(e), counts)
    for i in range(e):
        r = np.nonzero(at == i)[0]
        if len(r):
            want[y_rows.cpu().numpy()[r]] = X[x_rows.cpu().numpy()[r] // 3] @ weights64(w[i], ws[i]).T
    y = torch.full((rows + 5, out + 3), 7.0, device="cuda")
    grouped(gpu, y[:, :out], x, xs, off, max(1, rows), wt, ws, inn, out, x_rows, 3, y_rows)
    assert np.array_equal(f64(y[:, :out]), want) and (y[:, out:] == 7).all()
    # in rows' own order, with more room than there are rows
    if rows:
        x, xs = acts(g, rows, inn, True)
        X = rows64(x, xs, inn)
        y = torch.full((rows + 9, out), 7.0, device="cuda")
        grouped(gpu, y, x, xs, off, rows + 1000, wt, ws, inn, out)
        want = np.full((rows + 9, out), 7.0)
        for i in range(e):
            r = np.nonzero(at == i)[0]
            if len(r):
                want[r] = X[r] @ weights64(w[i], ws[i]).T
        assert np.array_equal(f64(y), want)


def test_grouped_bounds(gpu):
    """Rows that name no row of x or y, and offsets that fall, leave what they would have written as it was."""
    g = gen(1)
    for n in (6, 200):
        w, ws = weights(g, 3, 64, 128, True)
        wt = tile(gpu, w)
        x, xs = acts(g, 10, 128, True)
        x_rows = torch.randint(-3, 14, (n,), device="cuda", generator=g, dtype=torch.int32)
        y_rows = torch.arange(n, device="cuda", dtype=torch.int32)
        y_rows[1], y_rows[3] = -1, n + 100
        y = torch.full((n, 64), 7.0, device="cuda")
        off = torch.tensor([0, n // 2, n // 2, n + 50], device="cuda", dtype=torch.int32)
        grouped(gpu, y, x, xs, off, n, wt, ws, 128, 64, x_rows, 1, y_rows)
        X, xr = rows64(x, xs, 128), x_rows.cpu().numpy()
        want = np.full((n, 64), 7.0)
        for r in range(n):
            if 0 <= xr[r] < 10 and r not in (1, 3):
                e = 0 if r < n // 2 else 2
                want[r] = X[xr[r]] @ weights64(w[e], ws[e]).T
        assert np.array_equal(f64(y), want)
        y.fill_(7.0)
        off = torch.tensor([-4, n + 7, 2, 1], device="cuda", dtype=torch.int32)
        grouped(gpu, y, x, xs, off, n, wt, ws, 128, 64)
        assert (y == 7).all()
        # rows in their own order of which x has only the first ten
        off = torch.tensor([0, n // 3, n // 2, n], device="cuda", dtype=torch.int32)
        grouped(gpu, y, x, xs, off, n, wt, ws, 128, 64)
        want = np.full((n, 64), 7.0)
        for r in range(min(n, 10)):
            want[r] = X[r] @ weights64(w[(r >= n // 3) + (r >= n // 2)], ws[(r >= n // 3) + (r >= n // 2)]).T
        assert np.array_equal(f64(y), want)


@pytest.mark.parametrize("y_type", [F32, BF16])
def test_grouped(gpu, y_type):
    g = gen(11)
    for counts, inn, out in ((rng_counts(g, 40, 3), 7168, 256), (rng_counts(g, 8, 60), 1000, 300), (rng_counts(g, 5, 300), 2048, 520)):
        rows, e = sum(counts), len(counts)
        off = counts_to_offsets(counts)
        w, ws = weights(g, e, out, inn)
        x, xs = acts(g, rows, inn)
        y = torch.empty(rows, out, device="cuda", dtype=y_type)
        grouped(gpu, y, x, xs, off, rows, tile(gpu, w), ws, inn, out)
        X, at = rows64(x, xs, inn), np.repeat(np.arange(e), counts)
        for i in range(e):
            r = np.nonzero(at == i)[0]
            if len(r):
                v, tol = product64(X[r], weights64(w[i], ws[i]), y_type == BF16)
                within(y[torch.from_numpy(r).cuda()], (v, tol + (np.abs(v) + tol) * HALF[y_type]))


def rng_counts(g, e, most):
    return torch.randint(0, 2 * most, (e,), device="cuda", generator=g).tolist()


MOE = [(1, 8, 16, 256, 128, SILU), (1, 1, 1, 100, 30, SITU), (1, 8, 3, 200, 130, SITU), (1, 64, 70, 300, 200, SILU), (5, 2, 4, 130, 200, SITU), (33, 8, 12, 512, 384, SILU), (64, 4, 3, 384, 256, SITU),
       (200, 2, 3, 256, 300, SILU)]


@pytest.mark.parametrize("T,k,experts,hidden,inter,act", MOE)
@pytest.mark.parametrize("out_type", [F32, BF16])
def test_moe(gpu, T, k, experts, hidden, inter, act, out_type):
    g = gen(T + hidden)
    x, xs = acts(g, T, hidden)
    w = [weights(g, experts, o, i) for o, i in ((inter, hidden), (inter, hidden), (hidden, inter))]
    bank = [(tile(gpu, q), s) for q, s in w]
    idx = torch.randint(-1, experts + 1, (T, k), device="cuda", generator=g, dtype=torch.int32)
    if T > 2:
        idx[2] = -1
    wt = torch.rand(T, k, device="cuda", generator=g)
    out = torch.full((T, hidden + 3), 7.0, device="cuda", dtype=out_type)
    moe8(gpu, x, xs, idx, wt, bank, hidden, inter, act, out=out[:, 1:hidden + 1])
    W = [np.stack([weights64(q[e], s[e]) for e in range(experts)]) for q, s in w]
    y, tol = moe64(rows64(x, xs, hidden), idx, wt, *W, act, 4.0, 25.0, out_type)
    within(out[:, 1:hidden + 1], (y, tol + (np.abs(y) + tol) * HALF[out_type]))
    assert (out[:, 0] == 7).all() and (out[:, hidden + 1:] == 7).all()
    if T > 2:
        assert (out[2, 1:hidden + 1] == 0).all()


def test_moe_is_its_parts(gpu):
    """The layer gives what its parts give one after another, rounded alike (sums of integers, exact in every instruction)."""
    from layer8_ops import quant
    g = gen(2)
    for T in (1, 3, 70, 400):
        k, experts, hidden, inter = 4, 6, 512, 256
        x, xs = acts(g, T, hidden, True)
        w = [weights(g, experts, o, i, True) for o, i in ((inter, hidden), (inter, hidden), (hidden, inter))]
        bank = [(tile(gpu, q), s) for q, s in w]
        idx = torch.stack([torch.randperm(experts, device="cuda", generator=g)[:k] for _ in range(T)]).to(torch.int32)
        wt = torch.rand(T, k, device="cuda", generator=g)
        out = moe8(gpu, x, xs, idx, wt, bank, hidden, inter, SITU)
        off, perm = group(gpu, idx, experts)
        gu = torch.empty(T * k, 2 * inter, device="cuda")
        grouped(gpu, gu[:, :inter], x, xs, off, T * k, *bank[0], hidden, inter, perm, k)
        grouped(gpu, gu[:, inter:], x, xs, off, T * k, *bank[1], hidden, inter, perm, k)
        hq, hs = quant(gpu, gu, act=SITU)
        y = torch.empty(T * k, hidden, device="cuda")
        grouped(gpu, y, hq, hs, off, T * k, *bank[2], inter, hidden, y_rows=perm)
        want = f64(y).reshape(T, k, hidden) * f64(wt)[:, :, None]
        S = np.abs(want).sum(1)
        assert (np.abs(f64(out) - want.sum(1)) <= S * 2.0 ** -20).all()


@pytest.mark.parametrize("T", [1, 5, 300])
@pytest.mark.parametrize("out_type", [F32, BF16])
def test_moe_values(gpu, T, out_type):
    """A token that is no number stays alone with it, a token without experts is zero, and the same expert twice counts twice."""
    g = gen(T)
    k, experts, hidden, inter = 3, 4, 384, 256
    x, xs = acts(g, T, hidden)
    bank = [(tile(gpu, q), s) for q, s in (weights(g, experts, o, i) for o, i in ((inter, hidden), (inter, hidden), (hidden, inter)))]
    idx = torch.randint(0, experts, (T, k), device="cuda", generator=g, dtype=torch.int32)
    wt = torch.rand(T, k, device="cuda", generator=g)
    at = T // 2
    idx[at] = torch.tensor([-1, experts, -2 ** 31], dtype=torch.int32)
    assert (moe8(gpu, x, xs, idx, wt, bank, hidden, inter, out_type=out_type)[at] == 0).all()
    idx[at] = torch.tensor([1, 1, -1], dtype=torch.int32)
    clean = moe8(gpu, x, xs, idx, wt, bank, hidden, inter, out_type=out_type)
    once, both = idx.clone(), wt.clone()
    once[at, 1], both[at, 0] = -1, wt[at, 0] + wt[at, 1]
    y = moe8(gpu, x, xs, once, both, bank, hidden, inter, out_type=out_type)
    # (the two weights' sum and the two products are rounded, and then the result)
    d = np.abs(f64(y[at]) - f64(clean[at]))
    assert (d <= np.abs(f64(clean[at])) * (2.0 ** -22 + 2 * HALF[out_type])).all()
    for bad in (float("nan"), float("inf")):
        s = xs.clone()
        s[at, 1] = bad
        y = moe8(gpu, x, s, idx, wt, bank, hidden, inter, out_type=out_type)
        assert torch.isnan(y[at]).all()
        y[at] = clean[at]
        assert torch.equal(y, clean)
