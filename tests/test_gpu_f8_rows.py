# SPDX-License-Identifier: Apache-2.0
"""k3d_add_norm and k3d_quant_f8 against 64 bits."""
import numpy as np
import pytest
import torch

from layer8_ops import (BF16, F32, HALF, NONE, SILU, SITU, add_norm, check_codes, codes_of, f64, glu64, nb, norm64, quant, rows_for)
from layer_ops import gen, within

pytestmark = pytest.mark.gpu
SIZES = (1, 7, 8, 100, 127, 128, 129, 511, 512, 513, 1000, 1024, 1536, 2048, 2050, 4096, 5001, 7168, 8192, 8200, 16384, 20001, 65536)


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("x_type,r_type", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
def test_norm(gpu, n, x_type, r_type):
    g = gen(n)
    for T in (1, 3, 600) if n <= 8200 else (1, 5):
        # views: rows of odd strides from odd places
        x = torch.randn(T, n + 3, device="cuda", generator=g).to(x_type)[:, 1:n + 1]
        res = (torch.randn(T, n + 1, device="cuda", generator=g) * 3).to(r_type)[:, :n]
        w = torch.randn(n + 1, device="cuda", generator=g)[1:] * 0.1 + 1
        q, qs = rows_for(T, n, nb(n) * 128 + 16, nb(n) + 3)
        y = torch.full((T, n + 5), 7.0, device="cuda", dtype=r_type)
        s = torch.full((T, n + 2), 7.0, device="cuda", dtype=r_type)
        add_norm(gpu, x, res, w, y=y[:, 2:n + 2], q=q, qs=qs, sum_=s[:, 1:n + 1], n=n)
        v, u, tol = norm64(x, res, w, 1e-6)
        within(s[:, 1:n + 1], (v, np.abs(v) * (HALF[r_type] + 2.0 ** -24) * 1.001))
        within(y[:, 2:n + 2], (u, tol + (np.abs(u) + tol) * HALF[r_type]))
        check_codes(q, qs, u, tol, n)
        # nothing but the rows
        for t, a, b in ((y, 2, n + 2), (s, 1, n + 1)):
            assert (t[:, :a] == 7).all() and (t[:, b:] == 7).all()
        assert (q[:, nb(n) * 128:] == 0x7f).all() and torch.isnan(qs[:, nb(n):]).all()


def test_norm_parts(gpu):
    """Without a residual, a weight, one or the other output; in place."""
    g = gen(5)
    x = torch.randn(9, 1000, device="cuda", generator=g)
    res = torch.randn(9, 1000, device="cuda", generator=g)
    v, u, tol = norm64(x, None, None, 1e-5)
    q, qs = rows_for(9, 1000)
    add_norm(gpu, x, eps=1e-5, q=q, qs=qs)
    check_codes(q, qs, u, tol, 1000)
    y = torch.empty(9, 1000, device="cuda", dtype=BF16)
    add_norm(gpu, x, eps=1e-5, y=y)
    within(y, (u, tol + (np.abs(u) + tol) * HALF[BF16]))
    s = torch.empty(9, 1000, device="cuda", dtype=BF16)
    add_norm(gpu, x, sum_=s)
    assert torch.equal(s, x.to(BF16))
    # the sum in the residual's place, in x's, and y in x's
    v, u, tol = norm64(x, res, None, 1e-6)
    for place in (res.clone(), x.clone()):
        q1, qs1 = rows_for(9, 1000)
        if torch.equal(place, res):
            add_norm(gpu, x, place, q=q1, qs=qs1, sum_=place)
        else:
            add_norm(gpu, place, res, q=q1, qs=qs1, sum_=place)
        assert torch.equal(place, x + res)
        check_codes(q1, qs1, u, tol, 1000)
    place = x.clone()
    add_norm(gpu, place, res, y=place)
    within(place, (u, tol + (np.abs(u) + tol) * HALF[F32]))


@pytest.mark.parametrize("n", [128, 1000, 7168])
def test_norm_values(gpu, n):
    """Zero rows, tiny and large ones, eps alone, NaN and infinities in one block."""
    g = gen(n)
    x = torch.randn(8, n, device="cuda", generator=g)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e15
    x[3] *= 1e-4
    q, qs = rows_for(8, n)
    add_norm(gpu, x, q=q, qs=qs)
    v, u, tol = norm64(x, None, None, 1e-6)
    check_codes(q, qs, u, tol + 2.0 ** -126, n)
    assert (q[0] == 0).all()
    x[5, 3] = float("nan")
    x[6, 100] = float("inf")
    add_norm(gpu, x, q=q, qs=qs)
    c = codes_of(q) * np.repeat(f64(qs), 128, 1)
    assert np.isnan(c[5, :n]).all()                     # the mean of its squares is NaN
    assert np.isnan(c[6, 100]) and (np.isnan(c[6, :128]).any())
    check_codes(q[:5], qs[:5], u[:5], tol[:5] + 2.0 ** -126, n)
    check_codes(q[7:], qs[7:], u[7:], tol[7:], n)


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("act", [NONE, SITU, SILU])
def test_quant(gpu, n, act):
    g = gen(n)
    for x_type in (F32, BF16):
        T = 37 if n <= 8200 else 3
        wide = n * (1 if act == NONE else 2)
        x = (torch.randn(T, wide + 3, device="cuda", generator=g) * 3).to(x_type)[:, 1:wide + 1]
        q, qs = rows_for(T, n, nb(n) * 128 + 32, nb(n) + 1)
        quant(gpu, x, n, act, q=q, qs=qs)
        v = f64(x)
        if act == NONE:
            u, tol = v, np.zeros_like(v)
        else:
            u = glu64(v[:, :n], v[:, n:], act, 4.0, 25.0)
            tol = 2.0 ** -20 * np.abs(u)
        check_codes(q, qs, u, tol, n)
        assert (q[:, nb(n) * 128:] == 0x7f).all() and torch.isnan(qs[:, nb(n):]).all()


def test_quant_exact(gpu):
    """Values that are codes times a power of two come back as they are; halves between two codes go to the even one; every finite
    code occurs."""
    from layer8_ops import F8
    codes = torch.arange(256, device="cuda", dtype=torch.uint8)
    fine = torch.cat((codes[:127], codes[128:255]))
    for e in (-90, -3, 0, 20):
        x = torch.full((1, 256), 448.0, device="cuda")
        x[0, :254] = fine.view(F8).float()
        q, qs = quant(gpu, x * 2.0 ** e)
        assert (qs == 2.0 ** e).all()
        assert torch.equal(q.view(F8).float(), x)
    v = codes[:126].view(F8).float()
    mid = (v[:-1] + v[1:]) / 2
    x = torch.full((1, 128), 448.0, device="cuda")
    x[0, :mid.numel() - 1] = mid[:-1]
    q, qs = quant(gpu, x)
    even = torch.where(codes[:124] % 2 == 0, codes[:124], codes[1:125])
    assert torch.equal(q[0, :124], even)


def test_quant_values(gpu):
    """Zeros, values below the least scale, subnormals, the largest, NaN and infinities, far gates."""
    x = torch.zeros(8, 256, device="cuda")
    x[1] = 2.0 ** -110
    x[2, 5] = 2.0 ** -140
    x[3] = 3e38
    x[4, 7] = float("nan")
    x[5, 200] = float("-inf")
    x[6] = torch.linspace(-1, 1, 256, device="cuda") * 1e-30
    q, qs = quant(gpu, x)
    keep = [0, 1, 2, 3, 6, 7]
    check_codes(q[keep], qs[keep], f64(x)[keep], np.zeros((6, 256)), 256)
    c = codes_of(q) * np.repeat(f64(qs), 128, 1)
    assert np.isnan(c[4, :128]).all() and (c[4, 128:] == 0).all()
    assert (c[5, :128] == 0).all() and np.isnan(c[5, 200])
    # gates past where e^-g leaves fp32, up large: silu(g) up is still a number of the range
    g = torch.tensor([-95.0, -90.0, -100.0, -50.0, 80.0, 100.0, 1e30, 0.0] * 16, device="cuda")
    u = torch.full((128,), 2.0 ** 100, device="cuda")
    u[4:7] = 1e-3
    u[6::8] = 1e-20
    x = torch.cat((g, u))[None]
    for act in (SILU, SITU):
        q, qs = quant(gpu, x, act=act)
        want = glu64(f64(x)[:, :128], f64(x)[:, 128:], act, 4.0, 25.0)
        check_codes(q, qs, want, 2.0 ** -19 * np.abs(want), 128)
    # tiny arguments keep their precision through tanh
    x = torch.randn(4, 256, device="cuda", generator=gen(3)) * 1e-5
    q, qs = quant(gpu, x, act=SITU)
    want = glu64(f64(x)[:, :128], f64(x)[:, 128:], SITU, 4.0, 25.0)
    check_codes(q, qs, want, 2.0 ** -20 * np.abs(want), 128)
