# SPDX-License-Identifier: Apache-2.0
"""k3d_linear on integers whose products and sums fp32 holds exactly in any order, so that one result only is right: a step of
the columns, a term or a stage that is lost, read too early or counted twice shows as a wrong number."""
import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)


def rows(n, inn, dtype, pad=0, off=0):
    """[n][inn] with `pad` elements between the rows and `off` before the first; NaN there."""
    b = torch.full((n * (inn + pad) + off + 8,), float("nan"), device="cuda", dtype=dtype)
    return b[off:off + n * (inn + pad)].view(n, inn + pad)[:, :inn]


@pytest.mark.parametrize("T,out", [(100, 130), (1500, 2000)])
@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("steps", list(range(1, 14)) + [31, 32, 33])
def test_any_number_of_steps(gpu, k3, T, out, x_type, steps):
    """Weights that are not 16-byte rows, through registers: every number of 64-column steps behind the rounds of a ring, in few
    tiles and in many, with the row's end inside the last step and at it."""
    for inn in (64 * steps, 64 * steps + 59 - 64 * (steps > 1)):
        say(f"case: {T} x {inn} -> {out} {x_type}")
        x, w = rows(T, inn, x_type, pad=1), rows(out, inn, BF16, pad=1, off=1)
        x.copy_(torch.randint(-60, 61, x.shape, device="cuda", generator=lo.gen(steps)))
        w.copy_(torch.randint(-3, 4, w.shape, device="cuda", generator=lo.gen(steps + 100)))
        for _ in range(2):
            assert torch.equal(lo.linear(k3, x, w).double(), x.double() @ w.double().T)


def terms(x):
    """fp32 as the sum of three of 8 significant bits each, by truncation."""
    cut = lambda v: (v.contiguous().view(torch.int32) & -65536).view(F32)
    h = cut(x)
    m = cut(x - h)
    return h, m, x - h - m


KERNELS = [(1, 7168, 7168), (6, 4096, 4096), (14, 2048, 8192), (22, 7168, 896), (30, 2048, 2048), (38, 12288, 4100), (46, 512, 16384),
           (60, 8192, 6400), (64, 7168, 7000), (96, 7168, 7168), (200, 7168, 2048), (1024, 2048, 2048), (1500, 1024, 3584),
           (2048, 2048, 4096), (4096, 1024, 4096), (300, 7168, 384), (1000, 7168, 130)]
FEW = [(T, inn, out) for T in (8, 13, 32, 48, 62) for inn, out in ((1024, 2000), (512, 5200), (1024, 8200), (8192, 6400), (4096, 12300), (16384, 3500))]
TAILS = [(8, 1032, 8200), (13, 4104, 12300), (30, 2056, 5200), (60, 8200, 6400), (46, 136, 130), (4100, 520, 2050), (1030, 1096, 12304),
         (1030, 1032, 4096), (700, 7176, 896), (200, 7176, 896), (300, 1032, 4096), (300, 264, 1160), (2000, 1024, 2051),
         (2001, 800, 4099), (513, 960, 1021)]
SMALL = [(1, 1, 1), (2, 31, 17), (9, 40, 48), (16, 48, 20), (100, 7, 9), (20, 128, 40), (1, 64, 64), (300, 1001, 77), (128, 72, 256)]


@pytest.mark.parametrize("T,inn,out,pad,off", [s + (0, 0) for s in KERNELS + FEW + TAILS + SMALL] + [s + (1, 1) for s in KERNELS[::2] + TAILS[::3] + SMALL] +
                         [s + (4, 0) for s in TAILS + SMALL])
def test_all_of_fp32(gpu, k3, T, inn, out, pad, off):
    """fp32 activations that need all 24 bits (or 21): integers of three parts, none of them zero, one for each term, and weights that are zero but for
    a few of a row, so that every sum is exact. Without the third term no result would be right, which is checked of the operands."""
    say(f"case: {T} x {inn} -> {out} pad {pad} off {off}")
    g = lo.gen(T + inn + out)
    x, w = rows(T, inn, F32, pad=pad), rows(out, inn, BF16, pad=8 * pad, off=off)
    o = torch.arange(out, device="cuda")
    part = lambda least, end: torch.randint(least, end, x.shape, device="cuda", generator=g)
    for low, count in ((8, 1), (5, 4)):                           # under 2^24, and 4 * 2^21 + residuals < 2^24
        v = (part(128, 256) << (low + 8)) + (part(128, 256) << low) + part(0, 1 << (low - 1)) * 2 + 1
        x.copy_(v * (torch.randint(0, 2, x.shape, device="cuda", generator=g) * 2 - 1))
        third = terms(x)[2]
        assert (third != 0).all()
        w.zero_()
        for i in range(count):
            at = torch.randint(0, inn, (out,), device="cuda", generator=g)
            if i % 2 == 0:                                        # (every other output out of the last columns of a row)
                at[1::2] = inn - 1 - at[1::2] % min(inn, 64)
            w[o, at] = (torch.randint(0, 2, (out,), device="cuda", generator=g) * 2 - 1).to(BF16)
        r = torch.randint(-1000, 1001, (T, out), device="cuda", generator=g).float() if count > 1 else None
        want = x.double() @ w.double().T
        lost = third.double() @ w.double().T
        assert (lost != 0).all() if count == 1 else (lost != 0).float().mean() > 0.5
        got = lo.linear(k3, x, w, res=r)
        assert torch.equal(got.double(), want if r is None else want + r)


@pytest.mark.parametrize("T,inn,out", [(1, 64, 16), (100, 64, 128), (300, 64, 256), (3, 40, 16), (90, 201, 70)])
@pytest.mark.parametrize("x_type", [F32, BF16])
def test_smallest_values(gpu, k3, T, inn, out, x_type):
    """Subnormal operands count in full, and of an fp32 one all bits down to bf16's least step of 2^-133."""
    say(f"case: {T} x {inn} -> {out} {x_type}")
    x, w = torch.zeros(T, inn, device="cuda", dtype=x_type), torch.zeros(out, inn, device="cuda", dtype=BF16)
    for e in (-133, -130, -127, -126, -110):
        x[:, inn - 1], w[:, inn - 1] = 2.0 ** e, 2.0 ** 100
        assert (lo.linear(k3, x, w) == 2.0 ** (e + 100)).all(), e
        x[:, inn - 1], w[:, inn - 1] = 2.0 ** 100, 2.0 ** e
        assert (lo.linear(k3, x, w) == 2.0 ** (e + 100)).all(), e
    if x_type == F32:
        x[:, inn - 1], w[:, inn - 1] = (1 + 2.0 ** -23) * 2.0 ** -110, 2.0 ** 100
        assert (lo.linear(k3, x, w) == (1 + 2.0 ** -23) * 2.0 ** -10).all()
