# SPDX-License-Identifier: Apache-2.0
"""k3d_linear against the product, bias, activation and residual in 64 bits, at the edges of its tiles,
types, strides and alignments. The bound is worst-case arithmetic (layer_ops.linear64); at the short
sums below it tells a lost bf16 term of fp32 activations (2^-16 relative)."""
import numpy as np
import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)


def operands(T, inn, out, x_type, y_type, seed, bias=True, res=True, padx=0, padw=0, offx=0, offw=0):
    """x, W as views with row padding (elements) and a start offset (elements)."""
    g = lo.gen(seed)
    bx = torch.full((T * (inn + padx) + offx + 8,), float("nan"), device="cuda", dtype=x_type)
    bw = torch.full((out * (inn + padw) + offw + 8,), float("nan"), device="cuda", dtype=BF16)
    x = bx[offx:offx + T * (inn + padx)].view(T, inn + padx)[:, :inn]
    w = bw[offw:offw + out * (inn + padw)].view(out, inn + padw)[:, :inn]
    x.copy_(torch.randn(T, inn, device="cuda", generator=g))
    w.copy_(torch.randn(out, inn, device="cuda", generator=g) * inn ** -0.5)
    b = torch.randn(out, device="cuda", generator=g) if bias else None
    r = torch.randn(T, out, device="cuda", generator=g).to(y_type) if res else None
    return x, w, b, r


def check(k3, T, inn, out, x_type, y_type, act="none", seed=1, **kw):
    x, w, b, r = operands(T, inn, out, x_type, y_type, seed, **kw)
    y = torch.full((T + 1, out + 3), 7.0, device="cuda", dtype=y_type)
    got = lo.linear(k3, x, w, b, act, r, y=y[:T, :out])
    lo.within(got, lo.linear64(x, w, b, act, r, y_type))
    assert (y[T] == 7).all() and (y[:, out:] == 7).all()          # nothing written beside the rows
    return got


@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("T,inn,out", [
    (1, 1, 1), (1, 8, 3), (1, 64, 64), (1, 1000, 257), (2, 31, 17), (3, 33, 16), (4, 256, 130), (5, 72, 129), (8, 40, 48),
    (9, 128, 63), (15, 65, 33), (16, 64, 128), (17, 96, 100), (31, 520, 31), (32, 264, 65), (33, 63, 255), (48, 200, 80),
    (63, 8, 64), (64, 1, 65), (65, 192, 127), (100, 7, 9), (127, 136, 128), (128, 64, 256), (129, 250, 257), (200, 321, 130),
    (256, 128, 256), (257, 72, 300), (300, 1001, 77), (511, 48, 33), (700, 24, 513)])
def test_sizes(gpu, k3, T, inn, out, x_type, y_type):
    say(f"case: {T} x {inn} -> {out} {x_type} {y_type}")
    check(k3, T, inn, out, x_type, y_type, act=lo.ACTS[(T + inn) % 5], seed=T)


# (from a handful of columns a worker to many stages, tiles by the hundred and a few)
@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("T,inn,out", [(1, 7168, 576), (7, 3584, 2048), (40, 7168, 384), (64, 12288, 130), (90, 2048, 4100),
                                       (130, 7168, 896), (300, 1536, 3584), (520, 2056, 1030), (1030, 520, 2050), (2100, 264, 1160)])
def test_longer(gpu, k3, T, inn, out, x_type):
    say(f"case: {T} x {inn} -> {out} {x_type}")
    check(k3, T, inn, out, x_type, F32, act="none", seed=T)


@pytest.mark.parametrize("act", lo.ACTS)
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("T,inn,out", [(3, 64, 40), (70, 64, 40), (300, 192, 300)])
def test_epilogue(gpu, k3, act, bias, res, T, inn, out):
    say(f"case: {act} bias={bias} res={res} {T}")
    check(k3, T, inn, out, BF16, BF16, act, 3, bias=bias, res=res)
    check(k3, T, inn, out, BF16, F32, act, 4, bias=bias, res=res)


@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("T", [1, 6, 40, 150, 600])
@pytest.mark.parametrize("padx,padw,offx,offw", [(8, 8, 0, 0), (3, 0, 0, 0), (0, 5, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 3, 5), (64, 16, 8, 8)])
def test_strides(gpu, k3, T, x_type, padx, padw, offx, offw):
    """Row strides and starts off every alignment; what lies between the rows is NaN and stays out."""
    say(f"case: {T} {x_type} {padx} {padw} {offx} {offw}")
    check(k3, T, 200, 136, x_type, BF16, "silu", 5, padx=padx, padw=padw, offx=offx, offw=offw)


@pytest.mark.parametrize("T", [1, 5, 70, 600])
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_in_place_residual(gpu, k3, T, y_type):
    """res may be y itself; a padded, odd y."""
    say(f"case: {T} {y_type}")
    x, w, b, r = operands(T, 520, 201, BF16, y_type, 8)
    y = torch.full((T, 207), 3.0, device="cuda", dtype=y_type)[:, 1:202]
    y.copy_(r)
    lo.linear(k3, x, w, b, "gelu", y, y=y)
    lo.within(y, lo.linear64(x, w, b, "gelu", r, y_type))


@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("T,inn,out", [(2, 64, 20), (20, 72, 40), (90, 200, 140), (300, 512, 260)])
def test_nonfinite(gpu, k3, x_type, T, inn, out):
    """Infinities and NaN of x stay in their own token, those of W in their own column."""
    say(f"case: {T} {x_type}")
    x, w, b, r = operands(T, inn, out, x_type, F32, 9)
    w[:, 3].abs_().add_(0.1)
    clean = lo.linear(k3, x, w, b, "none", r)
    x[1, 3], x[0, 5] = float("inf"), float("nan")
    w[7, 2] = float("nan")
    y = lo.linear(k3, x, w, b, "none", r)
    assert torch.isnan(y[0]).all() and torch.isnan(y[:, 7]).all()
    keep = torch.arange(out, device="cuda") != 7
    assert (y[1][keep] == float("inf")).all()
    assert torch.equal(y[2:][:, keep], clean[2:][:, keep])


@pytest.mark.parametrize("act", lo.ACTS)
def test_activation_range(gpu, k3, act):
    """From subnormal to infinite arguments of the activations: one weight of 1, sums exact. v / (1 + e^-z) in fp32
    is 0 once e^-z passes the largest fp32 number, at z < -88.73: there it is less than |v| 2^-128, which for
    silu falls with v (|v| e^v) and for gelu_tanh is at |v| < 10 (z = 1.6 v (1 + .045 v^2)): 89 * 2^-128 at most."""
    say(f"case: {act}")
    m = torch.logspace(-40, 38.4, 3000, device="cuda", dtype=torch.float64).float()
    v = torch.cat([m, -m, torch.linspace(-100, 100, 4001, device="cuda"), torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan")], device="cuda")])
    x = torch.zeros(v.numel(), 64, device="cuda")
    x[:, 0] = v
    w = torch.zeros(1, 64, device="cuda", dtype=BF16)
    w[0, 0] = 1
    got = lo.f64(lo.linear(k3, x, w, act=act))[:, 0]
    with np.errstate(all="ignore"):
        want = lo.act64(lo.f64(v), act)
    fin = np.isfinite(want)
    size = np.abs(lo.f64(v) if act == "gelu" else want)[fin]
    tol = 2.0 ** -21 * size + 2.0 ** -126 * 1.01
    if act in ("silu", "gelu_tanh"):
        tol = np.maximum(tol, 89 * 2.0 ** -128)
    if act == "gelu_tanh":      # z comes out of three roundings, each of which moves e^-z by 2^-24 |z| of itself, |z| < 89 where it counts
        tol = tol + 3 * 89 * 2.0 ** -24 * size
    assert (np.abs(got[fin] - want[fin]) <= tol).all()
    assert np.isnan(got[-1])
    if act != "gelu" and act != "gelu_tanh" and act != "silu":
        assert got[-2] == (0 if act == "relu" else -np.inf)
    assert got[-3] == np.inf


@pytest.mark.parametrize("T,inn,out", [(1, 512, 96), (24, 512, 96), (200, 2048, 260), (900, 512, 300)])
def test_repeats_and_graph(gpu, k3, T, inn, out):
    """The same bits from call to call, on another stream and from a captured graph replayed on new inputs."""
    say(f"case: {T}")
    L = k3.lib()
    x, w, b, r = operands(T, inn, out, BF16, BF16, 10)
    first = lo.linear(k3, x, w, b, "silu", r)
    assert torch.equal(first, lo.linear(k3, x, w, b, "silu", r))
    ws = torch.empty(max(1, L.k3d_linear_ws(T, inn, out, 1)), device="cuda", dtype=torch.uint8)
    y = torch.zeros_like(first)
    torch.cuda.synchronize()
    st = L.k3d_stream_create()
    import ctypes as C
    ex = C.c_void_p()
    try:
        k3.check(L.k3d_graph_begin(st))
        lo.linear(k3, x, w, b, "silu", r, y=y, ws=ws, st=st)
        k3.check(L.k3d_graph_end(st, C.byref(ex)))
        for i in range(4):
            x.copy_(torch.randn(T, inn, device="cuda", generator=lo.gen(20 + i)))
            y.zero_()
            want = lo.linear(k3, x, w, b, "silu", r)
            torch.cuda.synchronize()
            k3.check(L.k3d_graph_launch(ex, st))
            k3.check(L.k3d_sync(st))
            assert torch.equal(y, want)
    finally:
        if ex:
            L.k3d_graph_destroy(ex)
        L.k3d_stream_destroy(st)


def test_far_rows(gpu, k3):
    """Rows of W and y past 2^32 bytes from their start."""
    say("case: far rows")
    ld, out = 1 << 21, 1100
    w = torch.zeros(out, ld, device="cuda", dtype=BF16)[:, :64]
    w.copy_(torch.randn(out, 64, device="cuda", generator=lo.gen(11)))
    y = torch.zeros(9, 1 << 28, device="cuda", dtype=BF16)[:, :out]
    x = torch.randn(9, 64, device="cuda", generator=lo.gen(12)).to(BF16)
    lo.within(lo.linear(k3, x, w, y=y), lo.linear64(x, w, None, "none", None, BF16))


@pytest.mark.parametrize("T,inn,out", [
    (1, 7168, 7168), (6, 4096, 4096), (14, 2048, 8192), (22, 7168, 896), (30, 2048, 2048), (38, 12288, 4100), (46, 512, 16384),
    (60, 8192, 6400), (64, 7168, 7000), (96, 7168, 7168), (200, 7168, 2048), (1024, 2048, 2048), (1500, 1024, 3584),
    (2048, 2048, 4096), (4096, 1024, 4096), (300, 7168, 384), (1000, 7168, 130)])
@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("off", [0, 1])
def test_every_kernel(gpu, k3, T, inn, out, x_type, off):
    """Large enough that each kernel, tile, slicing and way of reading W is some shape's choice, with W aligned and not. Operands
    are integers whose sums stay below 2^24, so fp32 forms them exactly in any order and the result is one only."""
    say(f"case: {T} x {inn} -> {out} {x_type} off {off}")
    x, w, b, r = operands(T, inn, out, x_type, F32, T, offw=off)
    big, one = (511, 1) if x_type == F32 else (3, 3)               # (of fp32 the two upper terms; 511 * 12288 < 2^23)
    x.copy_(torch.randint(-big, big + 1, x.shape, device="cuda", generator=lo.gen(T)))
    w.copy_(torch.randint(-one, one + 1, w.shape, device="cuda", generator=lo.gen(T + 1)))
    for t in (b, r):
        t.copy_((t * 100).round())
    y = torch.full((T + 1, out + 3), 7.0, device="cuda", dtype=F32)
    got = lo.linear(k3, x, w, b, "relu", r, y=y[:T, :out])
    want = (x.double() @ w.double().T + b).clamp(min=0) + r
    assert torch.equal(got.double(), want)
    assert (y[T] == 7).all() and (y[:, out:] == 7).all()


@pytest.mark.parametrize("inn,out", [(1024, 2000), (512, 5200), (1024, 8200), (8192, 6400), (4096, 12300), (16384, 3500)])
@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("T", [8, 13, 32, 48, 62])
def test_every_few(gpu, k3, T, inn, out, x_type):
    """Each group of tokens with each number of rows of W a workgroup takes, and with W past the caches."""
    test_every_kernel(gpu, k3, T, inn, out, x_type, 0)


@pytest.mark.parametrize("T,inn,out", [(2, 64, 20), (20, 128, 40), (90, 256, 140), (90, 200, 140), (3, 40, 20)])
def test_nan_payloads(gpu, k3, T, inn, out):
    """An fp32 NaN whose payload lies in any of its three parts makes its row NaN, an infinity infinite, and no other row either."""
    say(f"case: {T} {inn} {out}")
    bits = [0x7f800001, 0xff800100, 0x7f810000, 0x7fc00000, 0xffffffff]
    for b in bits + [0x7f800000]:
        x = torch.ones(T, inn, device="cuda")
        x.view(torch.int32)[T - 1, inn - 1] = b - (1 << 32) if b >> 31 else b
        w = torch.ones(out, inn, device="cuda", dtype=BF16)
        y = lo.linear(k3, x, w)
        assert (y[T - 1] == float("inf")).all() if b == 0x7f800000 else torch.isnan(y[T - 1]).all()
        assert (y[:T - 1] == inn).all()


@pytest.mark.parametrize("T,inn,out", [(2, 72, 20), (9, 200, 40), (20, 520, 70), (48, 136, 33), (64, 1096, 64), (90, 200, 140), (300, 1160, 260),
                                       (700, 328, 513), (90, 201, 140), (3, 40, 20), (3, 201, 20), (1500, 777, 999)])
def test_infinite_weight(gpu, k3, T, inn, out):
    """An infinite weight in any column, those at the end of a row among them, makes its own outputs infinite and no other; so does an
    infinite activation, in bf16 and in fp32."""
    say(f"case: {T} {inn} {out}")
    for x_type in (BF16, F32):
        x, w, b, r = operands(T, inn, out, x_type, F32, 3)
        x.abs_().add_(0.5)
        w.abs_().add_(0.125)
        clean = lo.linear(k3, x, w, b, "none", r)
        for k in sorted({0, 1, inn // 2, max(0, inn - 64), max(0, inn - 57), inn - inn % 64 - 1 if inn > 64 else 0, inn - 8, inn - 1}):
            if x_type == BF16:                                     # (with fp32 x it meets the terms that are zero)
                keep = w[7, k].clone()
                w[7, k] = float("inf")
                y = lo.linear(k3, x, w, b, "none", r)
                w[7, k] = keep
                assert (y[:, 7] == float("inf")).all(), k
                on = torch.arange(out, device="cuda") != 7
                assert torch.equal(y[:, on], clean[:, on])
            keep = x[1, k].clone()
            x[1, k] = float("-inf")
            y = lo.linear(k3, x, w, b, "none", r)
            x[1, k] = keep
            assert (y[1] == float("-inf")).all(), k
            on = torch.arange(T, device="cuda") != 1
            assert torch.equal(y[on], clean[on])


@pytest.mark.parametrize("T,inn,out", [
    (8, 1032, 8200), (13, 4104, 12300), (30, 2056, 5200), (60, 8200, 6400), (46, 136, 130), (4100, 520, 2050), (1030, 1096, 12304), (1030, 1032, 4096),
    (700, 7176, 896), (200, 7176, 896), (300, 1032, 4096), (300, 264, 1160), (2000, 1024, 2051), (2001, 800, 4099), (513, 960, 1021)])
@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_every_tail(gpu, k3, T, inn, out, x_type, y_type):
    """Rows that end inside a step, and edges of the outputs with residuals, on the kernels for few tokens and on every tile. Integers again: the
    fp32 result is exact, a bf16 one its one rounding."""
    say(f"case: {T} x {inn} -> {out} {x_type} {y_type}")
    x, w, b, r = operands(T, inn, out, x_type, y_type, T, padx=8, padw=16)
    big, one = (511, 1) if x_type == F32 else (3, 3)
    x.copy_(torch.randint(-big, big + 1, x.shape, device="cuda", generator=lo.gen(T)))
    w.copy_(torch.randint(-one, one + 1, w.shape, device="cuda", generator=lo.gen(T + 1)))
    b.copy_((b * 100).round())
    r.copy_((r.float() * 10).round())
    y = torch.full((T + 1, out + 3), 7.0, device="cuda", dtype=y_type)
    got = lo.linear(k3, x, w, b, "relu", r, y=y[:T, :out])
    want = (x.double() @ w.double().T + b).clamp(min=0) + r.double()
    assert torch.equal(got, want.float().to(y_type))
    assert (y[T] == 7).all() and (y[:, out:] == 7).all()
    y[:T, :out] = r                                                # the residual in the result's place
    assert torch.equal(lo.linear(k3, x, w, b, "relu", y[:T, :out], y=y[:T, :out]), want.float().to(y_type))
    assert (y[T] == 7).all() and (y[:, out:] == 7).all()
