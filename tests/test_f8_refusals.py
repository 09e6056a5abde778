# SPDX-License-Identifier: Apache-2.0
"""What the entry points of a layer's 8-bit path refuse: every call here returns an error with its reason before anything
reaches a device (the pointers are none)."""
import pytest

A = 4096            # addresses that nothing reads
BIG = 1 << 40


def refused(k3, rc, word):
    assert rc != 0
    assert word in k3.lib().k3d_error().decode()


NORM = dict(y=A, y_type=1, ldy=200, q=2 * A, ldq=256, qs=3 * A, ldqs=2, sum=4 * A, ldsum=200, x=5 * A, x_type=0, ldx=200, res=6 * A,
            r_type=1, ldr=200, T=4, n=200, w=7 * A, eps=1e-6)


@pytest.mark.parametrize("change,word", [
    (dict(x_type=2), "x_type"), (dict(y_type=-1), "x_type"), (dict(r_type=2), "x_type"), (dict(T=-1), "T >= 0"), (dict(n=0), "n <="),
    (dict(n=65537, ldx=1 << 20), "NORM_MAX_N"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(T=(1 << 24) + 1), "MAX_TOKENS"),
    (dict(x=None), "must be given"), (dict(y=None, q=None, sum=None), "must be given"), (dict(ldx=199), "stride"), (dict(ldy=199), "stride"),
    (dict(ldsum=199), "stride"), (dict(ldr=199), "stride"), (dict(x=A * 5 + 2), "aligned"), (dict(y=A + 1), "aligned"),
    (dict(res=6 * A + 1), "aligned"), (dict(sum=4 * A + 1), "aligned"), (dict(w=A + 2), "aligned"), (dict(q=2 * A + 8), "aligned"),
    (dict(ldq=264), "aligned"), (dict(ldq=240), "whole blocks"), (dict(qs=None), "scales must be given"), (dict(qs=A + 2), "aligned"),
    (dict(ldqs=1), "scales' stride"), (dict(sum=6 * A, ldsum=201), "res's place"), (dict(sum=5 * A), "x's place"),
    (dict(y=5 * A), "x's place"), (dict(y=6 * A, ldy=300), "res's place"), (dict(y=4 * A), "one place"), (dict(sum=2 * A), "one place"),
    (dict(y=2 * A), "one place"), (dict(q=5 * A), "operand"), (dict(q=6 * A), "operand")])
def test_norm(k3, change, word):
    refused(k3, k3.lib().k3d_add_norm(*dict(NORM, **change).values(), None), word)


QUANT = dict(q=A, ldq=256, qs=2 * A, ldqs=2, x=3 * A, x_type=0, ldx=400, T=4, n=200, act=1, b1=1.0, b2=1.0)


@pytest.mark.parametrize("change,word", [
    (dict(x_type=3), "x_type"), (dict(act=2), "activation"), (dict(act=-2), "activation"), (dict(act=0, b1=0.0), "limits"),
    (dict(act=0, b2=-1.0), "limits"), (dict(act=0, b2=float("nan")), "limits"),
    (dict(act=0, b1=float("inf")), "limits"), (dict(act=0, b2=1e30), "limits"), (dict(act=0, b1=1e-30), "limits"), (dict(T=-1), "T >= 0"), (dict(n=0), "n <="),
    (dict(n=65537, ldx=1 << 20), "NORM_MAX_N"), (dict(T=(1 << 24) + 1), "MAX_TOKENS"), (dict(x=None), "must be given"),
    (dict(ldx=399), "stride"), (dict(act=-1, ldx=199), "stride"), (dict(x=3 * A + 1), "aligned"), (dict(q=None), "must be given"),
    (dict(qs=None), "must be given"), (dict(q=A + 4), "aligned"), (dict(ldq=248), "aligned"), (dict(ldq=128), "whole blocks"),
    (dict(ldqs=1), "scales' stride"), (dict(q=3 * A), "operand")])
def test_quant(k3, change, word):
    refused(k3, k3.lib().k3d_quant_f8(*dict(QUANT, **change).values(), None), word)


@pytest.mark.parametrize("change,word", [
    (dict(rows=0), "rows >= 1"), (dict(inn=0), "in >= 1"), (dict(mats=-1), "mats >= 0"), (dict(inn=(1 << 20) + 1, ldw=1 << 21), "MAX_IN"),
    (dict(rows=(1 << 18) + 1), "MAX_OUT"), (dict(ldw=127), "stride"), (dict(t=None), "must be given"), (dict(W=None), "must be given"),
    (dict(t=A + 8), "aligned"), (dict(t=2 * A), "place"), (dict(rows=1 << 18, inn=1 << 20, ldw=1 << 20, mats=64), "2^43")])
def test_tile(k3, change, word):
    a = dict(dict(t=A, W=2 * A, ldw=128, rows=100, inn=128, mats=1), **change)
    refused(k3, k3.lib().k3d_f8_tile(*a.values(), None), word)


LINEAR = dict(y=A, y_type=1, ldy=64, x=2 * A, ldx=256, xs=3 * A, ldxs=2, T=4, W=4 * A, Ws=5 * A, ldws=2, inn=200, out=64, bias=6 * A, act=0,
              res=7 * A, ldr=64, ws=8 * A, ws_bytes=BIG)


@pytest.mark.parametrize("change,word", [
    (dict(inn=0), "in >= 1"), (dict(out=-1), "out >= 0"), (dict(inn=(1 << 20) + 1), "MAX_IN"), (dict(out=(1 << 18) + 1), "MAX_OUT"),
    (dict(y_type=2), "y_type"), (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(T=-1), "T >= 0"),
    (dict(T=(1 << 24) + 1), "MAX_TOKENS"), (dict(T=1 << 24, out=(1 << 13) + 1, ldy=1 << 14, ldr=1 << 14), "MAX_RESULTS"), (dict(x=None), "must be given"),
    (dict(xs=None), "must be given"), (dict(x=2 * A + 8), "aligned"), (dict(ldx=264), "aligned"), (dict(ldx=240), "whole blocks"),
    (dict(ldxs=1), "scales' stride"), (dict(xs=3 * A + 2), "aligned"), (dict(ldx=(1 << 22) + 16), "MAX_LD"), (dict(ldxs=(1 << 20) + 1), "MAX_LD"),
    (dict(y=None), "must be given"), (dict(W=None), "must be given"), (dict(Ws=None), "must be given"), (dict(ldy=63), "stride"),
    (dict(ldr=63), "stride"), (dict(ldws=1), "stride"), (dict(y=A + 1), "aligned"), (dict(res=7 * A + 1), "aligned"),
    (dict(bias=A + 1), "aligned"), (dict(Ws=A + 2), "aligned"), (dict(W=4 * A + 8), "16-byte"), (dict(res=A, ldr=65), "y's stride"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=16), "workspace"), (dict(ws=8 * A + 8), "workspace"), (dict(y=2 * A), "operand"),
    (dict(y=3 * A), "operand"), (dict(y=4 * A), "operand"), (dict(y=5 * A), "operand"), (dict(y=6 * A), "operand"), (dict(y=8 * A), "operand")])
def test_linear(k3, change, word):
    a = dict(LINEAR, T=100) if "ws" in change or "ws_bytes" in change else LINEAR
    refused(k3, k3.lib().k3d_linear_f8(*dict(a, **change).values(), None), word)


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "T >= 0"), (dict(topk=0), "topk"), (dict(topk=65), "topk"), (dict(n=0), "2048"), (dict(n=2049), "2048"),
    (dict(T=1 << 23, topk=3), "MAX_SLOTS"), (dict(offsets=None), "must be given"), (dict(perm=None), "must be given"),
    (dict(idx=None), "must be given"), (dict(offsets=A + 1), "aligned"), (dict(perm=A + 2), "aligned"), (dict(idx=A + 3), "aligned"),
    (dict(perm=A), "place"), (dict(idx=A), "place"), (dict(idx=2 * A), "place"), (dict(T=1000, ws=None), "workspace"),
    (dict(T=1000, ws_bytes=8), "workspace"), (dict(T=1000, ws=A + 2), "aligned")])
def test_group(k3, change, word):
    a = dict(dict(offsets=A, perm=2 * A, idx=3 * A, T=4, topk=8, n=64, ws=4 * A, ws_bytes=BIG), **change)
    refused(k3, k3.lib().k3d_group(*a.values(), None), word)


GROUPED = dict(y=A, y_type=1, ldy=64, y_rows=2 * A, y_cap=10, x=3 * A, ldx=256, xs=4 * A, ldxs=2, x_rows=5 * A, x_div=2, x_cap=10,
               offsets=6 * A, rows=10, n=4, W=7 * A, Ws=8 * A, inn=200, out=64)


@pytest.mark.parametrize("change,word", [
    (dict(inn=0), "in >= 1"), (dict(out=-1), "out >= 0"), (dict(inn=(1 << 20) + 1), "MAX_IN"), (dict(out=(1 << 18) + 1), "MAX_OUT"),
    (dict(y_type=2), "y_type"), (dict(n=0), "2048"), (dict(n=2049), "2048"), (dict(rows=-1), "x_div"), (dict(x_cap=-1), "x_div"),
    (dict(y_cap=-1), "x_div"), (dict(x_div=0), "x_div"), (dict(rows=(1 << 24) + 1), "MAX_SLOTS"), (dict(x_cap=(1 << 24) + 1), "MAX_TOKENS"),
    (dict(y_cap=(1 << 24) + 1), "MAX_TOKENS"), (dict(rows=1 << 24, out=1 << 14, ldy=1 << 14), "MAX_RESULTS"), (dict(x=None), "must be given"),
    (dict(ldx=240), "whole blocks"), (dict(ldx=(1 << 22) + 16), "MAX_LD"), (dict(ldxs=(1 << 20) + 1), "MAX_LD"),
    (dict(x_cap=1 << 23, ldx=272), "MAX_X"), (dict(x_cap=1 << 20, ldxs=600), "MAX_X"), (dict(y=None), "must be given"),
    (dict(offsets=None), "must be given"), (dict(W=None), "must be given"), (dict(Ws=None), "must be given"), (dict(ldy=63), "stride"),
    (dict(y=A + 1), "aligned"), (dict(offsets=A + 1), "aligned"), (dict(x_rows=A + 1), "aligned"), (dict(y_rows=A + 2), "aligned"),
    (dict(Ws=A + 2), "aligned"), (dict(W=A + 8), "16-byte"), (dict(y=2 * A), "operand"), (dict(y=3 * A), "operand"), (dict(y=4 * A), "operand"),
    (dict(y=5 * A), "operand"), (dict(y=6 * A), "operand"), (dict(y=7 * A), "operand"), (dict(y=8 * A), "operand")])
def test_grouped(k3, change, word):
    refused(k3, k3.lib().k3d_grouped_f8(*dict(GROUPED, **change).values(), None), word)


MOE = dict(out=A, out_type=1, ldo=256, idx=2 * A, wt=3 * A, x=4 * A, ldx=256, xs=5 * A, ldxs=2, T=4, w1=6 * A, s1=7 * A, w3=8 * A, s3=9 * A,
           w2=10 * A, s2=11 * A, hidden=256, inter=128, n=16, topk=4, act=1, b1=1.0, b2=1.0, ws=12 * A, ws_bytes=BIG)


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "T >= 0"), (dict(topk=0), "topk"), (dict(topk=65), "topk"), (dict(n=0), "2048"), (dict(n=2049), "2048"),
    (dict(T=1 << 23), "MAX_SLOTS"), (dict(out_type=2), "out_type"), (dict(act=2), "activation"), (dict(act=-1), "activation"),
    (dict(act=0, b1=0.0), "limits"), (dict(hidden=0), "hidden"), (dict(inter=65537), "hidden"), (dict(x=None), "must be given"),
    (dict(ldx=128), "whole blocks"), (dict(ldx=(1 << 22) + 16), "MAX_LD"), (dict(T=1 << 20, ldx=4096), "MAX_X"),
    (dict(T=1 << 22, inter=256), "MAX_X"), (dict(out=None), "must be given"), (dict(idx=None), "must be given"), (dict(wt=None), "must be given"),
    (dict(w1=None), "must be given"), (dict(s2=None), "must be given"), (dict(ldo=255), "stride"), (dict(out=A + 1), "aligned"),
    (dict(idx=A + 2), "aligned"), (dict(wt=A + 2), "aligned"), (dict(s3=A + 2), "aligned"), (dict(w3=A + 8), "16-byte"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=100), "workspace"), (dict(ws=12 * A + 8), "workspace"), (dict(out=4 * A), "operand"),
    (dict(out=12 * A), "operand"), (dict(out=2 * A), "operand")])
def test_moe(k3, change, word):
    refused(k3, k3.lib().k3d_moe_f8(*dict(MOE, **change).values(), None), word)


def test_nothing_to_do(k3):
    """No tokens, rows or outputs: done, without a device."""
    L = k3.lib()
    assert L.k3d_add_norm(*dict(NORM, T=0).values(), None) == 0
    assert L.k3d_quant_f8(*dict(QUANT, T=0).values(), None) == 0
    assert L.k3d_f8_tile(A, 2 * A, 128, 64, 128, 0, None) == 0
    for ch in (dict(T=0), dict(out=0, ldy=0)):
        assert L.k3d_linear_f8(*dict(LINEAR, **ch).values(), None) == 0
    for ch in (dict(rows=0), dict(x_cap=0), dict(y_cap=0), dict(out=0)):
        assert L.k3d_grouped_f8(*dict(GROUPED, **ch).values(), None) == 0
    assert L.k3d_moe_f8(*dict(MOE, T=0).values(), None) == 0


def test_sizes(k3):
    """A workspace of T tokens holds any fewer; a tiled matrix is whole 128 x 128 blocks."""
    L = k3.lib()
    for rows, inn in ((1, 1), (128, 128), (129, 128), (300, 1000)):
        assert L.k3d_f8_tiled_bytes(rows, inn) == -(-rows // 128) * -(-inn // 128) * 16384
    assert L.k3d_f8_tiled_bytes(0, 5) == 0 and L.k3d_linear_f8_ws(0, 64, 64) == 0 and L.k3d_moe_f8_ws(0, 1, 1, 1, 1) == 0
    sizes = list(range(1, 70)) + [127, 128, 129, 255, 256, 257, 500, 512, 513, 1000, 1024, 2048, 4097]
    for f in (lambda T: L.k3d_linear_f8_ws(T, 7168, 384), lambda T: L.k3d_linear_f8_ws(T, 1001, 2047),
              lambda T: L.k3d_moe_f8_ws(T, 7168, 2048, 384, 8), lambda T: L.k3d_moe_f8_ws(T, 100, 30, 2048, 64),
              lambda T: L.k3d_group_ws(T, 8, 384)):
        last = 0
        for T in sizes:
            assert f(T) >= last
            last = f(T)
