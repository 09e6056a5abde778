# SPDX-License-Identifier: Apache-2.0
"""What k3d_linear, k3d_route and k3d_qk_norm_rope refuse: every call here returns an error with its
reason before anything reaches a device (the pointers are none)."""
import pytest

A = 4096            # an address that nothing reads


def refused(k3, rc, word):
    assert rc != 0
    assert word in k3.lib().k3d_error().decode()


LINEAR = dict(y=A, y_type=1, ldy=64, x=A, x_type=1, ldx=32, T=4, W=A, ldw=32, inn=32, out=64, bias=None, act=0, res=None, ldr=0,
              ws=A, ws_bytes=1 << 40)


@pytest.mark.parametrize("change,word", [
    (dict(y_type=2), "x_type"), (dict(x_type=-1), "x_type"), (dict(act=5), "activation"), (dict(act=-1), "activation"),
    (dict(T=-1), "T >= 0"), (dict(inn=0), "in >= 1"), (dict(out=-3), "out >= 0"), (dict(ldx=31), "stride"),
    (dict(ldw=31), "stride"), (dict(ldy=63), "stride"), (dict(res=A, ldr=63), "stride"), (dict(ldx=(1 << 22) + 1), "MAX_LD"),
    (dict(ldw=(1 << 22) + 1), "MAX_LD"), (dict(inn=(1 << 20) + 1, ldx=1 << 21, ldw=1 << 21), "MAX_IN"), (dict(y=None), "must be given"), (dict(x=None), "must be given"),
    (dict(W=None), "must be given"), (dict(res=A, ldr=65), "y's stride"), (dict(y=A + 1), "aligned"),
    (dict(x=A + 1), "aligned"), (dict(W=A + 1), "aligned"), (dict(bias=A + 2), "aligned"), (dict(res=A + 1, ldr=64), "aligned"),
    (dict(y_type=0, y=A + 2), "aligned"), (dict(x_type=0, x=A + 2), "aligned")])
def test_linear(k3, change, word):
    a = dict(LINEAR, **change)
    refused(k3, k3.lib().k3d_linear(*a.values(), None), word)


ROUTE = dict(idx=A, wt=A, logits=A, type=0, ld=64, T=4, n=64, bias=None, score=0, groups=8, top_groups=4, group_top=2, topk=8,
             renorm=1, scale=1.0)


@pytest.mark.parametrize("change,word", [
    (dict(type=2), "type"), (dict(score=2), "score"), (dict(T=-1), "T >= 0"), (dict(n=0), "2048"), (dict(n=2049), "2048"),
    (dict(groups=0), "n_groups"), (dict(groups=7), "n_groups"), (dict(n=650, ld=650, groups=65), "n_groups"),
    (dict(top_groups=0), "top_groups"), (dict(top_groups=9), "top_groups"), (dict(group_top=3), "group_top"),
    (dict(group_top=0), "group_top"), (dict(topk=0), "topk"), (dict(topk=33), "topk"),
    (dict(n=128, ld=128, top_groups=8, topk=65), "topk"), (dict(ld=63), "ld"), (dict(idx=None), "must be given"),
    (dict(wt=None), "must be given"), (dict(logits=None), "must be given"), (dict(bias=A + 1), "aligned"),
    (dict(logits=A + 2), "aligned"), (dict(type=1, logits=A + 1), "aligned"), (dict(idx=A + 2), "aligned")])
def test_route(k3, change, word):
    a = dict(ROUTE, **change)
    refused(k3, k3.lib().k3d_route(*a.values(), None), word)


HEADS = dict(qo=A, ldqo=256, hsqo=64, ko=A, ldko=128, hsko=64, q=2 * A, ldq=256, hsq=64, k=2 * A, ldk=128, hsk=64, type=1, T=4,
             hq=4, hk=2, dim=64, qw=None, kw=None, eps=1e-6, pos=A, freq=A, rot=64, off=0, pairs=0, scale=1.0)


@pytest.mark.parametrize("change,word", [
    (dict(type=3), "type"), (dict(pairs=2), "pairs"), (dict(T=-1), "T >= 0"), (dict(hq=-1), "heads"), (dict(hk=65537), "heads"),
    (dict(dim=0), "dim"), (dict(dim=1025), "dim"), (dict(rot=63), "rot"), (dict(rot=66), "rot"), (dict(off=2), "rot"),
    (dict(rot=32, off=-1), "rot"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(pos=None), "pos"),
    (dict(freq=None), "inv_freq"), (dict(q=None), "without"), (dict(qo=None), "without"), (dict(k=None), "without"),
    (dict(ko=None), "without"), (dict(hsq=63), "heads overlap"), (dict(hsko=63), "heads overlap"), (dict(ldq=63), "tokens overlap"),
    (dict(ldko=1), "tokens overlap"), (dict(qo=2 * A, ldqo=512), "in place"), (dict(ko=2 * A, hsko=65), "in place"),
    (dict(q=A + 1), "aligned"), (dict(ko=A + 1), "aligned"), (dict(pos=A + 1), "aligned"), (dict(freq=A + 4), "aligned"),
    (dict(qw=A + 2), "aligned")])
def test_heads(k3, change, word):
    a = dict(HEADS, **change)
    refused(k3, k3.lib().k3d_qk_norm_rope(*a.values(), None), word)


def test_nothing_to_do(k3):
    """No tokens, rows or heads: done, without a device."""
    L = k3.lib()
    for ch in (dict(T=0), dict(out=0, ldy=0)):
        assert L.k3d_linear(*dict(LINEAR, **ch).values(), None) == 0
    assert L.k3d_route(*dict(ROUTE, T=0).values(), None) == 0
    for ch in (dict(T=0), dict(hq=0, hk=0)):
        assert L.k3d_qk_norm_rope(*dict(HEADS, **ch).values(), None) == 0


def test_linear_workspace(k3):
    """One too small, missing or unaligned is refused; the size for T tokens holds any fewer."""
    L = k3.lib()
    for x_type in (0, 1):
        for inn, out in ((64, 64), (7168, 384), (1001, 2047), (12288, 7168), (32, 16384)):
            last = 0
            for T in list(range(1, 70)) + [100, 127, 128, 129, 255, 256, 257, 500, 1000, 2048, 5000]:
                need = L.k3d_linear_ws(T, inn, out, x_type)
                assert need >= last
                last = need
            if last:
                a = dict(LINEAR, x_type=x_type, T=5000, inn=inn, out=out, ldx=inn, ldw=inn, ldy=out)
                refused(k3, L.k3d_linear(*dict(a, ws_bytes=last - 1).values(), None), "workspace")
                refused(k3, L.k3d_linear(*dict(a, ws=None).values(), None), "workspace")
                refused(k3, L.k3d_linear(*dict(a, ws=A + 8).values(), None), "aligned")
    assert L.k3d_linear_ws(0, 64, 64, 0) == 0


APART = dict(LINEAR, x=2 * A, W=3 * A, bias=4 * A, ws=5 * A)


@pytest.mark.parametrize("change,word", [
    (dict(T=(1 << 24) + 1), "MAX_TOKENS"), (dict(out=(1 << 28) + 1, ldy=1 << 30), "MAX_OUT"),
    (dict(T=1 << 20, out=(1 << 13) + 1, ldy=1 << 14), "2^33"), (dict(y=2 * A), "operand"), (dict(y=3 * A), "operand"), (dict(y=4 * A), "operand"),
    (dict(y=5 * A), "operand")])
def test_linear_places(k3, change, word):
    refused(k3, k3.lib().k3d_linear(*dict(APART, **change).values(), None), word)


def test_route_tokens(k3):
    refused(k3, k3.lib().k3d_route(*dict(ROUTE, T=(1 << 24) + 1).values(), None), "MAX_TOKENS")


@pytest.mark.parametrize("change,word", [
    (dict(T=(1 << 24) + 1), "MAX_TOKENS"),
    (dict(qo=3 * A, ko=3 * A), "one place"), (dict(ldqo=255), "token and of a head"), (dict(ldqo=64, hsqo=255), "token and of a head"),
    (dict(ldko=64, hsko=64), "token and of a head"), (dict(ldqo=1 << 62, hsqo=1 << 62), "token and of a head")])
def test_heads_places(k3, change, word):
    refused(k3, k3.lib().k3d_qk_norm_rope(*dict(HEADS, **change).values(), None), word)
