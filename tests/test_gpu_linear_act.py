# SPDX-License-Identifier: Apache-2.0
"""The activations of k3d_linear to the last units of fp32, under results of either type. x has one column that counts, with a weight
of 1, so the argument is x itself and every sum exact. Of a bf16 result a residual takes off nearly all of the activation's value, so that
the result's rounding does not hide the fp32 that it is formed in.

The bounds count roundings of half a step (a unit: 2^-24 of the value) and hardware exponentials and reciprocals, two units each."""
import numpy as np
import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24


def say(msg):
    print(msg, flush=True)


def arguments(lo_, hi, n, seed):
    g = np.random.default_rng(seed)
    v = np.concatenate([g.uniform(lo_, hi, n), np.linspace(lo_, hi, 999)]).astype(np.float32)
    return v[v != 0]


def apply(k3, v, act, res=None, y_type=F32):
    x = torch.zeros(len(v), 64, device="cuda")
    x[:, 0] = torch.from_numpy(v).cuda()
    w = torch.zeros(1, 64, device="cuda", dtype=BF16)
    w[0, 0] = 1
    return lo.f64(lo.linear(k3, x, w, act=act, res=res, y_type=y_type))[:, 0]


def units_of_gate(v, act):
    """Of v / (1 + e^-z): the exponential 2, its correction 1, the sum 1, the reciprocal 2, the product with v 1, and nothing worth a
    unit from the correction's own error (2^-24 of a correction under 2^-16). For gelu_tanh z = c v (1 + d v^2) first: c, d and four
    operations move it by 6 units (d v^2 counts at most once), and e^-z by |z| times that, which counts by e^-z / (1 + e^-z)."""
    if act == "silu":
        return 8.0
    z = 2 * np.sqrt(2 / np.pi) * v * (1 + 0.044715 * v * v)
    with np.errstate(over="ignore"):
        return 8.0 + 6 * np.abs(z) / (1 + np.exp(z))


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("span", [(-85, -20), (-20, -1), (-1, 0), (0, 3), (3, 85)])
def test_gate_of_bf16_results(gpu, k3, act, span):
    if act == "gelu_tanh":
        span = tuple(s / 10 for s in span)
    say(f"case: {act} {span}")
    v = arguments(*span, 400000, 1)
    a = lo.act64(v.astype(np.float64), act)
    r = torch.from_numpy(a).cuda().to(BF16)
    near = np.abs(a - lo.f64(r)) <= 2.0 ** -17 * np.abs(a)         # (values next to a bf16 number: the residual's other sign)
    v, a, r = v[near], a[near], -r[torch.from_numpy(near).cuda()].unsqueeze(1)
    assert len(v) > 1000
    got, want = apply(k3, v, act, r, BF16), a + lo.f64(r)[:, 0]
    tol = units_of_gate(v.astype(np.float64), act) * UNIT * np.abs(a)
    half = np.maximum((np.abs(want) + tol) * lo.HALF[BF16], 2.0 ** -134)        # (the least step of bf16 is 2^-133)
    assert (np.abs(got - want) <= tol + half).all(), (np.abs(got - want) / np.abs(a) / UNIT).max()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("span", [(-99, -80), (-80, -20), (-20, -1), (-1, 0), (0, 3), (3, 99)])
def test_gate_of_fp32_results(gpu, k3, act, span):
    """Down to the subnormals, past where e^-z alone leaves fp32."""
    if act == "gelu_tanh":
        span = tuple(s / 10 for s in span)
    say(f"case: {act} {span}")
    v = arguments(*span, 100000, 2)
    a = lo.act64(v.astype(np.float64), act)
    tol = units_of_gate(v.astype(np.float64), act) * UNIT * np.abs(a) + 2.0 ** -148      # (two roundings of a subnormal result)
    got = apply(k3, v, act)
    assert (np.abs(got - a) <= tol).all(), (np.abs(got - a) / np.abs(a) / UNIT).max()


def off_of_gelu(v, a, y_type):
    """How far v (1 - h) or v h may be off, h = erfc(|v| / sqrt 2) / 2, a the value.
    fp32 results, past |v| = 1: t 2 units and its correction's 1, with at most 2.5 times their weight in h, the polynomial 4, its products 2, the
    exponential 2 with its correction 1: 16.5, and v's product 1, of v h; of 1 - h, h < 0.16, 3.2 and 2. Up to 1: the series 3, under .342 of
    a sum of at least .158 (v < 0) or .5, and 2.
    bf16 results before their rounding: t 3 with up to 3 times its weight, the polynomial 4, products 2, the exponential 2 and 1.5 v^2 for its
    argument's roundings: 17 + 1.5 v^2 of h, and v's product. Of 1 - h: at most 8.5 |v| (where h is a half) and 1 |v|."""
    if y_type == F32:
        return UNIT * np.abs(a) * np.where(np.abs(v) <= 1, np.where(v > 0, 5.0, 9.0), np.where(v > 0, 6.0, 17.5))
    return UNIT * np.where(v > 0, 10 * np.abs(v), (18 + 1.5 * v * v) * np.abs(a))


@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("span", [(-13, -5), (-5, -1), (-1, 0), (0, 1), (1, 3), (3, 20)])
def test_gelu(gpu, k3, span, y_type):
    say(f"case: {span} {y_type}")
    v = arguments(*span, 100000 if y_type == F32 else 400000, 3)
    a = lo.act64(v.astype(np.float64), "gelu")
    if y_type == F32:
        got, want, r = apply(k3, v, "gelu"), a, None
    else:
        r = torch.from_numpy(a).cuda().to(BF16)
        near = np.abs(a - lo.f64(r)) <= 2.0 ** -17 * np.abs(a)
        v, a, r = v[near], a[near], -r[torch.from_numpy(near).cuda()].unsqueeze(1)
        assert len(v) > 1000
        got, want = apply(k3, v, "gelu", r, BF16), a + lo.f64(r)[:, 0]
    tol = off_of_gelu(v.astype(np.float64), a, y_type) + 2.0 ** -145        # (h may be a subnormal: v 2^-149)
    half = 0 if r is None else np.maximum((np.abs(want) + tol) * lo.HALF[BF16], 2.0 ** -134)
    assert (np.abs(got - want) <= tol + half).all(), (np.abs(got - want) / np.abs(a) / UNIT).max()
