# SPDX-License-Identifier: Apache-2.0
"""k3d_route with finite biases that mask or force experts: up to the lowest and the largest fp32 values, whose sums in a
group are past fp32 and not past 64 bits. Experts exactly and weights within their one rounding, as the definition has them."""
import itertools

import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

pytestmark = pytest.mark.gpu
LOW, INF = torch.finfo(F32).min, float("inf")


def say(msg):
    print(msg, flush=True)


def masks(n, gs):
    """Biases of n experts in groups of gs: name -> tensor."""
    e = torch.arange(n, device="cuda")
    some = torch.randn(n, device="cuda", generator=lo.gen(n)) * 0.05
    put = lambda where, value, rest: torch.where(where, torch.as_tensor(value, device="cuda", dtype=F32), torch.as_tensor(rest, device="cuda", dtype=F32))
    yield "all but the first group at the lowest value", put(e >= gs, LOW, 0.0)
    yield "all but the last group, others near zero", put(e < n - gs, LOW, some)
    yield "all at the lowest value", torch.full((n,), LOW, device="cuda")
    yield "all but one expert of each group", put(e % gs != gs // 2, LOW, some)
    yield "one expert in the middle left", put(e != n // 2 + 1, LOW, 0.0)
    yield "the lowest value and -inf in turns of a group", put(e // gs % 2 == 0, LOW, -INF)
    yield "-inf but for two groups of the lowest value", put((e // gs == 1) | (e // gs == n // gs - 1), LOW, -INF)
    yield "pairs just past the lowest sum, by group", -1.7e38 - 1e36 * (e // gs % 5).float()
    yield "pairs on both sides of the lowest sum", put(e // gs % 2 == 0, -1.69e38, -1.72e38)
    yield "half of each group at the lowest value", put(e % gs < (gs + 1) // 2, LOW, some)
    yield "pairs past the largest sum, by group", 1.7e38 + 1e36 * (e // gs % 5).float()
    yield "the largest value in one group and past it in the next", put(e // gs == 0, 3.4e38, put(e // gs == 1, 1.75e38, 0.0))
    yield "the largest and the lowest in one group", put(e % gs == 0, -LOW, put(e % gs == 1, LOW, some))
    yield "an infinite one beside the lowest", put(e == n - 1, INF, LOW)
    yield "-1e9 on a tenth", put(e % 10 == 3, -1e9, some)
    yield "-1e9 on all but a few", put(e % gs > 1, -1e9, some)
    yield "1e4 on one group", put(e // gs == n // gs // 2, 1e4, some)


@pytest.mark.parametrize("score,dtype", itertools.product([0, 1], [F32, BF16]))
@pytest.mark.parametrize("n,groups,top_groups,topk", [
    (16, 4, 2, 8), (64, 8, 2, 12), (64, 1, 1, 12), (64, 64, 9, 9), (128, 1, 1, 64), (160, 8, 3, 6), (192, 3, 2, 64), (257, 1, 1, 12),
    (384, 8, 4, 8), (513, 27, 4, 9), (896, 8, 4, 16), (2048, 64, 7, 64), (2046, 2, 1, 5)])
def test_finite_masks(gpu, k3, n, groups, top_groups, topk, score, dtype):
    lg = (torch.randn(5, n, device="cuda", generator=lo.gen(topk)) * 1.5).to(dtype)
    lg[1] = 0.25
    lg[2, ::3] = -INF
    lg[3] = LOW if dtype == F32 else torch.finfo(BF16).min
    for name, bias in masks(n, n // groups):
        for group_top, renorm in ((1, 1), (2, 0), (2, 1)):
            say(f"case: {n} {groups} {top_groups} {topk} score {score} {dtype} top {group_top}: {name}")
            got = lo.route(k3, lg, bias, score, groups, top_groups, group_top, topk, renorm, 2.5)
            lo.check_route(got, lo.route64(lg, bias, score, groups, top_groups, group_top, topk, renorm, 2.5))


def test_masked_groups_are_taken(gpu, k3):
    """Eight experts without a mask, four more out of groups whose two largest choices sum to less than any fp32 number."""
    say("case: 64 experts, 8 unmasked, top 12 of 2 groups")
    lg = torch.randn(3, 64, device="cuda", generator=lo.gen(5))
    bias = torch.full((64,), LOW, device="cuda")
    bias[:8] = 0
    idx, wt = lo.route(k3, lg, bias, 0, 8, 2, 2, 12, 0, 1.0)
    assert (idx[:, :8].sort(1).values == torch.arange(8, device="cuda")).all()
    assert idx[:, 8:].tolist() == [[8, 9, 10, 11]] * 3
    s = torch.sigmoid(lg.double()).gather(1, idx.long())
    assert ((wt.double() - s).abs() <= 2.0 ** -23 * s).all()
