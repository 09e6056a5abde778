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
