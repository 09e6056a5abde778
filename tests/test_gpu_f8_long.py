# SPDX-License-Identifier: Apache-2.0
"""The tiles of k3d_linear_f8 and k3d_grouped_f8 over long rows: scales of x in their second half and back, of W past the 64 column
blocks that a wave holds, on integers whose sums are exact (a bf16 result is their rounding)."""
import pytest
import torch

from layer8_ops import BF16, F32, F8, acts, grouped, linear8, nb, tile, weights
from layer_ops import gen

pytestmark = pytest.mark.gpu


def rows(q, s, n):
    return (q.view(F8).double() * s.double().repeat_interleave(128, 1))[:, :n]


def matrix(q, s):
    out, inn = q.shape
    return q.view(F8).double() * s.double().repeat_interleave(128, 0)[:out].repeat_interleave(128, 1)[:, :inn]


# tokens and outputs whose tiles fill 256 CUs in one slice: as 256 x 256, 128 x 256, 128 x 128
@pytest.mark.parametrize("T,out,y_type", [(4000, 4090, BF16), (2000, 4090, BF16), (2000, 2040, BF16), (2000, 4090, F32)])
@pytest.mark.parametrize("blocks", [9, 17, 56, 66, 130])
def test_linear(gpu, T, out, y_type, blocks):
    inn, g = blocks * 128 - 5, gen(T + blocks)
    x, xs = acts(g, T, inn, True)
    w, ws = weights(g, 1, out, inn, True)
    y = torch.full((T + 1, out), 7.0, device="cuda", dtype=y_type)
    linear8(gpu, x, xs, tile(gpu, w), ws, inn, out, y=y[:T])
    want = rows(x, xs, inn) @ matrix(w[0], ws[0]).T
    assert torch.equal(y[:T], want.to(y_type)) and (y[T:] == 7).all()


@pytest.mark.parametrize("y_type", [BF16, F32])
@pytest.mark.parametrize("blocks", [9, 17, 66, 130])
def test_grouped(gpu, y_type, blocks):
    """Experts on both sides of half a tile and of a tile."""
    counts = [127, 128, 129, 255, 256, 257, 300, 0, 385]
    inn, out, g, n = blocks * 128 - 5, 520, gen(blocks), sum(counts)
    x, xs = acts(g, n, inn, True)
    w, ws = weights(g, len(counts), out, inn, True)
    off = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
    y = torch.full((n + 1, out), 7.0, device="cuda", dtype=y_type)
    grouped(gpu, y[:n], x, xs, off, n, tile(gpu, w), ws, inn, out)
    X, o = rows(x, xs, inn), off.tolist()
    assert nb(inn) == blocks and (y[n:] == 7).all()
    for e in range(len(counts)):
        r = slice(o[e], o[e + 1])
        assert torch.equal(y[r], (X[r] @ matrix(w[e], ws[e]).T).to(y_type)), e
