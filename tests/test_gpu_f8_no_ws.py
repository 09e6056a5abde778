# SPDX-License-Identifier: Apache-2.0
"""k3d_linear_f8 of few tokens without a workspace."""
import pytest
import torch

from layer8_ops import BF16, F32, acts, addr, linear8, nb, tile, weights
from layer_ops import TYPE, gen, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,inn,out", [(1, 640, 300), (37, 1001, 130), (64, 256, 64)])
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_none(gpu, T, inn, out, y_type):
    g = gen(T)
    x, xs = acts(g, T, inn)
    w, ws = weights(g, 1, out, inn)
    wt = tile(gpu, w)
    want = linear8(gpu, x, xs, wt, ws, inn, out, y_type=y_type)
    y = torch.full_like(want, 7.0)
    gpu.check(gpu.lib().k3d_linear_f8(addr(y), TYPE[y_type], out, addr(x), x.stride(0), addr(xs), nb(inn), T, addr(wt), addr(ws), nb(inn), inn,
                                      out, None, 0, None, 0, None, 0, stream()), "k3d_linear_f8")
    assert torch.equal(y, want)
