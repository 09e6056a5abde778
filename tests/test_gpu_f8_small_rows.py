# SPDX-License-Identifier: Apache-2.0
"""k3d_add_norm of rows whose squares are small, with an eps of 0."""
import numpy as np
import pytest
import torch

from layer8_ops import F32, add_norm, norm64
from layer_ops import HALF, gen, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [128, 1000, 7168])
def test_eps_zero(gpu, n):
    """As exact as any down to squares of 2^-126; rows whose squares all vanish, and rows of zeros, are NaN."""
    x = torch.randn(6, n, device="cuda", generator=gen(n))
    x = x.sign() * (x.abs() + 0.25)
    x *= torch.tensor([1.0, 2.0 ** -20, 2.0 ** -60, 2.0 ** -85, 0.0, 1.0], device="cuda")[:, None]
    y = torch.full_like(x, 7.0)
    add_norm(gpu, x, eps=0.0, y=y)
    ok = [0, 1, 2, 5]
    _, u, tol = norm64(x[ok], None, None, 0.0)
    within(y[ok], (u, tol + (np.abs(u) + tol) * HALF[F32]))
    assert torch.isnan(y[[3, 4]]).all()
