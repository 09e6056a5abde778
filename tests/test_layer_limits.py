# SPDX-License-Identifier: Apache-2.0
"""k3d_linear at the most work that a launch takes: refused with its reason, or done in several."""
import pytest
import torch

import layer_ops as lo
from layer_ops import BF16, F32

A = 4096            # an address that nothing reads


@pytest.mark.parametrize("T,out", [(1 << 24, (1 << 13) + 1), (1 << 24, 1 << 28), ((1 << 9) + 1, 1 << 28)])
@pytest.mark.parametrize("inn", [64, 72, 101])
@pytest.mark.parametrize("x_type", [0, 1])
def test_results(k3, T, inn, out, x_type):
    rc = k3.lib().k3d_linear(A, 1, out, 2 * A, x_type, inn, T, 3 * A, inn, inn, out, None, 0, None, 0, 5 * A, 1 << 60, None)
    assert rc != 0 and "MAX_RESULTS" in k3.lib().k3d_error().decode()


@pytest.mark.gpu
def test_rows_laid_out_in_two_launches(gpu, k3):
    """2^32 pieces of x, more than one launch has work-items: rows of 2041 columns, which the workspace takes in another form."""
    T, inn, out = 1 << 24, 2041, 3
    if torch.cuda.mem_get_info()[0] < 170 << 30:
        pytest.skip("needs 170 GiB of device memory")
    print(f"case: {T} x {inn} -> {out}", flush=True)
    x = torch.ones(T, inn, device="cuda", dtype=BF16)
    w = torch.randint(-3, 4, (out, inn), device="cuda", generator=lo.gen(1)).to(BF16)
    at = torch.tensor([0, 1, 63, 64, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 23) + 64, T - 65, T - 1], device="cuda")
    x[at] = torch.randint(-9, 10, (len(at), inn), device="cuda", generator=lo.gen(2)).to(BF16)
    try:
        y = lo.linear(k3, x, w, y_type=F32)
        assert torch.equal(y[at].double(), x[at].double() @ w.double().T)
        y[at] = w.float().sum(1)
        assert (y == w.float().sum(1)).all()
    finally:
        del x
        torch.cuda.empty_cache()
