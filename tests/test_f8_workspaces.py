# SPDX-License-Identifier: Apache-2.0
"""What the 8-bit path's workspaces hold: nothing that no call uses."""
import pytest


def up(n, m):
    return -(-n // m) * m


@pytest.mark.parametrize("T,hidden,inter,experts,topk", [(1, 7168, 2048, 64, 8), (64, 7168, 2048, 384, 8), (2048, 7168, 2048, 64, 8),
                                                         (65536, 4096, 1408, 128, 8), (100, 100, 1000, 4, 2)])
def test_moe(k3, T, hidden, inter, experts, topk):
    """The slots' rows take the place of gate and up's sums, which are codes by then."""
    L, N = k3.lib(), T * topk
    parts = [(experts + 1) * 4, N * 4, L.k3d_group_ws(T, topk, experts), N * up(inter, 128), N * up(inter, 128) // 32,
             N * max(2 * inter, up(hidden, 64)) * 4]
    assert L.k3d_moe_f8_ws(T, hidden, inter, experts, topk) == sum(up(p, 256) for p in parts)


def test_linear(k3):
    """Up to 64 tokens a dense product has no sums of slices."""
    L = k3.lib()
    for inn, out in ((7168, 12288), (128, 16), (1 << 20, 1 << 18)):
        assert all(L.k3d_linear_f8_ws(T, inn, out) == 0 for T in (1, 16, 17, 63, 64))
        assert L.k3d_linear_f8_ws(65, inn, out) > 0
