# SPDX-License-Identifier: Apache-2.0
"""Outputs and workspaces of the 8-bit path that are another argument's place: refused before anything reaches a device."""
import pytest

from test_f8_refusals import A, BIG, LINEAR, MOE, NORM, QUANT, refused


@pytest.mark.parametrize("change,word", [
    (dict(qs=A), "one place"), (dict(qs=2 * A), "one place"), (dict(qs=4 * A), "one place"), (dict(qs=5 * A), "operand"),
    (dict(qs=6 * A), "operand"), (dict(qs=7 * A), "operand"), (dict(q=7 * A), "operand"), (dict(y=7 * A), "operand"), (dict(sum=7 * A), "operand")])
def test_norm(k3, change, word):
    refused(k3, k3.lib().k3d_add_norm(*dict(NORM, **change).values(), None), word)


@pytest.mark.parametrize("change,word", [(dict(qs=A), "one place"), (dict(qs=3 * A), "operand")])
def test_quant(k3, change, word):
    refused(k3, k3.lib().k3d_quant_f8(*dict(QUANT, **change).values(), None), word)


@pytest.mark.parametrize("ws", [2 * A, 3 * A, 4 * A, 5 * A, 6 * A, 7 * A])
def test_linear(k3, ws):
    refused(k3, k3.lib().k3d_linear_f8(*dict(LINEAR, T=100, ws=ws).values(), None), "workspace lies")


@pytest.mark.parametrize("ws", [A, 2 * A, 3 * A])
def test_group(k3, ws):
    refused(k3, k3.lib().k3d_group(A, 2 * A, 3 * A, 1000, 8, 64, ws, BIG, None), "workspace lies")


@pytest.mark.parametrize("change,word", [(dict(out=i * A), "operand") for i in range(2, 13)] + [(dict(ws=i * A), "workspace lies") for i in range(2, 12)])
def test_moe(k3, change, word):
    refused(k3, k3.lib().k3d_moe_f8(*dict(MOE, **change).values(), None), word)
