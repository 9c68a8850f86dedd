# SPDX-License-Identifier: Apache-2.0
"""The activations of the gated feed-forward block on CUDA, value by value.

``x = [g, 1]`` with ``w_gate = [1, 0]``, ``w_up = [0, 1]`` and ``w_down = 1`` gives ``y = act(g)``, ``dx[0] = act'(g)`` and
``dx[1] = act(g)``: every product of the chain is one number times one, and exact.  Bounds, in half steps of float32 (2^-24): an exponential
2, its argument 1, a quotient 4, a polynomial of one sign's size 5, three products 3: 16 of the value, and for a derivative of the
sum of the magnitudes of its terms.  16-bit results add half a step of their type for h and one for the result, with 1e-5 of the value for the fast functions."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import feedforward as ff
from tests.test_feedforward import _half_step

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
pytestmark = pytest.mark.gpu


def _values(g):
    """``act, act', |terms of act'|`` of both activations in float64."""
    s, r = torch.sigmoid(g), torch.sigmoid(-g)
    p, phi = torch.special.erfc(-g / 2 ** 0.5) / 2, torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    return {"silu": (g * s, s + g * s * r, s + (g * s * r).abs()), "gelu": (g * p, p + g * phi, p + (g * phi).abs())}


def _call(g, act):
    """``act(g), act'(g), act(g)`` by the operator, for a vector ``g``."""
    dt = g.dtype
    x = torch.stack([g, torch.ones_like(g)], 1)
    wg, wu = torch.tensor([[1.0], [0.0]], device="cuda", dtype=dt), torch.tensor([[0.0], [1.0]], device="cuda", dtype=dt)
    one = torch.ones(1, 1, device="cuda", dtype=dt)
    dx = ff.gated_feed_forward_backward(torch.ones(len(g), 1, device="cuda", dtype=dt), x, wg, wu, one, act)[0]
    return ff.gated_feed_forward(x, wg, wu, one, act)[:, 0], dx[:, 0], dx[:, 1]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [8, 200, 100001])
def test_float32_values(act, rows):
    g = torch.linspace(-10, 10, rows, device="cuda", dtype=F64).to(F32)
    a, da, terms = _values(g.double())[act]
    y, d, h = _call(g, act)
    unit = 16 * 2.0 ** -24
    for got in (y, h):
        assert float(((got.double() - a).abs() - unit * a.abs()).max()) <= 0
    assert float(((d.double() - da).abs() - unit * terms).max()) <= 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_float32_far_values(act):
    """Past the exponential's range: results below 2^-126 may become zero, nothing else changes."""
    g = torch.tensor([s * v for v in (11.0, 14.0, 30.0, 86.0, 87.5, 90.0, 104.0, 1e3, 1e10, 1e20, 1e37, 3e38) for s in (1, -1)], device="cuda")
    a, da, terms = _values(g.double())[act]
    for rows in (g, g[:8], g[-8:]):
        y, d, h = _call(rows, act)
        i = 0 if rows is g or len(rows) == 8 and torch.equal(rows, g[:8]) else len(g) - 8
        want, slope, size = a[i:i + len(rows)], da[i:i + len(rows)], terms[i:i + len(rows)]
        for got in (y, h):
            assert float(((got.double() - want).abs() - 16 * 2.0 ** -24 * want.abs()).max()) <= 128 * 2.0 ** -126
        assert float(((d.double() - slope).abs() - 16 * 2.0 ** -24 * size).max()) <= 128 * 2.0 ** -126


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [200, 100001])
def test_16_bit_values(act, dtype, rows):
    g = torch.linspace(-10, 10, rows, device="cuda", dtype=F64).to(dtype)
    a, da, terms = _values(g.double())[act]
    y, d, h = _call(g, act)
    for got, want, size in ((y, a, a), (h, a, a), (d, da, terms)):
        assert got.dtype == dtype
        bound = 2 * _half_step(want, dtype) + 1e-5 * size.abs()
        assert float(((got.double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_nan_and_infinity(act):
    g = torch.tensor([float("nan"), float("inf"), 1.0] * 4, device="cuda")
    for n in (3, 12):
        y, d, h = _call(g[:n], act)
        assert y[0].isnan() and d[0].isnan() and h[0].isnan() and not y[1].isfinite() and not h[1].isfinite() and y[2].isfinite()
