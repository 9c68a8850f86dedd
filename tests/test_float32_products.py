# SPDX-License-Identifier: Apache-2.0
"""Single float32 products of the gated feed-forward block on the tensor cores, by parts of 8 bits.

With gelu, ``x = [16, a]``, ``w_gate = [1, 0]``, ``w_up = [0, b]`` and ``w_down`` the unit matrix, ``y = 16 a b``: gelu(16) is 16 in
float32 and every other product has a factor that is a power of two.  Bound, in half steps (2^-24 of the value): the partial
products left out 1, the cuts of the sum of the others (their largest and the sum of the small ones) 2 each."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import feedforward as ff

F32 = torch.float32
pytestmark = pytest.mark.gpu


def _products(a, b):
    n = len(b)
    x = torch.stack([torch.full_like(a, 16.0), a], 1)
    wg = torch.zeros(2, n, device="cuda")
    wg[0] = 1
    wu = torch.stack([torch.zeros_like(b), b])
    return ff.gated_feed_forward(x, wg, wu, torch.eye(n, device="cuda"), "gelu").double() / 16


@pytest.mark.parametrize("rows", [8, 9, 50000])
@pytest.mark.parametrize("signs", [False, True])
def test_every_product_to_float32_accuracy(rows, signs):
    g = torch.Generator(device="cuda").manual_seed(rows)
    a, b = (1 + torch.rand(n, generator=g, device="cuda") for n in (rows, 64))
    b[:8] = torch.tensor([1.0, 1.9999999, 1.0039061, 1.0039062, 1.9960937, 1.9980469, 1.0078124, 1.5], device="cuda")
    a[:4] = torch.tensor([1.9999999, 1.0039061, 1.0078124, 1.0], device="cuda")
    if signs:
        a, b = a * (1 - 2 * (torch.arange(rows, device="cuda") % 2)), b * (1 - 2 * (torch.arange(64, device="cuda") % 3 % 2))
    want = a.double()[:, None] * b.double()
    rel = ((_products(a, b) - want) / want).abs()
    assert float(rel.max()) <= 5 * 2.0 ** -24, float(rel.max()) * 2 ** 24


def test_the_ends_of_the_range():
    """The largest float32 values, and infinities and NaN, survive the split."""
    top = torch.finfo(F32).max
    a = torch.tensor([top, -top, top * (1 - 2.0 ** -9), top * (1 - 2.0 ** -8), 1.0] * 4, device="cuda")
    b = torch.tensor([2.0 ** -6, -0.75 * 2.0 ** -5, 1.9999999 * 2.0 ** -7], device="cuda")
    want = a.double()[:, None] * b.double()
    assert float(((_products(a, b) - want) / want).abs().max()) <= 5 * 2.0 ** -24
    for bad in (float("inf"), -float("inf"), float("nan")):
        a[7] = bad
        y = _products(a, b)
        assert not y[7].isfinite().any() and y[:7].isfinite().all() and y[8:].isfinite().all()
