# SPDX-License-Identifier: Apache-2.0
"""Newton-Schulz orthogonalisation at extreme scales, of zero matrices and with NaN in one matrix of a batch, on every route:
matrices inside one SM (48 x 80), tiled products (300 x 260 in pairs and mirrored tiles, tall 260 x 100 with remainders)."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import orthogonalize as ortho
from tests.test_orthogonalize import _exact, _matrices, _near

F32 = torch.float32
SHAPES = [(48, 80), (80, 48), (300, 260), (260, 100), (100, 300), (1, 5)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("scale", [1e-27, 1e30, 2.0 ** 60])
def test_the_result_does_not_depend_on_the_scale(m, n, scale, device):
    """Without eps; the scaled entries are normal float32 values, so nothing is lost before the first product."""
    g = _matrices(3, m, n, "gauss", F32, device)
    base = ortho.newton_schulz(g, eps=0.0)
    _near(base, _exact(g, eps=0.0))
    scaled = g * scale
    _near(ortho.newton_schulz(scaled, eps=0.0), _exact(scaled, eps=0.0))


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("eps", [0.0, 1e-7])
def test_zero_and_nan_stay_in_their_matrix(m, n, eps, device):
    g = _matrices(4, m, n, "gauss", F32, device)
    base = ortho.newton_schulz(g, eps=eps)
    g[1] = 0
    g[2, m // 2, n // 3] = float("nan")
    o = ortho.newton_schulz(g, eps=eps)
    assert torch.equal(o[1], torch.zeros_like(o[1])) and o[2].isnan().all()
    assert torch.equal(o[0], base[0]) and torch.equal(o[3], base[3])
    g[2, m // 2, n // 3] = float("inf")
    assert ortho.newton_schulz(g, eps=eps)[2].isnan().all()
    zeros = torch.zeros_like(g[:1])
    assert torch.equal(ortho.newton_schulz(zeros, eps=eps), torch.zeros_like(o[:1]))
