# SPDX-License-Identifier: Apache-2.0
"""Newton-Schulz orthogonalisation of matrices with one very long side: the bounds of ``tests/test_orthogonalize.py``, which do
not grow with the length."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import orthogonalize as ortho
from tests.test_orthogonalize import _exact, _matrices, _near

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "noise"])
@pytest.mark.parametrize("batch,m,n,dtype", [
    (1, 64, 1000000, F32), (1, 1000000, 64, BF16), (1, 300, 400000, F32), (3, 9, 70001, F32), (2, 70000, 257, F16), (2, 129, 65600, BF16),
    (1, 1, 4200000, F32)])
def test_long_sides_against_float64(batch, m, n, dtype, kind):
    g = _matrices(batch, m, n, kind, dtype, "cuda")
    if dtype == F16:
        g = g * 64
    _near(ortho.newton_schulz(g), _exact(g))
    assert ortho.check_errors(g) == 0
