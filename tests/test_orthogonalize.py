# SPDX-License-Identifier: Apache-2.0
"""Newton-Schulz orthogonalisation against its formula in float64.

Tolerances.  The bfloat16 result is off by at most half a step of each entry (2^-8 of it), about 2^-8 / sqrt(3) of the norm.  On
top of that comes the rounding of the float16 operands, 2^-11 of their entries each; every step forms three products of them
and the polynomial has a slope of up to 3.45 where singular values are small and up to about 2 near 1, so relative errors of a
few 2^-12 from one step reach the result a few times enlarged: 2e-3 of the norm bounds the float16 arithmetic restated on the
CPU over Gaussian, noisy low-rank and low-rank matrices of 1 to 1024 rows, and is what is allowed here; an element may be off
by 12 times the root mean square error."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import orthogonalize as ortho

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
A, B, C = ortho.COEFFICIENTS


def _matrices(batch, m, n, kind, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * m + n)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if kind == "gauss":
        x = r(batch, m, n)
    else:
        k = max(1, min(m, n) // 8)
        x = (r(batch, m, k) * torch.logspace(0, -2, k)) @ r(batch, k, n) / k ** 0.5
        if kind == "noise":
            x = x + 0.02 * r(batch, m, n)
    return (1e-3 * x).to(dtype).to(device)


def _exact(g, steps=5, eps=1e-7):
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    eye = torch.eye(min(g.shape[-2:]), dtype=x.dtype, device=x.device)
    for _ in range(steps):
        if g.shape[-2] > g.shape[-1]:
            a = x.mT @ x
            x = x @ (A * eye + B * a + C * a @ a)
        else:
            a = x @ x.mT
            x = (A * eye + B * a + C * a @ a) @ x
    return x


def _near(got, want):
    assert got.dtype == BF16 and got.shape == want.shape
    d = got.double() - want
    # the result's own rounding (uniform errors: 1 / sqrt(3) of half a step) and the products', added as squares; a matrix of a
    # few entries averages nothing: both at their bounds
    norm = (2.0 ** -16 / 3 + 2e-3 ** 2) ** 0.5 if want.shape[-1] * want.shape[-2] >= 64 else 2.0 ** -8 + 2e-3
    rel = (torch.linalg.matrix_norm(d) / torch.linalg.matrix_norm(want)).max()
    rms = torch.linalg.matrix_norm(want)[..., None, None] / (want.shape[-1] * want.shape[-2]) ** 0.5
    worst = ((d.abs() - 2.0 ** -8 * want.abs()) / rms).max()
    assert float(rel) <= norm and float(worst) <= 12 * 2e-3, (float(rel), float(worst))


SHAPES = [(1, 1, 1), (3, 1, 9), (2, 9, 1), (5, 8, 8), (2, 33, 35), (4, 64, 64), (24, 128, 128), (3, 100, 128), (2, 128, 40), (1, 17, 300),
          (2, 300, 17), (1, 129, 129), (2, 130, 257), (1, 257, 130), (1, 515, 700), (3, 640, 64), (2, 128, 513), (1, 1024, 1024),
          (1, 7, 2000), (1, 1537, 515), (2, 1000, 1001), (1, 512, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["gauss", "noise", "low"])
@pytest.mark.parametrize("batch,m,n", SHAPES)
def test_kernels_against_float64(batch, m, n, kind):
    for dtype in (F32, BF16, F16):
        g = _matrices(batch, m, n, kind, dtype, "cuda")
        if dtype == F16:
            g = g * 64   # float16 gradients are scaled away from its smallest values
        _near(ortho.newton_schulz(g), _exact(g))
    assert ortho.check_errors(g) == 0


@pytest.mark.parametrize("batch,m,n", SHAPES[:12])
def test_formula_on_cpu(batch, m, n):
    g = _matrices(batch, m, n, "noise", F32, "cpu")
    _near(ortho.newton_schulz(g), _exact(g))


def test_singular_values_go_to_one_and_vectors_stay(device):
    g = _matrices(3, 40, 60, "gauss", F32, device)
    o = ortho.newton_schulz(g).float()
    s = torch.linalg.svdvals(o)
    assert float(s.min()) > 0.3 and float(s.max()) < 1.3
    u, _, vt = torch.linalg.svd(g, full_matrices=False)
    mid = u.mT @ o @ vt.mT
    off = mid - torch.diag_embed(torch.diagonal(mid, dim1=-2, dim2=-1))
    assert float(off.norm() / mid.norm()) < 1e-2   # twice the allowed error of the result


def test_scale_zero_and_nan(device):
    g = _matrices(4, 48, 80, "gauss", F32, device)
    base = ortho.newton_schulz(g, eps=0.0)
    for s in (1e-30, 1e30):                                         # squares leave the float32 range
        assert torch.equal(ortho.newton_schulz(g * s * 1e3, eps=0.0).isnan(), torch.zeros_like(base, dtype=torch.bool))
    assert torch.equal(ortho.newton_schulz(g * 2.0 ** 60, eps=0.0), base)   # a power of two changes nothing
    g[1] = 0
    g[2, 3, 4] = float("nan")
    o = ortho.newton_schulz(g)
    assert torch.equal(o[1], torch.zeros_like(o[1])) and o[2].isnan().all() and o[0].isfinite().all() and o[3].isfinite().all()


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 4, 4), (2, 3, 6, 10)])
def test_shapes(device, shape):
    g = torch.randn(shape, device=device)
    o = ortho.newton_schulz(g)
    assert o.shape == g.shape and o.dtype == BF16
    if len(shape) == 4:
        assert torch.equal(o[1, 2], ortho.newton_schulz(g[1, 2]))
        t = torch.randn(10, 6, device=device).t()                   # not contiguous
        assert torch.equal(ortho.newton_schulz(t), ortho.newton_schulz(t.contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(65537, 2, 3), (65536, 1, 260)])
def test_more_matrices_than_one_launch_takes(shape):
    g = torch.randn(shape, device="cuda")
    o = ortho.newton_schulz(g)
    assert torch.equal(o[-3:], ortho.newton_schulz(g[-3:])) and torch.equal(o[:3], ortho.newton_schulz(g[:3]))
    assert bool(o.isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6, 96, 128), (1, 400, 260)])
def test_captured_and_repeated(shape):
    g = torch.randn(shape, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ortho.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ortho.newton_schulz(g)
    for _ in range(2):
        g.copy_(torch.randn(shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ortho.newton_schulz(g))


def test_refusals(device):
    g = torch.randn(4, 4, device=device)
    with pytest.raises(ValueError, match="batch of matrices"):
        ortho.newton_schulz(g[0])
    with pytest.raises(TypeError, match="is needed"):
        ortho.newton_schulz(g.double())
    for steps in (0, 2.5, 101):
        with pytest.raises(ValueError, match="steps"):
            ortho.newton_schulz(g, steps=steps)
    with pytest.raises(ValueError, match="coefficients"):
        ortho.newton_schulz(g, coefficients=(1.0, float("nan"), 0.0))
    with pytest.raises(ValueError, match="grow beyond"):
        ortho.newton_schulz(g, coefficients=(10.0, 0.0, 0.0))
    with pytest.raises(ValueError, match="eps"):
        ortho.newton_schulz(g, eps=-1.0)
