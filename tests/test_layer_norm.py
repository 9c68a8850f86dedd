# SPDX-License-Identifier: Apache-2.0
"""Layer norm against the definition in float64: values, gradients, second derivatives, strides, refusals, graphs.

Tolerances.  A stored result is off by at most half a step of its type, ``finfo.eps / 2`` relative.  In 32-bit arithmetic
the normalised value carries the rounding of the mean and of ``x - mean`` (each 2^-24 of ``|x|`` at most, divided by the
row's deviation) and a handful of operations of 2^-24 each; row sums of n terms add at most about log2(n) + n / 32 more.
With rows whose mean is at most ``3`` deviations that stays under 64 * 2^-24 of the row's largest term, which is what
``_BASE`` counts; column sums over R rows get sqrt(R) + 16 roundings of the root mean square term on top."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import norm

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
_BASE = 64 * 2.0 ** -24


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(rows, cols, dtype, wdtype, device, step=1, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 31 + cols)
    x = (torch.randn(rows, 1, generator=g) + (0.5 + torch.rand(rows, 1, generator=g)) * torch.randn(rows, step * cols, generator=g))
    x = x.to(dtype).to(device)[:, :cols]
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(wdtype).to(device)
    b = (0.2 * torch.randn(cols, generator=g)).to(wdtype).to(device)
    dy = torch.randn(rows, cols, generator=g).to(dtype).to(device)
    return x, w, b, dy


def _exact(x, w, b, dy, eps=1e-5):
    ts = [t.double().detach().requires_grad_() for t in (x, w, b)]
    var, mean = torch.var_mean(ts[0], -1, unbiased=False, keepdim=True)
    y = (ts[0] - mean) * (var + eps) ** -0.5 * ts[1] + ts[2]
    return (y.detach(), *torch.autograd.grad(y, ts, dy.double()))


def _check_all(got, want, rows, dtype, wdtype, terms):
    acc = _BASE if dtype != F64 else 64 * 2.0 ** -53
    for k, (a, e) in enumerate(zip(got, want)):
        t = dtype if k < 2 else wdtype
        assert a.dtype == t and a.shape == e.shape
        scale = terms[k]
        extra = acc * scale * (1 if k < 2 else (rows ** 0.5 + 16) * max(1.0, rows ** 0.5) / 16)
        assert ((a.double() - e).abs() <= _half_step(t) * e.abs() + extra).all(), (k, float((a.double() - e).abs().max()))


SHAPES = [(1, 1), (1, 7), (3, 64), (21, 64), (5, 128), (130, 256), (17, 333), (9, 1000), (33, 1024), (4, 1032), (3, 2048),
          (7, 4096), (2, 5001), (2, 8192), (700, 24), (1, 513), (2048, 8)]
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F64, F64)]


def _run(rows, cols, dtype, wdtype, device, step=1):
    x, w, b, dy = _inputs(rows, cols, dtype, wdtype, device, step)
    y, mean, rstd = norm.layer_norm_forward(x, w, b)
    grads = norm.layer_norm_backward(dy, x, mean, rstd, w)
    want = _exact(x, w, b, dy)
    r = rstd.double()[:, None]
    xm = (x.double().abs().amax(-1, keepdim=True) * r).clamp(min=1)      # the largest normalised value, mean included
    gw = (dy.double() * w.double()).abs().amax(-1, keepdim=True)
    terms = [xm * (1 + w.double().abs().max()), r * gw * xm * (2 + xm), (dy.double().abs() * xm).amax(0), dy.double().abs().amax(0)]
    _check_all((y, *grads), want, rows, dtype, wdtype, terms)


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES[:8])
def test_formulas_on_cpu(rows, cols, dtype, wdtype):
    _run(rows, cols, dtype, wdtype, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_kernels_against_float64(rows, cols, dtype, wdtype):
    _run(rows, cols, dtype, wdtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(200, 128), (3000, 333), (100003, 64)])
def test_strided_rows_and_many_rows(rows, cols, dtype):
    _run(rows, cols, dtype, F32, "cuda", step=4)


def test_autograd_matches_formula_and_differences(device):
    x, w, b, dy = _inputs(6, 10, F64, F64, device)
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    assert torch.autograd.gradcheck(lambda *a: norm.layer_norm(*a, 1e-3), args)
    assert torch.autograd.gradgradcheck(lambda *a: norm.layer_norm(*a, 1e-3), args)
    assert torch.autograd.gradcheck(lambda a: norm.layer_norm(a, None, None, 1e-3), args[:1])
    assert torch.autograd.gradgradcheck(lambda a, c: norm.layer_norm(a, None, c, 1e-3), [args[0], args[2]])


def test_force_training_step_differentiates_twice(device):
    """Energy -> force -> gradient of a force loss, float32: against the same graph in float64."""
    def grads(dt):
        g = torch.Generator().manual_seed(4)
        x = torch.randn(12, 3, generator=g, dtype=F64).to(device, dt).requires_grad_()
        win = torch.randn(3, 40, generator=g, dtype=F64).to(device, dt)
        w = (1 + 0.1 * torch.randn(40, generator=g, dtype=F64)).to(device, dt).requires_grad_()
        b = torch.zeros(40, device=device, dtype=dt, requires_grad=True)
        e = torch.tanh(norm.layer_norm(x @ win, w, b)).pow(2).sum()
        (f,) = torch.autograd.grad(e, x, create_graph=True)
        return torch.autograd.grad(f.pow(2).sum(), [w, b])
    for a, e in zip(grads(F32), grads(F64)):
        # a chain of about twenty 32-bit operations on sums of 40 terms, three derivatives deep
        assert float((a.double() - e).norm() / e.norm()) < 2000 * 2.0 ** -24


@pytest.mark.parametrize("rows", [0, 1])
def test_empty_and_expanded(device, rows):
    x = torch.randn(rows, 16, device=device, requires_grad=True)
    w = torch.ones(16, device=device, requires_grad=True)
    norm.layer_norm(x, w, None).sum().backward()                       # the gradient arrives expanded from one number
    assert x.grad.shape == x.shape and w.grad.shape == (16,) and torch.isfinite(w.grad).all()
    row = torch.randn(1, 16, device=device, requires_grad=True)
    y = norm.layer_norm(row.expand(5, 16), w, None)
    assert torch.equal(y[0], y[4])
    y[:3].square().sum().backward()                                    # a broadcast input collects its copies' gradients
    assert row.grad.shape == (1, 16)


@pytest.mark.gpu
def test_other_layouts_equal_the_contiguous_ones():
    x, w, b, dy = _inputs(60, 96, F32, F32, "cuda")
    y, m, r = norm.layer_norm_forward(x, w, b)
    t = x.t().contiguous().t()                                         # columns contiguous: copied
    assert torch.equal(norm.layer_norm(t, w, b), y)
    off = torch.empty(60 * 96 + 1, device="cuda")[1:].view(60, 96).copy_(x)   # rows off the 16-byte boundary
    assert torch.allclose(norm.layer_norm(off, w, b), y, rtol=0, atol=32 * 2.0 ** -24 * float(y.abs().max()))
    assert torch.equal(norm.layer_norm(x.view(3, 20, 96), w, b), y.view(3, 20, 96))
    wide = torch.randn(2, 96, device="cuda").repeat_interleave(2, dim=1)[:, ::2]
    assert torch.equal(norm.layer_norm(x, wide[0], wide[1]), norm.layer_norm(x, wide[0].contiguous(), wide[1].contiguous()))
    a = norm.layer_norm_backward(dy, x, m, r, w)
    assert all(torch.equal(p, q) for p, q in zip(a, norm.layer_norm_backward(dy, x, m, r, w)))   # the same bits again


@pytest.mark.gpu
def test_constant_rows_infinities_and_nan():
    x = torch.randn(4, 64, device="cuda")
    x[0] = 3.0
    x[1, 5] = float("inf")
    x[2, 9] = float("nan")
    y = norm.layer_norm(x, None, None)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and y[1].isnan().all() and y[2].isnan().all() and y[3].isfinite().all()
    big = torch.randn(3, 64, device="cuda") + 1e4                        # a mean far above the deviation
    want = torch.nn.functional.layer_norm(big.double(), (64,))
    assert float((norm.layer_norm(big).double() - want).abs().max()) < 4 * 1e4 * 2.0 ** -24 * 8


@pytest.mark.gpu
def test_captured_passes_replay_on_new_inputs():
    x, w, b, dy = _inputs(300, 128, BF16, F32, "cuda")
    out = {}

    def step():
        y, m, r = norm.layer_norm_forward(x, w, b)
        out["v"] = (y, *norm.layer_norm_backward(dy, x, m, r, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    captured = out["v"]
    for seed in (1, 2):
        nx, _, _, ndy = _inputs(300, 128, BF16, F32, "cuda", seed=seed)
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        step()
        assert all(torch.equal(p, q) for p, q in zip(captured, out["v"]))


def test_refusals(device):
    x, w = torch.randn(4, 8, device=device), torch.ones(8, device=device)
    with pytest.raises(TypeError, match="must be float32"):
        norm.layer_norm(x.long(), w)
    with pytest.raises(ValueError, match="last axis"):
        norm.layer_norm(torch.zeros((), device=device))
    with pytest.raises(ValueError, match="last axis"):
        norm.layer_norm(torch.zeros(3, 0, device=device))
    with pytest.raises(ValueError, match="last axis"):
        norm.layer_norm(torch.zeros(1, norm.MAX_COLS + 1, device=device))
    with pytest.raises(ValueError, match="weight has shape"):
        norm.layer_norm(x, torch.ones(1, device=device))
    with pytest.raises(TypeError, match="weight of type"):
        norm.layer_norm(x, w.double())
    with pytest.raises(TypeError, match="weight of type"):
        norm.layer_norm(x.bfloat16(), w.half())
    with pytest.raises(TypeError, match="one type"):
        norm.layer_norm(x.bfloat16(), w, w.bfloat16())
    y, m, r = norm.layer_norm_forward(x, w)
    with pytest.raises(ValueError, match="does not match x"):
        norm.layer_norm_backward(y[:2], x, m, r, w)
    with pytest.raises(ValueError, match="mean must be"):
        norm.layer_norm_backward(y, x, m[:2], r, w)
    with pytest.raises(TypeError, match="param_dtype"):
        norm.layer_norm_backward(y, x, m, r, None, param_dtype=torch.float64)
    if device == "cuda":
        with pytest.raises(ValueError, match="weight is on"):
            norm.layer_norm(x, w.cpu())
