# SPDX-License-Identifier: Apache-2.0
"""Second derivatives of layer norm and the gated block form only what an incoming gradient reaches.  The autograd functions of
the CUDA path are called directly, with the formulas in the place of the kernels where there is no GPU."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from nvalchemi_toolkit_b200.ops import feedforward as ff, norm
from tests.test_feedforward import _inputs

F64 = torch.float64


class _Count(TorchDispatchMode):
    def __init__(self, *names):
        super().__init__()
        self.names, self.n = names, 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.n += func.overloadpacket.__name__ in self.names
        return func(*args, **(kwargs or {}))


@pytest.fixture
def block(monkeypatch):
    monkeypatch.setattr(ff, "_forward_kernel", ff._forward_formula)
    return lambda *ts: ff._GatedFeedForward.apply(*ts, "silu")


def _force(y, x):
    return torch.autograd.grad(y.square().sum(), x, create_graph=True)[0]


def test_a_force_loss_through_the_block(block):
    ts = [t.requires_grad_() for t in _inputs(5, 6, 7, 4, F64, "cpu")[:4]]
    (f,) = torch.autograd.grad(block(*ts).square().sum(), ts[0], create_graph=True)
    with _Count("mm") as count:
        got = torch.autograd.grad(f.square().sum(), ts)
    # of the function's own derivative: g, u, dh, dx of two products, and both operands' gradients of these five: 15.  Around it
    # the second pass reaches y once more: its backward pass of 8 products
    assert count.n <= 15 + 8, count.n
    y = ff._forward_formula(*ts, "silu")
    for a, b in zip(got, torch.autograd.grad(_force(y, ts[0]).square().sum(), ts)):
        assert float((a - b).abs().max()) <= 1e-12 * max(1.0, float(b.abs().max()))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_each_gradient_alone_differentiates(block, which):
    """The second derivative through one first derivative only, whichever it is."""
    ts = [t.requires_grad_() for t in _inputs(5, 6, 7, 4, F64, "cpu")[:4]]
    dy = torch.randn(5, 4, dtype=F64, generator=torch.Generator().manual_seed(1))
    first = torch.autograd.grad(block(*ts), ts, dy, create_graph=True)[which]
    want = torch.autograd.grad(ff._forward_formula(*ts, "silu"), ts, dy, create_graph=True)[which]
    for a, b in zip(torch.autograd.grad(first.sin().sum(), ts, allow_unused=True),
                    torch.autograd.grad(want.sin().sum(), ts, allow_unused=True)):
        assert (a is None and b is None) or torch.allclose(torch.zeros_like(b) if a is None else a, torch.zeros_like(a) if b is None else b,
                                                            rtol=1e-12, atol=1e-12)


def test_a_force_loss_through_the_norm():
    x, w, b = (torch.randn(s, dtype=F64, generator=torch.Generator().manual_seed(i)).requires_grad_() for i, s in enumerate(((5, 8), (8,), (8,))))
    args = []
    formula = norm._backward_formula

    def spy(*a, **k):
        args.append(k.get("want", a[4] if len(a) > 4 else (True, True, True)))
        return formula(*a, **k)

    norm_backward, norm._backward_formula = norm._backward_formula, spy
    try:
        y = norm._LayerNorm.apply(x, w, b, 1e-5)
        f = _force(y, x)
        got = torch.autograd.grad(f.square().sum(), [x, w, b], allow_unused=True)
    finally:
        norm._backward_formula = norm_backward
    assert args == [(True, False, False)]
    want = torch.autograd.grad(_force(norm._forward_formula(x, w, b, 1e-5)[0], x).square().sum(), [x, w, b], allow_unused=True)
    for p, q in zip(got, want):
        assert float((p - q).abs().max()) <= 1e-10 * max(1.0, float(q.abs().max()))
