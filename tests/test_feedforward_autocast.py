# SPDX-License-Identifier: Apache-2.0
"""The gated feed-forward block inside ``torch.autocast`` regions."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import feedforward as ff
from tests.test_feedforward import _inputs

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


def test_what_autocast_casts():
    ts = _inputs(6, 16, 24, 8, F64, "cpu")[:4]
    want = ff.gated_feed_forward(*ts)
    with torch.autocast("cpu", dtype=BF16):
        y = ff.gated_feed_forward(*ts)
        assert (ts[0] @ ts[1]).dtype == F64 and y.dtype == F64 and torch.equal(y, want)   # float64 stays, as in a product
        with pytest.raises(TypeError, match="not supported"):
            ff.gated_feed_forward(*(t.long() for t in ts))
        with pytest.raises(TypeError, match="w_gate of type"):
            ff.gated_feed_forward(ts[0], *(t.float() for t in ts[1:]))
        assert ff.gated_feed_forward(*(t.float() for t in ts)).dtype == BF16


@pytest.mark.gpu
def test_float64_is_refused_inside_autocast_too():
    ts = _inputs(6, 16, 24, 8, F64, "cuda")[:4]
    with torch.autocast("cuda", dtype=BF16), pytest.raises(TypeError, match="float64 is not supported"):
        ff.gated_feed_forward(*ts)


def _force_step(ts, region):
    """Energy, force and the gradients of a force loss, all of it inside ``region``."""
    x, wg, wu, wd = (t.clone().requires_grad_() for t in ts)
    with region:
        e = ff.gated_feed_forward(x, wg, wu, wd).float().tanh().square().sum()
        (f,) = torch.autograd.grad(e, x, create_graph=True)
        return [e, f, *torch.autograd.grad(f.float().square().sum(), [x, wg, wu, wd])]


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_formulas_stay_wide_inside_autocast(act, device):
    """The formulas behind the CPU path and the second derivative have 32-bit products whatever the region asks for.  Sums of up
    to 24 terms, two dozen 32-bit operations in a chain, magnitudes sqrt(24) above the results: 500 half steps; bfloat16 products are
    off by more than 60,000 of them."""
    x, wg, wu, wd, dy = (t.requires_grad_() for t in _inputs(6, 16, 24, 8, F32, device))
    want = ff._backward_formula(dy, x, wg, wu, wd, act)
    wide = torch.autograd.grad(want[0].square().sum(), [dy, x, wg, wu, wd])
    with torch.autocast(device, dtype=BF16):
        y = ff._forward_formula(x, wg, wu, wd, act)
        got = ff._backward_formula(dy, x, wg, wu, wd, act)
        (first,) = torch.autograd.grad((y * dy).sum(), x, create_graph=True)
        again = torch.autograd.grad(got[0].square().sum(), [dy, x, wg, wu, wd])
        twice = torch.autograd.grad(first.square().sum(), [dy, x, wg, wu, wd])
    near = lambda a, b: float(((a - b).norm() / b.norm()).detach()) < 500 * 2.0 ** -24  # noqa: E731
    assert near(y, ff._forward_formula(x, wg, wu, wd, act)) and near(first, want[0])
    assert all(near(a, b) for a, b in zip(got, want)) and all(near(a, b) for a, b in zip(again, wide))
    assert all(near(a, b) for a, b in zip(twice, wide))


def test_force_training_inside_autocast(device):
    """The operator rounds its arguments and results to bfloat16 and nothing between: inside the region a step equals the same
    step on rounded arguments up to the roundings of y, of the force and of the gradients (each 2^-8, the force's counted twice in
    its square, second derivatives magnify them by the ratio of the magnitudes, 8 here)."""
    ts = [t.bfloat16().float() for t in _inputs(6, 16, 24, 8, F32, device)[:4]]
    got = _force_step(ts, torch.autocast(device, dtype=BF16))
    want = _force_step([t.double().cpu() for t in ts], torch.autocast("cpu", enabled=False))
    for a, b in zip(got, want):
        assert float(((a.double().cpu() - b).norm() / b.norm()).detach()) < 8 * 2.0 ** -8


def test_devices_without_autocast():
    """Shapes of a model on the meta device, as they are asked for before weights are loaded."""
    from nvalchemi_toolkit_b200.models import GatedBlock

    with torch.device("meta"):
        block = GatedBlock(8, 12)
        x = torch.empty(3, 8, requires_grad=True)
    y = block(x)
    assert y.shape == (3, 8) and y.device.type == "meta"
    assert [g.shape for g in torch.autograd.grad(y.sum(), [x, block.feed_forward.w_down])] == [(3, 8), (12, 8)]
