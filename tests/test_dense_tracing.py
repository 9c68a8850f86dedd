# SPDX-License-Identifier: Apache-2.0
"""Layer norm, the gated block and Newton-Schulz on tensors without memory (``FakeTensorMode``): tracing a model must not reach
the kernels, which would read and write where nothing is."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from nvalchemi_toolkit_b200.ops import _native, feedforward as ff, norm, orthogonalize as ortho

OPS = ["layer_norm_apply", "layer_norm_fwd", "layer_norm_bwd", "gated_ff_fwd", "gated_ff_bwd", "gated_ff_error_status", "newton_schulz",
       "newton_schulz_error_status"]


@pytest.fixture(autouse=True)
def _library():
    if not _native.available():
        pytest.skip("native library not built")


@pytest.mark.parametrize("name", OPS)
def test_tracing_does_not_enter_the_operator(name):
    """An operator that tracing decomposes would run its C++ on tensors without memory."""
    assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"nvalchemi::{name}", "CompositeImplicitAutograd")
    if not name.endswith("status"):
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"nvalchemi::{name}", "Meta")


def _same(a, shape, dtype):
    assert tuple(a.shape) == shape and a.dtype == dtype and a.is_contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_and_types(dtype):
    if torch._C._dispatch_has_kernel_for_dispatch_key("nvalchemi::layer_norm_apply", "CompositeImplicitAutograd"):
        pytest.fail("not safe to call")
    with FakeTensorMode():
        e = lambda *s, dt=dtype: torch.empty(*s, device="cuda", dtype=dt)  # noqa: E731
        x, w = e(3, 5, 8), e(8, dt=torch.float32)
        _same(norm.layer_norm(x, w, w), (3, 5, 8), dtype)
        y, m, r = norm.layer_norm_forward(x, w)
        _same(m, (15,), torch.float32)
        for a, s, t in zip(norm.layer_norm_backward(y, x, m, r, w), ((3, 5, 8), (8,), (8,)), (dtype, torch.float32, torch.float32)):
            _same(a, s, t)
        assert norm.layer_norm_backward(y, x, m, r, w, param_grads=False)[1:] == (None, None)
        _same(norm.layer_norm_backward(y, x, m, r)[1], (8,), dtype)
        wg, wd = e(8, 12), e(12, 4)
        z = ff.gated_feed_forward(x, wg, wg, wd)
        _same(z, (3, 5, 4), dtype)
        for a, s in zip(ff.gated_feed_forward_backward(z, x, wg, wg, wd), ((3, 5, 8), (8, 12), (8, 12), (12, 4))):
            _same(a, s, dtype)
        dx, *dw = ff.gated_feed_forward_backward(z, x, wg, wg, wd, input_grad=False)
        assert dx is None and tuple(dw[0].shape) == (8, 12)
        _same(ortho.newton_schulz(x), (3, 5, 8), torch.bfloat16)
        with pytest.raises(ValueError, match="weight has shape"):
            norm.layer_norm(x, w[:3])
        with pytest.raises(ValueError, match="do not fit"):
            ff.gated_feed_forward(x, wg, wg, wg)
        with pytest.raises(ValueError, match="activation"):
            ff.gated_feed_forward(x, wg, wg, wd, "relu")


@pytest.mark.gpu
def test_a_traced_training_step_has_the_operators_as_nodes():
    """``make_fx`` over forward and backward pass on fake tensors, then the graph on real ones: the eager results."""
    from torch.fx.experimental.proxy_tensor import make_fx

    g = torch.Generator().manual_seed(0)
    ts = [torch.randn(s, generator=g).cuda() for s in ((20, 16), (16,), (16, 24), (16, 24), (24, 16), (20, 16))]

    def step(x, w, wg, wu, wd, dy):
        y, m, r = norm.layer_norm_forward(x, w)
        z = ff.gated_feed_forward(y, wg, wu, wd)
        dn, *dw = ff.gated_feed_forward_backward(dy, y, wg, wu, wd)
        return z, *norm.layer_norm_backward(dn, x, m, r, w), *dw, ortho.newton_schulz(dw[0])

    graph = make_fx(step, tracing_mode="fake")(*ts)
    names = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    assert all(any(f"nvalchemi.{op}" in n for n in names) for op in ("layer_norm_fwd", "layer_norm_bwd", "gated_ff_fwd", "gated_ff_bwd", "newton_schulz"))
    assert all(torch.equal(a, b) for a, b in zip(graph(*ts), step(*ts)))
