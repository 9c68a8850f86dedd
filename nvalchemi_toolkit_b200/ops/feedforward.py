# SPDX-License-Identifier: Apache-2.0
"""Gated feed-forward block ``y = (act(x @ w_gate) * (x @ w_up)) @ w_down``, forward and backward.

Weights are ``[in, out]`` like those of :func:`~nvalchemi_toolkit_b200.ops.gemm.matmul`; a transposed view
(``linear.weight.t()``) is read in place as well.  ``gated_feed_forward`` is differentiable;
``gated_feed_forward_backward`` is the backward pass on its own, for hand-written steps and for capture into CUDA graphs (it
involves no autograd graph).  CUDA tensors run ``csrc/feedforward.cu`` on the tensor cores: bfloat16 and float16 with 32-bit
sums (``h`` and its gradients are rounded to the type once, as the operands of the next product; in float16 a value of ``h``
past 65504 becomes infinite, from 9 rows on), float32 to 32-bit accuracy by exact splits into three bfloat16 parts.  Sums of any
length keep their accuracy.  Infinities and NaN give non-finite results (float32: an infinity may come out as NaN).  CPU tensors run the same formulas in PyTorch, float64 among them.

Forces are gradients, so training on them differentiates the backward pass once more: the second derivative is the formula of
the backward pass differentiated by PyTorch, in 32 bits.
"""
from __future__ import annotations

import torch

from nvalchemi_toolkit_b200.ops import _native
from nvalchemi_toolkit_b200.ops._native_counter import ops as _nops

ACTIVATIONS = {"silu": 0, "gelu": 1}  # gelu: g * Phi(g), by the error function
_CUDA_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_feed_forward: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or any(w.dim() != 2 for w in (w_gate, w_up, w_down)):
        raise ValueError("gated_feed_forward: x must have an axis of features and the weights must be matrices")
    k, h = w_gate.shape
    if x.shape[-1] != k or tuple(w_up.shape) != (k, h) or w_down.shape[0] != h:
        raise ValueError(f"gated_feed_forward: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and "
                         f"w_down {tuple(w_down.shape)} do not fit: x [..., K], w_gate and w_up [K, H], w_down [H, N]")
    if min(k, h, w_down.shape[1]) < 1:
        raise ValueError("gated_feed_forward: every feature axis needs at least one element")
    for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if w.device != x.device:
            raise ValueError(f"gated_feed_forward: {name} is on {w.device}, x on {x.device}")
        if w.dtype != x.dtype:
            raise TypeError(f"gated_feed_forward: {name} of type {w.dtype} with x of type {x.dtype}")
    if not x.dtype.is_floating_point or (x.is_cuda and x.dtype not in _CUDA_TYPES):
        raise TypeError(f"gated_feed_forward: {x.dtype} is not supported on {x.device.type}"
                        + (" (float32, bfloat16, float16)" if x.is_cuda else ""))


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


class _Product(torch.autograd.Function):
    """``a @ b`` in the type of its arguments inside an autocast region too, and so are its derivatives."""

    generate_vmap_rule = True

    @staticmethod
    def forward(a, b):
        with torch.autocast(a.device.type, enabled=False):
            return a @ b

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.save_for_backward(*inputs)
        ctx.save_for_forward(*inputs)

    @staticmethod
    def backward(ctx, grad):
        a, b = ctx.saved_tensors
        need = ctx.needs_input_grad
        return _Product.apply(grad, b.mT) if need[0] else None, _Product.apply(a.mT, grad) if need[1] else None

    @staticmethod
    def jvp(ctx, da, db):
        a, b = ctx.saved_tensors
        terms = [_Product.apply(*t) for t in ((da, b), (a, db)) if t[0] is not None and t[1] is not None]
        return sum(terms[1:], terms[0])


def _in_autocast(t: torch.Tensor) -> bool:
    kind = t.device.type
    return (t.is_cuda or torch.amp.is_autocast_available(kind)) and torch.is_autocast_enabled(kind)


def _product(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    return _Product.apply(a, b) if _in_autocast(a) else a @ b


def _activate(g: torch.Tensor, activation: str) -> tuple[torch.Tensor, torch.Tensor]:
    """``act(g)`` and ``act'(g)``, both differentiable."""
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.erfc(-0.7071067811865476 * g)
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * 0.3989422804014327


def _forward_formula(x, w_gate, w_up, w_down, activation):
    xf = _wide(x)
    h = _activate(_product(xf, _wide(w_gate)), activation)[0] * _product(xf, _wide(w_up))
    return _product(h, _wide(w_down)).to(x.dtype)


def _backward_formula(dy, x, w_gate, w_up, w_down, activation, want=(True,) * 4):
    """``(dx, dw_gate, dw_up, dw_down)`` in differentiable operations, at least 32 bits wide; matrices only.  ``None`` where
    ``want`` says so."""
    dy, x, wg, wu, wd = (_wide(t) for t in (dy, x, w_gate, w_up, w_down))
    u = _product(x, wu)
    a, da = _activate(_product(x, wg), activation)
    dh = _product(dy, wd.t())
    dg, du = dh * u * da, dh * a
    return (_product(dg, wg.t()) + _product(du, wu.t()) if want[0] else None, _product(x.t(), dg) if want[1] else None,
            _product(x.t(), du) if want[2] else None, _product((a * u).t(), dy) if want[3] else None)


def gated_feed_forward_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                                activation: str = "silu", *, input_grad: bool = True, weight_grads: bool = True
                                ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """``(dx, dw_gate, dw_up, dw_down)`` for the gradient ``dy`` of ``y``; nothing of the forward pass is needed.
    ``input_grad=False`` / ``weight_grads=False`` leave the first / the other three out (``None``)."""
    with torch.no_grad():
        if x.is_cuda:
            try:
                dx, *dw = _nops.gated_ff_bwd(dy, x, w_gate, w_up, w_down, ACTIVATIONS.get(activation, -1),
                                             (1 if input_grad else 0) | (6 if weight_grads else 0))
            except RuntimeError:  # the operator refuses what the checks refuse; they say it in Python's exceptions
                _check_backward(dy, x, w_gate, w_up, w_down, activation)
                raise
        else:
            _check_backward(dy, x, w_gate, w_up, w_down, activation)
            dx, *dw = (t.to(x.dtype) for t in _backward_formula(dy.reshape(-1, w_down.shape[1]), x.reshape(-1, x.shape[-1]), w_gate, w_up,
                                                                w_down, activation))
            dx = dx.reshape(x.shape)
        return (dx if input_grad else None, *(dw if weight_grads else (None,) * 3))


def _check_backward(dy, x, w_gate, w_up, w_down, activation) -> None:
    _check(x, w_gate, w_up, w_down, activation)
    if dy.shape != (*x.shape[:-1], w_down.shape[1]) or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError(f"gated_feed_forward_backward: dy ({tuple(dy.shape)}, {dy.dtype}, {dy.device}) does not match y "
                         f"({(*x.shape[:-1], w_down.shape[1])}, {x.dtype}, {x.device})")


def _forward_kernel(x, w_gate, w_up, w_down, activation):
    try:
        return _nops.gated_ff_fwd(x, w_gate, w_up, w_down, ACTIVATIONS.get(activation, -1))
    except RuntimeError:
        _check(x, w_gate, w_up, w_down, activation)
        raise


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        ctx.save_for_backward(x, w_gate, w_up, w_down)
        ctx.activation = activation
        return _forward_kernel(x, w_gate, w_up, w_down, activation)

    @staticmethod
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        grads = _GatedFeedForwardGrad.apply(dy, *ctx.saved_tensors, ctx.activation, need[0], any(need[1:4]))
        return (*(g if n else None for g, n in zip(grads, need)), None)


class _GatedFeedForwardGrad(torch.autograd.Function):
    """The backward pass as a function of ``(dy, x, w_gate, w_up, w_down)``; its derivative differentiates the formula."""

    @staticmethod
    def forward(ctx, dy, x, w_gate, w_up, w_down, activation, input_grad, weight_grads):
        ctx.save_for_backward(dy, x, w_gate, w_up, w_down)
        ctx.set_materialize_grads(False)  # None, not zeros, for the gradients that were not used
        ctx.activation = activation
        return gated_feed_forward_backward(dy, x, w_gate, w_up, w_down, activation, input_grad=input_grad, weight_grads=weight_grads)

    @staticmethod
    def backward(ctx, *dd):
        saved, need = ctx.saved_tensors, ctx.needs_input_grad[:5]
        again = torch.is_grad_enabled()  # a third derivative is wanted: keep the graph of this one
        with torch.enable_grad():
            args = [t if again else t.detach().requires_grad_(n) for t, n in zip(saved, need)]
            dy, x = args[:2]
            dx, *dw = _backward_formula(dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1]), *args[2:], ctx.activation,
                                        [d is not None for d in dd])
            outs = (None if dx is None else dx.reshape(x.shape), *dw)
            pairs = [(o, d) for o, d in zip(outs, dd) if d is not None and o.requires_grad]
            wanted = [t for t, n in zip(args, need) if n]
            got = torch.autograd.grad([o for o, _ in pairs], wanted, [d.to(o.dtype) for o, d in pairs], create_graph=again,
                                      allow_unused=True) if pairs and wanted else [None] * len(wanted)
        it = iter(got)
        return (*(next(it) if n else None for n in need), None, None, None)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "silu"
                       ) -> torch.Tensor:
    """``(act(x @ w_gate) * (x @ w_up)) @ w_down`` for ``x [..., K]``, ``w_gate`` and ``w_up`` ``[K, H]``, ``w_down [H, N]``;
    ``activation`` is ``"silu"`` or ``"gelu"``.  Differentiable (twice and more).  Under ``torch.autocast`` the arguments are
    cast to its type first, as those of a matrix product are: floating types but float64."""
    if _in_autocast(x):
        dt = torch.get_autocast_dtype(x.device.type)
        x, w_gate, w_up, w_down = (t.to(dt) if t.is_floating_point() and t.dtype != torch.float64 else t for t in (x, w_gate, w_up, w_down))
    if not x.is_cuda:
        _check(x, w_gate, w_up, w_down, activation)
        return _forward_formula(x, w_gate, w_up, w_down, activation)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        return _GatedFeedForward.apply(x, w_gate, w_up, w_down, activation)
    return _forward_kernel(x, w_gate, w_up, w_down, activation)


def check_errors(like: torch.Tensor) -> int:
    """Status word of the kernels on ``like``'s device (0 = fine; non-zero = a bounded wait expired and NaN stands where nothing was
    formed).  Covers work launched on the current stream, or on streams it has waited for; waits for it and clears the word."""
    if like.is_cuda and _native.available():
        return int(_nops.gated_ff_error_status(like))
    return 0
