# SPDX-License-Identifier: Apache-2.0
"""Layer norm over the last axis, forward and backward.

``layer_norm(x, weight, bias, eps)`` is differentiable; ``layer_norm_forward`` / ``layer_norm_backward`` are the two passes
on their own, for hand-written steps and for capture into CUDA graphs (they involve no autograd graph).  CUDA tensors run
``csrc/layer_norm.cu``: float32, bfloat16 and float16 rows with weights of the same type or float32, float64 rows with
float64 weights, statistics and sums in 32 bits (64 for float64), rows of up to 8192 elements at any row stride.  CPU tensors
run the same formulas in PyTorch.

Forces are gradients, so training on them differentiates the backward pass once more: the second derivative is the formula
of the backward pass differentiated by PyTorch, in at least 32 bits.
"""
from __future__ import annotations

import torch

from nvalchemi_toolkit_b200.ops._native_counter import ops as _nops

MAX_COLS = 8192
_ROW_TYPES = (torch.float32, torch.float64, torch.bfloat16, torch.float16)


def _check(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None) -> None:
    if x.dtype not in _ROW_TYPES:
        raise TypeError(f"layer_norm: x must be float32, float64, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > MAX_COLS:
        raise ValueError(f"layer_norm: the last axis of x must have 1..{MAX_COLS} elements, got shape {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"layer_norm: {name} has shape {tuple(t.shape)}, expected {tuple(x.shape[-1:])}")
        if t.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {t.device}, x on {x.device}")
        if t.dtype != x.dtype and (t.dtype != torch.float32 or x.dtype == torch.float64):
            raise TypeError(f"layer_norm: {name} of type {t.dtype} with x of type {x.dtype}; use the type of x"
                            + ("" if x.dtype == torch.float64 else " or float32"))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight ({weight.dtype}) and bias ({bias.dtype}) must have one type")


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def _forward_formula(x, weight, bias, eps):
    xf = _wide(x)
    mean = xf.mean(-1, keepdim=True)
    d = xf - mean
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)
    y = d * rstd
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y.to(x.dtype), mean.reshape(-1), rstd.reshape(-1)


def _backward_formula(grad, x, weight, eps, want=(True,) * 3):
    """``(dx, dweight, dbias)`` from ``grad`` and ``x`` in differentiable operations, in at least 32 bits.  ``None`` where ``want``
    says so."""
    xf, g = _wide(x), _wide(grad)
    d = xf - xf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)
    xh = d * rstd
    dx, n = None, x.shape[-1]
    if want[0]:
        gw = g if weight is None else g * _wide(weight)
        dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return dx, (g * xh).reshape(-1, n).sum(0) if want[1] else None, g.reshape(-1, n).sum(0) if want[2] else None


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                       eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)``: the normalised rows and the statistics the backward pass takes, one value per row (float32;
    float64 rows: float64).  Not recorded by autograd."""
    with torch.no_grad():
        if x.is_cuda:
            try:
                return _nops.layer_norm_fwd(x, weight, bias, eps)
            except RuntimeError:  # the operator refuses what _check refuses; _check says it in Python's exceptions
                _check(x, weight, bias)
                raise
        _check(x, weight, bias)
        return _forward_formula(x, weight, bias, eps)


def layer_norm_backward(grad: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None = None, *, param_grads: bool = True, param_dtype: torch.dtype | None = None
                        ) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """``(dx, dweight, dbias)`` for the gradient ``grad`` of ``y``.  The parameters' gradients have the type of ``weight``
    (without a weight: ``param_dtype``, by default that of ``x``); ``param_grads=False`` leaves them out (``None``).  Their
    sums over the rows are added in a fixed order: the same inputs give the same bits."""
    ptype = weight.dtype if weight is not None else (param_dtype or x.dtype)
    with torch.no_grad():
        if x.is_cuda:
            try:
                dx, dw, db = _nops.layer_norm_bwd(grad, x, mean, rstd, weight, param_grads, ptype)
            except RuntimeError:
                _check_backward(grad, x, mean, rstd, weight, param_dtype)
                raise
            return (dx, dw, db) if param_grads else (dx, None, None)
        _check_backward(grad, x, mean, rstd, weight, param_dtype)
        n = x.shape[-1]
        xf, g = _wide(x).reshape(-1, n), _wide(grad).reshape(-1, n)
        xh = (xf - mean[:, None]) * rstd[:, None]
        gw = g if weight is None else g * _wide(weight)
        dx = rstd[:, None] * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
        dx = dx.to(x.dtype).reshape(x.shape)
        return (dx, (g * xh).sum(0).to(ptype), g.sum(0).to(ptype)) if param_grads else (dx, None, None)


def _check_backward(grad, x, mean, rstd, weight, param_dtype) -> None:
    _check(x, weight, None)
    if grad.shape != x.shape or grad.dtype != x.dtype or grad.device != x.device:
        raise ValueError(f"layer_norm_backward: grad ({tuple(grad.shape)}, {grad.dtype}, {grad.device}) does not match x "
                         f"({tuple(x.shape)}, {x.dtype}, {x.device})")
    n_rows, stat_type = x.numel() // x.shape[-1], torch.float64 if x.dtype == torch.float64 else torch.float32
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.shape != (n_rows,) or t.dtype != stat_type or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"layer_norm_backward: {name} must be what layer_norm_forward returned for x")
    if param_dtype is not None and param_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"layer_norm_backward: param_dtype {param_dtype} with x of type {x.dtype}")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.eps = eps
        return y

    @staticmethod
    def backward(ctx, grad):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = _LayerNormGrad.apply(grad, x, weight, bias, mean, rstd, ctx.eps,
                                          ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return dx if ctx.needs_input_grad[0] else None, dw if ctx.needs_input_grad[1] else None, \
            db if ctx.needs_input_grad[2] else None, None


class _LayerNormGrad(torch.autograd.Function):
    """The backward pass as a function of ``(grad, x, weight)``; its own derivative differentiates the formula."""

    @staticmethod
    def forward(ctx, grad, x, weight, bias, mean, rstd, eps, param_grads):
        ctx.save_for_backward(grad, x, weight)
        ctx.set_materialize_grads(False)  # None, not zeros, for the gradients that were not used
        ctx.eps, ctx.param_grads = eps, param_grads
        ptype = None if weight is not None or bias is None else bias.dtype
        dx, dw, db = layer_norm_backward(grad, x, mean, rstd, weight, param_grads=param_grads, param_dtype=ptype)
        return dx, dw if weight is not None else None, db if bias is not None else None

    @staticmethod
    def backward(ctx, ddx, ddw, ddb):
        saved = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        again = torch.is_grad_enabled()  # a third derivative is wanted: keep the graph of this one
        with torch.enable_grad():
            args = [t if t is None or again else t.detach().requires_grad_(n) for t, n in zip(saved, need)]
            outs = _backward_formula(*args, ctx.eps, tuple(d is not None for d in (ddx, ddw, ddb)))
            pairs = [(o, d) for o, d in zip(outs, (ddx, ddw, ddb)) if d is not None and o.requires_grad]
            wanted = [t for t, n in zip(args, need) if n]
            got = torch.autograd.grad([o for o, _ in pairs], wanted, [d.to(o.dtype) for o, d in pairs], create_graph=again,
                                      allow_unused=True) if pairs and wanted else [None] * len(wanted)
        it = iter(got)
        return (*(next(it) if n else None for n in need), None, None, None, None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5
               ) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, in the type of ``x``; differentiable (twice and
    more in ``x``, ``weight`` and ``grad``).  ``weight`` and ``bias`` may be absent and may be float32 beside 16-bit rows."""
    if not x.is_cuda:
        _check(x, weight, bias)
        return _forward_formula(x, weight, bias, eps)[0]
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    try:
        return _nops.layer_norm_apply(x, weight, bias, eps)
    except RuntimeError:
        _check(x, weight, bias)
        raise
