# SPDX-License-Identifier: Apache-2.0
"""Orthogonalising matrices by Newton-Schulz products, the update rule of the Muon optimiser.

``newton_schulz(g)`` maps ``G = U S V^T`` to ``U p(S / |G|_F) V^T``, where the odd polynomial ``p`` (``steps`` times
``s -> a s + b s^3 + c s^5``) takes every singular value that is not tiny to about 1.  Leading axes are a batch.  CUDA tensors
run ``csrc/orthogonalize.cu`` on the tensor cores (float16 operands scaled by powers of two, fp32 sums, the iterate as a float16
value and a float16 remainder, 22 bits); CPU tensors run the formula in float32.  The result is a direction, not a sum: it is returned in bfloat16.
"""
from __future__ import annotations

import functools
import math

import torch

from nvalchemi_toolkit_b200.ops import _native
from nvalchemi_toolkit_b200.ops._native_counter import ops as _nops

COEFFICIENTS = (3.4445, -4.775, 2.0315)
#: Bound of the iterate's singular values for which the float16 operands (X and A times 2^12, B times 2^11) cannot overflow.
_MAX_VALUE = 2.5
_MAX_BATCH = 65535  # matrices of one launch


def _check(g: torch.Tensor, steps: int, coefficients: tuple[float, float, float], eps: float) -> None:
    if g.dim() < 2:
        raise ValueError(f"newton_schulz: a matrix or a batch of matrices is needed, got shape {tuple(g.shape)}")
    if g.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"newton_schulz: float32, bfloat16 or float16 is needed, got {g.dtype}")
    if int(steps) != steps or not 1 <= steps <= 100:
        raise ValueError(f"newton_schulz: steps must be a whole number in 1..100, got {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"newton_schulz: three finite coefficients are needed, got {coefficients}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"newton_schulz: eps must be finite and not negative, got {eps}")
    if not _bounded(int(steps), *(float(v) for v in coefficients)):
        raise ValueError(f"newton_schulz: with coefficients {coefficients} singular values grow beyond {_MAX_VALUE}")


@functools.lru_cache(maxsize=64)
def _bounded(steps: int, a: float, b: float, c: float) -> bool:
    """Whether singular values from [0, 1] stay below ``_MAX_VALUE`` in every step, and the entries of ``B`` below 30."""
    top = 1.0
    for _ in range(steps):
        grid = [top * i / 256 for i in range(257)]
        top = max(abs(a * s + b * s ** 3 + c * s ** 5) for s in grid)
        if top > _MAX_VALUE or max(abs(b * s * s + c * s ** 4) for s in grid) > 30:
            return False
    return True


def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients: tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7
                  ) -> torch.Tensor:
    """``X = G / (|G|_F + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` (transposed for matrices
    with more rows than columns), for every matrix of ``g [..., m, n]`` (float32, bfloat16 or float16); bfloat16 result.

    A zero matrix stays zero; a matrix with an infinity or NaN comes back as NaN.  Not recorded by autograd."""
    _check(g, steps, coefficients, eps)
    a, b, c = (float(v) for v in coefficients)
    with torch.no_grad():
        if not g.is_cuda:
            return _formula(g.detach().float(), int(steps), a, b, c, float(eps)).to(torch.bfloat16)
        _native.require(g)
        batch = g.reshape(math.prod(g.shape[:-2]), *g.shape[-2:]).contiguous()
        parts = batch.split(_MAX_BATCH) if batch.shape[0] > _MAX_BATCH else (batch,)
        outs = [_nops.newton_schulz(p, int(steps), a, b, c, float(eps)) for p in parts]
        return (outs[0] if len(outs) == 1 else torch.cat(outs)).view(g.shape)


def _formula(x: torch.Tensor, steps: int, a: float, b: float, c: float, eps: float) -> torch.Tensor:
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt() + eps
    x = (x / torch.where(norm == 0, 1.0, norm)).float()  # a zero matrix stays zero without eps too
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(-2, -1) if tall else x).contiguous()


def check_errors(like: torch.Tensor) -> int:
    """Status word of the kernels on ``like``'s device (0 = fine; non-zero = a bounded wait expired and NaN stands where nothing was
    formed).  Covers work launched on the current stream, or on streams it has waited for; waits for it and clears the word."""
    if like.is_cuda and _native.available():
        return int(_nops.newton_schulz_error_status(like))
    return 0
