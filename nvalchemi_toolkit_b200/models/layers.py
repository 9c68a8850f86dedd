# SPDX-License-Identifier: Apache-2.0
"""Dense building blocks of per-atom networks, as modules over the package's operators (``ops.norm``, ``ops.feedforward``).

All of them are differentiable as often as needed (forces are gradients, force losses differentiate those), run the
hand-written kernels on CUDA and the same formulas in PyTorch on a CPU."""
from __future__ import annotations

import torch
from torch import nn

from nvalchemi_toolkit_b200.ops.feedforward import ACTIVATIONS, gated_feed_forward
from nvalchemi_toolkit_b200.ops.norm import layer_norm


class LayerNorm(nn.Module):
    """Layer norm over the last axis; parameters are named and shaped like those of ``torch.nn.LayerNorm(width)``."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True) -> None:
        super().__init__()
        self.width, self.eps = int(width), float(eps)
        self.weight = nn.Parameter(torch.ones(self.width))
        self.bias = nn.Parameter(torch.zeros(self.width)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.width}, eps={self.eps}, bias={self.bias is not None}"


class GatedFeedForward(nn.Module):
    """``(act(x @ w_gate) * (x @ w_up)) @ w_down``; weights are ``[in, out]`` and start as ``N(0, 1 / in)``."""

    def __init__(self, width: int, hidden: int, out: int | None = None, activation: str = "silu") -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        self.activation = activation
        self.w_gate = nn.Parameter(torch.randn(width, hidden) / width ** 0.5)
        self.w_up = nn.Parameter(torch.randn(width, hidden) / width ** 0.5)
        self.w_down = nn.Parameter(torch.randn(hidden, width if out is None else out) / hidden ** 0.5)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_feed_forward(x, self.w_gate, self.w_up, self.w_down, self.activation)

    def extra_repr(self) -> str:
        return f"{self.w_gate.shape[0]}, hidden={self.w_gate.shape[1]}, out={self.w_down.shape[1]}, activation={self.activation!r}"


class GatedBlock(nn.Module):
    """Pre-norm residual block ``x + feed_forward(norm(x))``."""

    def __init__(self, width: int, hidden: int, activation: str = "silu") -> None:
        super().__init__()
        self.norm = LayerNorm(width)
        self.feed_forward = GatedFeedForward(width, hidden, activation=activation)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.feed_forward(self.norm(x))
