# SPDX-License-Identifier: Apache-2.0
"""Status words of the tensor-core kernels.

Every wait inside those kernels is bounded.  When one runs out, the kernel records a code in a status word and returns; the
gated feed-forward block and the Newton-Schulz iteration leave NaN in the results that were not formed.  The words are read where
a program waits for the GPU anyway: ``TrainingStrategy`` does so before it writes a checkpoint (not an asynchronous one), after a
validation run and at the end of a run."""
from __future__ import annotations

import torch

from nvalchemi_toolkit_b200.ops import feedforward, gemm, orthogonalize

_KERNELS = {"gemm": gemm, "feedforward": feedforward, "orthogonalize": orthogonalize}


def kernel_errors(like: torch.Tensor) -> dict[str, int]:
    """Codes of the bounded waits that ran out since the words were last read, by family of kernels; empty when all is well.
    Waits for the current stream of ``like``'s device and covers what was launched on it, or on streams it has waited for.  The
    words are cleared."""
    codes = {name: module.check_errors(like) for name, module in _KERNELS.items()}
    return {name: code for name, code in codes.items() if code}


def raise_on_kernel_errors(like: torch.Tensor) -> None:
    """``RuntimeError`` when :func:`kernel_errors` finds any."""
    codes = kernel_errors(like)
    if codes:
        raise RuntimeError(f"a bounded wait ran out in kernels on {like.device}: {codes}; results since the last check are not valid")
