# SPDX-License-Identifier: Apache-2.0
"""State of the Muon optimiser: when it is made, its types, and what a saved copy of it brings back."""
import torch

from nvalchemi_toolkit_b200.training import Muon


def test_momentum_buffers_are_made_once(monkeypatch, device):
    p = torch.nn.Parameter(torch.randn(6, 10, device=device))
    opt = Muon([p], lr=0.1)
    made = []
    zeros_like = torch.zeros_like
    monkeypatch.setattr(torch, "zeros_like", lambda *a, **k: made.append(a) or zeros_like(*a, **k))
    for _ in range(3):
        p.grad = torch.ones_like(p)
        opt.step()
    assert len(made) == 1
