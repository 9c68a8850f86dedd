# SPDX-License-Identifier: Apache-2.0
"""State of the Muon optimiser: when it is made, its types, and what a saved copy of it brings back."""
import copy

import pytest
import torch

from nvalchemi_toolkit_b200.ops.orthogonalize import newton_schulz
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


def _grad(shape, step, device, size):
    return (size * torch.randn(shape, generator=torch.Generator().manual_seed(step))).to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1.0, 1e-3])
def test_adam_steps_of_16_bit_parameters(dtype, size, device):
    """Every step is AdamW's float32 step from the same parameter, rounded once to its type: off by half a step of the type
    and a few float32 roundings (64 of the largest term).  float16: the squares of gradients of 1e-3 are below its smallest
    value."""
    p = torch.nn.Parameter(_grad((40,), 100, device, 1.0).to(dtype))
    opt = Muon([p], lr=0.05, weight_decay=0.1)
    q = torch.nn.Parameter(p.detach().float())
    ref = torch.optim.AdamW([q], lr=0.05, weight_decay=0.1)
    for step in range(20):
        g = _grad(p.shape, step, device, size).to(dtype)
        if step % 3 == 0:
            g[:5] = 0
        p.grad, q.grad = g, g.float()
        with torch.no_grad():
            q.copy_(p)
        opt.step()
        ref.step()
        bound = torch.finfo(dtype).eps / 2 * q.detach().abs() + 64 * 2.0 ** -24
        assert ((p.detach().float() - q.detach()).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_second_moments_of_16_bit_parameters_decay(dtype):
    """One large gradient, then small ones: the running mean of squares follows its formula (each step two float32 roundings)."""
    p = torch.nn.Parameter(torch.ones(3, dtype=dtype))
    opt = Muon([p], lr=0.0)
    n, want = 400, 0.0
    for step in range(n):
        p.grad = torch.full_like(p, 1.0 if step == 0 else 2.0 ** -10)
        opt.step()
        want = 0.999 * want + 0.001 * float(p.grad[0]) ** 2
    got = opt.state[p]["exp_avg_sq"].double()
    assert float((got / want - 1).abs().max()) <= 2 * n * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_matrix_steps_of_16_bit_parameters(dtype, device):
    """The momentum is a float32 sum (two roundings a step), the parameter is rounded once a step.  The last bit of the argument may
    move an entry of the bfloat16 direction by one step of it."""
    p = torch.nn.Parameter(_grad((2, 6, 10), 100, device, 1.0).to(dtype))
    opt = Muon([p], lr=0.1, momentum=0.9, weight_decay=0.2)
    buf = torch.zeros(p.shape, dtype=torch.float64, device=device)
    for step in range(8):
        g = _grad(p.shape, step, device, 1.0 if step == 0 else 2.0 ** -9).to(dtype)
        before = p.detach().double()
        p.grad = g
        opt.step()
        buf = 0.9 * buf + g.double()
        assert float((opt.state[p]["momentum_buffer"].double() - buf).abs().max()) <= 16 * 2.0 ** -24 * float(buf.abs().max())
        kept = opt.state[p]["momentum_buffer"]
        o = 0.1 * 0.2 * 10 ** 0.5 * newton_schulz(torch.add(g.float(), kept, alpha=0.9)).double()
        want = before * (1 - 0.1 * 0.2) - o
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 16 * 2.0 ** -24 * 4 + 2.0 ** -7 * o.abs()
        assert ((p.detach().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_state_survives_a_saved_copy(dtype, device):
    torch.manual_seed(0)
    make = lambda: [torch.nn.Parameter(t.to(device, dtype)) for t in (torch.randn(5), torch.randn(4, 6), torch.randn(2))]  # noqa: E731
    opt = Muon(make()[:2], lr=0.1)
    opt.add_param_group({"params": [make()[2]], "lr": 0.01})
    ps = [p for g in opt.param_groups for p in g["params"]]
    for step in range(3):
        for i, p in enumerate(ps):
            p.grad = _grad(p.shape, 10 * step + i, device, 1e-2).to(dtype)
        opt.step()
    other = Muon([torch.nn.Parameter(p.detach().clone()) for p in ps[:2]], lr=0.1)
    other.add_param_group({"params": [torch.nn.Parameter(ps[2].detach().clone())], "lr": 0.01})
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    qs = [q for g in other.param_groups for q in g["params"]]
    for p, q in zip(ps, qs):
        assert opt.state[p].keys() == other.state[q].keys()
        for k, v in opt.state[p].items():
            w = other.state[q][k]
            assert type(v) is type(w)
            if isinstance(v, torch.Tensor):
                assert v.dtype == w.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
                assert torch.equal(v, w)
        p.grad = torch.full_like(p, 1e-3)
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize("bad", [dict(ns_steps=101), dict(ns_steps=2.5), dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1),
                                 dict(betas=(0.9, 1.0)), dict(adam_eps=0.0)])
def test_refused_before_the_first_step(bad):
    """What the step could not carry out is refused when the optimiser, or one of its groups, is made."""
    p, q = (torch.nn.Parameter(torch.randn(4, 4)) for _ in range(2))
    with pytest.raises(ValueError, match="Muon"):
        Muon([p], **bad)
    with pytest.raises(ValueError, match="Muon"):
        Muon([{"params": [p]}, {"params": [q], **bad}])
    opt = Muon([p])
    with pytest.raises(ValueError, match="Muon"):
        opt.add_param_group({"params": [q], **bad})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [q], "lr": 0.0, "ns_steps": 100, "orthogonalize": False})
