# SPDX-License-Identifier: Apache-2.0
"""Layer norm, gated feed-forward block and orthogonalised updates together: modules, the Muon optimiser, a training run."""
import copy

import pytest
import torch

from nvalchemi_toolkit_b200 import Batch
from nvalchemi_toolkit_b200.models import DemoModel, DemoModelWrapper, GatedBlock, GatedFeedForward, LayerNorm
from nvalchemi_toolkit_b200.ops.orthogonalize import newton_schulz
from nvalchemi_toolkit_b200.training import EnergyMSELoss, ForceMSELoss, Muon, OptimizerConfig, TrainingStrategy
from nvalchemi_toolkit_b200.training.optimizers import ParamGroupSpec
from tests.helpers import random_molecule


def _batches(device, n=6):
    data = []
    for i in range(n):
        d = random_molecule(5 + i % 3, i)
        g = torch.Generator().manual_seed(100 + i)
        d.__dict__["energy"] = torch.randn(1, 1, generator=g)
        d.__dict__["forces"] = torch.randn(d.positions.shape, generator=g)
        data.append(d)
    return [Batch.from_data_list(data[i:i + 3], device=device) for i in range(0, n, 3)]


def _model(device, seed=0):
    torch.manual_seed(seed)
    return DemoModelWrapper(hidden_dim=32, gated_hidden=48).to(device)


def test_modules(device):
    torch.manual_seed(0)
    norm, ref = LayerNorm(24).to(device), torch.nn.LayerNorm(24).to(device)
    ref.load_state_dict(norm.state_dict())
    x = torch.randn(7, 24, device=device)
    assert float((norm(x) - ref(x)).detach().abs().max()) < 64 * 2.0 ** -24 * 4
    assert [n for n, _ in LayerNorm(3, bias=False).named_parameters()] == ["weight"]
    ffn = GatedFeedForward(24, 40, 8, activation="gelu").to(device)
    want = (torch.nn.functional.gelu(x.double() @ ffn.w_gate.double()) * (x.double() @ ffn.w_up.double())) @ ffn.w_down.double()
    assert ffn(x).shape == (7, 8) and float(((ffn(x) - want).norm() / want.norm()).detach()) < 64 * 2.0 ** -24
    block = GatedBlock(24, 40).to(device)
    assert torch.equal(block(x), x + block.feed_forward(block.norm(x)))
    with pytest.raises(ValueError, match="activation"):
        GatedFeedForward(4, 4, activation="relu")


def test_demo_model_without_the_block_is_unchanged():
    torch.manual_seed(3)
    a = DemoModel(16)
    torch.manual_seed(3)
    b = DemoModel(16, gated_hidden=8)
    assert not any("gated" in k for k in a.state_dict())
    assert all(torch.equal(v, b.state_dict()[k]) for k, v in a.state_dict().items())
    assert DemoModelWrapper(hidden_dim=16).checkpoint_spec()["config"] == {"hidden_dim": 16}
    assert DemoModelWrapper(hidden_dim=16, gated_hidden=8).checkpoint_spec()["config"] == {"hidden_dim": 16, "gated_hidden": 8}


def test_muon_step_is_its_formula(device):
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, device=device)) for s in ((6, 10), (3, 6, 10), (10, 6), (7,), (1, 5))]
    before = [p.detach().clone() for p in ps]
    opt = Muon(ps, lr=0.1, momentum=0.5, weight_decay=0.2)
    bufs = [torch.zeros_like(p) for p in ps]
    for step in range(2):
        grads = [torch.randn(p.shape, generator=torch.Generator().manual_seed(step)).to(device) for p in ps]
        for p, g in zip(ps, grads):
            p.grad = g.clone()
        opt.step()
        for i in range(3):
            bufs[i] = 0.5 * bufs[i] + grads[i]
            o = newton_schulz(grads[i] + 0.5 * bufs[i]).float()
            before[i] = before[i] * (1 - 0.1 * 0.2) - 0.1 * 0.2 * 10 ** 0.5 * o
            assert float((ps[i] - before[i]).abs().max()) < 16 * 2.0 ** -24 * 4
    ref = torch.optim.AdamW([torch.nn.Parameter(b) for b in before[3:]], lr=0.1, weight_decay=0.2)
    for step in range(2):
        grads = [torch.randn(p.shape, generator=torch.Generator().manual_seed(step)).to(device) for p in ps]
        for p, g in zip(ref.param_groups[0]["params"], grads[3:]):
            p.grad = g
        ref.step()
    for p, q in zip(ps[3:], ref.param_groups[0]["params"]):
        assert float((p - q).abs().max()) < 64 * 2.0 ** -24 * 4
    state = copy.deepcopy(opt.state_dict())
    other = Muon([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=0.1, momentum=0.5, weight_decay=0.2)
    other.load_state_dict(state)
    for p, q in zip(ps, other.param_groups[0]["params"]):
        p.grad = torch.ones_like(p)
        q.grad = torch.ones_like(q)
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, other.param_groups[0]["params"]))


def test_muon_refusals_and_groups():
    p = torch.nn.Parameter(torch.randn(4, 4))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)), dict(ns_steps=0), dict(adam_eps=0.0)):
        with pytest.raises(ValueError, match="Muon"):
            Muon([p], **kw)
    cfg = OptimizerConfig(cls="nvalchemi_toolkit_b200.training.optimizers.Muon", kwargs={"lr": 1e-2},
                          param_groups=[ParamGroupSpec(pattern="embedding", options={"orthogonalize": False})])
    model = _model("cpu")
    opt, _ = cfg.build([(f"main.{n}", q) for n, q in model.named_parameters()])
    table = model.model.embedding.weight
    assert any(table is q for q in opt.param_groups[1]["params"]) and opt.param_groups[1]["orthogonalize"] is False
    assert OptimizerConfig(cls=Muon, kwargs={"lr": 1e-2}).to_spec()["cls"].endswith("Muon")
    with pytest.raises(ValueError, match="does not accept"):
        OptimizerConfig(cls=Muon, kwargs={"learning_rate": 1e-2})


def test_training_run_with_all_of_them(device):
    """Energy + force loss (second derivatives through norm and block) with Muon steps: runs, stays finite, and the first step
    moves the block's matrices by the size of an orthogonal update."""
    loss = EnergyMSELoss() + ForceMSELoss()
    model = _model(device)
    cfg = OptimizerConfig(cls=Muon, kwargs={"lr": 1e-2})
    batches = _batches(device)
    strategy = TrainingStrategy(model, cfg, loss, num_epochs=2, devices=[device])
    start = {n: p.detach().clone() for n, p in model.named_parameters()}
    strategy.train_batch(batches[0])
    first = {n: p.detach().clone() for n, p in model.named_parameters()}
    strategy.run(batches)
    assert strategy.step_count == 4 and all(torch.isfinite(p).all() for p in model.parameters())

    moved = {n: float((first[n] - start[n]).norm()) for n in start}
    for n, p in model.named_parameters():
        if n.endswith(("w_gate", "w_up", "w_down")):
            # between one and all singular values of the update are near 1 (0.68 .. 1.14, the largest surely): the last layer's
            # gradient has rank one, its readout being linear
            unit = 1e-2 * 0.2 * max(p.shape) ** 0.5
            assert 0.5 * unit < moved[n] < 1.3 * unit * min(p.shape) ** 0.5, (n, moved[n], unit)


@pytest.mark.gpu
def test_gpu_gradients_of_the_model_equal_the_cpus():
    """Gradients of an energy + force loss through the gated model: float32 kernels against float64 on the CPU."""
    def grads(model, dev, dt):
        data = _batches(dev)[0]
        model = copy.deepcopy(model).to(dev, dt)
        pos = data.positions.to(dt).requires_grad_()
        energy, _ = model.model(data.atomic_numbers, pos, data.batch_idx, 3)
        (f,) = torch.autograd.grad(energy.sum(), pos, create_graph=True)
        total = (energy - data.energy.to(dt)).square().sum() + (f + data.forces.to(dt)).square().sum()
        ps = dict(model.named_parameters())
        return dict(zip(ps, torch.autograd.grad(total, list(ps.values()), allow_unused=True)))
    model = _model("cpu")
    want, got = grads(model, "cpu", torch.float64), grads(model, "cuda", torch.float32)
    for n, e in want.items():
        if e is None or float(e.norm()) == 0:
            continue
        # about a hundred dependent float32 operations, sums of up to 64 terms with magnitudes sqrt(64) above the results
        assert float((got[n].double().cpu() - e).norm() / e.norm()) < 2e4 * 2.0 ** -24, n
