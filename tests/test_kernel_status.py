# SPDX-License-Identifier: Apache-2.0
"""What a training run does when a kernel reports an expired wait: the status words are replaced by stand-ins here."""
import pytest
import torch

from nvalchemi_toolkit_b200.models import DemoModelWrapper
from nvalchemi_toolkit_b200.ops import feedforward, orthogonalize, status
from nvalchemi_toolkit_b200.training import EnergyMSELoss, Muon, OptimizerConfig, TrainingStrategy, ValidationConfig
from tests.test_gated_training import _batches


def _strategy(device, **kw):
    torch.manual_seed(0)
    return TrainingStrategy(DemoModelWrapper(hidden_dim=16, gated_hidden=8), OptimizerConfig(cls=Muon, kwargs={"lr": 1e-3}),
                            EnergyMSELoss(), num_epochs=1, devices=[device], **kw)


def test_nothing_to_report(device):
    like = torch.zeros(3, device=device)
    assert status.kernel_errors(like) == {}
    status.raise_on_kernel_errors(like)


@pytest.mark.parametrize("module,name", [(feedforward, "feedforward"), (orthogonalize, "orthogonalize")])
def test_an_expired_wait_ends_the_run(monkeypatch, device, tmp_path, module, name):
    strategy = _strategy(device)
    word = [0]
    monkeypatch.setattr(module, "check_errors", lambda like: word[0] if like.device.type == torch.device(device).type else 99)
    strategy.train_batch(_batches(device)[0])
    strategy.save_checkpoint(tmp_path / "good")
    assert (tmp_path / "good").exists()
    word[0] = 15
    with pytest.raises(RuntimeError, match=f"bounded wait ran out.*{name}.: 15"):
        strategy.save_checkpoint(tmp_path / "bad")
    assert not (tmp_path / "bad").exists()
    with pytest.raises(RuntimeError, match="bounded wait ran out"):
        strategy.run(_batches(device))


def test_validation_results_are_not_kept(monkeypatch, device):
    strategy = _strategy(device, validation_config=ValidationConfig(data=_batches(device)))
    strategy.train_batch(_batches(device)[0])
    monkeypatch.setattr(feedforward, "check_errors", lambda like: 13)
    with pytest.raises(RuntimeError, match="feedforward.: 13"):
        strategy.validate()
    assert strategy.last_validation is None
