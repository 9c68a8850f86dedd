# SPDX-License-Identifier: Apache-2.0
"""Demo models saved as whole objects before they could have a gated block."""
import torch

from nvalchemi_toolkit_b200.models import DemoModelWrapper
from tests.test_gated_training import _batches


def test_a_model_without_the_attribute_still_runs():
    torch.manual_seed(0)
    model, data = DemoModelWrapper(hidden_dim=16), _batches("cpu")[0]
    want = model(data)
    del model.model.gated_block, model.model.gated_hidden     # as an older object comes out of torch.load
    got = model(data)
    # every call scales embeddings of norm 1 back to norm 1, which may move their last bits: a chain of a hundred operations
    assert all(float((got[k] - want[k]).abs().max()) <= 100 * 2.0 ** -24 * float(want[k].abs().max()) for k in ("energy", "forces"))
    assert model.checkpoint_spec()["config"] == {"hidden_dim": 16}
