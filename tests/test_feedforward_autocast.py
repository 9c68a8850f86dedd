# SPDX-License-Identifier: Apache-2.0
"""The gated feed-forward block inside ``torch.autocast`` regions."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import feedforward as ff
from tests.test_feedforward import _inputs

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


def test_what_autocast_casts():
    ts = _inputs(6, 16, 24, 8, F64, "cpu")[:4]
    want = ff.gated_feed_forward(*ts)
    with torch.autocast("cpu", dtype=BF16):
        y = ff.gated_feed_forward(*ts)
        assert (ts[0] @ ts[1]).dtype == F64 and y.dtype == F64 and torch.equal(y, want)   # float64 stays, as in a product
        with pytest.raises(TypeError, match="not supported"):
            ff.gated_feed_forward(*(t.long() for t in ts))
        with pytest.raises(TypeError, match="w_gate of type"):
            ff.gated_feed_forward(ts[0], *(t.float() for t in ts[1:]))
        assert ff.gated_feed_forward(*(t.float() for t in ts)).dtype == BF16


@pytest.mark.gpu
def test_float64_is_refused_inside_autocast_too():
    ts = _inputs(6, 16, 24, 8, F64, "cuda")[:4]
    with torch.autocast("cuda", dtype=BF16), pytest.raises(TypeError, match="float64 is not supported"):
        ff.gated_feed_forward(*ts)
