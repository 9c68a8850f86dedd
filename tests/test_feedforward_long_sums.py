# SPDX-License-Identifier: Apache-2.0
"""Long contraction axes of the gated feed-forward block: sums of terms of one sign, where an accumulator that is cut towards
zero shows, against float64.

Bounds, none of which grows with the length of the axis.  16-bit products: the mean error stays under an eighth of half a step of
the result (rounding the operands and the result averages to nothing over the elements: four standard errors).  float32: a sum
of at most 32 instructions loses about 27 half steps of a float32 value (2^-24) where all terms have one sign; three such sums
in a chain (u, act(g), the product that follows) make 81, the other roundings fit between that and 96."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import feedforward as ff
from tests.test_feedforward import _exact, _run

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
pytestmark = pytest.mark.gpu


def _positive(m, k, h, n, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(m + k)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").abs_()  # noqa: E731
    return [t.to(dtype) for t in (r(m, k), r(k, h) / k, r(k, h) / k, r(h, n) / h, r(m, n) * scale)]


@pytest.mark.parametrize("dtype,rows", [(F16, 262144), (BF16, 1048576)])
def test_weight_gradients_of_many_rows_16_bit(dtype, rows):
    x, wg, wu, wd, dy = _positive(rows, 32, 1024, 2560, dtype, 2.0 ** -8)
    dwd = ff.gated_feed_forward_backward(dy, x, wg, wu, wd)[3]
    want = torch.zeros(1024, 2560, dtype=torch.float64, device="cuda")
    for i in range(0, rows, 65536):
        p, d = x[i:i + 65536].double(), dy[i:i + 65536].double()
        want += (torch.nn.functional.silu(p @ wg.double()) * (p @ wu.double())).t() @ d
    half = torch.finfo(dtype).eps / 2
    mean = float(((dwd.double() - want) / want).mean())
    assert abs(mean) <= half * (1 / 8 + 4 / want.numel() ** 0.5), mean / half


def test_weight_gradients_of_many_rows_float32():
    x, wg, wu, wd, dy = _positive(1 << 20, 64, 64, 64, F32)
    got = ff.gated_feed_forward_backward(dy, x, wg, wu, wd)[1:]
    for g, e in zip(got, _exact(x, wg, wu, wd, dy, "silu")[2:]):
        assert float((g.double() - e).norm() / e.norm()) <= 48 * 2.0 ** -24  # 27, and g and u of 64 terms


@pytest.mark.parametrize("width", [1024, 2048, 8192])
def test_wide_projections_float32(width):
    x, wg, wu, wd, dy = _positive(200, width, 64, 64, F32)
    got = [ff.gated_feed_forward(x, wg, wu, wd), *ff.gated_feed_forward_backward(dy, x, wg, wu, wd)]
    for g, e in zip(got, _exact(x, wg, wu, wd, dy, "silu")):
        assert float((g.double() - e).norm() / e.norm()) <= 96 * 2.0 ** -24


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,h,n,dtype,layout", [
    (130, 2500, 257, 129, F32, None), (1000, 2000, 257, 129, F32, None), (130, 1025, 130, 70, F32, "mixed"), (20, 2049, 40, 24, F32, "linear"), (300, 2100, 33, 2100, F32, "sliced"),
    (200, 9000, 72, 40, F16, None), (300, 40, 72, 9000, F16, "mixed"), (300, 8200, 65, 8200, F16, "linear"),
    (130, 70000, 64, 16, BF16, None), (20, 16, 64, 70000, BF16, None)])
def test_axes_past_the_accumulators(m, k, h, n, dtype, layout, act):
    """Against float64, element by element; only the bounds of `tests/test_feedforward.py`, which count the length, apply here."""
    _run(m, k, h, n, dtype, "cuda", act, layout)


def test_partial_sums_take_bounded_memory():
    """float16 over 262,144 rows splits into 32 parts of 134 MB; beyond h, dg, du (2.1 GB each) and the gradients no more than
    1.5 GB is held."""
    x, wg, wu, wd, dy = _positive(262144, 32, 4096, 8192, F16, 2.0 ** -8)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = ff.gated_feed_forward_backward(dy, x, wg, wu, wd)
    torch.cuda.synchronize()
    held = torch.cuda.max_memory_allocated() - before - 3 * 262144 * 4096 * 2 - sum(g.numel() * g.element_size() for g in grads)
    assert held <= 1.5 * 2 ** 30, held / 2 ** 30
    rows = torch.arange(0, 4096, 512, device="cuda")
    h = torch.nn.functional.silu(x.double() @ wg[:, rows].double()) * (x.double() @ wu[:, rows].double())
    want = torch.cat([h.t() @ dy[:, i:i + 1024].double() for i in range(0, 8192, 1024)], 1)
    mean = float(((grads[3][rows].double() - want) / want).mean())
    assert abs(mean) <= 2.0 ** -11 * (1 / 8 + 4 / want.numel() ** 0.5)
