# SPDX-License-Identifier: Apache-2.0
"""The gated feed-forward block against its formula in float64: values, gradients, layouts, refusals, graphs.

Tolerances.  Element by element, with ``|.|`` matrices of magnitudes: a product of n terms
is off by ``e = (n / 16 + 8) * 2^-23`` of the product of magnitudes (the tensor core adds 16 products at a time and may cut the
sum; the split of float32 values leaves out less than 2^-24); what that does to g, u and dh goes through the derivatives of the
activation (first at most 1.13, second at most 0.8) into h, dg and du; 16-bit tensors add half a step (``eps / 2``) of h, dg and
du, and of the stored result; below the smallest normal value ``tiny`` of a type its step stays ``eps * tiny``, so half a step is
``eps / 2 * max(|v|, tiny)`` (float16 gradients get there).  Where every sum has 64 terms or more, rounding errors also average out: the norm of the error
stays under ``eps / 2`` of the norm of the result (two uniform errors: sqrt(2 / 3) * eps / 2 at most)."""
import pytest
import torch

from nvalchemi_toolkit_b200.ops import feedforward as ff

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16


def _inputs(m, k, h, n, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed + m + 3 * k + 5 * h)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ts = (r(m, k), r(k, h) / k ** 0.5, r(k, h) / k ** 0.5, r(h, n) / h ** 0.5, r(m, n))
    return [t.to(dtype).to(device) for t in ts]


def _exact(x, wg, wu, wd, dy, act):
    ts = [t.double().detach().requires_grad_() for t in (x, wg, wu, wd)]
    gate = ts[0] @ ts[1]
    gate = torch.nn.functional.silu(gate) if act == "silu" else torch.nn.functional.gelu(gate)
    y = (gate * (ts[0] @ ts[2])) @ ts[3]
    return [y.detach(), *torch.autograd.grad(y, ts, dy.double())]


def _half_step(v, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * v.abs().clamp(min=f.tiny)


def _bounds(x, wg, wu, wd, dy, act, dtype):
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    n = max(*x.shape, *wd.shape)
    e = (n / 16 + 8) * 2.0 ** -23 if dtype != F64 else 64 * n * 2.0 ** -53
    half = (lambda v: _half_step(v, dtype)) if dtype in (BF16, F16) else (lambda v: e * v)
    g = (x @ wg).requires_grad_()
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    (da,) = torch.autograd.grad(a.sum(), g)
    g, a, da, u, dh = g.detach(), a.detach(), da.abs(), (x @ wu).abs(), (dy @ wd.t()).abs()
    a = a.abs()
    eg, eu, ed = e * (x.abs() @ wg.abs()), e * (x.abs() @ wu.abs()), e * (dy.abs() @ wd.abs().t())
    h, dg, du = a * u, dh * u * da, dh * a
    eh = 1.13 * eg * u + (a + 1.13 * eg) * eu + half(h)
    edg = ed * u * da + (dh + ed) * eu * da + 0.8 * (dh + ed) * (u + eu) * eg + half(dg)
    edu = ed * a + 1.13 * (dh + ed) * eg + half(du)
    y = dy.abs()
    return [eh @ wd.abs() + e * (h @ wd.abs()), edg @ wg.abs().t() + edu @ wu.abs().t() + e * (dg @ wg.abs().t() + du @ wu.abs().t()),
            x.abs().t() @ edg + e * (x.abs().t() @ dg), x.abs().t() @ edu + e * (x.abs().t() @ du), eh.t() @ y + e * (h.t() @ y)]


def _near(got, want, bound, dtype, least):
    assert got.dtype == dtype and got.shape == want.shape
    d, bound = got.double() - want, 1.01 * (_half_step(want, dtype) + bound)
    worst = float((d.abs() / bound).max())
    assert worst <= 1, worst
    if least >= 64 and dtype in (BF16, F16):
        assert float(d.norm() / want.norm()) <= torch.finfo(dtype).eps / 2


def _run(m, k, h, n, dtype, device, act="silu", layout=None):
    x, wg, wu, wd, dy = _inputs(m, k, h, n, dtype, device)
    want, bounds = _exact(x, wg, wu, wd, dy, act), _bounds(x, wg, wu, wd, dy, act, dtype)
    if layout == "linear":  # weights of linear layers, passed as transposed views
        wg, wu, wd = (w.t().contiguous().t() for w in (wg, wu, wd))
    elif layout == "mixed":
        wu = wu.t().contiguous().t()
        x, dy = x.t().contiguous().t(), torch.cat([dy, dy], 1)[:, :n]
    elif layout == "sliced":  # rows of wider tensors, and every second column
        x, wg = torch.cat([x, x], 1)[:, :k], wg.repeat_interleave(2, dim=1)[:, ::2]
        wd = torch.cat([wd, wd], 1)[:, n:]
    got = [ff.gated_feed_forward(x, wg, wu, wd, act), *ff.gated_feed_forward_backward(dy, x, wg, wu, wd, act)]
    for p, q, b in zip(got, want, bounds):
        _near(p, q, b, dtype, min(m, k, h, n))
    assert ff.check_errors(x) == 0
    return got


SHAPES = [(1, 1, 1, 1), (1, 64, 128, 64), (3, 5, 7, 2), (21, 64, 128, 64), (128, 64, 64, 64), (129, 72, 136, 40), (130, 65, 257, 129),
          (300, 128, 512, 128), (1000, 200, 777, 200), (2, 1024, 512, 1024), (4097, 40, 24, 8), (17, 1000, 96, 33),
          (5, 120, 72, 56), (8, 513, 130, 96), (8, 2048, 512, 264), (1, 1024, 4096, 1024)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,h,n", SHAPES[:7])
def test_formulas_on_cpu(m, k, h, n, act):
    for dtype in (F32, F64):
        _run(m, k, h, n, dtype, "cpu", act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,h,n", SHAPES)
def test_kernels_against_float64(m, k, h, n, dtype):
    _run(m, k, h, n, dtype, "cuda", "gelu" if m % 2 else "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k,h,n", [(20011, 128, 512, 128), (5000, 512, 1500, 512), (2048, 1024, 4096, 1024)])
def test_large_products(m, k, h, n, dtype):
    _run(m, k, h, n, dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["linear", "mixed", "sliced"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k,h,n", [(200, 96, 160, 96), (3, 96, 160, 96), (77, 50, 90, 34), (20, 1, 33, 1), (200, 1, 40, 7), (30, 16, 1, 16)])
def test_layouts(m, k, h, n, dtype, layout):
    _run(m, k, h, n, dtype, "cuda", layout=layout)


def test_one_row_without_a_batch_axis_and_more_axes(device):
    x, wg, wu, wd, dy = _inputs(6, 16, 24, 8, F32, device)
    y = ff.gated_feed_forward(x, wg, wu, wd)
    dx, *_ = ff.gated_feed_forward_backward(dy, x, wg, wu, wd)
    one = ff.gated_feed_forward(x[2], wg, wu, wd)
    assert one.shape == (8,) and float((one - y[2]).abs().max()) < 64 * 2.0 ** -23 * float(y.abs().max())
    deep = ff.gated_feed_forward(x.view(3, 1, 2, 16), wg, wu, wd)
    assert deep.shape == (3, 1, 2, 8) and torch.equal(deep.view(6, 8), y)
    again, *_ = ff.gated_feed_forward_backward(dy.view(3, 2, 8), x.view(3, 2, 16), wg, wu, wd)
    assert again.shape == (3, 2, 16) and torch.equal(again.view(6, 16), dx)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls on two streams share nothing: each gives what it gives alone."""
    a, b = _inputs(700, 96, 160, 96, BF16, "cuda"), _inputs(500, 64, 256, 64, F32, "cuda")
    want = [[ff.gated_feed_forward(*t[:4]), *ff.gated_feed_forward_backward(t[4], *t[:4])] for t in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = [ff.gated_feed_forward(*t[:4]), *ff.gated_feed_forward_backward(t[4], *t[:4])]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for x, y in zip(want, got) for p, q in zip(x, y))
    assert ff.check_errors(a[0]) == 0


@pytest.mark.gpu
def test_same_bits_again_and_rows_do_not_mix():
    a = _run(500, 128, 384, 128, BF16, "cuda")
    assert all(torch.equal(p, q) for p, q in zip(a, _run(500, 128, 384, 128, BF16, "cuda")))
    x, wg, wu, wd, _ = _inputs(300, 64, 96, 64, BF16, "cuda")
    x[17], x[200, 3] = float("nan"), float("inf")
    y = ff.gated_feed_forward(x, wg, wu, wd)
    bad = ~torch.isfinite(y).all(1)
    assert bad.nonzero().flatten().tolist() == [17, 200]


@pytest.mark.gpu
def test_float32_range():
    """Values near both ends of the float32 range survive the split into three parts."""
    x, wg, wu, wd, _ = _inputs(130, 64, 64, 64, F32, "cuda")
    y = ff.gated_feed_forward(x, wg, wu, wd)
    h = torch.nn.functional.silu(x.double() @ wg.double()) * (x.double() @ wu.double())
    for s in (2.0 ** 100, 2.0 ** -60):
        # scaling by a power of two changes nothing but the parts of wd / s below 2^-126, the smallest normal bfloat16: of each
        # element at most 2^-126 is lost, times h * s <= |h| * 2^100, summed over h: 2^-26 * sum |h|
        d = (ff.gated_feed_forward(x, wg, wu * s, wd / s).double() - y.double()).abs()
        assert bool((d <= 2.0 ** -26 * h.abs().sum(1, keepdim=True)).all())
    one = torch.eye(64, device="cuda")
    big = torch.full((1, 64), torch.finfo(F32).max, device="cuda")
    ok = ff.gated_feed_forward(torch.ones(1, 64, device="cuda"), one, one * big, one * 2.0 ** -3)
    want = torch.sigmoid(torch.ones(1, device="cuda", dtype=F64)) * torch.finfo(F32).max / 8
    assert float(((ok.double() - want) / want).abs().max()) < 16 * 2.0 ** -23


def test_gradients_against_differences_and_second_derivatives():
    ts = [t.requires_grad_() for t in _inputs(4, 3, 5, 2, F64, "cpu")[:4]]
    for act in ("silu", "gelu"):
        assert torch.autograd.gradcheck(lambda *a: ff.gated_feed_forward(*a, act), ts)
        assert torch.autograd.gradgradcheck(lambda *a: ff.gated_feed_forward(*a, act), ts)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_autograd_and_force_training_on_gpu(act):
    """First and second derivatives through autograd (energy -> force -> gradient of a force loss), float32 against float64."""
    def grads(dt, dev):
        x, wg, wu, wd, _ = _inputs(33, 24, 40, 16, F64, dev)
        x, wg, wu, wd = (t.to(dt).requires_grad_() for t in (x, wg, wu, wd))
        e = torch.tanh(ff.gated_feed_forward(x, wg, wu, wd, act)).pow(2).sum()
        first = torch.autograd.grad(e, [x, wg, wu, wd], create_graph=True)
        return [*first, *torch.autograd.grad(first[0].pow(2).sum(), [x, wg, wu, wd])]
    for a, e in zip(grads(F32, "cuda"), grads(F64, "cpu")):
        # sums of at most 40 terms, two levels of about ten 32-bit operations each, magnitudes sqrt(40) above the results
        assert float((a.double().cpu() - e).norm().detach() / e.norm().detach()) < 500 * 2.0 ** -23
    x, wg, wu, wd, _ = _inputs(8, 16, 16, 16, F32, "cuda")
    wg.requires_grad_()
    ff.gated_feed_forward(x.expand(2, 8, 16), wg, wu, wd, act).sum().backward()   # dy expanded from one number, x broadcast
    both = wg.grad.clone()
    wg.grad = None
    ff.gated_feed_forward(x, wg, wu, wd, act).sum().backward()
    assert float((both - 2 * wg.grad).abs().max()) <= 64 * 2.0 ** -23 * float(both.abs().max())


@pytest.mark.gpu
def test_autocast_and_captured_passes():
    x, wg, wu, wd, dy = _inputs(200, 64, 128, 64, F32, "cuda")
    with torch.autocast("cuda", dtype=BF16):
        y = ff.gated_feed_forward(x, wg, wu, wd)
    assert y.dtype == BF16 and torch.equal(y, ff.gated_feed_forward(*(t.bfloat16() for t in (x, wg, wu, wd))))
    out = {}

    def step():
        out["v"] = [ff.gated_feed_forward(x, wg, wu, wd), *ff.gated_feed_forward_backward(dy, x, wg, wu, wd)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    captured = out["v"]
    for seed in (1, 2):
        for t, new in zip((x, wg, wu, wd, dy), _inputs(200, 64, 128, 64, F32, "cuda", seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        step()
        assert all(torch.equal(p, q) for p, q in zip(captured, out["v"]))


def test_empty_batch(device):
    x, wg, wu, wd, dy = _inputs(0, 8, 16, 4, F32, device)
    assert ff.gated_feed_forward(x, wg, wu, wd).shape == (0, 4)
    dx, *dw = ff.gated_feed_forward_backward(dy, x, wg, wu, wd)
    assert dx.shape == (0, 8) and all(not t.any() for t in dw) and [tuple(t.shape) for t in dw] == [(8, 16), (8, 16), (16, 4)]


def test_refusals(device):
    x, wg, wu, wd, dy = _inputs(4, 8, 16, 4, F32, device)
    with pytest.raises(ValueError, match="activation"):
        ff.gated_feed_forward(x, wg, wu, wd, "relu")
    with pytest.raises(ValueError, match="do not fit"):
        ff.gated_feed_forward(x, wg, wu[:, :8], wd)
    with pytest.raises(ValueError, match="do not fit"):
        ff.gated_feed_forward(x[:, :7], wg, wu, wd)
    with pytest.raises(ValueError, match="matrices"):
        ff.gated_feed_forward(x, wg[None], wu, wd)
    with pytest.raises(ValueError, match="at least one"):
        ff.gated_feed_forward(x[:, :0], wg[:0], wu[:0], wd)
    with pytest.raises(TypeError, match="w_up of type"):
        ff.gated_feed_forward(x, wg, wu.double(), wd)
    with pytest.raises(TypeError, match="not supported"):
        ff.gated_feed_forward(*(t.long() for t in (x, wg, wu, wd)))
    with pytest.raises(ValueError, match="does not match y"):
        ff.gated_feed_forward_backward(dy[:2], x, wg, wu, wd)
    if device == "cuda":
        with pytest.raises(TypeError, match="float64 is not supported"):
            ff.gated_feed_forward(*(t.double() for t in (x, wg, wu, wd)))
        with pytest.raises(ValueError, match="w_down is on"):
            ff.gated_feed_forward(x, wg, wu, wd.cpu())
