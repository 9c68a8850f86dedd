# SPDX-License-Identifier: Apache-2.0
"""Workloads of the dense training operators: layer norm, the gated feed-forward block, Newton-Schulz orthogonalisation.

``listed()`` names fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes the inputs of a case on the GPU,
``run`` makes one pass through the operator (the framework's kernels where ``own`` is true, elementary torch operations
otherwise), ``work`` counts what a pass cannot do without, ``exact`` evaluates the definition in float64.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_NS = (3.4445, -4.775, 2.0315)  # coefficients of the quintic iteration
_STEPS = 5
_NS_EPS = 1e-7
_LN_EPS = 1e-5


def listed():
    return [
        # layer norm of the embeddings of a few small molecules (21 atoms, width 64 as in the demo model): latency
        {"name": "norm_small_f32", "op": "norm", "train": False, "rows": 21, "cols": 64, "dtype": "f32", "wdtype": "f32", "step": 1},
        # one training step's norm over 131,072 atoms (the share of one GPU in an 8-GPU run) with 128 channels
        {"name": "norm_train_atoms_bf16", "op": "norm", "train": True, "rows": 131072, "cols": 128, "dtype": "bf16", "wdtype": "f32",
         "step": 1},
        # the scalar channels of features laid out [atoms, 4, C]: rows four widths apart; an odd width
        {"name": "norm_train_odd_f32", "op": "norm", "train": True, "rows": 20011, "cols": 333, "dtype": "f32", "wdtype": "f32", "step": 4},
        # a wide hidden state (the joint width of a large readout)
        {"name": "norm_train_wide_f16", "op": "norm", "train": True, "rows": 16384, "cols": 4096, "dtype": "f16", "wdtype": "f16",
         "step": 1},
        # one atom (a single token) through a wide block: bound by the weights' bytes
        {"name": "ff_single_bf16", "op": "ff", "train": False, "rows": 1, "width": 1024, "hidden": 4096, "act": "silu", "dtype": "bf16"},
        # per-atom block of a 128-channel model over 131,072 atoms, inference
        {"name": "ff_atoms_bf16", "op": "ff", "train": False, "rows": 131072, "width": 128, "hidden": 512, "act": "silu", "dtype": "bf16"},
        # training step of a wide block over a batch of 8192 atoms
        {"name": "ff_train_wide_bf16", "op": "ff", "train": True, "rows": 8192, "width": 1024, "hidden": 4096, "act": "silu",
         "dtype": "bf16"},
        # ragged sizes: an odd batch, widths that fill no tile
        {"name": "ff_train_odd_f16", "op": "ff", "train": True, "rows": 3001, "width": 200, "hidden": 777, "act": "gelu", "dtype": "f16"},
        # float32 training, the default type of the framework's models
        {"name": "ff_train_f32", "op": "ff", "train": True, "rows": 4096, "width": 256, "hidden": 1024, "act": "silu", "dtype": "f32"},
        # the stacked channel mixes of a 128-channel model: many small matrices, latency
        {"name": "ortho_channel_mixes_f32", "op": "ortho", "batch": 24, "m": 128, "n": 128, "dtype": "f32"},
        # projections of a wide block, several layers stacked
        {"name": "ortho_projections_bf16", "op": "ortho", "batch": 4, "m": 1024, "n": 4096, "dtype": "bf16"},
        # one odd matrix, taller than wide
        {"name": "ortho_tall_odd_f32", "op": "ortho", "batch": 1, "m": 1537, "n": 515, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "ff", "ff", "ff", "ortho", "ortho"])
    if op == "norm":
        cols = _log(rng, 16, 4096)
        if rng.random() < 0.5:
            cols = -(-cols // 8) * 8
        rows = min(_log(rng, 1, 200000), (1 << 26) // cols)
        dtype = rng.choice(["f32", "bf16", "f16"])
        return {"op": op, "train": rng.random() < 0.7, "rows": rows, "cols": cols, "dtype": dtype,
                "wdtype": rng.choice(["f32", dtype]), "step": rng.choice([1, 1, 4])}
    if op == "ff":
        width, hidden = _log(rng, 32, 1024), _log(rng, 64, 4096)
        if rng.random() < 0.6:
            width, hidden = -(-width // 8) * 8, -(-hidden // 8) * 8
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        cap = (1 << 35) // (4 if dtype == "f32" else 1) // (width * hidden)
        rows = _log(rng, 1, 131072)
        return {"op": op, "train": rng.random() < 0.6, "rows": max(1, min(rows, cap)), "width": width, "hidden": hidden,
                "act": rng.choice(["silu", "gelu"]), "dtype": dtype}
    m, n = _log(rng, 16, 2048), _log(rng, 16, 2048)
    cap = int(1e11 / (6.0 * min(m, n) ** 2 * max(m, n)))
    return {"op": op, "batch": max(1, min(_log(rng, 1, 32), cap)), "m": m, "n": n, "dtype": rng.choice(["f32", "bf16", "f16"])}


def _flops_ortho(c):
    m, n = min(c["m"], c["n"]), max(c["m"], c["n"])
    return c["batch"] * _STEPS * (1.0 * m * m * n + 1.0 * m ** 3 + 2.0 * m * m * n)  # the Gram matrix and its square are symmetric


def work(case):
    c = case
    if c["op"] == "ortho":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["batch"] * c["m"] * c["n"] * (size + 2), "flops": _flops_ortho(c)}
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        wsize = 4 if c["wdtype"] == "f32" else 2
        elems = c["rows"] * c["cols"]
        if not c["train"]:
            return {"bytes": 2 * elems * size + 2 * c["cols"] * wsize, "flops": 8 * elems}
        return {"bytes": 4 * elems * size + 4 * c["cols"] * wsize, "flops": 20 * elems}
    m, k, h = c["rows"], c["width"], c["hidden"]
    if not c["train"]:
        return {"bytes": size * (2 * m * k + 3 * k * h), "flops": 6.0 * m * k * h}
    return {"bytes": size * (4 * m * k + 6 * k * h), "flops": 18.0 * m * k * h}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = _DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["op"] == "norm":
        r, n = c["rows"], c["cols"]
        x = (randn(r, 1) + (0.5 + torch.rand(r, 1, generator=g, device="cuda")) * randn(r, c["step"] * n)).to(dt)[:, :n]
        wdt = _DTYPES[c["wdtype"]]
        s = {"x": x, "w": (1 + 0.2 * randn(n)).to(wdt), "b": (0.2 * randn(n)).to(wdt)}
        if c["train"]:
            s["dy"] = randn(r, n).to(dt)
    elif c["op"] == "ff":
        m, k, h = c["rows"], c["width"], c["hidden"]
        s = {"x": randn(m, k).to(dt), "wg": (randn(k, h) / k ** 0.5).to(dt), "wu": (randn(k, h) / k ** 0.5).to(dt),
             "wd": (randn(h, k) / h ** 0.5).to(dt)}
        if c["train"]:
            s["dy"] = randn(m, k).to(dt)
    else:  # an averaged gradient: activations times errors of a decaying spectrum, over a floor of noise
        b, m, n = c["batch"], c["m"], c["n"]
        r = max(1, min(m, n) // 2)
        decay = torch.logspace(0, -1.5, r, device="cuda")
        low = (randn(b, m, r) * decay) @ randn(b, r, n) / r ** 0.5
        s = {"g": (1e-3 * (low + 0.1 * randn(b, m, n))).to(dt)}
    s["case"] = dict(c)
    return s


def run(state):
    c = state["case"]
    if c["op"] == "norm":
        return _norm(state, c["train"])
    if c["op"] == "ff":
        return _ff(state, c["act"], c["train"])
    return _ortho(state)


def _norm(s, train):
    x, w, b = s["x"], s["w"], s["b"]
    if own:
        from nvalchemi_toolkit_b200.ops import norm

        if not train:
            return norm.layer_norm(x, w, b, eps=_LN_EPS)
        y, mean, rstd = norm.layer_norm_forward(x, w, b, eps=_LN_EPS)
        return (y, *norm.layer_norm_backward(s["dy"], x, mean, rstd, w))
    xf, wf = x.float(), w.float()
    mean = xf.mean(-1, keepdim=True)
    d = xf - mean
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + _LN_EPS)
    xh = d * rstd
    y = (xh * wf + b.float()).to(x.dtype)
    if not train:
        return y
    g = s["dy"].float()
    gw = g * wf
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), (g * xh).sum(0).to(w.dtype), g.sum(0).to(b.dtype)


def _ff(s, act, train):
    x, wg, wu, wd = s["x"], s["wg"], s["wu"], s["wd"]
    if own:
        from nvalchemi_toolkit_b200.ops import feedforward

        y = feedforward.gated_feed_forward(x, wg, wu, wd, activation=act)
        if not train:
            return y
        return (y, *feedforward.gated_feed_forward_backward(s["dy"], x, wg, wu, wd, activation=act))
    xf, wgf, wuf, wdf = x.float(), wg.float(), wu.float(), wd.float()
    g, u = xf @ wgf, xf @ wuf
    if act == "silu":
        sg = torch.sigmoid(g)
        a, da = g * sg, sg * (1 + g * (1 - sg))
    else:
        cdf = 0.5 * (1 + torch.erf(g * 0.7071067811865476))
        a, da = g * cdf, cdf + g * torch.exp(-0.5 * g * g) * 0.3989422804014327
    h = a * u
    y = (h @ wdf).to(x.dtype)
    if not train:
        return y
    dy = s["dy"].float()
    dh = dy @ wdf.t()
    dg, du = dh * u * da, dh * a
    dx = dg @ wgf.t() + du @ wuf.t()
    return (y, dx.to(x.dtype), (xf.t() @ dg).to(x.dtype), (xf.t() @ du).to(x.dtype), (h.t() @ dy).to(x.dtype))


def _ortho(s):
    g = s["g"]
    if own:
        from nvalchemi_toolkit_b200.ops import orthogonalize

        return orthogonalize.newton_schulz(g, steps=_STEPS, coefficients=_NS, eps=_NS_EPS)
    a, b, c = _NS
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + _NS_EPS)
    x = _ns_step(_ns_step(_ns_step(_ns_step(_ns_step(x, a, b, c), a, b, c), a, b, c), a, b, c), a, b, c)
    return (x.transpose(-2, -1) if tall else x).to(torch.bfloat16).contiguous()


def _ns_step(x, a, b, c):
    gram = x @ x.transpose(-2, -1)
    return a * x + (b * gram + c * (gram @ gram)) @ x


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "ortho":
        g = s["g"].double()
        x = g / (torch.linalg.matrix_norm(g).reshape(-1, 1, 1) + _NS_EPS)
        a, b, cc = _NS
        if c["m"] > c["n"]:  # the Gram matrix of the shorter side, multiplied from that side
            eye = torch.eye(c["n"], dtype=x.dtype, device=x.device)
            for _ in range(_STEPS):
                gram = torch.einsum("bki,bkj->bij", x, x)
                x = torch.bmm(x, a * eye + b * gram + cc * torch.bmm(gram, gram))
        else:
            eye = torch.eye(c["m"], dtype=x.dtype, device=x.device)
            for _ in range(_STEPS):
                gram = torch.einsum("bik,bjk->bij", x, x)
                x = torch.bmm(a * eye + b * gram + cc * torch.bmm(gram, gram), x)
        return x
    with torch.enable_grad():
        leaves = [s[k].double().requires_grad_(c["train"]) for k in (("x", "w", "b") if c["op"] == "norm" else ("x", "wg", "wu", "wd"))]
        if c["op"] == "norm":
            x, w, b = leaves
            var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
            y = (x - mean) / (var + _LN_EPS) ** 0.5 * w + b
        else:
            x, wg, wu, wd = leaves
            gate = x.matmul(wg)
            gate = gate / (1 + torch.exp(-gate)) if c["act"] == "silu" else gate * torch.special.ndtr(gate)
            y = (gate * x.matmul(wu)).matmul(wd)
        if not c["train"]:
            return y.detach()
        grads = torch.autograd.grad(y, leaves, s["dy"].double())
    return (y.detach(), *grads)
