# SPDX-License-Identifier: Apache-2.0
"""Declarative optimiser / scheduler configuration (reference ``nvalchemi/training/optimizers.py:111-447``)."""
from __future__ import annotations

import inspect
import re
from typing import Any, Callable, Mapping

import torch
from pydantic import BaseModel, ConfigDict, Field, model_validator

from nvalchemi_toolkit_b200._serialization import import_from_path, type_to_path


def check_kwargs(cls: Any, kwargs: Mapping[str, Any], label: str) -> None:
    """Reject keyword arguments the constructor does not accept at configuration time (reference
    ``training/optimizers.py:56-82``): a typo such as ``weight_decy`` should fail when the recipe is read, not after the data
    pipeline and the model are built.  Constructors that take ``**kwargs`` accept everything."""
    try:
        params = inspect.signature(cls.__init__ if isinstance(cls, type) else cls).parameters
    except (TypeError, ValueError):
        return
    if any(p.kind is inspect.Parameter.VAR_KEYWORD for p in params.values()):
        return
    unknown = sorted(k for k in kwargs if k not in params)
    if unknown:
        accepted = sorted(k for k in params if k not in ("self", "params", "optimizer"))
        raise ValueError(f"{label} {getattr(cls, '__name__', cls)} does not accept {unknown}; accepted: {accepted}")


def _state_type(p: torch.Tensor) -> torch.dtype:
    """Type of a parameter's optimiser state: 16 bits are too few for running means (a mean of squares stops decaying in bfloat16
    and vanishes in float16)."""
    return torch.float32 if p.dtype in (torch.bfloat16, torch.float16) else p.dtype


class Muon(torch.optim.Optimizer):
    """Momentum whose matrix updates are orthogonalised by Newton-Schulz products (``ops.orthogonalize.newton_schulz``).

    For a parameter with two axes or more (its last two are the matrix, the others a batch: MACE's stacked ``[l, C, C]`` channel
    mixes are ``l`` matrices)::

        buf <- momentum * buf + grad;   u = grad + momentum * buf  (nesterov)  or  buf
        p   <- p * (1 - lr * weight_decay) - lr * 0.2 * sqrt(max(m, n)) * newton_schulz(u)

    The factor gives an update of the root mean square size of an AdamW step, so ``lr`` and ``weight_decay`` are AdamW's.
    Parameters with fewer axes, matrices with a side of one, and groups with ``orthogonalize=False`` (embedding tables, for
    instance, by a ``ParamGroupSpec``) take AdamW steps with ``betas`` and ``adam_eps``.  Matrices of one shape are
    orthogonalised together, one call for all of them.  The state of 16-bit parameters is float32, their steps are formed in float32
    and rounded once."""

    def __init__(self, params: Any, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 ns_steps: int = 5, betas: tuple[float, float] = (0.9, 0.999), adam_eps: float = 1e-8, orthogonalize: bool = True) -> None:
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, ns_steps=ns_steps,
                                      betas=tuple(betas), adam_eps=adam_eps, orthogonalize=orthogonalize))

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        o = {**self.defaults, **param_group}
        if not o["lr"] >= 0.0:
            raise ValueError(f"Muon: lr must not be negative, got {o['lr']}")
        if not 0.0 <= o["momentum"] < 1.0:
            raise ValueError(f"Muon: momentum must lie in [0, 1), got {o['momentum']}")
        if not o["weight_decay"] >= 0.0:
            raise ValueError(f"Muon: weight_decay must not be negative, got {o['weight_decay']}")
        if not all(0.0 <= b < 1.0 for b in o["betas"]) or not o["adam_eps"] > 0.0:
            raise ValueError(f"Muon: betas must lie in [0, 1) and adam_eps be positive, got {o['betas']}, {o['adam_eps']}")
        if int(o["ns_steps"]) != o["ns_steps"] or not 1 <= o["ns_steps"] <= 100:
            raise ValueError(f"Muon: ns_steps must be a whole number in 1..100, got {o['ns_steps']}")
        super().add_param_group(param_group)

    @staticmethod
    def _is_matrix(p: torch.Tensor) -> bool:
        return p.dim() >= 2 and min(p.shape[-2:]) > 1

    @torch.no_grad()
    def step(self, closure: Callable[[], Any] | None = None) -> Any:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_shape: dict[tuple, list[torch.Tensor]] = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse or p.is_complex():
                    raise RuntimeError("Muon: sparse gradients and complex parameters are not supported")
                if group["orthogonalize"] and self._is_matrix(p):
                    by_shape.setdefault((tuple(p.shape[-2:]), p.dtype, p.device), []).append(p)
                else:
                    self._adam_step(p, group)
            for (shape, _, _), ps in by_shape.items():
                self._matrix_step(ps, shape, group)
        return loss

    def _matrix_step(self, ps: list[torch.Tensor], shape: tuple[int, int], group: dict[str, Any]) -> None:
        from nvalchemi_toolkit_b200.ops.orthogonalize import newton_schulz

        grads = [p.grad.to(_state_type(p)) for p in ps]
        bufs = [self._buffer(p, "momentum_buffer") for p in ps]
        torch._foreach_mul_(bufs, group["momentum"])
        torch._foreach_add_(bufs, grads)
        updates = torch._foreach_add(grads, bufs, alpha=group["momentum"]) if group["nesterov"] else bufs
        stacked = torch.cat([u.reshape(-1, *shape) for u in updates])
        if stacked.dtype == torch.float64:
            stacked = stacked.float()
        o = newton_schulz(stacked, steps=group["ns_steps"])
        scale = 0.2 * max(shape) ** 0.5
        wide = [p.to(_state_type(p)) for p in ps]  # the parameters themselves, unless they have 16 bits
        if group["weight_decay"]:
            torch._foreach_mul_(wide, 1.0 - group["lr"] * group["weight_decay"])
        row = 0
        for p, w in zip(ps, wide):
            count = p.numel() // (shape[0] * shape[1])
            w.add_(o[row: row + count].reshape(p.shape).to(w.dtype), alpha=-group["lr"] * scale)
            row += count
            if w.dtype != p.dtype:
                p.copy_(w)

    def _buffer(self, p: torch.Tensor, name: str) -> torch.Tensor:
        """The state tensor ``name`` of ``p``, zeros when it is first asked for."""
        st = self.state[p]
        if name not in st:
            st[name] = torch.zeros_like(p, dtype=_state_type(p), memory_format=torch.preserve_format)
        return st[name]

    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        super().load_state_dict(state_dict)  # casts the state to the types of the parameters
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            if _state_type(p) != p.dtype:
                for name, v in state_dict["state"].get(i, {}).items():
                    if isinstance(v, torch.Tensor):
                        self.state[p][name] = v.to(p.device, _state_type(p))

    def _adam_step(self, p: torch.Tensor, group: dict[str, Any]) -> None:
        avg, avg_sq = self._buffer(p, "exp_avg"), self._buffer(p, "exp_avg_sq")
        b1, b2 = group["betas"]
        step = self.state[p]["adam_step"] = self.state[p].get("adam_step", 0) + 1
        w, grad = p.to(avg.dtype), p.grad.to(avg.dtype)  # p itself, unless it has 16 bits
        avg.lerp_(grad, 1 - b1)
        avg_sq.mul_(b2).addcmul_(grad, grad, value=1 - b2)
        denom = (avg_sq / (1 - b2 ** step)).sqrt_().add_(group["adam_eps"])
        if group["weight_decay"]:
            w.mul_(1.0 - group["lr"] * group["weight_decay"])
        w.addcdiv_(avg, denom, value=-group["lr"] / (1 - b1 ** step))
        if w.dtype != p.dtype:
            p.copy_(w)


class ParamGroupSpec(BaseModel):
    """Parameters whose qualified name matches ``pattern`` (``re.search``) form a group with their own optimiser options,
    e.g. ``ParamGroupSpec(pattern=r"bias$|norm", options={"weight_decay": 0.0})`` or a smaller ``lr`` for a pretrained trunk.
    The first matching spec wins; parameters no spec matches use the config's ``kwargs``."""

    pattern: str
    options: dict[str, Any] = Field(default_factory=dict)


class OptimizerConfig(BaseModel):
    """``cls(params, **kwargs)`` plus an optional scheduler.  ``scheduler_metric`` names the validation-summary key fed
    to metric-driven schedulers such as ``ReduceLROnPlateau``."""

    model_config = ConfigDict(arbitrary_types_allowed=True)
    cls: Any = torch.optim.Adam
    kwargs: dict[str, Any] = Field(default_factory=lambda: {"lr": 1e-3})
    scheduler_cls: Any = None
    scheduler_kwargs: dict[str, Any] = Field(default_factory=dict)
    scheduler_metric: str | None = None
    scheduler_interval: str = "step"  # "step" | "epoch" | "validation"
    #: maps the validation summary to the number a metric-driven scheduler steps on (default: ``summary[scheduler_metric]``)
    scheduler_metric_adapter: Callable[[Mapping[str, Any]], float] | None = None
    param_groups: list[ParamGroupSpec] = Field(default_factory=list)

    @model_validator(mode="after")
    def _validate(self) -> "OptimizerConfig":
        if self.scheduler_interval not in ("step", "epoch", "validation"):
            raise ValueError(f"scheduler_interval must be 'step', 'epoch' or 'validation', got {self.scheduler_interval!r}")
        cls = import_from_path(self.cls) if isinstance(self.cls, str) else self.cls
        check_kwargs(cls, self.kwargs, "optimizer")
        for g in self.param_groups:
            re.compile(g.pattern)
            check_kwargs(cls, g.options, "optimizer (parameter group)")
        if self.scheduler_cls is not None:
            scls = import_from_path(self.scheduler_cls) if isinstance(self.scheduler_cls, str) else self.scheduler_cls
            check_kwargs(scls, self.scheduler_kwargs, "scheduler")
        return self

    def group_parameters(self, named: list[tuple[str, torch.nn.Parameter]]) -> Any:
        """``named`` parameters split into optimiser parameter groups according to ``param_groups``."""
        if not self.param_groups:
            return [p for _, p in named]
        buckets: list[list[torch.nn.Parameter]] = [[] for _ in self.param_groups]
        rest: list[torch.nn.Parameter] = []
        for name, p in named:
            for i, g in enumerate(self.param_groups):
                if re.search(g.pattern, name):
                    buckets[i].append(p)
                    break
            else:
                rest.append(p)
        groups = [{"params": b, **g.options} for b, g in zip(buckets, self.param_groups) if b]
        return ([{"params": rest}] if rest else []) + groups

    def build(self, params: Any) -> tuple[torch.optim.Optimizer, Any]:
        cls = import_from_path(self.cls) if isinstance(self.cls, str) else self.cls
        if params and isinstance(params[0], tuple):  # (name, parameter) pairs: apply the group specs
            params = self.group_parameters(list(params))
        opt = cls(params, **self.kwargs)
        sched = None
        if self.scheduler_cls is not None:
            scls = import_from_path(self.scheduler_cls) if isinstance(self.scheduler_cls, str) else self.scheduler_cls
            sched = scls(opt, **self.scheduler_kwargs)
        return opt, sched

    def to_spec(self) -> dict[str, Any]:
        return {"cls": self.cls if isinstance(self.cls, str) else type_to_path(self.cls), "kwargs": dict(self.kwargs),
                "scheduler_cls": None if self.scheduler_cls is None else (
                    self.scheduler_cls if isinstance(self.scheduler_cls, str) else type_to_path(self.scheduler_cls)),
                "scheduler_kwargs": dict(self.scheduler_kwargs), "scheduler_metric": self.scheduler_metric,
                "scheduler_interval": self.scheduler_interval,
                "param_groups": [g.model_dump() for g in self.param_groups]}


def setup_optimizers(models: dict[str, torch.nn.Module], configs: dict[str, list[OptimizerConfig]],
                     name_filter: set[str] | None = None) -> tuple[list, list, list[str]]:
    """One optimiser (and scheduler slot) per configured (model, config); returns flat lists plus their model keys."""
    opts, scheds, keys = [], [], []
    for key, cfgs in configs.items():
        if key not in models:
            raise KeyError(f"optimizer configured for unknown model '{key}'")
        named = [(n, p) for n, p in models[key].named_parameters() if p.requires_grad]
        if name_filter is not None:
            named = [(n, p) for n, p in named if f"{key}.{n}" in name_filter or n in name_filter]
        for cfg in cfgs if isinstance(cfgs, (list, tuple)) else [cfgs]:
            o, s = cfg.build([(f"{key}.{n}", p) for n, p in named] if cfg.param_groups else [p for _, p in named])
            opts.append(o)
            scheds.append(s)
            keys.append(key)
    return opts, scheds, keys


def zero_gradients(opts: list) -> None:
    for o in opts:
        o.zero_grad(set_to_none=True)


def step_optimizers(opts: list) -> None:
    for o in opts:
        o.step()


def step_schedulers(scheds: list, configs: list[OptimizerConfig], interval: str, metrics: dict | None = None) -> None:
    for s, c in zip(scheds, configs):
        if s is None or c.scheduler_interval != interval:
            continue
        if isinstance(s, torch.optim.lr_scheduler.ReduceLROnPlateau):
            if metrics is not None and c.scheduler_metric_adapter is not None:
                s.step(float(c.scheduler_metric_adapter(metrics)))
            elif metrics is not None and c.scheduler_metric in metrics:
                s.step(float(metrics[c.scheduler_metric]))
        else:
            s.step()


def step_lr_schedulers(scheds: list, configs: "list[OptimizerConfig] | None" = None, interval: str = "step",
                       metrics: dict | None = None) -> None:
    """Step learning-rate schedulers (the reference's name, ``training/optimizers.py:404-447``).  With their
    ``OptimizerConfig`` list only those of the given ``interval`` step, metric-driven ones with ``metrics``; without it
    every scheduler that is not metric-driven steps once."""
    if configs is not None:
        step_schedulers(scheds, configs, interval, metrics)
        return
    for s in scheds:
        if s is not None and not isinstance(s, torch.optim.lr_scheduler.ReduceLROnPlateau):
            s.step()
