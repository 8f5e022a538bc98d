"""AdamW for the training of the block modules, one fused step over all parameters.

Stands where the reference's training loop clips its gradients and steps its optimizer
(train.py:1163-1170).  ``torch.ops``-level form: :func:`strata_amd.ops.adamw_step`.
"""

from __future__ import annotations

from itertools import chain
from typing import Optional

import torch
from torch import Tensor

from . import ops


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay over the parameters of one GPU.

    state_bits  32: fp32 moments.  8: codes with a scale for every 256 elements (2.03 bytes a
                parameter instead of 8); tensors under ``min_8bit`` elements keep fp32 moments.
    master      fp32 weights kept beside bf16 parameters, which are rounded from them (without
                them an update below half a bf16 step of its weight is lost).
    max_norm    clips the gradients by the norm of all of them together; ``grad_norm`` then holds
                the last norm (fp64 ``[1]``, on the GPU), and a step whose norm is not finite is
                left out whole.

    ``lr`` and ``weight_decay`` may differ between parameter groups, ``betas`` and ``eps`` are
    the optimizer's.  A parameter counts the steps that it took (with a gradient), for its bias corrections;
    parameters that have taken the same ones share a count, which lives on the GPU.  A step can be
    captured in a graph, after one eager step with the same gradients has made the states and counts (the
    rates are those of the capture).

    A master weight stands for its parameter once it exists, at the first step: a value written
    into the parameter later (loaded weights, an average) goes into ``state[p]["master"]`` too, or
    the next step takes it back."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, master: bool = True,
                 max_norm: Optional[float] = None, min_8bit: int = 4096):
        if state_bits not in (32, 8):
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {state_bits}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps >= 0.0:
            raise ValueError(f"AdamW: betas must lie in [0, 1) and eps be at least 0, got {betas}, {eps}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"AdamW: max_norm must be positive, got {max_norm}")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))
        self.betas, self.eps, self.max_norm = (float(betas[0]), float(betas[1])), float(eps), max_norm
        self.state_bits, self.master, self.min_8bit = state_bits, master, int(min_8bit)
        self.grad_norm: Optional[Tensor] = None

    def __getstate__(self) -> dict:  # copies and pickles: torch's own keeps the groups and states alone
        own = ("betas", "eps", "max_norm", "state_bits", "master", "min_8bit", "grad_norm")
        return {**super().__getstate__(), **{k: self.__dict__[k] for k in own}}

    def add_param_group(self, group) -> None:
        for k in ("betas", "eps", "max_norm"):
            if isinstance(group, dict) and k in group:
                raise ValueError(f"AdamW: {k} is the optimizer's, not a parameter group's")
        super().add_param_group(group)

    def _new_state(self, p: Tensor, step: Tensor) -> dict:
        n = p.numel()
        s = {"step": step}
        if self.state_bits == 8 and n >= self.min_8bit:
            blocks = -(-n // ops.STATE_BLOCK)
            s["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
            s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
            s["exp_avg_scale"], s["exp_avg_sq_scale"] = torch.zeros(2, blocks, device=p.device).unbind()
        else:
            s["exp_avg"], s["exp_avg_sq"] = (torch.zeros(p.shape, device=p.device) for _ in range(2))
        if self.master and p.dtype == torch.bfloat16:
            s["master"] = p.detach().float()
        return s

    def _uncaptured(self) -> None:
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a step is captured after an eager one with the same gradients, which makes its states")

    def _split_counts(self, states: list[dict]) -> None:
        """States that this step leaves out keep their count: a copy of one that they share with others."""
        taking, counts, kept = set(map(id, states)), {id(s["step"]) for s in states}, {}
        for s in self.state.values():
            step = s.get("step")
            if step is None or id(s) in taking or id(step) not in counts:
                continue
            if id(step) not in kept:
                self._uncaptured()
                kept[id(step)] = step.clone()
            s["step"] = kept[id(step)]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ps, lrs, wds = [], [], []
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("AdamW: sparse gradients are not supported")
                ps.append(p)
                lrs.append(group["lr"])
                wds.append(group["weight_decay"])
        if not ps:
            return loss
        new = [p for p in ps if not self.state[p]]
        if new:
            self._uncaptured()
            step = torch.zeros(1, dtype=torch.int64, device=ps[0].device)
            for p in new:
                self.state[p].update(self._new_state(p, step))
        states = [self.state[p] for p in ps]
        if len(self.state) > len(ps):
            self._split_counts(states)
        self.grad_norm = ops.adamw_step(
            ps, [p.grad.contiguous() for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
            [s["step"] for s in states], lr=lrs, betas=self.betas, eps=self.eps, weight_decay=wds, max_norm=self.max_norm,
            masters=[s.get("master") for s in states], exp_avg_scales=[s.get("exp_avg_scale") for s in states],
            exp_avg_sq_scales=[s.get("exp_avg_sq_scale") for s in states])
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but every state keeps the type it was saved in (torch's would round the fp32
        moments and master weights of a bf16 parameter to bf16), and equal counts become one."""
        super().load_state_dict(state_dict)
        saved = chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        counts, values = {}, {}
        for i, p in zip(saved, chain.from_iterable(g["params"] for g in self.param_groups)):
            if i not in state_dict["state"]:
                continue
            s = {k: v.detach().to(p.device, copy=True) for k, v in state_dict["state"][i].items()}
            one = state_dict["state"][i]["step"]
            if id(one) not in values:
                values[id(one)] = int(one)
            s["step"] = counts.setdefault(values[id(one)], s["step"])
            self.state[p] = s
