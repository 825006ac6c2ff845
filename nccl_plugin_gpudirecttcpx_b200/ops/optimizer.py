"""AdamW as a torch optimizer, on top of `adamw_step`: a few launches for each 380 parameters of a group and type."""
from __future__ import annotations

import itertools
import math
from typing import Optional

import torch

from .train import STATE_BLOCK, adamw_step, grad_norm


class AdamW(torch.optim.Optimizer):
    """AdamW over bfloat16, float16 or float32 CUDA parameters, with states in 32 or 8 bits.

    `state_bits`: 32 keeps float32 states.  8 keeps float8 codes with a scale for each 256 elements: a
    quarter of the memory and of the states' traffic; a state is off by up to 2^-4 of its value, small ones of a
    block by up to 2^-10 (a root that is raised to the smallest code: 2^-9) of the block's largest over 448.
    `master_weights`: float32 weights behind 16-bit parameters, which then are their rounded copies: they are
    taken from the parameters at the first step and part of the state, which is loaded with the model's.
    `max_grad_norm`: gradients are scaled, while they are read, by min(1, max_grad_norm / (norm + 1e-6))
    with the norm over all groups; `grad_norm` is the last step's, a device scalar.  Parameters without a
    gradient are left alone and their counters stand still, as in torch.optim.AdamW.

    Nothing is copied to or from the host, so a step can be captured into a graph once a first one has
    made the states; the graph keeps the learning rate it was captured with."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, master_weights: bool = False, max_grad_norm: Optional[float] = None):
        if state_bits not in (8, 32):
            raise ValueError(f"states have 8 or 32 bits, not {state_bits}")
        if max_grad_norm is not None and not 0 <= max_grad_norm < math.inf:
            raise ValueError(f"max_grad_norm has to be finite and not below zero, got {max_grad_norm}")
        self.state_bits, self.master_weights, self.max_grad_norm = state_bits, bool(master_weights), max_grad_norm
        self.grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), **{n: getattr(self, n) for n in ("state_bits", "master_weights", "max_grad_norm", "grad_norm")}}

    def add_param_group(self, group: dict) -> None:
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
        except (TypeError, ValueError):
            del self.param_groups[-1]  # a group that is refused is not there
            raise

    @staticmethod
    def _check_group(group: dict) -> None:
        if isinstance(group["lr"], torch.Tensor):
            raise TypeError("the learning rate has to be a number")
        (beta1, beta2), numbers = group["betas"], (group["lr"], group["eps"], group["weight_decay"])
        if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and all(0 <= x < math.inf for x in numbers)):
            raise ValueError(f"bad numbers: lr {group['lr']}, betas {group['betas']}, eps {group['eps']}, weight_decay {group['weight_decay']}")
        for p in group["params"]:
            if p.dtype not in (torch.bfloat16, torch.float16, torch.float32):
                raise TypeError(f"parameters have to be bfloat16, float16 or float32, got {p.dtype}")
            if not p.is_contiguous():
                raise ValueError("parameters have to be contiguous")

    def _state_of(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        if state:
            return state
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a parameter without states cannot be updated inside a capture, which would clear them at every replay: "
                               "run one step before")
        state["step"] = torch.zeros((), dtype=torch.int32, device=p.device)
        kind = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        blocks = -(-p.numel() // STATE_BLOCK)
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros(p.shape, dtype=kind, device=p.device)
            if self.state_bits == 8:
                state[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        if self.master_weights and p.dtype is not torch.float32:
            state["master"] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lists = []
        for group in self.param_groups:
            kinds: dict = {}
            for p in group["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise TypeError("gradients have to be dense")
                    kinds.setdefault((p.device, p.dtype), []).append(p)
            lists += [(group, ps, [p.grad.contiguous() for p in ps]) for ps in kinds.values()]
        norm = None
        if self.max_grad_norm is not None and len(lists) > 1:
            # one norm for lists of several types, groups or devices, on the first one's
            norms = [grad_norm(grads) for _, _, grads in lists]
            norm = torch.linalg.vector_norm(torch.stack([n.to(norms[0].device) for n in norms]))
        total = norm
        for group, ps, grads in lists:
            states = [self._state_of(p) for p in ps]
            more = {}
            if self.state_bits == 8:
                more = {"exp_avg_scales": [s["exp_avg_scale"] for s in states], "exp_avg_sq_scales": [s["exp_avg_sq_scale"] for s in states]}
            if "master" in states[0]:
                more["masters"] = [s["master"] for s in states]
            got = adamw_step(ps, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], [s["step"] for s in states], lr=group["lr"],
                             betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], max_grad_norm=self.max_grad_norm,
                             norm=None if norm is None else norm.to(ps[0].device), **more)
            total = got if total is None else total
        if total is None and self.max_grad_norm is not None:
            total = torch.zeros((), device=next((p.device for g in self.param_groups for p in g["params"]), None))  # of no gradients
        self.grad_norm = total
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As the base class does it, but states keep their own types (it gives them the parameters')."""
        saved = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        own = list(itertools.chain.from_iterable(g["params"] for g in self.param_groups))
        states = [state_dict["state"].get(n) for n in saved]
        names = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if self.state_bits == 8 else set())
        for p, s in zip(own, states):
            if s and set(s) != names | ({"master"} if self.master_weights and p.dtype is not torch.float32 else set()):
                raise ValueError(f"the states hold {sorted(s)}: they are of another state_bits or master_weights")
            for name, t in (s or {}).items():
                kind = torch.int32 if name == "step" else torch.float32 if self.state_bits == 32 or name not in ("exp_avg", "exp_avg_sq") else torch.float8_e4m3fn
                size = 1 if name == "step" else -(-p.numel() // STATE_BLOCK) if name.endswith("_scale") else p.numel()
                if not isinstance(t, torch.Tensor) or t.dtype is not kind or t.numel() != size or not t.is_contiguous():
                    raise ValueError(f"the state {name} has to be a contiguous {kind} tensor of {size}: these are another optimizer's or of other parameters")
        super().load_state_dict(state_dict)
        for p, s in zip(own, states):
            if s:
                self.state[p] = {name: t.detach().clone().to(p.device) for name, t in s.items()}
