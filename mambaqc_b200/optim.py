"""AdamW for the LM's training step, with moments in 32 or in 8 bits.

``AdamW`` takes the place of ``torch.optim.AdamW`` that the reference trainer uses
(mambaqc train.py): the same update, over all tensors in a few launches
(``kernels.adamw_step``), with gradient clipping folded into it. With
``state_bits=8`` the two moments take 2 bytes a parameter instead of 8, which is
what lets the base preset's weights, gradients and moments share one GPU.
"""

from __future__ import annotations

from collections.abc import Callable

import torch

from . import _lib
from .kernels.adamw import adamw_moments, adamw_step, grad_norm

__all__ = ["AdamW"]


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on CUDA fp32 or bf16 parameters.

    ``state_bits``: 32 keeps fp32 moments; 8 keeps a byte each of m and sqrt(v) and
    two bytes for every 256 of them (see ``kernels.adamw``). bf16 parameters, and
    8-bit moments, are rounded up or down by a hash that ``seed`` chooses, so that
    small updates are not lost; the same seed gives the same bits. ``step(closure,
    max_grad_norm=...)`` clips by the global norm of all gradients without rewriting
    them and leaves the norm, a device scalar, in ``grad_norm``. A gradient that is
    infinite or NaN makes the moments and parameters NaN, as it would in 32 bits; in
    8 bits it takes its block of 256 with it at the next step. One whose square is
    infinite in fp32 (above 1.8e19) makes v infinite: the parameter takes no step from
    it, and in 8 bits, where that marks the block, the block is NaN at the next step."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 seed: int = 0):
        if lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError("AdamW: lr, eps and weight_decay must not be negative")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas}")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits = state_bits
        self.seed = seed
        self.grad_norm: torch.Tensor | None = None

    def __getstate__(self) -> dict:
        """What a copy or a pickle keeps (the base class would leave these three out)."""
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed,
                "grad_norm": self.grad_norm}

    def _state_of(self, p: torch.Tensor) -> dict:
        s = self.state[p]
        if s:
            return s
        s["step"] = 0
        if self.state_bits == 32:
            s["exp_avg"] = torch.zeros(p.numel(), dtype=torch.float32, device=p.device)
            s["exp_avg_sq"] = torch.zeros_like(s["exp_avg"])
        else:
            blocks = -(-p.numel() // _lib.MQC_ADAMW_BLOCK)
            for name, n in (("exp_avg", p.numel()), ("exp_avg_sq", p.numel()),
                            ("exp_avg_exponent", blocks), ("exp_avg_sq_exponent", blocks)):
                s[name] = torch.zeros(n, dtype=torch.uint8, device=p.device)
        return s

    @torch.no_grad()
    def step(self, closure: Callable | None = None, *, max_grad_norm: float | None = None):
        """One update of every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # (group, place in the whole list, parameter, gradient), gradients flat and dense
        work = []
        place = 0
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise RuntimeError("AdamW: sparse gradients are not supported")
                    work.append((group, place, p, p.grad.contiguous()))
                place += 1
        self.grad_norm = None
        clips = {}
        if max_grad_norm is not None and work:
            devices = {g.device for _, _, _, g in work}
            if len(devices) > 1:
                raise RuntimeError("AdamW: clipping needs all parameters on one device")
            got = grad_norm([g for _, _, _, g in work], max_grad_norm)
            self.grad_norm = got[0]
            clips[work[0][3].device] = got[1]
        # parameters that share hyperparameters and step go in one call
        calls: dict[tuple, list] = {}
        for group, place, p, g in work:
            s = self._state_of(p)
            key = (id(group), s["step"] + 1, p.device)
            calls.setdefault(key, [group]).append((place, p, g, s))
        for (_, step, device), (group, *members) in calls.items():
            dense = [p if p.is_contiguous() else p.contiguous() for _, p, _, _ in members]
            states = [s for _, _, _, s in members]
            exponents = None
            if self.state_bits == 8:
                exponents = ([s["exp_avg_exponent"] for s in states],
                             [s["exp_avg_sq_exponent"] for s in states])
            adamw_step(dense, [g for _, _, g, _ in members], [s["exp_avg"] for s in states],
                       [s["exp_avg_sq"] for s in states], step=step, lr=float(group["lr"]),
                       betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], exponents=exponents, seed=self.seed, carry=True,
                       clip=clips.get(device), ordinals=[k for k, _, _, _ in members])
            for d, (_, p, _, s) in zip(dense, members):
                s["step"] = step        # counted when done: not by a call that is refused
                if d is not p:
                    p.copy_(d)
        return loss

    @torch.no_grad()
    def moments(self, p: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(m, sqrt(v)) of one parameter as they stand, shaped like it: fp32 from 32-bit
        moments, bf16 (exact) from 8-bit ones."""
        s = self._state_of(p)
        if self.state_bits == 32:
            return s["exp_avg"].view(p.shape).clone(), s["exp_avg_sq"].sqrt().view(p.shape)
        (m,), (root,) = adamw_moments([s["exp_avg"]], [s["exp_avg_sq"]],
                                      ([s["exp_avg_exponent"]], [s["exp_avg_sq_exponent"]]))
        return m.view(p.shape), root.view(p.shape)

    def state_dict(self) -> dict:
        return {**super().state_dict(), "state_bits": self.state_bits, "seed": self.seed}

    def load_state_dict(self, state_dict: dict) -> None:
        """Loads a state as it was saved. (The base class would cast the moments to the
        parameters' type.) A state of ``torch.optim.AdamW`` is one with 32-bit moments:
        its steps become numbers, its moments flat and fp32."""
        bits = state_dict.get("state_bits", 32)
        for option in ("amsgrad", "maximize"):
            if any(g.get(option) for g in state_dict["param_groups"]):
                raise ValueError(f"AdamW: the state is one with {option}, which this optimizer "
                                 "does not have")
        if bits != self.state_bits:
            raise ValueError(f"AdamW: the state has {bits}-bit moments, "
                             f"the optimizer {self.state_bits}-bit ones")
        super().load_state_dict({k: state_dict[k] for k in ("state", "param_groups")})
        self.seed = state_dict.get("seed", self.seed)
        places = [k for g in state_dict["param_groups"] for k in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for k, p in zip(places, params):
            for name, value in state_dict["state"].get(k, {}).items():
                if name == "step":
                    value = int(value)
                elif torch.is_tensor(value):
                    value = value.detach().reshape(-1)      # in the order of p's elements
                    dtype = torch.float32 if value.is_floating_point() else value.dtype
                    value = value.to(p.device, dtype, copy=True)
                self.state[p][name] = value
