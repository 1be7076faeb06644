"""AdamW over many tensors in few launches, with moments in float32 or in 8 bits.

``adamw_step`` is the step on lists of tensors (``gs_adamw_step`` of libgruscan.so, its
checks in csrc/torch_ops.cpp: a tensor's take under 0.1 us there, over 1 us in Python);
``AdamW`` is the optimizer around it. No counterpart in the reference.
"""

from __future__ import annotations

from typing import Any, Callable, Iterable, Optional, Sequence, Tuple

import torch

from . import _lib

STATE_BLOCK = 256  # elements of a tensor that share a scale where moments are held in 8 bits
_ROUNDINGS = {"nearest": _lib.ROUND_NEAREST, "unbiased": _lib.ROUND_UNBIASED}


def _rounding(who: str, rounding: Any) -> int:
    try:
        return _ROUNDINGS[rounding]
    except (KeyError, TypeError):
        raise ValueError(f"{who}: rounding must be 'nearest' or 'unbiased'; got {rounding!r}") from None


def _blocks(n: int) -> int:
    return -(-n // STATE_BLOCK)


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    *,
    step: int,
    lr: float,
    betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    masters: Optional[Sequence[torch.Tensor]] = None,
    exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
    exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
    grad_scale: Optional[torch.Tensor] = None,
    rounding: str = "nearest",
) -> None:
    """One AdamW step in place, the ``step``-th (from 1), on contiguous tensors of one device.

    ``params`` are float32, or bfloat16 with float32 ``masters`` of which they are the
    rounding (without masters, updates under half a bfloat16 unit are lost); all of one
    type, and ``grads`` too. The moments are float32, or, with ``exp_avg_scales`` and
    ``exp_avg_sq_scales`` (float32, one number per 256 elements), int8 and uint8 codes (see
    ``adamw_dequantize_state``). ``grad_scale``: a float32 tensor of one element on the
    device that multiplies the gradients; where it is not finite the step does nothing.

    ``rounding`` of 8-bit moments: "nearest" stores the nearest code and loses every change of
    less than half a code. While a block's largest magnitude holds and betas are (0.9, 0.999), a second
    moment then never falls, rises only where g^2 passes 9 to 40 times it, and a first moment of
    code 9 or less (0.5 % of the largest) stays for good. "unbiased" stores one of the two codes
    around a value so that the average over steps is right; which one is a hash of ``step``,
    the tensor's place in the list and the element, so that results repeat."""
    how = _rounding("adamw_step", rounding)
    try:
        (_lib._ops or _lib.ops()).adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas[0], betas[1], eps,
                                             weight_decay, masters, exp_avg_scales, exp_avg_sq_scales, grad_scale, how)
    except TypeError as e:
        raise ValueError(f"adamw_step: params, grads and states must be lists of tensors ({e})") from None


def adamw_dequantize_state(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 values of a moment held in 8 bits: int8 ``codes`` c stand for
    A sign(c) (c / 127)^2 (the first moment), uint8 ones for A (c / 255)^4 (the second),
    with A = ``scales`` [ceil(n / 256)], one for each 256 elements."""
    try:
        return (_lib._ops or _lib.ops()).adamw_dequantize_state(codes, scales)
    except TypeError as e:
        raise ValueError(f"adamw_dequantize_state: codes and scales must be tensors ({e})") from None


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is ``adamw_step``: one launch for up to 48 parameters.

    ``state_bits`` 32 keeps float32 moments, 8 keeps codes of 8 bits with a float32 scale
    per 256 elements (2 bytes an element instead of 8). ``state_rounding`` is the ``rounding`` of
    those codes: "unbiased" follows gradients that grow, shrink or end, with a noise of a few per
    cent of an update where gradients are within a hundredth of their block's largest and as large as the
    update under a ten thousandth; elements under 1.5e-5 of it move less than they should. "nearest"
    has no noise, but does not follow such changes (``adamw_step``), and an element
    under four millionths of the largest keeps a second moment of 0: an ``eps`` of the size of such
    gradients keeps its updates small. bfloat16 parameters get float32
    masters unless ``master_weights`` is off (taken at a parameter's first step; from then on
    a parameter is its master's rounding, whatever else is written to it). ``step(grad_scale=...)`` multiplies the
    gradients by a device scalar (a clipping factor, an inverse loss scale); where that is
    not finite, parameters and moments stay as they are (the count of steps still advances:
    the host does not read the scalar)."""

    def __init__(self, params: Iterable[Any], lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *, state_bits: int = 32,
                 master_weights: bool = True, state_rounding: str = "unbiased") -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32; got {state_bits}")
        _rounding("AdamW", state_rounding)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, state_rounding=state_rounding))

    def _init_state(self, p: torch.Tensor, group: dict) -> None:
        s = self.state[p]
        s["step"] = 0
        n = p.numel()
        if group["state_bits"] == 8:
            s["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
            s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
            s["exp_avg_scale"] = torch.zeros(_blocks(n), device=p.device)
            s["exp_avg_sq_scale"] = torch.zeros(_blocks(n), device=p.device)
        else:
            s["exp_avg"] = torch.zeros(p.shape, device=p.device)
            s["exp_avg_sq"] = torch.zeros(p.shape, device=p.device)
        if p.dtype == torch.bfloat16 and group["master_weights"]:
            s["master"] = p.detach().float()

    @torch.no_grad()
    def step(self, closure: Optional[Callable[[], Any]] = None, *,
             grad_scale: Optional[torch.Tensor] = None) -> Any:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls: dict = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise ValueError("AdamW: sparse gradients are not supported")
                s = self.state[p]
                if not s:
                    self._init_state(p, group)
                calls.setdefault((s["step"], p.dtype, g.dtype, p.device, "master" in s), []).append((p, g, s))
            for (count, _, _, _, master), rows in calls.items():
                states = [s for _, _, s in rows]
                scales = {}
                if group["state_bits"] == 8:
                    scales = dict(exp_avg_scales=[s["exp_avg_scale"] for s in states],
                                  exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states])
                adamw_step([p for p, _, _ in rows], [g for _, g, _ in rows], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], step=count + 1, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"],
                           masters=[s["master"] for s in states] if master else None, grad_scale=grad_scale,
                           rounding=group.get("state_rounding", "unbiased"), **scales)
                for s in states:
                    s["step"] = count + 1
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, with moments, codes, scales and masters kept in their own types (torch
        casts a state to its parameter's type)."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if i in saved:
                self.state[p] = {k: v.to(device=p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                 for k, v in saved[i].items()}
