"""Linear with bias, activation and residual in one call: ``act(x W^T + bias) + residual``.

In bfloat16 the product runs on the bf16 matrix units with float32 sums, in float32 on
the fp32 ones (``gs_linear_fwd`` / ``gs_linear_bwd`` of libgruscan.so; checks and
autograd in csrc/torch_ops.cpp). No counterpart in the reference, whose projections are
``input_projection``'s.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_ACTIVATIONS = {"none": _lib.ACT_NONE, "tanh": _lib.ACT_TANH, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
                "silu": _lib.ACT_SILU, "sigmoid": _lib.ACT_SIGMOID}


def linear_act(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    activation: str = "none",
    residual: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` for ``x`` [..., K], ``weight`` [N, K], ``bias``
    [N] and ``residual`` [..., N], all float32 or all bfloat16 on one GPU; returns [..., N] in
    that type, every sum in float32. ``activation``: "none", "relu", "gelu" (of erf), "silu",
    "tanh" or "sigmoid". Differentiable in all four tensors (once). With an activation, a training
    forward keeps its argument [..., N], in bfloat16 as halves, and a bfloat16 backward rounds the
    argument's gradient to bfloat16, as an operand of the products for x and weight, whose error that
    takes from 0.0017 of their size (their own rounding) to 0.0024."""
    try:
        act = _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"linear_act: activation must be one of {', '.join(_ACTIVATIONS)}; got {activation!r}") from None
    try:
        return (_lib._ops or _lib.ops()).linear_act(x, weight, bias, residual, act)
    except TypeError as e:
        raise ValueError(f"linear_act: x, weight, bias and residual must be tensors ({e})") from None
