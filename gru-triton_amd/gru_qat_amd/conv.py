"""Short causal convolution of each channel over time, ``y_t = act(bias + sum_k w_k x_{t-W+1+k})``,
as layers around a recurrence use it to mix a few neighbouring steps. The kernels are
``gs_conv_fwd``, ``gs_conv_bwd`` and ``gs_conv_step`` of libgruscan.so, their checks and autograd
in csrc/torch_sequence_ops.cpp. No counterpart in the reference.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple

import torch

from . import _lib

_ACTIVATIONS = {"none": _lib.ACT_NONE, "silu": _lib.ACT_SILU}


def _activation(who: str, activation: Any) -> int:
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"{who}: activation must be 'none' or 'silu'; got {activation!r}") from None


def causal_conv(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    state: Optional[torch.Tensor] = None,
    *,
    activation: str = "silu",
    reset: Optional[torch.Tensor] = None,
    batch_first: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(y, last)`` for ``x`` [T, B, C] (``[B, T, C]`` when ``batch_first``), ``weight`` [C, W] with
    W from 2 to 4 (``weight[:, -1]`` for the step itself) and ``bias`` [C]. ``state`` [B, W - 1, C]
    holds the inputs before the first step, oldest first (zeros when None), and ``last`` those of the
    last W - 1 steps, with which a following call continues. ``reset`` [T, B] bool starts a new
    sequence at a step: whatever is before counts as zero. All tensors are float32 or all bfloat16,
    sums float32. Differentiable in x, weight, bias and state, from y and last (once)."""
    act = _activation("causal_conv", activation)
    try:
        return (_lib._ops or _lib.ops()).causal_conv(x, weight, bias, state, reset, act, batch_first)
    except TypeError as e:
        raise ValueError(f"causal_conv: x, weight, bias, state and reset must be tensors ({e})") from None


def causal_conv_step(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    state: torch.Tensor,
    slots: Optional[torch.Tensor] = None,
    *,
    activation: str = "silu",
) -> torch.Tensor:
    """One token for each row of ``x`` [B, C]: ``y`` [B, C], with the inputs before it in row
    ``slots[b]`` of ``state`` [S, W - 1, C] (x's type), which moves on in place. ``slots`` as in
    ``gated_linear_step``: distinct int32 rows, row b when None, a negative one for an empty row
    of the batch (its output is zero), NaN for one past the cache. At most 65535 rows. No autograd."""
    act = _activation("causal_conv_step", activation)
    try:
        return (_lib._ops or _lib.ops()).causal_conv_step(x, weight, bias, state, slots, act)
    except TypeError as e:
        raise ValueError(f"causal_conv_step: x, weight, bias, state and slots must be tensors ({e})") from None
