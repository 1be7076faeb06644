"""Gated linear recurrence: the GRU update without a hidden map, so that a sequence
is a scan over independent channels instead of T dependent matrix products.

``z = sigmoid(gi_z)``, ``n = tanh(gi_n)`` (or ``gi_n``),
``h_t = z h_{t-1} + (1 - z) n`` with ``gi = [gi_z, gi_n]`` [T, B, 2H] from an input
projection. Activations are float32 or bfloat16; states and sums are float32. The
kernels are ``gs_glr_fwd``, ``gs_glr_bwd`` and ``gs_glr_step`` of libgruscan.so, their
checks and autograd in csrc/torch_ops.cpp. No counterpart in the reference.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple

import torch

from . import _lib

_ACTIVATIONS = {"identity": _lib.ACT_NONE, "tanh": _lib.ACT_TANH}


def _activation(who: str, activation: Any) -> int:
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"{who}: activation must be 'tanh' or 'identity'; got {activation!r}") from None


def gated_linear_scan(
    gi: torch.Tensor,
    h0: Optional[torch.Tensor] = None,
    *,
    activation: str = "tanh",
    reset: Optional[torch.Tensor] = None,
    batch_first: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(out, h_T)`` of the recurrence over ``gi`` [T, B, 2H] (``[B, T, 2H]`` when
    ``batch_first``): ``out`` [T, B, H] in gi's type (float32 or bfloat16), ``h_T`` [B, H]
    in float32, with which a following call continues. ``h0`` [B, H] float32 (zeros when
    None). ``reset`` [T, B] bool starts a new sequence at a step: the state before it is
    taken as zero, whatever it is. Differentiable in gi and h0 (once).

    On few channels and a long axis workgroups wait for each other, for seconds at most; a wait
    that runs out leaves NaN from there on, and the next scan on the device, or ``check_faults``,
    raises ``PersistentScanFault``."""
    act = _activation("gated_linear_scan", activation)
    try:
        return (_lib._ops or _lib.ops()).gated_linear_scan(gi, h0, reset, act, batch_first)
    except TypeError as e:
        raise ValueError(f"gated_linear_scan: gi, h0 and reset must be tensors ({e})") from None


def gated_linear_step(
    gi: torch.Tensor,
    state: torch.Tensor,
    slots: Optional[torch.Tensor] = None,
    *,
    activation: str = "tanh",
) -> torch.Tensor:
    """One token for each row of ``gi`` [B, 2H]: advances row ``slots[b]`` of ``state``
    [S, H] (float32, in place) and returns ``out`` [B, H] in gi's type. ``slots`` [B] int32
    holds distinct rows of the cache (row b uses state b when None); a negative one marks
    an empty row of the batch, whose output is zero. A slot past the cache gives NaN and
    touches no state. No autograd."""
    act = _activation("gated_linear_step", activation)
    try:
        return (_lib._ops or _lib.ops()).gated_linear_step(gi, state, slots, act)
    except TypeError as e:
        raise ValueError(f"gated_linear_step: gi, state and slots must be tensors ({e})") from None
