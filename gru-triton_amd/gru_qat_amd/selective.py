"""Selective state space scan: a recurrence whose decay and input depend on the step.

``dt = softplus(delta + delta_bias)``, ``h_t[n] = exp(dt A[n]) h_{t-1}[n] + dt u B_t[n]``,
``y = (sum_n C_t[n] h_t[n] + D u) silu(z)`` for every channel, with N states each. Activations are
float32 or bfloat16; A, D, delta_bias, states and sums are float32. The kernels are
``gs_ssm_fwd``, ``gs_ssm_bwd`` and ``gs_ssm_step`` of libgruscan.so, their checks and autograd in
csrc/torch_sequence_ops.cpp. No counterpart in the reference.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def selective_scan(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    h0: Optional[torch.Tensor] = None,
    *,
    delta_bias: Optional[torch.Tensor] = None,
    reset: Optional[torch.Tensor] = None,
    batch_first: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(y, h_T)`` of the recurrence over ``u`` and ``delta`` [T, B, H] with ``B`` and ``C`` [T, B, N],
    all ``[B, T, ...]`` when ``batch_first``, and ``A`` [H, N], N from 1 to 32: ``y`` [T, B, H] in u's
    type, ``h_T`` [B, H, N] in float32, with which a following call continues. ``D`` and
    ``delta_bias`` [H] and ``h0`` [B, H, N] are float32 (zeros when None), ``z`` [T, B, H] gates the output
    (no gate when None). ``reset`` [T, B] bool starts a new sequence at a step: the state before it is
    taken as zero, whatever it is. An infinite state stays one until then, or until a step whose decay is zero
    in float32 (exp(dt A) below 1e-38), which makes it NaN. Differentiable in all of them but reset (once); a training forward
    keeps the states before every 16th step and, with z, the outputs before their gate, in float32."""
    try:
        return (_lib._ops or _lib.ops()).selective_scan(u, delta, A, B, C, D, z, h0, delta_bias, reset, batch_first)
    except TypeError as e:
        raise ValueError(f"selective_scan: arguments must be tensors ({e})") from None


def selective_step(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    state: torch.Tensor,
    slots: Optional[torch.Tensor] = None,
    *,
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    delta_bias: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One token for each row of ``u``, ``delta`` and ``z`` [B, H], ``B`` and ``C`` [B, N]: advances row
    ``slots[b]`` of ``state`` [S, H, N] (float32, in place) and returns ``y`` [B, H] in u's type.
    ``slots`` as in ``gated_linear_step``: distinct int32 rows, row b when None, a negative one for an
    empty row of the batch (its output is zero), NaN for one past the cache. At most 65535 rows. No autograd."""
    try:
        return (_lib._ops or _lib.ops()).selective_step(u, delta, A, B, C, state, slots, D, z, delta_bias)
    except TypeError as e:
        raise ValueError(f"selective_step: arguments must be tensors ({e})") from None
