"""Linear with bias, activation and residual in one call: ``act(x W^T + bias) + residual``.

In bfloat16 the product runs on the bf16 matrix units with float32 sums, in float32 on
the fp32 ones (``gs_linear_fwd`` / ``gs_linear_bwd`` of libgruscan.so). No counterpart in
the reference, whose projections are ``input_projection``'s.
"""

from __future__ import annotations

import functools
from typing import Any, Optional, cast

import torch

from . import _lib
from .gated_linear import _DTYPES

_ACTIVATIONS = {"none": _lib.ACT_NONE, "tanh": _lib.ACT_TANH, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
                "silu": _lib.ACT_SILU, "sigmoid": _lib.ACT_SIGMOID}


@functools.lru_cache(maxsize=4096)
def _fwd_scratch(M: int, N: int, K: int, dtype: int) -> int:
    return _lib.raw_size(_lib.load(), "gs_linear_scratch_bytes",
                         _lib.LINEAR_ARGS.pack(*[0] * 8, M, N, K, K, N, N, dtype, _lib.ACT_NONE))


@functools.lru_cache(maxsize=4096)
def _bwd_scratch(M: int, N: int, K: int, dtype: int, act: int, dx: bool, dw: bool, dbias: bool) -> int:
    return _lib.raw_size(_lib.load(), "gs_linear_bwd_scratch_bytes",
                         _lib.LINEAR_BWD_ARGS.pack(0, 0, 0, 0, dx, dw, dbias, 0, 0, M, N, K, K, N, dtype, act))


def _forward(x2: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], res2: Optional[torch.Tensor], act: int,
             pre: Optional[torch.Tensor]) -> torch.Tensor:
    M, K = x2.shape
    N = w.shape[0]
    y = x2.new_empty((M, N))
    dtype = _DTYPES[x2.dtype]
    nbytes = _fwd_scratch(M, N, K, dtype)
    buf = torch.empty(nbytes, dtype=torch.uint8, device=x2.device) if nbytes else None
    _lib.call_on("gs_linear_fwd", _lib.LINEAR_ARGS.pack(
        x2.data_ptr(), w.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if res2 is None else res2.data_ptr(),
        y.data_ptr(), 0 if pre is None else pre.data_ptr(), 0 if buf is None else buf.data_ptr(), nbytes, M, N, K,
        x2.stride(0), 0 if res2 is None else res2.stride(0), N, dtype, act), x2.get_device())
    return y  # buf goes back to the caching allocator, which keeps it until the stream's work is done


class LinearActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x2, w, bias, res2, act):  # type: ignore[override]
        pre = x2.new_empty((x2.shape[0], w.shape[0])) if act else None
        y = _forward(x2, w, bias, res2, act, pre)
        ctx.save_for_backward(x2, w, pre)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx: Any, dy: torch.Tensor):  # type: ignore[override]
        x2, w, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        M, K = x2.shape
        N = w.shape[0]
        dres = dy if need[3] else None
        if not any(need[:3]):
            return None, None, None, dres, None
        if dy.stride(1) != 1 and N > 1:
            dy = dy.contiguous()
        dx = x2.new_empty((M, K)) if need[0] else None
        dw = x2.new_empty((N, K)) if need[1] else None
        dbias = x2.new_empty((N,)) if need[2] else None
        dtype = _DTYPES[x2.dtype]
        nbytes = _bwd_scratch(M, N, K, dtype, ctx.act, *need[:3])
        buf = torch.empty(nbytes, dtype=torch.uint8, device=x2.device) if nbytes else None
        _lib.call_on("gs_linear_bwd", _lib.LINEAR_BWD_ARGS.pack(
            x2.data_ptr(), w.data_ptr(), _lib.ptr(pre), dy.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(dbias),
            _lib.ptr(buf), nbytes, M, N, K, x2.stride(0), dy.stride(0), dtype, ctx.act), x2.get_device())
        return dx, dw, dbias, dres, None


def _require(who: str, x: torch.Tensor, **tensors: Any) -> None:
    for k, t in dict(x=x, **tensors).items():
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{who}: {k} must be a CUDA (HIP) tensor; got "
                             f"{t.device if isinstance(t, torch.Tensor) else type(t).__name__}")
        if t.get_device() != x.get_device():
            raise ValueError(f"{who}: all tensors must be on {x.device}; {k} is on {t.device}")
        if t.dtype != x.dtype or t.dtype not in _DTYPES:
            raise ValueError(f"{who}: all tensors must be float32 or all bfloat16; {k} is {t.dtype}, x {x.dtype}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


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
    "tanh" or "sigmoid". Differentiable in all four tensors; with an activation, a training
    forward keeps its argument [..., N] in x's type."""
    who = "linear_act"
    try:
        act = _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"{who}: activation must be one of {', '.join(_ACTIVATIONS)}; got {activation!r}") from None
    try:
        d, kind = x.get_device(), x.dtype
        ready = (d >= 0 and kind in _DTYPES and weight.get_device() == d and weight.dtype is kind
                 and (bias is None or (bias.get_device() == d and bias.dtype is kind))
                 and (residual is None or (residual.get_device() == d and residual.dtype is kind)))
    except AttributeError:
        ready = False
    if not ready:
        _require(who, x, weight=weight, **{k: t for k, t in (("bias", bias), ("residual", residual)) if t is not None})
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{who}: weight must be [N, K] with K = x.shape[-1]; got x {tuple(x.shape)}, weight "
                         f"{tuple(weight.shape)}")
    if x.numel() == 0 or weight.numel() == 0:
        raise ValueError(f"{who}: x and weight must be non-empty; got x {tuple(x.shape)}, weight {tuple(weight.shape)}")
    N = weight.shape[0]
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"{who}: bias must be [{N}]; got {tuple(bias.shape)}")
    shape = (*x.shape[:-1], N)
    if residual is not None and residual.shape != shape:
        raise ValueError(f"{who}: residual must be {shape}; got {tuple(residual.shape)}")
    x2, w = _rows(x), weight if weight.is_contiguous() else weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    res2 = _rows(residual) if residual is not None else None
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        y = LinearActFunction.apply(x2, w, bias, res2, act)
    else:
        y = _forward(x2, w, bias, res2, act, None)
    return cast(torch.Tensor, y if len(shape) == 2 else y.view(shape))
