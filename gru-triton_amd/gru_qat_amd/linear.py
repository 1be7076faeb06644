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


def _buffer(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _forward(x2: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], res2: Optional[torch.Tensor], act: int,
             pre: Optional[torch.Tensor]) -> torch.Tensor:
    lib = _lib.load()
    M, K = x2.shape
    N = w.shape[0]
    y = torch.empty((M, N), dtype=x2.dtype, device=x2.device)
    dtype = _DTYPES[x2.dtype]
    nbytes = _fwd_scratch(M, N, K, dtype)
    buf = _buffer(nbytes, x2.device)
    a = _lib.LINEAR_ARGS.pack(x2.data_ptr(), w.data_ptr(), _lib.ptr(bias), _lib.ptr(res2), y.data_ptr(), _lib.ptr(pre),
                              _lib.ptr(buf), nbytes, M, N, K, x2.stride(0), res2.stride(0) if res2 is not None else 0, N,
                              dtype, act)
    _lib.raw_call(lib, "gs_linear_fwd", a, x2.device)
    return y  # buf goes back to the caching allocator, which keeps it until the stream's work is done


class LinearActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x2, w, bias, res2, act):  # type: ignore[override]
        pre = torch.empty((x2.shape[0], w.shape[0]), dtype=x2.dtype, device=x2.device) if act else None
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
        dev, kind = x2.device, x2.dtype
        dx = torch.empty((M, K), dtype=kind, device=dev) if need[0] else None
        dw = torch.empty((N, K), dtype=kind, device=dev) if need[1] else None
        dbias = torch.empty(N, dtype=kind, device=dev) if need[2] else None
        dtype = _DTYPES[kind]
        nbytes = _bwd_scratch(M, N, K, dtype, ctx.act, *need[:3])
        buf = _buffer(nbytes, dev)
        a = _lib.LINEAR_BWD_ARGS.pack(x2.data_ptr(), w.data_ptr(), _lib.ptr(pre), dy.data_ptr(), _lib.ptr(dx),
                                      _lib.ptr(dw), _lib.ptr(dbias), _lib.ptr(buf), nbytes, M, N, K, x2.stride(0),
                                      dy.stride(0), dtype, ctx.act)
        _lib.raw_call(_lib.load(), "gs_linear_bwd", a, dev)
        return dx, dw, dbias, dres, None


def _rows(t: torch.Tensor) -> torch.Tensor:
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
    given = [("x", x), ("weight", weight)]
    if bias is not None:
        given.append(("bias", bias))
    if residual is not None:
        given.append(("residual", residual))
    for k, t in given:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{who}: {k} must be a CUDA (HIP) tensor; got "
                             f"{t.device if isinstance(t, torch.Tensor) else type(t).__name__}")
        if t.get_device() != x.get_device():
            raise ValueError(f"{who}: all tensors must be on {x.device}; {k} is on {t.device}")
        if t.dtype != x.dtype or t.dtype not in _DTYPES:
            raise ValueError(f"{who}: all tensors must be float32 or all bfloat16; {k} is {t.dtype}, x {x.dtype}")
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
    x2, w = _rows(x), weight.contiguous()
    bias = bias.contiguous() if bias is not None else None
    res2 = _rows(residual) if residual is not None else None
    if torch.is_grad_enabled() and any([t.requires_grad for _, t in given]):
        y = LinearActFunction.apply(x2, w, bias, res2, act)
    else:
        y = _forward(x2, w, bias, res2, act, None)
    return cast(torch.Tensor, y.view(shape))
