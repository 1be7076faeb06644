"""Gated linear recurrence: the GRU update without a hidden map, so that a sequence
is a scan over independent channels instead of T dependent matrix products.

``z = sigmoid(gi_z)``, ``n = tanh(gi_n)`` (or ``gi_n``),
``h_t = z h_{t-1} + (1 - z) n`` with ``gi = [gi_z, gi_n]`` [T, B, 2H] from an input
projection. Activations are float32 or bfloat16; states and sums are float32. The
kernels are ``gs_glr_fwd``, ``gs_glr_bwd`` and ``gs_glr_step`` of libgruscan.so. No
counterpart in the reference.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_ACTIVATIONS = {"identity": _lib.ACT_NONE, "tanh": _lib.ACT_TANH}
_SCRATCH: dict = {}  # scratch bytes per size query, sizes and strides
_F32 = torch.float32


def _activation(who: str, activation: str) -> int:
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"{who}: activation must be 'tanh' or 'identity'; got {activation!r}") from None


def _ready(gi: torch.Tensor, a: Optional[torch.Tensor], b: Optional[torch.Tensor]) -> bool:
    """Whether gi is of a supported type and all are on its GPU: the common case, in few calls. The
    callers run _require where not, for its messages."""
    try:
        d = gi.get_device()
        return (d >= 0 and gi.dtype in _DTYPES and (a is None or a.get_device() == d)
                and (b is None or b.get_device() == d))
    except AttributeError:
        return False


def _require(who: str, ref: torch.Tensor, **tensors: Any) -> None:
    """Every tensor on ref's GPU."""
    for k, t in dict(gi=ref, **tensors).items():
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{who}: {k} must be a CUDA (HIP) tensor; got "
                             f"{t.device if isinstance(t, torch.Tensor) else type(t).__name__}")
        if t.get_device() != ref.get_device():
            raise ValueError(f"{who}: all tensors must be on {ref.device}; {k} is on {t.device}")
    if ref.dtype not in _DTYPES:
        raise ValueError(f"{who}: gi dtype must be float32 or bfloat16; got {ref.dtype}")


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _scratch(query: str, pack: Any, pointers: int, sizes: tuple, device: torch.device) -> Tuple[Any, int, int]:
    """The scratch tensor (None when none is needed), its address and its bytes, by the sizes alone."""
    need = _SCRATCH.get((query, sizes))
    if need is None:
        if len(_SCRATCH) > 4096:
            _SCRATCH.clear()
        need = _SCRATCH[query, sizes] = _lib.raw_size(_lib.load(), query, pack(*[0] * pointers, 0, 0, *sizes))
    if need == 0:
        return None, 0, 0
    t = torch.empty(need, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), need


def _forward(gi: torch.Tensor, h0: Optional[torch.Tensor], reset: Optional[torch.Tensor], act: int,
             batch_first: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """gi [T, B, 2H] with unit last stride, already checked; out as [T, B, H] (batch rows outermost in
    memory when batch_first) and h_T [B, H] in float32."""
    T, B, H = gi.shape
    H //= 2
    dtype = gi.dtype
    if batch_first:
        out = gi.new_empty((B, T, H)).transpose(0, 1)
    else:
        out = gi.new_empty((T, B, H))
    h_last = gi.new_empty((B, H)) if dtype is _F32 else gi.new_empty((B, H), dtype=_F32)
    sr = reset.stride() if reset is not None else (0, 0)
    sizes = (T, B, H, *gi.stride()[:2], h0.stride(0) if h0 is not None else 0, *sr, *out.stride()[:2], _DTYPES[dtype], act)
    keep, scratch, nbytes = _scratch("gs_glr_scratch_bytes", _lib.GLR_ARGS.pack, 5, sizes, gi.device)
    _lib.call_on("gs_glr_fwd", _lib.GLR_ARGS.pack(
        gi.data_ptr(), 0 if h0 is None else h0.data_ptr(), 0 if reset is None else reset.data_ptr(), out.data_ptr(),
        h_last.data_ptr(), scratch, nbytes, *sizes), gi.get_device())
    return out, h_last  # the caching allocator keeps the scratch until the stream's work is done


class GatedLinearScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, gi, h0, reset, act, batch_first):  # type: ignore[override]
        out, h_last = _forward(gi, h0, reset, act, batch_first)
        ctx.save_for_backward(gi, h0, reset, out)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return out, h_last

    @staticmethod
    def backward(ctx: Any, dout, dh_last):  # type: ignore[override]
        gi, h0, reset, out = ctx.saved_tensors
        T, B, H = out.shape
        if dout is None:
            if dh_last is None:
                return None, None, None, None, None
            dout = out.new_zeros(H).expand(T, B, H)
        elif dout.stride(2) != 1 and H > 1:
            dout = dout.contiguous()
        if dh_last is not None and not dh_last.is_contiguous():
            dh_last = dh_last.contiguous()
        so = out.stride()
        dgi = gi.new_empty((T, B, 2 * H)) if so[0] >= so[1] else gi.new_empty((B, T, 2 * H)).transpose(0, 1)
        dh0 = out.new_empty((B, H), dtype=_F32) if ctx.needs_input_grad[1] else None
        sr = reset.stride() if reset is not None else (0, 0)
        sizes = (T, B, H, *gi.stride()[:2], h0.stride(0) if h0 is not None else 0, *sr, so[0], so[1], *dout.stride()[:2],
                 *dgi.stride()[:2], _DTYPES[gi.dtype], ctx.act)
        keep, scratch, nbytes = _scratch("gs_glr_bwd_scratch_bytes", _lib.GLR_BWD_ARGS.pack, 8, sizes, gi.device)
        _lib.call_on("gs_glr_bwd", _lib.GLR_BWD_ARGS.pack(
            gi.data_ptr(), _lib.ptr(h0), _lib.ptr(reset), out.data_ptr(), dout.data_ptr(), _lib.ptr(dh_last),
            dgi.data_ptr(), _lib.ptr(dh0), scratch, nbytes, *sizes), gi.get_device())
        return dgi, dh0, None, None, None


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
    taken as zero, whatever it is. Differentiable in gi and h0."""
    who = "gated_linear_scan"
    act = _activation(who, activation)
    if not _ready(gi, h0, reset):
        _require(who, gi, **{k: t for k, t in (("h0", h0), ("reset", reset)) if t is not None})
    if gi.dim() != 3 or gi.shape[2] % 2 or gi.shape[2] == 0:
        raise ValueError(f"{who}: gi must be [T, B, 2H] with H > 0; got shape {tuple(gi.shape)}")
    if batch_first:
        gi = gi.transpose(0, 1)
        reset = reset.transpose(0, 1) if reset is not None and reset.dim() == 2 else reset
    T, B, H2 = gi.shape
    if T == 0:
        raise ValueError(f"seq length T must be > 0; got T={T}")
    if B == 0:
        raise ValueError(f"batch size B must be > 0; got B={B}")
    if h0 is not None:
        if h0.shape != (B, H2 // 2) or h0.dtype != torch.float32:
            raise ValueError(f"h0 must be float32 of shape (B, H)=({B}, {H2 // 2}); got {h0.dtype} "
                             f"{tuple(h0.shape)}")
        h0 = _unit(h0)
    if reset is not None and (reset.shape != (T, B) or reset.dtype != torch.bool):
        raise ValueError(f"{who}: reset must be bool with one flag a step and row; got {reset.dtype} "
                         f"{tuple(reset.shape)}")
    gi = _unit(gi)
    if torch.is_grad_enabled() and (gi.requires_grad or (h0 is not None and h0.requires_grad)):
        out, h_last = GatedLinearScanFunction.apply(gi, h0, reset, act, batch_first)
    else:
        out, h_last = _forward(gi, h0, reset, act, batch_first)
    return (out.transpose(0, 1) if batch_first else out), h_last


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
    who = "gated_linear_step"
    act = _activation(who, activation)
    if not _ready(gi, state, slots):
        _require(who, gi, state=state, **({} if slots is None else {"slots": slots}))
    if gi.dim() != 2 or gi.shape[1] % 2 or gi.shape[1] == 0 or gi.shape[0] == 0:
        raise ValueError(f"{who}: gi must be [B, 2H] with B, H > 0; got shape {tuple(gi.shape)}")
    B, H = gi.shape[0], gi.shape[1] // 2
    if state.dim() != 2 or state.shape[1] != H or state.dtype != torch.float32 or state.shape[0] == 0:
        raise ValueError(f"{who}: state must be float32 [S, H] with H={H}; got {state.dtype} {tuple(state.shape)}")
    if state.stride(1) != 1 and H > 1:
        raise ValueError(f"{who}: state is updated in place and must have unit stride along H; got strides "
                         f"{state.stride()}")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError(f"{who}: {state.shape[0]} states for B={B} rows")
    elif slots.shape != (B,) or slots.dtype != torch.int32:
        raise ValueError(f"{who}: slots must be int32 [B]=[{B}]; got {slots.dtype} {tuple(slots.shape)}")
    else:
        slots = slots.contiguous()
    gi = _unit(gi)
    out = gi.new_empty((B, H))
    _lib.call_on("gs_glr_step", _lib.GLR_STEP_ARGS.pack(
        gi.data_ptr(), state.data_ptr(), 0 if slots is None else slots.data_ptr(), out.data_ptr(), B, H, state.shape[0],
        gi.stride(0), state.stride(0), H, _DTYPES[gi.dtype], act), gi.get_device())
    return out
