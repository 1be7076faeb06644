"""AdamW over many tensors in few launches, with moments in float32 or in 8 bits.

``adamw_step`` is the step on lists of tensors (``gs_adamw_step`` of libgruscan.so);
``AdamW`` is the optimizer around it. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import operator
import struct
from typing import Any, Callable, Iterable, List, Optional, Sequence, Tuple

import torch

from . import _lib

STATE_BLOCK = 256  # elements of a tensor that share a scale where moments are held in 8 bits

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_F32 = {torch.float32}
# over lists of tensors, in C: these calls are most of a small step's time
_NUMEL, _PTR, _ORDINAL, _CONTIGUOUS = (torch.Tensor.numel, torch.Tensor.data_ptr, torch.Tensor.get_device,
                                       torch.Tensor.is_contiguous)
_DTYPE = operator.attrgetter("dtype")
_ONLY = [{i} for i in range(64)]


def _blocks(n: int) -> int:
    return -(-n // STATE_BLOCK)


def _check_list(who: str, name: str, tensors: Sequence[torch.Tensor], counts: List[int], dtypes: set,
                device: int) -> None:
    """One contiguous tensor of counts[i] elements for each parameter, of one of the dtypes, on the device."""
    if len(tensors) != len(counts):
        raise ValueError(f"{who}: {len(tensors)} tensors in {name} for {len(counts)} parameters")
    if (list(map(_NUMEL, tensors)) == counts and dtypes.issuperset(map(_DTYPE, tensors))
            and _ONLY[device] == set(map(_ORDINAL, tensors)) and all(map(_CONTIGUOUS, tensors))):
        return
    for i, (t, n) in enumerate(zip(tensors, counts)):
        if t.get_device() != device:
            raise ValueError(f"{who}: every tensor must be on one CUDA (HIP) device; {name}[{i}] is on {t.device}")
        if t.dtype not in dtypes:
            raise ValueError(f"{who}: {name}[{i}] dtype must be {' or '.join(sorted(map(str, dtypes)))}; got {t.dtype}")
        if t.numel() != n:
            raise ValueError(f"{who}: {name}[{i}] must have {n} elements; got shape {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{who}: {name}[{i}] must be contiguous; got strides {t.stride()}")


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
) -> None:
    """One AdamW step in place, the ``step``-th (from 1), on contiguous tensors of one device.

    ``params`` are float32, or bfloat16 with float32 ``masters`` of which they are the
    rounding (without masters, updates under half a bfloat16 unit are lost); all of one
    type, and ``grads`` too. The moments are float32, or, with ``exp_avg_scales`` and
    ``exp_avg_sq_scales`` (float32, one number per 256 elements), int8 and uint8 codes (see
    ``adamw_dequantize_state``). ``grad_scale``: a float32 tensor of one element on the
    device that multiplies the gradients; where it is not finite the step does nothing."""
    who = "adamw_step"
    if not len(params):
        return
    if not isinstance(params[0], torch.Tensor) or not params[0].is_cuda:
        raise ValueError(f"{who}: params must be CUDA (HIP) tensors")
    dev = params[0].get_device()
    counts = list(map(_NUMEL, params))
    bits = 32 if exp_avg_scales is None else 8
    if (exp_avg_sq_scales is None) != (exp_avg_scales is None):
        raise ValueError(f"{who}: exp_avg_scales and exp_avg_sq_scales belong together")
    for name, ts in (("params", params), ("grads", grads)):
        if len(ts) and ts[0].dtype not in _DTYPES:
            raise ValueError(f"{who}: {name} must be float32 or bfloat16; got {ts[0].dtype}")
    _check_list(who, "params", params, counts, {params[0].dtype}, dev)
    if len(grads) == len(params) and not all(map(_CONTIGUOUS, grads)):
        grads = [g.contiguous() for g in grads]
    _check_list(who, "grads", grads, counts, {grads[0].dtype} if len(grads) else set(), dev)
    _check_list(who, "exp_avgs", exp_avgs, counts, _F32 if bits == 32 else {torch.int8}, dev)
    _check_list(who, "exp_avg_sqs", exp_avg_sqs, counts, _F32 if bits == 32 else {torch.uint8}, dev)
    if exp_avg_scales is not None and exp_avg_sq_scales is not None:
        blocks = [_blocks(n) for n in counts]
        _check_list(who, "exp_avg_scales", exp_avg_scales, blocks, _F32, dev)
        _check_list(who, "exp_avg_sq_scales", exp_avg_sq_scales, blocks, _F32, dev)
    if masters is not None:
        if params[0].dtype != torch.bfloat16:
            raise ValueError(f"{who}: masters belong to bfloat16 parameters; got {params[0].dtype}")
        _check_list(who, "masters", masters, counts, _F32, dev)
    if grad_scale is not None and (grad_scale.get_device() != dev or grad_scale.dtype != torch.float32
                                   or grad_scale.numel() != 1):
        raise ValueError(f"{who}: grad_scale must be one float32 number on the parameters' device; got "
                         f"{grad_scale.dtype} {tuple(grad_scale.shape)} on {grad_scale.device}")
    # one row of eight words a tensor (GsAdamwTensor), column by column
    words = [0] * (8 * len(counts))
    words[0::8], words[1::8], words[2::8], words[3::8], words[7::8] = (
        map(_PTR, params), map(_PTR, grads), map(_PTR, exp_avgs), map(_PTR, exp_avg_sqs), counts)
    if bits == 8:
        words[4::8], words[5::8] = map(_PTR, exp_avg_scales), map(_PTR, exp_avg_sq_scales)  # type: ignore[arg-type]
    if masters is not None:
        words[6::8] = map(_PTR, masters)
    table = struct.pack(f"<{len(words)}Q", *words)
    a = _lib.ADAMW_ARGS.pack(ctypes.cast(ctypes.c_char_p(table), ctypes.c_void_p).value, len(counts), lr, betas[0],
                             betas[1], eps, weight_decay, step, _lib.ptr(grad_scale), _DTYPES[params[0].dtype],
                             _DTYPES[grads[0].dtype], bits, masters is not None)
    _lib.call_on("gs_adamw_step", a, dev)  # `table` is read during the call


def adamw_dequantize_state(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float32 values of a moment held in 8 bits: int8 ``codes`` c stand for
    A sign(c) (c / 127)^2 (the first moment), uint8 ones for A (c / 255)^4 (the second),
    with A = ``scales`` [ceil(n / 256)], one for each 256 elements."""
    who = "adamw_dequantize_state"
    if codes.dtype not in (torch.int8, torch.uint8) or not codes.is_cuda or not codes.is_contiguous():
        raise ValueError(f"{who}: codes must be a contiguous int8 or uint8 CUDA (HIP) tensor; got {codes.dtype} on "
                         f"{codes.device}")
    n = codes.numel()
    _check_list(who, "scales", [scales], [_blocks(n)], _F32, codes.get_device())
    out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
    lib = _lib.load()
    with _lib.on_device(codes.device):
        rc = lib.gs_adamw_dequantize(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), n, codes.dtype is torch.uint8,
                                     _lib.current_stream_handle(codes.device))
    _lib.raise_for(rc, lib)
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is ``adamw_step``: one launch for up to 48 parameters.

    ``state_bits`` 32 keeps float32 moments, 8 keeps codes of 8 bits with a float32 scale
    per 256 elements (2 bytes an element instead of 8). bfloat16 parameters get float32
    masters unless ``master_weights`` is off. ``step(grad_scale=...)`` multiplies the
    gradients by a device scalar (a clipping factor, an inverse loss scale); where that is
    not finite, parameters and moments stay as they are (the count of steps still advances:
    the host does not read the scalar)."""

    def __init__(self, params: Iterable[Any], lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *, state_bits: int = 32,
                 master_weights: bool = True) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32; got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights))

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
                           masters=[s["master"] for s in states] if master else None, grad_scale=grad_scale, **scales)
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
