"""The gated linear recurrence, the linear operator and AdamW without a GPU: what the C ABI
refuses before any device work, its size queries, and the Python entry points' errors on
CPU tensors and non-tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

import gru_qat_amd as G
from gru_qat_amd import _lib

FAKE = 4096  # never dereferenced: validation fails before any device access


def _glr(**kw):
    a = _lib.GsGlrArgs(gi=FAKE, out=FAKE, T=4, B=3, H=8, sg_t=48, sg_b=16, so_t=24, so_b=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _glr_bwd(**kw):
    a = _lib.GsGlrBwdArgs(gi=FAKE, out=FAKE, dout=FAKE, dgi=FAKE, T=4, B=3, H=8, sg_t=48, sg_b=16, so_t=24, so_b=8,
                          sd_t=24, sd_b=8, sdg_t=48, sdg_b=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _step(**kw):
    a = _lib.GsGlrStepArgs(gi=FAKE, state=FAKE, out=FAKE, B=3, H=8, S=3, sg_b=16, ss=8, so_b=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _linear(**kw):
    a = _lib.GsLinearArgs(x=FAKE, w=FAKE, y=FAKE, M=4, N=3, K=8, sx=8, sr=3, sy=3)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _linear_bwd(**kw):
    a = _lib.GsLinearBwdArgs(x=FAKE, w=FAKE, dy=FAKE, dx=FAKE, dw=FAKE, dbias=FAKE, M=4, N=3, K=8, sx=8, sdy=3)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _adamw(tensor=None, **kw):
    t = _lib.GsAdamwTensor(param=FAKE, grad=FAKE, exp_avg=FAKE, exp_avg_sq=FAKE, n=4)
    for k, v in (tensor or {}).items():
        setattr(t, k, v)
    a = _lib.GsAdamwArgs(tensors=ctypes.pointer(t), count=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
                         step=1, state_bits=32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SIZES = [dict(T=0), dict(B=0), dict(H=0), dict(T=-1), dict(T=2 ** 31), dict(H=2 ** 21), dict(dtype=2), dict(dtype=-1)]
REFUSED = (
    [("gs_glr_fwd", _glr, kw) for kw in SIZES + [dict(gi=0), dict(out=0), dict(activation=2), dict(sg_t=-1), dict(so_t=7),
                                                 dict(so_b=7), dict(so_t=8), dict(sh0_b=-1), dict(sr_t=-1)]]
    + [("gs_glr_bwd", _glr_bwd, kw) for kw in SIZES + [dict(gi=0), dict(out=0), dict(dout=0), dict(dgi=0), dict(sd_b=-1),
                                                       dict(sdg_t=15), dict(sdg_b=15), dict(activation=5)]]
    + [("gs_glr_step", _step, kw) for kw in [dict(B=0), dict(H=0), dict(gi=0), dict(state=0), dict(out=0), dict(S=0),
                                             dict(S=2), dict(ss=7), dict(so_b=7), dict(B=70000, S=70000), dict(dtype=3)]]
    + [("gs_linear_fwd", _linear, kw) for kw in [dict(M=0), dict(N=0), dict(K=0), dict(N=2 ** 25), dict(x=0), dict(w=0),
                                                 dict(y=0), dict(sy=2), dict(sx=-1), dict(dtype=2), dict(activation=6),
                                                 dict(activation=-1)]]
    + [("gs_linear_bwd", _linear_bwd, kw) for kw in [dict(M=0), dict(dy=0), dict(x=0), dict(w=0), dict(activation=1),
                                                     dict(sdy=-1), dict(dtype=9)]]
    + [("gs_adamw_step", _adamw, kw) for kw in [dict(step=0), dict(lr=-1.0), dict(lr=float("nan")), dict(beta1=1.0),
                                                dict(beta2=-0.1), dict(eps=-1.0), dict(weight_decay=float("inf")),
                                                dict(state_bits=16), dict(param_dtype=2), dict(grad_dtype=-1), dict(count=-1),
                                                dict(has_master=1), dict(tensor=dict(param=0)), dict(tensor=dict(grad=0)),
                                                dict(tensor=dict(n=-1)), dict(state_bits=8),
                                                dict(param_dtype=1, has_master=1)]]
)


@pytest.mark.parametrize("fn,make,kw", REFUSED, ids=[f"{f}-{k}" for f, _, k in REFUSED])
def test_refused_before_any_device_work(fn, make, kw):
    lib = _lib.load()
    assert getattr(lib, fn)(ctypes.byref(make(**kw)), None) == _lib.GS_ERR_INVALID
    assert fn.encode() in lib.gs_last_error() or b"must be > 0" in lib.gs_last_error()


@pytest.mark.parametrize("fn", ["gs_glr_fwd", "gs_glr_bwd", "gs_glr_step", "gs_linear_fwd", "gs_linear_bwd",
                                "gs_adamw_step"])
def test_null_arguments(fn):
    assert getattr(_lib.load(), fn)(None, None) == _lib.GS_ERR_INVALID


def test_missing_scratch():
    lib = _lib.load()
    for fn, query, a in (
        ("gs_glr_fwd", "gs_glr_scratch_bytes", _glr(T=5000, sg_t=48, so_t=24)),
        ("gs_glr_bwd", "gs_glr_bwd_scratch_bytes", _glr_bwd(T=5000)),
        ("gs_linear_bwd", "gs_linear_bwd_scratch_bytes", _linear_bwd()),
    ):
        need = getattr(lib, query)(ctypes.byref(a))
        assert need > 0
        for scratch, nbytes in ((0, 0), (FAKE, 16), (FAKE + 8, need)):
            a.scratch, a.scratch_bytes = scratch, nbytes
            assert getattr(lib, fn)(ctypes.byref(a), None) == _lib.GS_ERR_INVALID
            assert b"scratch" in lib.gs_last_error()


def test_size_queries():
    lib = _lib.load()
    for query, make, kw in (("gs_glr_scratch_bytes", _glr, dict(T=0)), ("gs_glr_bwd_scratch_bytes", _glr_bwd, dict(H=0)),
                            ("gs_linear_scratch_bytes", _linear, dict(K=0)),
                            ("gs_linear_bwd_scratch_bytes", _linear_bwd, dict(N=0))):
        assert getattr(lib, query)(ctypes.byref(make(**kw))) == _lib.GS_ERR_INVALID
    assert lib.gs_glr_scratch_bytes(ctypes.byref(_glr())) == 0  # short axes need none
    # the most that any pointers may need covers what aligned ones do
    big = dict(dtype=_lib.DTYPE_BF16, M=8000, N=1001, K=1003, sx=1003, sy=1001, sr=0)
    assert lib.gs_linear_scratch_bytes(ctypes.byref(_linear(**big, x=0))) >= lib.gs_linear_scratch_bytes(ctypes.byref(_linear(**big))) > 0


def test_dequantize_refusals():
    lib = _lib.load()
    assert lib.gs_adamw_dequantize(None, None, None, -1, 0, None) == _lib.GS_ERR_INVALID
    assert lib.gs_adamw_dequantize(None, None, None, 4, 0, None) == _lib.GS_ERR_INVALID
    assert lib.gs_adamw_dequantize(None, None, None, 0, 0, None) == _lib.GS_OK


@pytest.mark.parametrize("call", [
    lambda t: G.gated_linear_scan(t(4, 2, 6), t(2, 3)),
    lambda t: G.gated_linear_scan(None),
    lambda t: G.gated_linear_scan(t(4, 2, 6), 0.0),
    lambda t: G.gated_linear_scan(t(4, 2, 6), activation="relu"),
    lambda t: G.gated_linear_step(t(2, 6), t(2, 3)),
    lambda t: G.gated_linear_step([1.0], t(2, 3)),
    lambda t: G.linear_act(t(2, 3), t(4, 3)),
    lambda t: G.linear_act(t(2, 3), None),
    lambda t: G.linear_act(t(2, 3), t(4, 3), activation="swish"),
    lambda t: G.adamw_step([t(3)], [t(3)], [t(3)], [t(3)], step=1, lr=1e-3),
    lambda t: G.adamw_step(t(3), [t(3)], [t(3)], [t(3)], step=1, lr=1e-3),
    lambda t: G.adamw_step([None], [t(3)], [t(3)], [t(3)], step=1, lr=1e-3),
    lambda t: G.adamw_dequantize_state(t(3), t(1)),
    lambda t: G.AdamW([t(3)], state_bits=4),
    lambda t: G.GatedLinearLayer(0, 3),
], ids=range(15))
def test_python_refusals_without_a_gpu(call):
    with pytest.raises(ValueError):
        call(torch.zeros)


def test_no_tensors_is_no_step():
    G.adamw_step([], [], [], [], step=1, lr=1e-3)
