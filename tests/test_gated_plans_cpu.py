"""Which layout the gated linear scan takes at sizes that no test runs, as its size queries and
refusals tell: chained layouts alone need scratch (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest

from gru_qat_amd import _lib

FAKE = 4096  # never dereferenced


def _args(back, T, B, H, dtype):
    kw = dict(gi=FAKE, out=FAKE, T=T, B=B, H=H, sg_t=2 * H * B, sg_b=2 * H, so_t=H * B, so_b=H, dtype=dtype)
    if not back:
        return _lib.GsGlrArgs(**kw)
    return _lib.GsGlrBwdArgs(dout=FAKE, dgi=FAKE, sd_t=H * B, sd_b=H, sdg_t=2 * H * B, sdg_b=2 * H, **kw)


def _scratch(back, *sizes):
    a = _args(back, *sizes)
    return getattr(_lib.load(), "gs_glr_bwd_scratch_bytes" if back else "gs_glr_scratch_bytes")(ctypes.byref(a))


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("dtype", [0, 1])
def test_axes_past_a_launch_are_not_chained(back, dtype):
    """Chained, 8 workgroups of 512 threads take 256 steps of up to 8 x 16 channels."""
    assert _scratch(back, 2 ** 28 - 256, 1, 16, dtype) > 0
    for T in (2 ** 28, 2 ** 29 + 7, 2 ** 30):
        assert _scratch(back, T, 1, 16, dtype) == 0


@pytest.mark.parametrize("back", [False, True])
def test_more_workgroups_than_a_launch_holds(back):
    """Refused with nothing launched: the pointers are no memory."""
    lib = _lib.load()
    a = _args(back, 3, 2 ** 24, 2 ** 20, 0)
    assert getattr(lib, "gs_glr_bwd" if back else "gs_glr_fwd")(ctypes.byref(a), None) == _lib.GS_ERR_INVALID
    assert b"T=3, B=16777216, H=1048576" in lib.gs_last_error()
