"""A chained gated linear scan whose bounded wait runs out is never silent.

The condition is forced from the host: a negative poll limit leaves the workgroups of the
axis' first tile out, so that the others wait for them in vain, run out of a small bound
through the kernel's own bounded wait and exit normally. What the first tile would have
written is untouched, everything after it is NaN, the fault mirror is set, and the next
scan on the device raises."""

from __future__ import annotations

import ctypes

import pytest
import torch

import gru_qat_amd as G
from gru_qat_amd import _lib
import test_gpu_gated_linear as scan

pytestmark = pytest.mark.gpu

LATE = -300  # polls
TILE = {40: 256, 70: 128}  # steps of a tile by H: 16 lanes, and 32 where there are more channels


def _call(dev, T, B, H, limit, mirror, back, size=4):
    """gs_glr_fwd or gs_glr_bwd through the C ABI: (oracle's arrays, the launch's)."""
    gi, h0, _, dout, dh = scan._inputs(T, B, H, torch.float32 if size == 4 else torch.bfloat16, seed=T)
    want = scan._oracle(gi, h0, None, "tanh", dout, dh)
    gi, h0, dout, dh = (t.to(dev) for t in (gi, h0, dout, dh))
    out, last = G.gated_linear_scan(gi, h0)
    kw = dict(gi=gi.data_ptr(), h0=h0.data_ptr(), T=T, B=B, H=H, sg_t=2 * B * H, sg_b=2 * H, sh0_b=H, so_t=B * H, so_b=H,
              dtype=0 if size == 4 else 1, activation=_lib.ACT_TANH, fault_mirror=mirror.data_ptr(), poll_limit=limit)
    if back:
        dgi, dh0 = torch.zeros_like(gi), torch.zeros_like(h0)
        a = _lib.GsGlrBwdArgs(out=out.data_ptr(), dout=dout.data_ptr(), dh_last=dh.data_ptr(), dgi=dgi.data_ptr(),
                              dh0=dh0.data_ptr(), sd_t=B * H, sd_b=H, sdg_t=2 * B * H, sdg_b=2 * H, **kw)
        name, got = "gs_glr_bwd", (dgi, dh0)
    else:
        out, last = torch.zeros_like(out), torch.zeros_like(last)
        a = _lib.GsGlrArgs(out=out.data_ptr(), h_last=last.data_ptr(), **kw)
        name, got = "gs_glr_fwd", (out, last)
    lib = _lib.load()
    need = getattr(lib, "gs_glr_bwd_scratch_bytes" if back else "gs_glr_scratch_bytes")(ctypes.byref(a))
    assert need > 0, "these sizes are not chained"
    scratch = torch.empty(need, dtype=torch.uint8, device=dev)
    a.scratch, a.scratch_bytes = scratch.data_ptr(), need
    assert getattr(lib, name)(ctypes.byref(a), _lib.current_stream_handle(dev)) == _lib.GS_OK
    torch.cuda.synchronize(dev)
    return want, got


@pytest.mark.parametrize("shape", [(1300, 1, 40), (5000, 1, 40), (1200, 8, 70)], ids=str)
def test_forward_gives_up_with_nan_and_a_word(dev, shape):
    T, B, H = shape
    mirror = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    ((o, e), (hl, el), *_), (out, last) = _call(dev, T, B, H, LATE, mirror, back=False)
    first = TILE[H]
    assert (out[:first] == 0).all()
    assert out[first:].isnan().all() and last.isnan().all() and mirror.item() != 0
    mirror.zero_()
    _, (out, last) = _call(dev, T, B, H, 0, mirror, back=False)
    scan._near(out, o, e, "out")
    scan._near(last, hl, el, "h_T")
    assert mirror.item() == 0


@pytest.mark.parametrize("shape", [(1300, 1, 40), (5000, 1, 40), (1200, 8, 70)], ids=str)
def test_backward_gives_up_with_nan_and_a_word(dev, shape):
    T, B, H = shape
    mirror = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    (_, _, (dg, e), (d0, e0), *_), (dgi, dh0) = _call(dev, T, B, H, LATE, mirror, back=True)
    first = TILE[H]  # from the end
    assert (dgi[-first:] == 0).all()
    assert dgi[:-first].isnan().all() and dh0.isnan().all() and mirror.item() != 0
    mirror.zero_()
    _, (dgi, dh0) = _call(dev, T, B, H, 0, mirror, back=True)
    scan._near(dgi, dg, e + 1e-38, "dgi")
    scan._near(dh0, d0, e0 + 1e-38, "dh0")
    assert mirror.item() == 0


def test_no_mirror_is_no_word(dev):
    class _None:
        def data_ptr(self):
            return 0

    _, (out, _) = _call(dev, 1300, 1, 40, LATE, _None(), back=False)
    assert out[256:].isnan().all()


def test_python_calls_raise_after_a_fault(dev):
    """The word that the kernels of the Python calls get: set, it makes the next scan raise, once."""
    gi = torch.randn(1300, 1, 80, device=dev, requires_grad=True)
    short = torch.randn(4, 1, 80, device=dev)
    want = G.gated_linear_scan(gi)[0]
    word = ctypes.c_int32.from_address(_lib.scan_fault_word(dev.index or 0))
    assert word.value == 0 and G.workspace_faults(dev) == 0
    for call in (lambda: G.gated_linear_scan(gi), lambda: G.gated_linear_scan(short), lambda: G.check_faults(dev)):
        word.value = 3
        with pytest.raises(G.PersistentScanFault, match="fault value 3"):
            call()
        assert word.value == 0
    word.value = 5
    assert G.workspace_faults(dev) == 1 and G.workspace_faults(dev) == 0
    out, _ = G.gated_linear_scan(gi)
    assert torch.equal(out, want)
    torch.autograd.grad(out.sum(), gi)
    G.check_faults(dev)
