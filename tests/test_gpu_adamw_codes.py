"""AdamW with moments in 8 bits: blocks that are not finite."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import test_gpu_adamw as adamw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 1e20])
def test_a_block_that_is_not_finite_is_nan_as_a_whole(dev, bad):
    """1e20 leaves the first moment finite and makes the second infinite."""
    s = adamw._make([700], 8, bits=8)
    s["grads"][0][300] = bad
    adamw._run(s, 2)
    m, v = (G.adamw_dequantize_state(s[k + "s"][0], s[k + "_scales"][0]).cpu() for k in ("exp_avg", "exp_avg_sq"))
    assert v[256:512].isnan().all() and v[:256].isfinite().all() and v[512:].isfinite().all()
    assert m[:256].isfinite().all() and m[512:].isfinite().all()
    assert m[256:512].isfinite().all() if bad == 1e20 else m[256:512].isnan().all()
