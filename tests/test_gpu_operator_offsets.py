"""The gated scan, the linear operator and AdamW where offsets pass 32 bits: rows far apart,
and tensors of more than 2^31 elements. Bounds are those of each operator's own tests."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import test_gpu_gated_linear as scan
import test_gpu_linear as linear

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def _far(values, strides):
    """`values` in a buffer with these strides (only its own elements are ever written)."""
    span = 1 + sum((n - 1) * s for n, s in zip(values.shape, strides))
    view = torch.empty(span, device="cuda", dtype=values.dtype).as_strided(values.shape, strides)
    return view.copy_(values)


# steps 1 GiB apart; rows of the batch; a chained axis of which each step is 16 MiB on
@pytest.mark.parametrize("case", [((12, 2, 33), lambda n: (1 << 28, n, 1)), ((9, 3, 34), lambda n: (n, 1 << 30, 1)),
                                  ((600, 1, 40), lambda n: (1 << 22, n, 1))], ids=["steps", "rows", "chained"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_scan_of_far_rows(dev, case, dtype):
    (T, B, H), strides = case
    gi, h0, reset, dout, dh = scan._inputs(T, B, H, dtype, seed=21, p_reset=0.02)
    scan._check(dev, _far(gi.to(dev), strides(2 * H)), h0, reset, dout, dh, "tanh")


@pytest.mark.parametrize("M", [20, 70])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_of_far_rows(dev, M, dtype):
    x, w, bias, res, dy = linear._inputs(dev, M, 72, 40, dtype, seed=22)
    far = _far(x, (1 << 26, 1))
    linear._check(far, w, bias, res, dy, "gelu", linear._call(far, w, bias, res, dy, "gelu"))


def test_linear_of_many_elements(dev):
    """y, pre, dy and dpre of more than 2^32 bytes: the last rows, and dw from rows that are mostly zero."""
    M, N, K = (1 << 17) + 5, (1 << 14) + 8, 8
    x, w, bias, _, _ = linear._inputs(dev, M, N, K, torch.bfloat16, seed=23, res=False)
    dy = torch.zeros(M, N, device=dev, dtype=torch.bfloat16)
    dy[-70:] = torch.randn(70, N, generator=torch.Generator().manual_seed(24)).to(dev)
    y, dx, dw, db = linear._call(x, w, bias, None, dy, "silu")
    linear._check(x[-70:], w, bias, None, dy[-70:], "silu", (y[-70:], dx[-70:], dw, db))
    assert not dx[:-70].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_many_elements(dev, bits):
    """The end of a tensor of more than 2^31 elements equals that end alone."""
    first, tail = 1 << 31, 700
    g = torch.Generator().manual_seed(25)

    def new(n):
        s = dict(p=torch.zeros(n, device=dev, dtype=torch.bfloat16), g=torch.zeros(n, device=dev, dtype=torch.bfloat16),
                 m=torch.zeros(n, device=dev, dtype=torch.int8 if bits == 8 else torch.float32),
                 v=torch.zeros(n, device=dev, dtype=torch.uint8 if bits == 8 else torch.float32))
        if bits == 8:
            s.update(a=torch.zeros(-(-n // 256), device=dev), b=torch.zeros(-(-n // 256), device=dev))
        return s

    def step(s):
        scales = dict(exp_avg_scales=[s["a"]], exp_avg_sq_scales=[s["b"]]) if bits == 8 else {}
        for t in (1, 2):
            G.adamw_step([s["p"]], [s["g"]], [s["m"]], [s["v"]], step=t, lr=0.01, **scales)

    large, small = new(first + tail), new(tail)
    for k in ("p", "g"):
        small[k].copy_(torch.randn(tail, generator=g))
        large[k][first:] = small[k]
    step(large)
    step(small)
    for k in small:
        assert torch.equal(large[k][-small[k].numel():], small[k]), k
    assert not large["p"][:first].any()
