"""The operators over sequences where sums are long, with the roundings of each result counted by itself: a result in
float32 that is rounded to bfloat16 on its way does not pass."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P
from test_gpu_selective_scan import _make, _run
from test_gpu_selective_scan_edges import check, roundings

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# rows, channels and steps enough for waves that share nothing, and states over the waves of a workgroup
@pytest.mark.parametrize("T,B,H,N", [(610, 60, 130, 3), (1100, 40, 65, 16), (2100, 12, 130, 5), (1060, 40, 70, 20), (700, 3, 130, 16),
                                     (300, 2, 64, 32)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_scan(dev, T, B, H, N, dtype):
    t, dy, dh = _make(T, B, H, N, dtype, dev, seed=50, reset=0.003)
    check(t, dy, dh)


def test_a_coarser_result_does_not_pass():
    """On the CPU, with the definition itself rounded to bfloat16 in the place of the kernel's result."""
    T, B, H, N = 200, 2, 20, 4
    t, dy, dh = _make(T, B, H, N, F32, "cpu", seed=51)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    kw = dict(delta_bias=t["delta_bias"], dy=dy, dh=dh)
    want, size = P.selective_scan(*args, **kw), P.selective_scan(*args, size=True, **kw)
    most = roundings(T, B, H, N)
    for k, w, s in [("y", want[0], size[0]), ("h_T", want[1], size[1])] + [(k, want[2][k], size[2][k]) for k in want[2]]:
        P.assert_within(w.float(), w, s, most[k], k)
        with pytest.raises(AssertionError):
            P.assert_within(w.to(BF16).float(), w, s, most[k], k)


@pytest.mark.parametrize("V", [30001, 32000])
def test_logprobs_of_many_elements(dev, V):
    """More than 2^31 logits, of which the last rows are looked at: the gradient is measured by the probabilities themselves."""
    M = (1 << 31) // V + 40
    x = torch.zeros(M, V, device=dev, dtype=BF16)
    x[-5:] = torch.randn(5, V, generator=torch.Generator().manual_seed(52)).to(dev)
    tokens = torch.arange(M, device=dev) % V
    leaf = x.requires_grad_(True)
    lp = G.token_logprobs(leaf, tokens)[0]
    dx, = torch.autograd.grad(lp, leaf, torch.ones_like(lp))
    logits, last = x.detach()[-5:], tokens[-5:]
    want = P.token_logprobs(logits, last, 0, torch.ones(5))
    hot = torch.nn.functional.one_hot(last.cpu(), V)
    # a sum of V terms in chains of V / 256 or fewer; log probabilities of 16 or less are off by 3 of that, as is the
    # argument of exp; exp and the sums 8
    roundings = V // 64 + 3 * 16 + 64
    P.assert_within(lp[-5:], want[0], 16 * torch.ones(5), V // 64 + 64, "logprobs")
    P.assert_within(dx[-5:], want[4], torch.softmax(logits.double().cpu(), -1) + hot, roundings, "dx")
    # every other row is uniform
    p = -dx.detach()[:3].float() + torch.nn.functional.one_hot(tokens[:3], V)
    assert torch.allclose(p[:, 5:], torch.full((), 1 / V, device=dev), rtol=2.0 ** -8)
