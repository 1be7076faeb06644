"""The operators over sequences of tokens where offsets pass 32 bits: rows far apart, and tensors of more than
2^31 elements. Bounds are those of each operator's own tests."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P
import test_gpu_causal_conv as conv
import test_gpu_selective_scan as scan
from test_gpu_operator_offsets import _far

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# steps 1 GiB apart; rows of the batch; an axis in chunks of which each step is 16 MiB on
@pytest.mark.parametrize("case", [((12, 2, 33), lambda n: (1 << 28, n, 1)), ((9, 3, 34), lambda n: (n, 1 << 30, 1)),
                                  ((600, 1, 40), lambda n: (1 << 22, n, 1))], ids=["steps", "rows", "chunks"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_far_rows(dev, case, dtype):
    (T, B, H), strides = case
    t, dy, dh = scan._make(T, B, H, 16, dtype, dev, seed=30, reset=0.02)
    for k in ("u", "B"):
        t[k] = _far(t[k], strides(t[k].shape[2]))
    scan._check(t, dy, dh, scan._roundings(T, B, H, 16))
    t, dy, dlast = conv._make(T, B, H, 4, dtype, dev, seed=31, reset=0.02)
    t["x"] = _far(t["x"], strides(H))
    conv._check(t, dy, dlast)


def test_conv_of_many_elements(dev):
    """x, y, dy and dx of more than 2^31 elements: the last rows equal a call of those alone."""
    T, B, C = 65, 16400, 2048
    g = torch.Generator().manual_seed(32)
    x = torch.zeros(T, B, C, device=dev, dtype=BF16)
    x[:, -3:] = torch.randn(T, 3, C, generator=g).to(dev)
    w = torch.randn(C, 4, generator=g).to(BF16).to(dev)
    dy = torch.zeros(T, B, C, device=dev, dtype=BF16)
    dy[:, -3:] = torch.randn(T, 3, C, generator=g).to(dev)
    leaf = x.requires_grad_(True)
    y, last = G.causal_conv(leaf, w)
    dx, = torch.autograd.grad(y, leaf, dy)
    small = x.detach()[:, -3:].contiguous().requires_grad_(True)
    y1, last1 = G.causal_conv(small, w)
    dx1, = torch.autograd.grad(y1, small, dy[:, -3:])
    assert torch.equal(y.detach()[:, -3:], y1) and torch.equal(last[-3:], last1) and torch.equal(dx[:, -3:], dx1)


def test_scan_of_many_elements(dev):
    T, B, H, N = 40, 26300, 2048, 1
    g = torch.Generator().manual_seed(33)
    u = torch.zeros(T, B, H, device=dev, dtype=BF16)
    u[:, -2:] = torch.randn(T, 2, H, generator=g).to(dev)
    bc = torch.randn(T, B, N, generator=g).to(BF16).to(dev)
    A = -torch.rand(H, N, generator=g).to(dev)
    y, h = G.selective_scan(u, u, A, bc, bc)
    y1, h1 = G.selective_scan(u[:, -2:], u[:, -2:], A, bc[:, -2:], bc[:, -2:])
    assert torch.allclose(y[:, -2:].float(), y1.float(), rtol=2.0 ** -7, atol=1e-5) and torch.allclose(h[-2:], h1, rtol=1e-5, atol=1e-6)


def test_embedding_of_many_elements(dev):
    V, K, M = (1 << 20) + 30, 2049, 3000
    w = torch.zeros(V, K, device=dev, dtype=BF16)
    w[-40:] = torch.randn(40, K, generator=torch.Generator().manual_seed(34)).to(dev)
    tokens = torch.randint(V - 40, V, (M,), generator=torch.Generator().manual_seed(35)).to(dev)
    dout = torch.randn(M, K, generator=torch.Generator().manual_seed(36)).to(BF16).to(dev)
    leaf = w.requires_grad_(True)
    out = G.embedding(tokens, leaf)
    dw, = torch.autograd.grad(out, leaf, dout)
    small = w.detach()[-40:].clone().requires_grad_(True)
    out1 = G.embedding(tokens - (V - 40), small)
    dw1, = torch.autograd.grad(out1, small, dout)
    assert torch.equal(out, out1) and torch.equal(dw[-40:], dw1) and not dw[:-40].any()


@pytest.mark.parametrize("V", [30001, 32000])
def test_logprobs_of_many_elements(dev, V):
    M = (1 << 31) // V + 40
    x = torch.zeros(M, V, device=dev, dtype=BF16)
    x[-5:] = torch.randn(5, V, generator=torch.Generator().manual_seed(37)).to(dev)
    tokens = torch.arange(M, device=dev) % V
    leaf = x.requires_grad_(True)
    lp, h, _, ids = G.token_logprobs(leaf, tokens, top=2)
    dx, = torch.autograd.grad(lp, leaf, torch.ones_like(lp))
    want = P.token_logprobs(x.detach()[-5:], tokens[-5:], 2, torch.ones(5))
    assert torch.equal(ids[-5:].cpu(), want[3])
    P.assert_within(lp[-5:], want[0], 8 * torch.ones(5), V // 64 + 64)
    P.assert_within(dx[-5:], want[4], 8 * torch.ones(5, V) / 100, V // 64 + 64)
    assert torch.allclose(lp[:-5], torch.full((), -float(torch.log(torch.tensor(float(V)))), device=dev), atol=1e-4)
