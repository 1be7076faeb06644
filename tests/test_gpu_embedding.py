"""The embedding and its gradient against the definition in 64 bits (sequence_plain)."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _check(tokens, w, dout, scale, most):
    w = w.detach().requires_grad_(True)
    out = G.embedding(tokens, w, scale=scale)
    dw, = torch.autograd.grad(out, w, dout)
    want, size = P.embedding(tokens, w, scale, dout), P.embedding(tokens, w, scale, dout, size=True)
    P.assert_within(out, want[0], want[0].abs().nan_to_num(), 2, "out")
    assert dw.dtype == w.dtype
    P.assert_within(dw, want[1], size[1], most + 2, "dw")
    again, = torch.autograd.grad(G.embedding(tokens, w, scale=scale), w, dout)
    assert torch.equal(dw, again)  # places in a list depend on timing, sums do not


# lists of none, one, up to 64 and more, chunks; rows aligned and not
@pytest.mark.parametrize("M,V", [(1, 1), (1, 50), (63, 1), (64, 1), (65, 1), (300, 7), (1000, 333), (5000, 3), (40000, 2)])
@pytest.mark.parametrize("K", [1, 33, 96, 520])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_forward_and_backward(dev, M, V, K, dtype):
    g = torch.Generator().manual_seed(M + V)
    # few tokens often, many seldom
    tokens = (V * torch.rand(M, generator=g) ** 3).long().clamp(max=V - 1).to(dev)
    w = torch.randn(V, K, generator=g).to(dtype).to(dev)
    dout = torch.randn(M, K, generator=g).to(dtype).to(dev)
    _check(tokens, w, dout, 1.5, M)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_padding_and_tokens_out_of_range(dev, kind):
    V, K = 9, 40
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(-2, V + 2, (4, 50), generator=g).to(kind).to(dev)
    tokens[0, :3] = torch.tensor([-(2 ** 31), 2 ** 31 - 1, V], device=dev).to(kind)
    if kind == torch.int64:
        tokens[1, 0], tokens[1, 1] = 2 ** 40 + 3, -(2 ** 40)
    w, dout = torch.randn(V, K, generator=g).to(dev), torch.randn(4, 50, K, generator=g).to(dev)
    dout[(tokens < 0) | (tokens >= V)] = float("nan")  # sends nothing
    _check(tokens, w, dout, 1.0, tokens.numel())


def test_no_token_counts(dev):
    w = torch.randn(5, 12, device=dev, requires_grad=True)
    tokens = torch.full((7,), -1, device=dev)
    out = G.embedding(tokens, w)
    dw, = torch.autograd.grad(out, w, torch.full((7, 12), float("inf"), device=dev))
    assert (out == 0).all() and (dw == 0).all()


def test_strides(dev):
    V, K = 20, 64
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, V, (30, 10), generator=g).to(dev)[:, ::2]
    w = torch.randn(V, K + 4, generator=g).to(dev)[:, 2:2 + K]
    wide = torch.randn(30, 5, K + 3, generator=g).to(dev)[..., 1:1 + K]
    _check(tokens, w, wide, 1.0, 150)
    _check(tokens, w, torch.ones((), device=dev).expand(30, 5, K), 1.0, 150)


def test_positions_past_a_window(dev):
    """A list over more positions than are ordered at a time (2^17), in chunks of more than 64."""
    M, K = 300_000, 8
    tokens = torch.zeros(M, dtype=torch.int32, device=dev)
    tokens[::3] = 1
    w = torch.zeros(2, K, device=dev)
    # whole numbers: sums are exact in any order
    dout = torch.randint(-3, 4, (M, K), generator=torch.Generator().manual_seed(2)).float().to(dev)
    w.requires_grad_(True)
    dw, = torch.autograd.grad(G.embedding(tokens, w), w, dout)
    assert torch.equal(dw.cpu(), P.embedding(tokens, w, 1.0, dout)[1].float())


def test_differences(dev):
    V, K, M = 6, 5, 20
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(-1, V, (M,), generator=g).to(dev)
    w, dout, d = (torch.randn(n, K, generator=g) for n in (V, M, V))
    leaf = w.to(dev).requires_grad_(True)
    dw, = torch.autograd.grad(G.embedding(tokens, leaf, scale=0.7), leaf, dout.to(dev))
    f = [(P.embedding(tokens, w.double() + s * d.double(), 0.7) * dout).sum() for s in (1, -1)]
    assert abs((dw.cpu() * d).sum() - (f[0] - f[1]) / 2) < 1e-4  # linear in w: the difference is exact
