"""What a bfloat16 linear_act keeps of its activation's argument for the backward: enough for the slope
to be as exact as float32 sums leave it, at every size of the argument.

A half has 11 bits, so the slope's argument is off by at most 2^-11 of itself, and by 2^-24 where it is small;
act' moves by that times act'' and is computed within 16 u of 1 + |argument| (u = 2^-24). The bias gradient of one
row is dy act' rounded once, to bfloat16 (2^-8)."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import test_gpu_linear as linear

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _slopes(pre, act):
    """act' and act'' in float64"""
    p = pre.double().requires_grad_(True)
    f = dict(gelu=torch.nn.functional.gelu, silu=torch.nn.functional.silu, tanh=torch.tanh, sigmoid=torch.sigmoid)[act]
    first, = torch.autograd.grad(f(p).sum(), p, create_graph=True)
    second, = torch.autograd.grad(first.sum(), p)
    return first.detach(), second


# few rows of a small layer; a single row through tiles, and through tiles whose sums are split
@pytest.mark.parametrize("shape", [(1, 517, 33), (1, 520, 2100), (1, 40, 16000)], ids=str)
@pytest.mark.parametrize("act", ["gelu", "silu", "tanh", "sigmoid"])
def test_slopes_of_arguments_of_every_size(dev, act, shape):
    M, N, K = shape
    g = torch.Generator().manual_seed(K)
    x = torch.randn(M, K, generator=g).bfloat16().to(dev)
    w = (torch.randn(N, K, generator=g) * (4.0 * K ** -0.5)).bfloat16().to(dev)
    b, dy = (torch.randn(n, generator=g).bfloat16().to(dev) for n in ((N,), (M, N)))
    bias = b.clone().requires_grad_(True)
    db, = torch.autograd.grad(G.linear_act(x, w, bias, activation=act), bias, dy)
    pre = (x.double() @ w.double().t() + b.double())[0]
    e = 2 * (K + 2) * U * (x.double().abs() @ w.double().abs().t())[0] + 2 * U * b.double().abs()
    first, second = (t.to(dev) for t in _slopes(pre.cpu(), act))
    step = e + 2.0 ** -11 * pre.abs() + 2.0 ** -24
    slack = step * second.abs() + step.square() + 16 * U * (1 + pre.abs())  # act''' is under 2
    want = dy[0].double() * first
    assert ((db.double() - want).abs() <= dy[0].double().abs() * slack * 1.01 + 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("act,large,small", [("relu", 1, None), ("gelu", 1, 0.5), ("silu", 1, 0.5), ("tanh", 0, 1),
                                             ("sigmoid", 0, 0.25)])
def test_arguments_past_a_half(dev, act, large, small):
    """Past its range the slope is that at infinity, under it that at 0, and relu's goes by the sign."""
    x = torch.tensor([[1e30], [1e5], [-1e30], [-7e4], [1e-30], [1e-9], [-1e-30], [-1e-9], [0.0], [float("nan")]],
                     device=dev).bfloat16().requires_grad_(True)
    one = torch.ones(1, 1, device=dev, dtype=torch.bfloat16)
    y = G.linear_act(x, one, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    got = dx[:, 0].tolist()
    assert got[:2] == [large, large] and got[2:4] == [0, 0]
    assert got[4:9] == ([1, 1, 0, 0, 0] if act == "relu" else [small] * 5)
    assert got[9] != got[9] or act == "relu"
    assert y[9, 0].isnan()
