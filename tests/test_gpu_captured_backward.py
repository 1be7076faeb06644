"""A backward captured while an eager graph of the same leaves is alive is an error, and the same capture
without one works."""

from __future__ import annotations

import gc

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu


def _conv(dev):
    x, w = torch.randn(20, 2, 12, device=dev, requires_grad=True), torch.randn(12, 4, device=dev, requires_grad=True)
    return (x, w), lambda: G.causal_conv(x, w)[0]


def _scan(dev):
    t = [torch.randn(s, device=dev, requires_grad=True) for s in ((40, 2, 33), (40, 2, 33), (40, 2, 5), (40, 2, 5))]
    A = (-torch.rand(33, 5, device=dev)).requires_grad_(True)
    return (*t, A), lambda: G.selective_scan(t[0], t[1], A, t[2], t[3])[0]


def _embedding(dev):
    tokens, w = torch.randint(0, 30, (50,), device=dev), torch.randn(30, 8, device=dev, requires_grad=True)
    return (w,), lambda: G.embedding(tokens, w)


def _logprobs(dev):
    tokens, x = torch.randint(0, 30, (50,), device=dev), torch.randn(50, 30, device=dev, requires_grad=True)
    return (x,), lambda: G.token_logprobs(x, tokens)[0]


def _linear(dev):
    x, w = torch.randn(20, 12, device=dev, requires_grad=True), torch.randn(16, 12, device=dev, requires_grad=True)
    return (x, w), lambda: G.linear_act(x, w, activation="silu")


@pytest.mark.parametrize("make", [_conv, _scan, _embedding, _logprobs, _linear])
def test_an_eager_graph_alive(dev, make):
    leaves, call = make(dev)
    y = call()
    want = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
    dy = torch.ones_like(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(call(), leaves, dy)
    del y
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaves, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), k
