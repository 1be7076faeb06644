"""A captured backward: a leaf whose eager graph is alive is refused also behind views, casts and other operators,
before anything is launched; one for which no gradient is asked does not matter."""

from __future__ import annotations

import gc

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu


def _r(*shape):
    return torch.randn(*shape, device="cuda", requires_grad=True)


def _conv():
    x, w = _r(2, 20, 12), _r(12, 4)
    return (x,), (w,), lambda: G.causal_conv(x, w, batch_first=True)[0]


def _scan():
    u, d, b, c = _r(40, 2, 33), _r(40, 2, 33), _r(40, 2, 5), _r(40, 2, 5)
    a = _r(33, 5)
    return (a,), (u, d, b, c), lambda: G.selective_scan(u, d, -torch.exp(a), b, c)[0]


def _embedding():
    tokens, w = torch.randint(0, 30, (50,), device="cuda"), _r(30, 8)
    return (w,), (), lambda: G.embedding(tokens, w.to(torch.bfloat16)).float()


def _logprobs():
    tokens, x = torch.randint(0, 30, (5, 10), device="cuda"), _r(5, 10, 30)
    return (x,), (), lambda: G.token_logprobs(x, tokens)[0]


def _linear():
    x, w = _r(4, 5, 12), _r(12, 16)
    return (w, x), (), lambda: G.linear_act(x, w.t(), activation="silu")


def _gated():
    gi, h0 = _r(2, 20, 24), _r(2, 12)
    return (gi,), (h0,), lambda: G.gated_linear_scan(gi, h0, batch_first=True)[0]


MAKE = [_conv, _scan, _embedding, _logprobs, _linear, _gated]


def _eager(call, leaves):
    y = call()
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dy)
    del y
    gc.collect()
    torch.cuda.synchronize()
    return dy, want


def _replays(graph, got, want):
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("make", MAKE)
def test_a_leaf_behind_another_node(dev, make):
    """Its accumulator is not next to the operator's node."""
    behind, beside, call = make()
    leaves = behind + beside
    dy, want = _eager(call, leaves)
    alive = [x * 2 for x in behind]  # the leaf's accumulator, made on the default stream, lives with these
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(call(), behind, dy)
    del alive
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaves, dy)
    _replays(graph, got, want)


@pytest.mark.parametrize("make", [m for m in MAKE if m not in (_embedding, _logprobs)])
def test_a_leaf_that_is_not_asked_for(dev, make):
    behind, beside, call = make()
    asked, other = (behind[:1], behind[1:]) if not beside else (behind, beside)
    dy, want = _eager(call, asked)
    alive = [x * 2 for x in other]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), asked, dy)
    _replays(graph, got, want)
    del alive


def test_a_graph_made_before(dev):
    x, w = _r(5, 12), _r(16, 12)
    before = x * 2
    G.linear_act(before, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="made on the default stream"):
        with torch.cuda.graph(graph):
            y = G.linear_act(before, w)
            torch.autograd.grad(y, w, torch.ones_like(y), retain_graph=True)  # w alone is fine
            torch.autograd.grad(y, x, torch.ones_like(y))
