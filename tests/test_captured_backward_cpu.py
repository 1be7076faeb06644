"""Which leaves the check before a captured backward sees: those that the backward reaches and runs, through views,
casts and other operators, and no others. On the CPU, where nothing can be captured."""

from __future__ import annotations

import pytest
import torch

from gru_qat_amd import _lib


def _leaf(*shape):
    return torch.randn(*shape, requires_grad=True)


def _found(t):
    return {x.data_ptr() for x in _lib.ops()._reached_leaves(t)}


def _are(*leaves):
    return {x.data_ptr() for x in leaves}


@pytest.mark.parametrize("route", [
    lambda x: x * 1, lambda x: x.transpose(0, 1) * 1, lambda x: x.reshape(-1) + 0, lambda x: x.to(torch.bfloat16),
    lambda x: -torch.exp(x), lambda x: x[::2, 1:].contiguous(), lambda x: (x.view(-1)[3:].double() * 2).float().split(2)[0],
], ids=range(7))
def test_leaves_behind_other_nodes(route):
    x, w = _leaf(4, 6), _leaf(3)
    y = route(x).sum() * w.exp().sum()
    assert _found(y) == _are(x, w)


def test_one_leaf_on_many_ways():
    x = _leaf(5)
    y = x
    for _ in range(40):  # 2^40 ways back, 120 nodes
        y = y * 0.5 + y.sin()
    assert _found(y.sum()) == _are(x) and len(_lib.ops()._reached_leaves(y.sum())) == 1


def test_no_leaf():
    assert _found(torch.ones(3)) == set()
    assert _found(_leaf(3).detach()) == set()


@pytest.mark.parametrize("asked", [("x",), ("w",), ("x", "w"), ("mid",), None], ids=str)
def test_only_what_the_backward_runs(asked):
    """torch.autograd.grad runs the accumulators of the inputs that it is asked for, backward() all."""
    x, w = _leaf(4, 6), _leaf(6, 3)
    mid = (x.t() * 2).t()
    y = mid @ w.double().float()
    seen = []
    y.register_hook(lambda g: seen.append(_found(y)))
    if asked is None:
        y.sum().backward()
        want = _are(x, w)
    else:
        torch.autograd.grad(y.sum(), [dict(x=x, w=w, mid=mid)[k] for k in asked])
        want = _are(*[dict(x=x, w=w)[k] for k in asked if k != "mid"])
    assert seen == [want]


def test_backward_with_inputs():
    x, w = _leaf(4), _leaf(4)
    y = x.exp() * w
    seen = []
    y.register_hook(lambda g: seen.append(_found(y)))
    y.sum().backward(inputs=[w])
    assert seen == [_are(w)] and x.grad is None
