"""What the operators over sequences of tokens do not differentiate, may not write or do not take is
refused before anything is launched."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import gru_qat_amd as G

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
T, B, H, N, W, V = 5, 2, 6, 4, 3, 11

SCAN = dict(u=(T, B, H), delta=(T, B, H), A=(H, N), B=(T, B, N), C=(T, B, N), D=(H,), z=(T, B, H), h0=(B, H, N), delta_bias=(H,))
STEP = dict(u=(B, H), delta=(B, H), A=(H, N), B=(B, N), C=(B, N), D=(H,), z=(B, H), delta_bias=(H,), state=(B, H, N))
CONV = dict(x=(T, B, H), weight=(H, W), bias=(H,), state=(B, W - 1, H))
CONV_STEP = dict(x=(B, H), weight=(H, W), bias=(H,), state=(B, W - 1, H))
EMBED = dict(weight=(V, H))
PROBS = dict(logits=(T, V))


def _values(shapes, **kw):
    return {k: torch.rand(s, device="cuda") for k, s in shapes.items()} | kw


def _scan(**kw):
    return G.selective_scan(**_values(SCAN, **kw))


def _step(**kw):
    return G.selective_step(**_values(STEP, **kw))


def _conv(**kw):
    return G.causal_conv(**_values(CONV, **kw))


def _conv_step(**kw):
    return G.causal_conv_step(**_values(CONV_STEP, **kw))


def _embed(**kw):
    return G.embedding(**(dict(tokens=torch.zeros(3, dtype=torch.long, device="cuda")) | _values(EMBED, **kw)))


def _probs(**kw):
    return G.token_logprobs(**(dict(tokens=torch.zeros(T, dtype=torch.long, device="cuda")) | _values(PROBS, **kw)))


CALLS = [(f, k, s) for f, shapes in ((_scan, SCAN), (_step, STEP), (_conv, CONV), (_conv_step, CONV_STEP), (_embed, EMBED),
                                     (_probs, PROBS)) for k, s in shapes.items()]


@pytest.mark.parametrize("call,name,shape", CALLS, ids=[f"{f.__name__}-{k}" for f, k, _ in CALLS])
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_is_refused(dev, call, name, shape, needs_grad):
    value = torch.ones(shape, device=dev, requires_grad=needs_grad)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(value, torch.ones(shape, device=dev))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(**{name: dual})
    assert (value == 1).all()


@pytest.mark.parametrize("call,name,shape", CALLS, ids=[f"{f.__name__}-{k}" for f, k, _ in CALLS])
def test_wrong_tensors_are_refused(dev, call, name, shape):
    wrong = [torch.ones((*shape, 2), device=dev), torch.ones(shape), torch.ones(shape, device=dev, dtype=torch.float64)]
    if len(shape) > 1:
        wrong.append(torch.ones((0, *shape[1:]), device=dev))
    if name not in ("u", "x", "weight", "logits"):
        other = BF16  # the others are float32
        wrong.append(torch.ones(shape, device=dev, dtype=other))
        wrong.append(torch.ones((shape[0] + 1, *shape[1:]), device=dev) if name != "state" or call in (_scan, _conv) else
                     torch.ones((shape[0], shape[1] + 1, shape[2]), device=dev))
    for t in wrong:
        with pytest.raises(ValueError):
            call(**{name: t})


@pytest.mark.parametrize("call", [_scan, _conv])
def test_wrong_resets_are_refused(dev, call):
    for r in (torch.zeros(T, B, device=dev), torch.zeros(T + 1, B, device=dev, dtype=torch.bool),
              torch.zeros(T, B, dtype=torch.bool), torch.zeros(T, device=dev, dtype=torch.bool)):
        with pytest.raises(ValueError):
            call(reset=r)


@pytest.mark.parametrize("call", [_step, _conv_step])
def test_wrong_caches_are_refused(dev, call):
    shape = STEP["state"] if call is _step else CONV_STEP["state"]
    for s in (torch.ones(4, *shape[1:], device=dev).transpose(1, 2).contiguous().transpose(1, 2),
              torch.ones(*shape[:2], 2 * shape[2], device=dev)[..., ::2], torch.ones(1, *shape[1:], device=dev)):
        with pytest.raises(ValueError):
            call(state=s)
    for slots in (torch.zeros(B, device=dev, dtype=torch.int64), torch.zeros(B + 1, device=dev, dtype=torch.int32),
                  torch.zeros(B, dtype=torch.int32)):
        with pytest.raises(ValueError):
            call(slots=slots)


def test_wrong_tokens_are_refused(dev):
    for tokens in (torch.zeros(T, device=dev), torch.zeros(T, dtype=torch.long), torch.zeros(T, dtype=torch.int16, device=dev)):
        with pytest.raises(ValueError):
            _embed(tokens=tokens)
        with pytest.raises(ValueError):
            _probs(tokens=tokens)
    with pytest.raises(ValueError):
        _probs(tokens=torch.zeros(T + 1, dtype=torch.long, device=dev))
    with pytest.raises(ValueError):
        _embed(tokens=torch.zeros(0, dtype=torch.long, device=dev))
    for top in (-1, 33, V + 1):
        with pytest.raises(ValueError):
            _probs(top=top)
    with pytest.raises(ValueError):
        _embed(scale=float("nan"))


@pytest.mark.parametrize("call,name", [(_scan, "u"), (_conv, "x"), (_embed, "weight"), (_probs, "logits")])
def test_second_derivatives_raise(dev, call, name):
    shape = (SCAN | CONV | EMBED | PROBS)[name]
    x = torch.rand(shape, device=dev, requires_grad=True)
    out = call(**{name: x})
    out = out[0] if isinstance(out, tuple) else out
    dx, = torch.autograd.grad(out, x, torch.ones_like(out).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        dx.sum().backward()


@pytest.mark.parametrize("call,name", [(_step, "state"), (_conv_step, "state")])
def test_a_cache_of_inference_mode_is_not_advanced_outside_it(dev, call, name):
    shape = STEP["state"] if call is _step else CONV_STEP["state"]
    with torch.inference_mode():
        state = torch.rand(shape, device=dev)
        before = state.clone()
    with pytest.raises(RuntimeError, match="inference mode"):
        call(state=state)
    assert torch.equal(state, before)
    with torch.inference_mode():
        call(state=state)
        assert not torch.equal(state, before)


def test_a_cache_updated_in_place_invalidates_its_graph(dev):
    state = torch.rand(B, H, N, device=dev)
    w = torch.rand(B, H, N, device=dev, requires_grad=True)
    y = (w * state).sum()
    _step(state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_the_likeliest_have_no_gradient(dev):
    x = torch.rand(T, V, device=dev, requires_grad=True)
    lp, h, top, ids = G.token_logprobs(x, torch.zeros(T, dtype=torch.long, device=dev), top=2)
    assert lp.requires_grad and h.requires_grad and not top.requires_grad and not ids.requires_grad


def test_an_embedding_may_change_between_forward_and_backward(dev):
    """Its gradient does not depend on it."""
    w = torch.rand(V, H, device=dev, requires_grad=True)
    out = _embed(weight=w)
    with torch.no_grad():
        w.add_(1.0)
    out.sum().backward()
    assert w.grad[0].eq(3).all() and not w.grad[1:].any()
