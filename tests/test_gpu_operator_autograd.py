"""What the gated scan, the step, the linear operator and AdamW do not differentiate or may
not write is refused before anything is launched."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import gru_qat_amd as G

pytestmark = pytest.mark.gpu


def _scan(**kw):
    a = dict(gi=torch.randn(4, 2, 6, device="cuda"), h0=torch.zeros(2, 3, device="cuda")) | kw
    return G.gated_linear_scan(a["gi"], a["h0"])


def _step(**kw):
    a = dict(gi=torch.randn(2, 6, device="cuda"), state=torch.zeros(2, 3, device="cuda")) | kw
    return G.gated_linear_step(a["gi"], a["state"])


def _linear(**kw):
    a = dict(x=torch.randn(6, 4, device="cuda"), weight=torch.randn(5, 4, device="cuda"), bias=torch.randn(5, device="cuda"),
             residual=torch.randn(6, 5, device="cuda")) | kw
    return G.linear_act(a["x"], a["weight"], a["bias"], residual=a["residual"], activation="tanh")


def _adamw(**kw):
    a = {k: torch.ones(7, device="cuda") for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")} | kw
    return G.adamw_step(*([a[k]] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")), step=1, lr=0.1,
                        grad_scale=kw.get("grad_scale"))


SHAPES = {"gi": (4, 2, 6), "h0": (2, 3), "state": (2, 3), "x": (6, 4), "weight": (5, 4), "bias": (5,), "residual": (6, 5),
          "params": (7,), "grads": (7,), "exp_avgs": (7,), "exp_avg_sqs": (7,), "grad_scale": (1,)}


@pytest.mark.parametrize("call,name", [(_scan, "gi"), (_scan, "h0"), (_step, "gi"), (_step, "state"), (_linear, "x"),
                                       (_linear, "weight"), (_linear, "bias"), (_linear, "residual"), (_adamw, "params"),
                                       (_adamw, "grads"), (_adamw, "exp_avgs"), (_adamw, "exp_avg_sqs"),
                                       (_adamw, "grad_scale")])
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_is_refused(dev, call, name, needs_grad):
    shape = (2, 6) if call is _step and name == "gi" else SHAPES[name]
    value = torch.ones(shape, device=dev, requires_grad=needs_grad)
    before = value.detach().clone()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(value, torch.ones(shape, device=dev))
        with pytest.raises(NotImplementedError, match=f"forward-mode.*{name}"):
            call(**{name: dual})
    assert torch.equal(value.detach(), before)
    with torch.no_grad():
        call(**{name: value})  # the same values without a tangent


@pytest.mark.parametrize("call", [lambda x: G.gated_linear_scan(x)[0], lambda x: G.gated_linear_scan(x)[1],
                                  lambda x: G.linear_act(x, torch.ones(3, 6, device="cuda"), activation="silu")],
                         ids=["out", "h_T", "linear"])
def test_a_tangent_of_the_gradient_is_refused(dev, call):
    x = torch.randn(4, 2, 6, device=dev, requires_grad=True)
    y = call(x)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dy, retain_graph=True)
    torch.autograd.grad(y, x, torch.ones_like(y))


def test_a_state_of_inference_mode_is_not_advanced_outside_it(dev):
    gi = torch.randn(2, 6, device=dev)
    with torch.inference_mode():
        state = torch.randn(2, 3, device=dev)
        before = state.clone()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="state was made in inference mode"):
            G.gated_linear_step(gi, state)
        assert torch.equal(state, before)
    with torch.inference_mode():
        G.gated_linear_step(gi, state)
        assert not torch.equal(state, before)


@pytest.mark.parametrize("name", ["params", "exp_avgs", "exp_avg_sqs", "masters", "exp_avg_scales", "exp_avg_sq_scales"])
def test_tensors_of_inference_mode_are_not_stepped_outside_it(dev, name):
    def make(dtype, n=300):
        return torch.ones(n, dtype=dtype, device=dev)

    bf = torch.bfloat16
    lists = dict(params=make(bf), grads=make(bf), exp_avgs=make(torch.int8), exp_avg_sqs=make(torch.uint8),
                 masters=make(torch.float32), exp_avg_scales=make(torch.float32, 2), exp_avg_sq_scales=make(torch.float32, 2))
    with torch.inference_mode():
        lists[name] = lists[name].clone()
        lists["grads"] = lists["grads"].clone()  # only read: one of inference mode is taken

    def step():
        G.adamw_step(*([lists[k]] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")), step=1, lr=0.1,
                     **{k: [lists[k]] for k in ("masters", "exp_avg_scales", "exp_avg_sq_scales")})

    before = {k: t.clone() for k, t in lists.items()}
    with pytest.raises(RuntimeError, match=f"{name} was made in inference mode"):
        step()
    assert all(torch.equal(t, before[k]) for k, t in lists.items())
    with torch.inference_mode():
        step()
    assert not torch.equal(lists["params"], before["params"])
