"""The gated linear layer and the example around it: training, and serving token by token."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("gated_linear_example", os.path.join(ROOT, "examples", "gated_linear.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _reference(layer, x, h0, reset):
    """The layer in float64, step by step."""
    wg, bg, wo, bo = (p.detach().double() for p in (layer.weight_g, layer.bias_g, layer.weight_o, layer.bias_o))
    H, h, out = layer.hidden, h0.double(), []
    for t in range(x.shape[0]):
        gi = x[t].double() @ wg.t() + bg
        z, n = torch.sigmoid(gi[:, :H]), torch.tanh(gi[:, H:])
        h = z * torch.where(reset[t][:, None], 0.0, h) + (1 - z) * n
        out.append(h @ wo.t() + bo + x[t].double())
    return torch.stack(out), h


@pytest.mark.parametrize("batch_first", [False, True])
def test_layer_against_its_formula(dev, batch_first):
    """float32, values of order 1: sums of 24 and 40 products, 50 steps whose gates pass errors on (under a
    hundred roundings of 2^-24 each way, weights of at most 0.3): 2^-14 covers all of it many times over, and no
    mistake in the formula."""
    torch.manual_seed(0)
    layer = G.GatedLinearLayer(24, 40, batch_first=batch_first, device=dev)
    x, h0 = torch.randn(50, 3, 24, device=dev), torch.randn(3, 40, device=dev)
    reset = torch.rand(50, 3, device=dev) < 0.1
    flip = (lambda t: t.transpose(0, 1)) if batch_first else (lambda t: t)
    y, h = layer(flip(x), h0, flip(reset))
    want, last = _reference(layer, x, h0, reset)
    assert (flip(y).double() - want).abs().max() < 2.0 ** -14 and (h.double() - last).abs().max() < 2.0 ** -14


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_tokens_one_by_one(dev, example, dtype):
    """Serving gives what the whole sequence gives: the same products and gates, the recurrence in
    another order (float32), and in bfloat16 roundings of the states' outputs that this can move by a unit,
    through two layers."""
    torch.manual_seed(1)
    model = [G.GatedLinearLayer(32, 48, device=dev, dtype=dtype) for _ in range(2)]
    head = torch.eye(32, device=dev, dtype=dtype)
    x = torch.randn(70, 5, 32, device=dev)
    y = x.to(dtype)
    with torch.no_grad():
        for layer in model:
            y, _ = layer(y)
    served = example.serve(model, head, x, dtype)
    bound = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -4
    assert (served.float() - G.linear_act(y, head).float()).abs().max() < bound


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.float32, 8), (torch.bfloat16, 8)],
                         ids=["f32", "f32-8bit", "bf16-8bit"])
def test_example_trains(dev, example, dtype, bits):
    """The target is in the layers' reach (one channel with z = 0.9 for each feature): the loss, which starts at
    the target's own size or above, falls to under half of what predicting zero gives."""
    _, _, data, losses = example.train(steps=150, dtype=dtype, state_bits=bits, say=None)
    zero = data[0][2].square().mean().item()
    assert all(v == v for v in losses) and losses[-1] < 0.5 * zero


def test_refusals(dev):
    for kw in (dict(size=0, hidden=4), dict(size=4, hidden=0), dict(size=4, hidden=4, activation="relu")):
        with pytest.raises(ValueError):
            G.GatedLinearLayer(**kw)
    layer = G.GatedLinearLayer(4, 6, device=dev)
    with pytest.raises(ValueError):
        layer(torch.randn(3, 2, 5, device=dev))
    with pytest.raises(ValueError):
        layer.step(torch.randn(2, 4, device=dev), torch.zeros(2, 5, device=dev))
