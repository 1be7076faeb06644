"""The causal convolution and its step against the definition in 64 bits (sequence_plain)."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("x", "weight", "bias", "state")


def _make(T, B, C, W, dtype, dev, seed=0, reset=0.0):
    g = torch.Generator().manual_seed(seed)

    def noise(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(dev)

    t = dict(x=noise(T, B, C), weight=noise(C, W), bias=noise(C), state=noise(B, W - 1, C))
    t["reset"] = (torch.rand(T, B, generator=g) < reset).to(dev) if reset else None
    return t, noise(T, B, C), noise(B, W - 1, C)


def _check(t, dy, dlast, activation="silu", batch_first=False):
    T, B, C = t["x"].shape
    leaves = {k: t[k].detach().requires_grad_(True) for k in NAMES if t[k] is not None}
    x, reset = leaves["x"], t["reset"]
    if batch_first:
        x, reset = x.transpose(0, 1), None if reset is None else reset.t()
    y, last = G.causal_conv(x, leaves["weight"], leaves.get("bias"), leaves.get("state"), activation=activation, reset=reset,
                            batch_first=batch_first)
    if batch_first:
        y = y.transpose(0, 1)
    kw = dict(activation=activation, reset=t["reset"], dy=dy, dlast=dlast)
    args = [t[k] for k in NAMES]
    want, size = P.causal_conv(*args, **kw), P.causal_conv(*args, size=True, **kw)
    # W + 1 terms, the activation (8 units); backwards also a sum over steps and rows
    P.assert_within(y, want[0], size[0], 16, "y")
    assert torch.equal(last.detach().cpu().double(), want[1])
    outs, grads = zip(*[(o, g) for o, g in ((y, dy), (last, dlast)) if g is not None])
    got = torch.autograd.grad(outs, list(leaves.values()), grads)
    for k, g in zip(leaves, got):
        P.assert_within(g, want[2][k], size[2][k], T * B + 32, "d" + k)


# fewer steps than taps, runs that end early and late; one channel a lane or four
@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 65, 200])
@pytest.mark.parametrize("C", [1, 5, 130, 132, 264])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_forward_and_backward(dev, T, C, W, dtype):
    t, dy, dlast = _make(T, 2, C, W, dtype, dev, reset=0.1)
    _check(t, dy, dlast)


@pytest.mark.parametrize("missing", [(), ("bias",), ("state",), ("bias", "state")], ids=str)
@pytest.mark.parametrize("reset", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("activation", ["silu", "none"])
def test_optional_inputs_and_resets(dev, missing, reset, activation):
    t, dy, dlast = _make(75, 3, 136, 4, F32, dev, seed=1, reset=reset)
    for k in missing:
        t[k] = None
    _check(t, dy, dlast, activation)


@pytest.mark.parametrize("which", ["y", "last"])
def test_one_gradient_alone(dev, which):
    t, dy, dlast = _make(20, 2, 30, 4, F32, dev, seed=2, reset=0.1)
    _check(t, dy if which == "y" else None, dlast if which == "last" else None)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("off", [0, 4, 5])
def test_batch_first_and_strides(dev, dtype, off):
    T, B, C = 70, 3, 136
    t, dy, dlast = _make(T, B, C, 4, dtype, dev, seed=3, reset=0.05)
    wide = torch.full((T, B, C + 12), float("nan"), device=dev, dtype=dtype)
    wide[..., off:off + C] = t["x"]
    t["x"] = wide[..., off:off + C]
    _check(t, dy, dlast, batch_first=True)
    _check(t, dy.transpose(0, 1).contiguous().transpose(0, 1), dlast)


def test_long_runs(dev):
    """Rows enough for runs of 64 steps."""
    t, dy, dlast = _make(130, 40, 512, 4, BF16, dev, seed=4, reset=0.02)
    T, B, C = t["x"].shape
    x = torch.cat([t["x"]] * 64, 1).requires_grad_(True)
    reset = torch.cat([t["reset"]] * 64, 1)
    y, last = G.causal_conv(x, t["weight"], t["bias"], torch.cat([t["state"]] * 64), reset=reset)
    dx, = torch.autograd.grad(y, x, torch.cat([dy] * 64, 1))
    one = t["x"].detach().requires_grad_(True)
    y1, last1 = G.causal_conv(one, t["weight"], t["bias"], t["state"], reset=t["reset"])
    dx1, = torch.autograd.grad(y1, one, dy)
    for k in (0, 31, 63):
        s = slice(k * B, (k + 1) * B)
        assert torch.equal(y[:, s], y1) and torch.equal(last[s], last1) and torch.equal(dx[:, s], dx1)


def test_nan_before_a_reset_stays_there(dev):
    T, B, C = 30, 2, 140
    t, dy, dlast = _make(T, B, C, 4, F32, dev, seed=5)
    t["reset"] = torch.zeros(T, B, dtype=torch.bool, device=dev)
    t["reset"][10, 0] = True
    t["reset"][0, 1] = True

    def run():
        x = t["x"].detach().requires_grad_(True)
        s = t["state"].detach().requires_grad_(True)
        y, last = G.causal_conv(x, t["weight"], t["bias"], s, reset=t["reset"])
        return (y, last, *torch.autograd.grad((y, last), (x, s), (dy, dlast)))

    clean = run()
    t["x"], t["state"] = t["x"].clone(), t["state"].clone()
    t["x"][9, 0] = float("nan")
    t["state"][1] = float("inf")
    odd = run()
    assert torch.equal(odd[0][10:, 0], clean[0][10:, 0]) and torch.equal(odd[0][:, 1], clean[0][:, 1])
    assert torch.equal(odd[1], clean[1])
    assert torch.equal(odd[2][10:, 0], clean[2][10:, 0]) and torch.equal(odd[2][:, 1], clean[2][:, 1])
    assert (odd[3][1] == 0).all() and odd[0][9, 0].isnan().all()


def test_split_in_two_calls(dev):
    T, B, C, cut = 50, 2, 40, 2
    t, dy, dlast = _make(T, B, C, 4, F32, dev, seed=6, reset=0.05)
    for k in NAMES:
        t[k] = t[k].detach().requires_grad_(True)
    s, ys = t["state"], []
    for part in (slice(0, cut), slice(cut, T)):
        y, s = G.causal_conv(t["x"][part], t["weight"], t["bias"], s, reset=t["reset"][part])
        ys.append(y)
    got = torch.autograd.grad((torch.cat(ys), s), [t[k] for k in NAMES], (dy, dlast))
    kw = dict(reset=t["reset"], dy=dy, dlast=dlast)
    args = [t[k] for k in NAMES]
    want, size = P.causal_conv(*args, **kw), P.causal_conv(*args, size=True, **kw)
    for k, g in zip(NAMES, got):
        P.assert_within(g, want[2][k], size[2][k], T * B + 32, "d" + k)


@pytest.mark.parametrize("B,C,W", [(1, 1, 2), (5, 70, 3), (3, 300, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("activation", ["silu", "none"])
def test_step(dev, B, C, W, dtype, activation):
    t, _, _ = _make(1, B, C, W, dtype, dev, seed=7)
    S = B + 2
    cache = torch.randn(S, W - 1, C, generator=torch.Generator().manual_seed(8)).to(dtype).to(dev)
    before = cache.clone()
    slots = torch.randperm(S, generator=torch.Generator().manual_seed(9))[:B].int().to(dev)
    y = G.causal_conv_step(t["x"][0], t["weight"], t["bias"], cache, slots, activation=activation)
    args = (t["x"], t["weight"], t["bias"], before[slots.long()])
    want, size = P.causal_conv(*args, activation=activation), P.causal_conv(*args, activation=activation, size=True)
    P.assert_within(y, want[0][0], size[0][0], 16, "y")
    assert torch.equal(cache[slots.long()].cpu().double(), want[1])
    rest = torch.ones(S, dtype=torch.bool, device=dev)
    rest[slots.long()] = False
    assert torch.equal(cache[rest], before[rest])


def test_step_empty_and_bad_slots(dev):
    t, _, _ = _make(1, 4, 20, 4, BF16, dev, seed=10)
    cache = torch.randn(6, 3, 20, device=dev).to(BF16)
    before = cache.clone()
    slots = torch.tensor([2, -1, 6, 0], dtype=torch.int32, device=dev)
    y = G.causal_conv_step(t["x"][0], t["weight"], None, cache, slots)
    assert (y[1] == 0).all() and y[2].isnan().all() and y[[0, 3]].isfinite().all()
    assert torch.equal(cache[[1, 3, 4, 5]], before[[1, 3, 4, 5]]) and not torch.equal(cache[2], before[2])
