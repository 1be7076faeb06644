"""The selective scan and its step against the definition in 64 bits (sequence_plain)."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
LEAVES = ("u", "delta", "A", "B", "C", "D", "z", "h0", "delta_bias")


def _make(T, B, H, N, dtype, dev, seed=0, reset=0.0, batch_first=False):
    g = torch.Generator().manual_seed(seed)

    def noise(*shape, kind=dtype):
        return torch.randn(shape, generator=g).to(kind).to(dev)

    t = dict(u=noise(T, B, H), delta=noise(T, B, H) - 1, z=noise(T, B, H), B=noise(T, B, N), C=noise(T, B, N),
             A=-torch.exp(noise(H, N, kind=F32)), D=noise(H, kind=F32), h0=noise(B, H, N, kind=F32),
             delta_bias=noise(H, kind=F32))
    t["reset"] = (torch.rand(T, B, generator=g) < reset).to(dev) if reset else None
    return t, noise(T, B, H), noise(B, H, N, kind=F32)


def _roundings(T, B, H, N):
    """On the way of any result: the chain over T, a sum over states, channels, or steps and rows, and what
    softplus, exp and the gate take (each within 8 units, at arguments whose error is 8 units)."""
    return T + N + max(H, T * B) + 64


def _run(t, dy=None, dh=None, batch_first=False):
    t = dict(t)
    if dy is not None or dh is not None:
        for k in LEAVES:
            if t[k] is not None:
                t[k] = t[k].detach().requires_grad_(True)
    args = [t[k].transpose(0, 1) if batch_first and t[k] is not None and k in "uBCz" or batch_first and k == "delta" else t[k]
            for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    reset = t["reset"].t() if batch_first and t["reset"] is not None else t["reset"]
    y, h = G.selective_scan(*args, delta_bias=t["delta_bias"], reset=reset, batch_first=batch_first)
    if batch_first:
        y = y.transpose(0, 1)
    if dy is None and dh is None:
        return y, h, {}
    outs, grads = zip(*[(o, g) for o, g in ((y, dy), (h, dh)) if g is not None])
    names = [k for k in LEAVES if t[k] is not None]
    return y, h, dict(zip(names, torch.autograd.grad(outs, [t[k] for k in names], grads)))


def _check(t, dy, dh, roundings, **kw):
    y, h, got = _run(t, dy, dh, **kw)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    kw = dict(delta_bias=t["delta_bias"], reset=t["reset"], dy=dy, dh=dh)
    want = P.selective_scan(*args, **kw)
    size = P.selective_scan(*args, size=True, **kw)
    P.assert_within(y, want[0], size[0], roundings, "y")
    P.assert_within(h, want[1], size[1], roundings, "h_T")
    for k in got:
        P.assert_within(got[k], want[2][k], size[2][k], roundings, "d" + k)


# a step, tiles of 16 that end early and late, chunks; channels around 64; states that fill waves or not
@pytest.mark.parametrize("T", [1, 15, 16, 33, 300])
@pytest.mark.parametrize("H,N", [(1, 1), (7, 3), (64, 4), (65, 8), (130, 16), (33, 13), (20, 32), (5, 17), (66, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_forward_and_backward(dev, T, H, N, dtype):
    B = 2
    t, dy, dh = _make(T, B, H, N, dtype, dev, reset=0.05)
    _check(t, dy, dh, _roundings(T, B, H, N))


# rows, channels and steps enough for waves that share nothing: several chunks, the last one short
@pytest.mark.parametrize("T,B,H,N", [(610, 60, 130, 3), (1100, 40, 65, 16), (2100, 12, 130, 5), (1060, 40, 70, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_many_channels(dev, T, B, H, N, dtype):
    t, dy, dh = _make(T, B, H, N, dtype, dev, seed=20, reset=0.003)
    _check(t, dy, dh, _roundings(T, B, H, N))


def test_nan_before_a_reset_among_many_channels(dev):
    T, B, H, N = 1100, 40, 65, 4
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=21)
    t["reset"] = torch.zeros(T, B, dtype=torch.bool, device=dev)
    t["reset"][700, 3] = True
    clean = _run(t, dy, dh)
    t["h0"] = t["h0"].clone()
    t["h0"][3, 7] = float("nan")
    y, h, grads = _run(t, dy, dh)
    assert y[:700, 3, 7].isnan().all() and torch.equal(y[700:], clean[0][700:]) and torch.equal(h, clean[1])
    for k in ("u", "delta", "z", "B", "C"):
        assert torch.equal(grads[k][700:], clean[2][k][700:]), k
        assert torch.equal(grads[k][:, 4:], clean[2][k][:, 4:]), k


@pytest.mark.parametrize("missing", [(), ("D",), ("z",), ("h0",), ("delta_bias",), ("D", "z", "h0", "delta_bias")], ids=str)
@pytest.mark.parametrize("reset", [0.0, 0.2, 1.0])
def test_optional_inputs_and_resets(dev, missing, reset):
    T, B, H, N = 150, 3, 40, 16
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=1, reset=reset)
    for k in missing:
        t[k] = None
    _check(t, dy, dh, _roundings(T, B, H, N))


@pytest.mark.parametrize("which", ["y", "h"])
def test_one_gradient_alone(dev, which):
    T, B, H, N = 140, 2, 20, 16
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=2, reset=0.02)
    _check(t, dy if which == "y" else None, dh if which == "h" else None, _roundings(T, B, H, N))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_batch_first_and_strides(dev, dtype):
    T, B, H, N = 70, 3, 37, 16
    t, dy, dh = _make(T, B, H, N, dtype, dev, seed=3, reset=0.05)
    for k, n in (("u", H), ("delta", H), ("z", H), ("B", N), ("C", N)):
        wide = torch.full((T, B, n + 11), float("nan"), device=dev, dtype=dtype)
        wide[..., 5:5 + n] = t[k]
        t[k] = wide[..., 5:5 + n]
    _check(t, dy, dh, _roundings(T, B, H, N), batch_first=True)
    t["u"] = t["u"].contiguous().transpose(0, 1).contiguous().transpose(0, 1)
    _check(t, dy.transpose(0, 1).contiguous().transpose(0, 1), dh, _roundings(T, B, H, N))


def test_large_decays_and_step_sizes(dev):
    """States that vanish in a step, step sizes of 1e-6 and of 30, decays of zero (A = 0)."""
    T, B, H, N = 100, 2, 24, 16
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=4)
    t["delta"][:, :, :8] -= 14.0
    t["delta"][:, :, 8:12] += 30.0
    t["A"][:, 0] = 0.0
    t["A"][:, 1] = -1000.0
    # with A = 0 sums grow by T terms; all of it is in `size`
    _check(t, dy, dh, _roundings(T, B, H, N))


@pytest.mark.parametrize("T,B,H", [(21, 2, 24), (150, 2, 24), (1061, 40, 70)])
def test_a_rate_of_minus_infinity(dev, T, B, H):
    """A state that forgets at once: exp(-infinity) is 0 at every step, also before the axis ends in a tile."""
    t, _, _ = _make(T, B, H, 4, F32, dev, seed=22)
    t["A"][:, 1] = -float("inf")
    y, h, _ = _run(t)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    want, size = P.selective_scan(*args, delta_bias=t["delta_bias"]), P.selective_scan(*args, delta_bias=t["delta_bias"], size=True)
    P.assert_within(y, want[0], size[0], _roundings(T, B, H, 4), "y")
    P.assert_within(h, want[1], size[1], _roundings(T, B, H, 4), "h_T")


def test_split_in_two_calls(dev):
    """h_T continues the sequence, and its gradient goes back through the first call."""
    T, B, H, N = 90, 2, 30, 16
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=5, reset=0.03)
    for k in LEAVES:
        t[k] = t[k].detach().requires_grad_(True)
    cut, h, ys = 41, t["h0"], []
    for s in (slice(0, cut), slice(cut, T)):
        y, h = G.selective_scan(t["u"][s], t["delta"][s], t["A"], t["B"][s], t["C"][s], t["D"], t["z"][s], h,
                                delta_bias=t["delta_bias"], reset=t["reset"][s])
        ys.append(y)
    got = torch.autograd.grad((torch.cat(ys), h), [t[k] for k in LEAVES], (dy, dh))
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    kw = dict(delta_bias=t["delta_bias"], reset=t["reset"], dy=dy, dh=dh)
    want, size = P.selective_scan(*args, **kw), P.selective_scan(*args, size=True, **kw)
    for k, g in zip(LEAVES, got):
        P.assert_within(g, want[2][k], size[2][k], _roundings(T, B, H, N), "d" + k)


@pytest.mark.parametrize("T", [20, 200])
def test_nan_before_a_reset_stays_there(dev, T):
    B, H, N = 2, 20, 16
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=6)
    t["reset"] = torch.zeros(T, B, dtype=torch.bool, device=dev)
    t["reset"][T // 2, 0] = True
    clean = _run(t, dy, dh)
    t["h0"] = t["h0"].clone()
    t["h0"][0, 3] = float("nan")
    t["h0"][0, 4] = float("inf")
    t["u"] = t["u"].clone()
    t["u"][T // 4, 0, 5] = float("inf")
    y, h, grads = _run(t, dy, dh)
    half = T // 2
    assert torch.equal(y[half:, 0], clean[0][half:, 0]) and torch.equal(y[:, 1], clean[0][:, 1])
    assert torch.equal(h, clean[1])
    for k in ("u", "delta", "z", "B", "C"):
        assert torch.equal(grads[k][half:, 0], clean[2][k][half:, 0]), k
        assert torch.equal(grads[k][:, 1], clean[2][k][:, 1]), k
    assert torch.equal(grads["h0"][1], clean[2]["h0"][1])
    assert y[:half, 0, 3].isnan().all()


def test_repeats_bit_for_bit(dev):
    t, dy, dh = _make(400, 3, 130, 16, BF16, dev, seed=7, reset=0.01)
    a, b = _run(t, dy, dh), _run(t, dy, dh)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(a[2][k], b[2][k]) for k in a[2])


def test_differences(dev):
    """The gradient along a direction against a difference of the function in 64 bits."""
    T, B, H, N = 40, 2, 10, 8
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=8, reset=0.05)
    _, _, got = _run(t, dy, dh)
    g = torch.Generator().manual_seed(9)

    def value(sign, k, d):
        s = {n: (None if v is None else v.cpu().double() if v.is_floating_point() else v.cpu()) for n, v in t.items()}
        s[k] = s[k] + sign * 1e-5 * d
        y, h = P.selective_scan(*[s[n] for n in ("u", "delta", "A", "B", "C", "D", "z", "h0")], delta_bias=s["delta_bias"],
                                reset=s["reset"])
        return (y * dy.cpu()).sum() + (h * dh.cpu()).sum()

    for k in LEAVES:
        d = torch.randn(t[k].shape, generator=g).double()
        want = (value(1, k, d) - value(-1, k, d)) / 2e-5
        have = (got[k].cpu().double() * d).sum()
        # the difference's own error is 1e-10 of third derivatives, the gradient's 2^-24 of its terms' sizes
        assert abs(have - want) <= 1e-4 * (got[k].cpu().double().abs() * d.abs()).sum() + 1e-6, (k, have, want)


# ---- the step -------------------------------------------------------------------------


@pytest.mark.parametrize("B,H,N", [(1, 1, 1), (5, 70, 16), (3, 65, 3), (2, 33, 32), (4, 64, 13)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bare", [False, True])
def test_step(dev, B, H, N, dtype, bare):
    t, _, _ = _make(1, B, H, N, dtype, dev, seed=10)
    if bare:
        t["D"] = t["z"] = t["delta_bias"] = None
    S = B + 3
    state = torch.randn(S, H, N, generator=torch.Generator().manual_seed(11)).to(dev)
    slots = torch.randperm(S, generator=torch.Generator().manual_seed(12))[:B].int().to(dev)
    before = state.clone()
    y = G.selective_step(t["u"][0], t["delta"][0], t["A"], t["B"][0], t["C"][0], state, slots, D=t["D"],
                         z=None if bare else t["z"][0], delta_bias=t["delta_bias"])
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z")]
    kw = dict(h0=before[slots.long()], delta_bias=t["delta_bias"])
    want, size = P.selective_scan(*args, **kw), P.selective_scan(*args, size=True, **kw)
    P.assert_within(y, want[0][0], size[0][0], _roundings(1, 1, 1, N), "y")
    P.assert_within(state[slots.long()], want[1], size[1], _roundings(1, 1, 1, N), "state")
    rest = torch.ones(S, dtype=torch.bool, device=dev)
    rest[slots.long()] = False
    assert torch.equal(state[rest], before[rest])


def test_step_empty_and_bad_slots(dev):
    B, H, N, S = 4, 20, 16, 6
    t, _, _ = _make(1, B, H, N, F32, dev, seed=13)
    state = torch.randn(S, H, N, device=dev)
    before, version = state.clone(), state._version
    slots = torch.tensor([2, -1, S, 0], dtype=torch.int32, device=dev)
    y = G.selective_step(t["u"][0], t["delta"][0], t["A"], t["B"][0], t["C"][0], state, slots)
    assert (y[1] == 0).all() and y[2].isnan().all() and y[0].isfinite().all() and y[3].isfinite().all()
    assert torch.equal(state[[1, 3, 4, 5]], before[[1, 3, 4, 5]])
    assert not torch.equal(state[2], before[2]) and state._version > version


def test_steps_equal_the_scan(dev):
    T, B, H, N = 30, 3, 40, 16
    t, _, _ = _make(T, B, H, N, F32, dev, seed=14)
    y, h, _ = _run(t)
    state = t["h0"].clone()
    for k in range(T):
        out = G.selective_step(t["u"][k], t["delta"][k], t["A"], t["B"][k], t["C"][k], state, D=t["D"], z=t["z"][k],
                               delta_bias=t["delta_bias"])
        # the sum over states is in another order
        assert torch.allclose(out, y[k], rtol=1e-5, atol=1e-5)
    assert torch.allclose(state, h, rtol=1e-5, atol=1e-6)
