"""The selective scan and its step at the ends of float32's range, against the definition in 64 bits
(sequence_plain). Roundings are counted for each result by itself."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P
from test_gpu_selective_scan import LEAVES, _make, _run

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")
LOWEST = torch.finfo(F32).min
# an axis within tiles, one in chunks, and one with channels enough for waves that share nothing; none ends with a tile
SIZES = [(21, 2, 24, 4), (150, 2, 24, 16), (1061, 40, 70, 4)]


def roundings(T, B, H, N):
    """On the way of each result: the chain of T states (y, h_T, dz), of T gradients (du, dh0) or of both (d delta), a sum
    over N states, over H channels (dB, dC) or over T B steps and rows (dA, dD and d delta_bias), and 64 for
    softplus, exp and the gate (each within 8 units, at arguments whose error is 8 units)."""
    own = dict.fromkeys(("y", "h_T", "z", "u", "h0"), T + N + 64)
    own["delta"] = 2 * T + N + 64
    own.update(dict.fromkeys(("B", "C"), 2 * T + H + 64))
    own.update(dict.fromkeys(("A", "D", "delta_bias"), 2 * T + N + T * B + 64))
    return own


def check(t, dy, dh):
    T, B, H = t["u"].shape
    most = roundings(T, B, H, t["A"].shape[1])
    y, h, got = _run(t, dy, dh)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    kw = dict(delta_bias=t["delta_bias"], reset=t["reset"], dy=dy, dh=dh)
    want, size = P.selective_scan(*args, **kw), P.selective_scan(*args, size=True, **kw)
    P.assert_within(y, want[0], size[0], most["y"], "y")
    P.assert_within(h, want[1], size[1], most["h_T"], "h_T")
    for k in got:
        P.assert_within(got[k], want[2][k], size[2][k], most[k], "d" + k)
    return y, h, got


@pytest.mark.parametrize("T,B,H,N", SIZES)
@pytest.mark.parametrize("reset", [0.0, 0.02])
def test_the_lowest_rate(dev, T, B, H, N, reset):
    """A finite rate whose product with log2 e is not: a state that lasts a step, with its gradients; -infinity is the same."""
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=40, reset=reset)
    t["A"][:, 1] = LOWEST
    t["A"][::3, 0] = -2.5e38
    y, h, got = check(t, dy, dh)
    t["A"] = torch.where(t["A"] < -1e38, -INF, t["A"])
    y1, h1, got1 = _run(t, dy, dh)
    assert torch.equal(y, y1) and torch.equal(h, h1)
    for k in LEAVES:
        assert torch.equal(got[k], got1[k]), k


def test_step_of_rates_and_no_step_size(dev):
    """A step size of zero (delta of -200) keeps the state, as in the scan, whatever the rate; a usual one drops what decays at once."""
    B, H, N = 2, 40, 4
    t, _, _ = _make(1, B, H, N, F32, dev, seed=41)
    t["A"][:, 1], t["A"][:, 2] = LOWEST, -INF
    t["delta"][0, 0] = -200.0
    t["delta_bias"] = None
    state = t["h0"].clone()
    y = G.selective_step(t["u"][0], t["delta"][0], t["A"], t["B"][0], t["C"][0], state, D=t["D"], z=t["z"][0])
    scan, h, _ = _run(t)
    assert torch.equal(state, h) and torch.equal(state[0], t["h0"][0])
    assert torch.allclose(y, scan[0], rtol=1e-6, atol=1e-6)  # four products in another order
    want = (torch.nn.functional.softplus(t["delta"][0, 1].double()) * t["u"][0, 1].double())[:, None] * t["B"][0, 1].double()
    assert torch.allclose(state[1, :, 1:3].double(), want[:, 1:3], rtol=1e-6)


def _steps_one_by_one(t):
    state, ys = t["h0"].clone(), []
    for k in range(t["u"].shape[0]):
        ys.append(G.selective_step(t["u"][k], t["delta"][k], t["A"], t["B"][k], t["C"][k], state, D=t["D"], z=t["z"][k],
                                   delta_bias=t["delta_bias"]))
    return torch.stack(ys), state


def _same_oddities(a, b):
    for odd in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(odd(a), odd(b)), odd.__name__
    keep = a.isfinite()
    assert torch.allclose(a[keep], b[keep], rtol=1e-4, atol=1e-4)


def _fast(T, B, H, N, dev, seed):
    """Channels 3 and 4 decay by e^-3.2 a step: to nothing in float32 over a chunk, and not in a step."""
    t, dy, dh = _make(T, B, H, N, F32, dev, seed=seed)
    t["A"][3:5] = -16.0
    t["delta"][..., 3:5] = -1.5  # step sizes of 0.2
    t["delta_bias"][3:5] = 0.0
    return t, dy, dh


@pytest.mark.parametrize("T,B,H,N", [(300, 2, 24, 4), (1061, 40, 70, 4)])
def test_an_infinite_state_is_the_steps(dev, T, B, H, N):
    """However an axis is cut, an infinite state is what one step after the other makes of it: infinite, and
    NaN behind a step whose own decay is zero."""
    t, _, _ = _fast(T, B, H, N, dev, 42)
    t["h0"][0, 3, 1], t["h0"][1, 3, 2], t["h0"][0, 4, 0] = INF, -INF, INF
    t["delta"][T // 2, 0, 4] = 30.0  # exp(-480)
    y, h, _ = _run(t)
    want, last = _steps_one_by_one(t)
    _same_oddities(y, want)
    _same_oddities(h, last)
    assert h[0, 3, 1] == INF and h[1, 3, 2] == -INF and h[0, 4, 0].isnan()
    assert y[:T // 2, 0, 4].isinf().all() and y[T // 2:, 0, 4].isnan().all()


@pytest.mark.parametrize("T,B,H,N", [(300, 2, 24, 4), (1061, 40, 70, 4)])
def test_an_infinite_gradient_goes_back(dev, T, B, H, N):
    t, dy, dh = _fast(T, B, H, N, dev, 43)
    dh[0, 3, 1], dh[1, 4, 2] = INF, -INF
    _, _, got = check(t, dy, dh)
    assert got["h0"][0, 3, 1] == INF and got["h0"][1, 4, 2] == -INF
    assert got["h0"].isfinite().sum() == got["h0"].numel() - 2


@pytest.mark.parametrize("T,B,H", [(192, 2, 24), (1100, 40, 70)])
def test_states_that_grow_past_a_chunk(dev, T, B, H):
    """Rates above zero: what a chunk makes of a state is outside float32, what becomes of the state is not;
    a state of zero stays zero."""
    t, _, _ = _make(T, B, H, 2, F32, dev, seed=44)
    t["A"][:] = 2.0
    t["delta"][:], t["delta_bias"] = -200.0, None  # steps that change nothing
    t["delta"][64:128] = 0.5413  # and 64 that take e^2 each
    t["u"][:], t["B"][:] = 0.0, 0.0
    t["h0"][:, :, 0], t["h0"][:, :, 1] = 1e-38, 0.0
    _, h, _ = _run(t)
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    want = P.selective_scan(*args)[1]
    # a step's exponent of 2 is off by some 10 units (8 of its size), its power and product by 2: 22 x 64;
    # a span's exponent of 185 by 3 of its own: 400
    P.assert_within(h, want, want, 2000, "h_T")
    assert (h[..., 1] == 0).all() and h[..., 0].min() > 1e16


# with the last step of a first chunk, and the first of one that is neither first nor second
@pytest.mark.parametrize("T,B,H,N,last,first", [(300, 2, 24, 4, 79, 160), (1061, 40, 70, 4, 47, 960)])
@pytest.mark.parametrize("large", [1e30, 1e38])
def test_a_large_state_decays_to_nothing(dev, T, B, H, N, last, first, large):
    """A finite state that a chunk's decay leaves nothing of is gone behind the chunk, however large it was, and so is a
    gradient on its way back."""
    t, dy, dh = _fast(T, B, H, N, dev, 45)
    t["u"][:, 0, 3], t["h0"][0, 3], dy[:, 1, 4], dh[1, 4] = 0.0, 0.0, 0.0, 0.0
    t["u"][last, 0, 3], dy[first, 1, 4] = large, large
    y, _, got = _run(t, dy, dh)
    # e^-3.2 a step: 60 steps leave 4e-84 of it
    assert y[last, 0, 3].abs() > 1e-6 * large and (y[last + 60:, 0, 3] == 0).all()
    assert got["u"][first - 1, 1, 4].abs() > 1e-6 * large and (got["u"][:first - 60, 1, 4] == 0).all()


@pytest.mark.parametrize("T,B,H,N", [(300, 2, 24, 4), (1061, 40, 70, 4)])
@pytest.mark.parametrize("large", [3e38, INF, float("nan")])
def test_channels_do_not_see_each_other(dev, T, B, H, N, large):
    """What is unusual in a channel changes no bit of another's results."""
    t, dy, dh = _fast(T, B, H, N, dev, 46)
    y, h, got = _run(t, dy, dh)
    t["h0"][0, 3, 1], dh[0, 4, 2] = large, large
    y1, h1, got1 = _run(t, dy, dh)
    others = [c for c in range(H) if c not in (3, 4)]
    assert torch.equal(y[..., others], y1[..., others]) and torch.equal(h[:, others], h1[:, others])
    for k in ("u", "delta", "z"):
        assert torch.equal(got[k][..., others], got1[k][..., others]), k
    assert torch.equal(got["h0"][:, others], got1["h0"][:, others])
    for k in ("A", "D", "delta_bias"):
        assert torch.equal(got[k][others], got1[k][others]), k
    assert torch.equal(y[:, 1:], y1[:, 1:]) and torch.equal(got["B"][:, 1:], got1["B"][:, 1:])
