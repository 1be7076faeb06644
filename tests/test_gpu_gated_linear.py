"""The gated linear recurrence (gs_glr_fwd / _bwd / _step) against the recurrence in
64 bits, step by step.

Tolerances carry a bound along with the recurrence. u is float32's unit roundoff; a
step's gates, products and sums round a small number of times relative to |h|, |n|
and |D| (16 in the bound: exponential and reciprocal of an ulp or two each, the
products, and one rounding per product of the composed maps), and what a step receives
it passes on times z:
  e_t = z e_{t-1} + 16 u (|h_{t-1}| + |n|),   and backwards alike.
In bfloat16 an output rounds once more (2^-8 relative), and the backward reads
h_{t-1} as stored.
"""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
C = 16 * U32


def _oracle(gi, h0, reset, act, dout=None, dh=None):
    """(out, h_T, dgi, dh0) in float64 on the CPU with a bound beside each."""
    gi, h0 = gi.detach().cpu().double(), h0.detach().cpu().double()
    low = gi.new_tensor(0.0)
    T, H = gi.shape[0], gi.shape[2] // 2
    z, n = torch.sigmoid(gi[..., :H]), gi[..., H:]
    n = torch.tanh(n) if act == "tanh" else n
    cut = (torch.zeros(gi.shape[:2], dtype=torch.bool) if reset is None else reset.cpu())[..., None]
    h, e = h0, torch.zeros_like(h0)
    out, err, prev = [], [], []
    for t in range(T):
        h, e = torch.where(cut[t], low, h), torch.where(cut[t], low, e)
        prev.append((h, e))
        e = z[t] * e + C * (h.abs() + n[t].abs())
        h = z[t] * h + (1 - z[t]) * n[t]
        out.append(h)
        err.append(e)
    out, err = torch.stack(out), torch.stack(err)
    if dout is None:
        return (out, err), (out[-1], err[-1])
    dout, E, eE = dout.detach().cpu().double(), dh.cpu().double(), torch.zeros_like(h0)
    dgi, bound = torch.empty_like(gi), torch.empty_like(gi)
    for t in range(T - 1, -1, -1):
        D, eD = dout[t] + E, eE + C * (dout[t].abs() + E.abs())
        (hp, ehp), s = prev[t], z[t] * (1 - z[t])
        slope = 1 - n[t] ** 2 if act == "tanh" else torch.ones_like(s)
        dgi[t, :, :H], dgi[t, :, H:] = D * (hp - n[t]) * s, D * (1 - z[t]) * slope
        bound[t, :, :H] = eD * (hp - n[t]).abs() * s + D.abs() * (ehp * s + C * (hp.abs() + n[t].abs()))
        bound[t, :, H:] = eD * (1 - z[t]) * slope + C * D.abs()
        E, eE = torch.where(cut[t], low, z[t] * D), torch.where(cut[t], low, z[t] * eD + C * D.abs())
    return (out, err), (out[-1], err[-1]), (dgi, bound), (E, eE), torch.stack([p[0] for p in prev]), z


def _near(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"{what}: {off.max()} off, {(off / bound.clamp(min=1e-300)).max()} of the bound"


def _inputs(T, B, H, dtype, seed, p_reset=0.0):
    g = torch.Generator().manual_seed(seed)
    gi = torch.randn(T, B, 2 * H, generator=g)
    gi[..., :H] += torch.rand(H, generator=g) * 6 - 1
    reset = torch.rand(T, B, generator=g) < p_reset if p_reset else None
    return (gi.to(dtype), torch.randn(B, H, generator=g), reset, torch.randn(T, B, H, generator=g).to(dtype),
            torch.randn(B, H, generator=g))


def _check(dev, gi, h0, reset, dout, dh, act, call=G.gated_linear_scan):
    dtype = gi.dtype
    x, s = gi.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    out, h_last = call(x, s, activation=act, reset=None if reset is None else reset.to(dev))
    dgi, dh0 = torch.autograd.grad((out, h_last), (x, s), (dout.to(dev), dh.to(dev)))
    (o, eo), (hl, ehl), (dg, edg), (d0, ed0), hp, z = _oracle(gi, h0, reset, act, dout, dh)
    if dtype == torch.bfloat16:
        H = h0.shape[1]
        # D, the gradient of h, from dgi_n's formula would divide by small slopes: bound it by a scan of |dout| instead
        Dabs, run = torch.empty_like(o), dh.double().abs()
        for t in range(o.shape[0] - 1, -1, -1):
            Dabs[t] = run = run * (z[t + 1] if t + 1 < o.shape[0] else 1.0) + dout[t].double().abs()
        edg[..., :H] += U16 * hp.abs() * Dabs * z * (1 - z)
        eo, edg = eo * (1 + U16) + U16 * o.abs(), edg * (1 + U16) + U16 * dg.abs()
    assert out.dtype == dgi.dtype == dtype and h_last.dtype == dh0.dtype == torch.float32
    _near(out, o, eo, "out")
    _near(h_last, hl, ehl, "h_T")
    _near(dgi, dg, edg + 1e-38, "dgi")
    _near(dh0, d0, ed0 + 1e-38, "dh0")
    with torch.no_grad():
        again, last = call(x, s, activation=act, reset=None if reset is None else reset.to(dev))
    assert torch.equal(again, out) and torch.equal(last, h_last)


# lengths around a tile (8 and 256 steps) and around where an axis is cut in segments; odd and
# even channel counts around a wave's share (16, 32, 64, 128)
SHAPES = [(1, 1, 1), (2, 3, 5), (8, 2, 64), (9, 1, 130), (16, 3, 31), (17, 2, 33), (64, 1, 16), (255, 1, 17),
          (256, 2, 32), (257, 1, 48), (513, 3, 15), (1025, 1, 20), (1300, 2, 34)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ["tanh", "identity"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_and_gradients(dev, shape, act, dtype):
    T, B, H = shape
    _check(dev, *_inputs(T, B, H, dtype, seed=T + H), act)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("p", [0.02, 0.4, 1.0])
@pytest.mark.parametrize("shape", [(1, 2, 3), (9, 1, 130), (257, 2, 34), (1300, 1, 20)], ids=str)
def test_resets(dev, shape, p, dtype):
    T, B, H = shape
    _check(dev, *_inputs(T, B, H, dtype, seed=T, p_reset=p), "tanh")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_channels(dev, dtype):
    """So many channels that a wave walks the axis alone (tiles of 8 steps)."""
    _check(dev, *_inputs(27, 2100, 258, dtype, seed=5, p_reset=0.1), "tanh")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_batch_first_and_strides(dev, dtype):
    T, B, H = 70, 3, 34
    gi, h0, reset, dout, dh = _inputs(T, B, H, dtype, seed=2, p_reset=0.1)
    whole = torch.empty(B, T, 2 * H + 5, dtype=dtype, device=dev)

    def batch_first(x, s, activation, reset):
        whole[..., 3:3 + 2 * H] = x.detach().transpose(0, 1)  # odd row starts and strides
        view = whole[..., 3:3 + 2 * H]
        y = G.gated_linear_scan(view.detach(), s.detach(), activation=activation, reset=reset.t(), batch_first=True)
        z = G.gated_linear_scan(x.transpose(0, 1), s, activation=activation, reset=reset.t(), batch_first=True)
        assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])
        return z[0].transpose(0, 1), z[1]

    _check(dev, gi, h0, reset, dout, dh, "tanh", batch_first)


def test_parts_continue_each_other(dev):
    gi, h0, reset, _, _ = _inputs(300, 2, 40, torch.float32, seed=3, p_reset=0.05)
    gi, h0, reset = gi.to(dev), h0.to(dev), reset.to(dev)
    whole, last = G.gated_linear_scan(gi, h0, reset=reset)
    a, h = G.gated_linear_scan(gi[:130], h0, reset=reset[:130])
    b, h = G.gated_linear_scan(gi[130:], h, reset=reset[130:])
    (o, e), _ = _oracle(gi, h0, reset, "tanh")
    _near(torch.cat([a, b]), o, e, "out")
    _near(h, o[-1], e[-1], "h_T")


@pytest.mark.parametrize("only", ["out", "last", "sum"])
def test_gradients_of_one_output(dev, only):
    gi, h0, _, dout, dh = _inputs(40, 2, 24, torch.float32, seed=4)
    x, s = gi.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    out, h = G.gated_linear_scan(x, s)
    if only == "out":
        grads, dh = torch.autograd.grad(out, (x, s), dout.to(dev)), torch.zeros_like(dh)
    elif only == "last":
        grads, dout = torch.autograd.grad(h, (x, s), dh.to(dev)), torch.zeros_like(dout)
    else:  # a gradient that is one number expanded
        grads, dout, dh = torch.autograd.grad(out.sum(), (x, s)), torch.ones_like(dout), torch.zeros_like(dh)
    _, _, (dg, e), (d0, e0), _, _ = _oracle(gi, h0, None, "tanh", dout, dh)
    _near(grads[0], dg, e + 1e-38, "dgi")
    _near(grads[1], d0, e0 + 1e-38, "dh0")


def test_gradient_against_differences(dev):
    """Central differences of a weighted sum of outputs, in float32 with a step of 2^-7: their own
    error is the third derivative's h^2 / 6 (under 2^-14 of the weights' scale) and 2 e / 2^-7 of
    rounding; the sum over 12 x 2 x 4 outputs of weight about 1 stays under 2^-8."""
    T, B, H = 12, 2, 4
    gi, h0, reset, dout, _ = _inputs(T, B, H, torch.float32, seed=6, p_reset=0.1)
    x, r, w = gi.to(dev).requires_grad_(True), reset.to(dev), dout.to(dev)
    out, _ = G.gated_linear_scan(x, h0.to(dev), reset=r)
    got, = torch.autograd.grad(out, x, w)
    step = 2.0 ** -7
    for at in range(0, gi.numel(), 7):
        d = torch.zeros(gi.numel(), device=dev)
        d[at] = step
        d = d.view(gi.shape)
        with torch.no_grad():
            up, dn = (G.gated_linear_scan(x + k * d, h0.to(dev), reset=r)[0].double() for k in (1, -1))
        assert abs(((up - dn) * w).sum().item() / (2 * step) - got.view(-1)[at].item()) < 2.0 ** -8


@pytest.mark.parametrize("T", [20, 300, 1300])
def test_nothing_passes_a_reset(dev, T):
    """NaN and infinities before a reset (in h0, gi or dout) leave what is on its other side alone."""
    gi, h0, _, dout, dh = _inputs(T, 2, 40, torch.float32, seed=7)
    cut = T // 2
    reset = torch.zeros(T, 2, dtype=torch.bool)
    reset[cut, 0] = True
    bad, bad_h0, bad_d = gi.clone(), h0.clone(), dout.clone()
    bad[3, 0, 5], bad[4, 0, 46] = float("nan"), float("inf")
    bad_h0[0, 7], bad_h0[0, 8] = float("inf"), float("nan")
    bad_d[cut + 2, 0, 9] = float("nan")
    r = reset.to(dev)

    def both(a, b, c):
        x, s = a.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)
        out, h = G.gated_linear_scan(x, s, activation="identity", reset=r)
        return (out, h, *torch.autograd.grad((out, h), (x, s), (c.to(dev), dh.to(dev))))

    out, h, dgi, dh0 = both(bad, bad_h0, bad_d)
    o, hl, dg, d0 = both(gi, h0, dout)
    assert torch.equal(out[cut:], o[cut:]) and torch.equal(h, hl) and torch.equal(out[:, 1], o[:, 1])
    assert not out[:cut, 0].isfinite().all() and out[:3, 0, [0, 1, 2, 3, 4, 6, 9, 39]].isfinite().all()
    # the gradient's NaN (channel 9, after the cut) stays after it; h0's and gi's stay before
    assert torch.equal(dgi[cut:, 0, :9], dg[cut:, 0, :9]) and torch.equal(dgi[:, 1], dg[:, 1])
    assert torch.equal(dgi[:cut, 0, 9], dg[:cut, 0, 9]) and dgi[cut:cut + 3, 0, 9].isnan().all()
    assert torch.equal(dh0[0, 9:], d0[0, 9:])


def test_nan_is_carried(dev):
    """A NaN stays in its channel to the end where nothing resets it, over tiles and segments."""
    gi, h0, _, _, _ = _inputs(1300, 1, 40, torch.float32, seed=8)
    gi[700, 0, 11] = float("nan")
    out, h = G.gated_linear_scan(gi.to(dev), h0.to(dev))
    assert out[700:, 0, 11].isnan().all() and h[0, 11].isnan() and out[:700].isfinite().all()
    keep = torch.arange(40, device=dev) != 11
    assert out[:, 0, keep].isfinite().all()


def test_other_stream(dev):
    gi, h0, _, _, _ = _inputs(1300, 1, 64, torch.float32, seed=9)
    a, b = gi.to(dev), h0.to(dev)
    want = G.gated_linear_scan(a, b)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = G.gated_linear_scan(a, b)[0]
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ["tanh", "identity"])
@pytest.mark.parametrize("H", [1, 33, 256, 700])
def test_step(dev, H, act, dtype):
    g = torch.Generator().manual_seed(H)
    S, slots = 9, [4, -1, 0, 8, 9, 2, -7]
    gi = torch.randn(len(slots), 2 * H, generator=g).to(dtype)
    state = torch.randn(S, H + 3, generator=g)
    cache = state.to(dev)[:, 1:1 + H]
    out = G.gated_linear_step(gi.to(dev), cache, torch.tensor(slots, dtype=torch.int32, device=dev), activation=act)
    before = state[:, 1:1 + H]
    after = before.double().clone()
    for b, s in enumerate(slots):
        if not 0 <= s < S:
            assert (out[b] == 0).all() if s < 0 else out[b].isnan().all()
            continue
        (o, e), _ = _oracle(gi[b][None, None], before[s][None], None, act)
        after[s] = o[0, 0]
        _near(cache[s], o[0, 0], e[0, 0], "state")
        _near(out[b], o[0, 0], e[0, 0] * 2 + (U16 * o[0, 0].abs() if dtype == torch.bfloat16 else 0), "out")
    rest = [s for s in range(S) if s not in slots]
    assert torch.equal(cache[rest].cpu(), before[rest])


# long axes of many channels: a tile of 128 steps by 32 lanes, the last one of each partly filled
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1025, 8, 65), (1100, 4, 258), (2100, 9, 130), (2200, 8, 135)], ids=str)
def test_long_axes_of_many_channels(dev, shape, dtype):
    _check(dev, *_inputs(*shape, dtype, seed=sum(shape), p_reset=0.01 if shape[0] % 2 else 0.0), "tanh")


def test_step_equals_a_scan_of_one(dev):
    gi = torch.randn(5, 80, device=dev)
    state = torch.randn(5, 40, device=dev)
    out, h = G.gated_linear_scan(gi[None], state)
    version = state._version
    got = G.gated_linear_step(gi, state)
    assert torch.equal(got, out[0]) and torch.equal(state, h) and state._version > version


def test_second_derivatives_are_refused(dev):
    gi, h0, _, _, _ = _inputs(5, 2, 7, torch.float32, seed=31)
    gi, h0 = gi.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    plain = torch.autograd.grad(G.gated_linear_scan(gi, h0)[0].sum(), (gi, h0))
    graph = torch.autograd.grad(G.gated_linear_scan(gi, h0)[0].sum(), (gi, h0), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graph))
    with pytest.raises(RuntimeError, match="gated_linear_scan: second derivatives"):
        torch.autograd.grad(graph[0].square().sum(), gi)
    alone, = torch.autograd.grad(G.gated_linear_scan(gi)[1].sum(), gi, create_graph=True)
    with pytest.raises(RuntimeError, match="gated_linear_scan: second derivatives"):
        alone.sum().backward()


def test_refusals(dev):
    gi, h0 = torch.randn(4, 2, 6, device=dev), torch.zeros(2, 3, device=dev)
    f, s = G.gated_linear_scan, G.gated_linear_step
    for call in (lambda: f(gi.cpu(), h0), lambda: f(gi, h0.cpu()), lambda: f(gi.half(), h0), lambda: f(gi[..., :5], h0),
                 lambda: f(gi[0], h0), lambda: f(gi[:0], h0), lambda: f(gi[:, :0], h0[:0]), lambda: f(gi, h0[:1]),
                 lambda: f(gi, h0.double()), lambda: f(gi, h0, activation="relu"), lambda: f(gi, h0, activation=None),
                 lambda: f(gi, h0, reset=torch.zeros(4, 2, device=dev)),
                 lambda: f(gi, h0, reset=torch.zeros(2, 4, dtype=torch.bool, device=dev)),
                 lambda: f(gi, h0, reset=torch.zeros(4, 2, dtype=torch.bool)),
                 lambda: s(gi, h0), lambda: s(gi[0], h0.double()), lambda: s(gi[0], h0[:1]),
                 lambda: s(gi[0], torch.zeros(3, 2, device=dev).t()),
                 lambda: s(gi[0], h0, torch.zeros(2, dtype=torch.int64, device=dev)),
                 lambda: s(gi[0], h0, torch.zeros(3, dtype=torch.int32, device=dev)),
                 lambda: s(gi[0], h0, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
