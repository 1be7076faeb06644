"""The gated linear recurrence where states, candidates or gradients are infinite, where
tiles follow each other, and where chained tiles hand states on. Bounds are those of the
operator's own tests."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import test_gpu_gated_linear as scan

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES, IDS = [F32, BF16], ["f32", "bf16"]


def _same_kind(got, want, what):
    """NaN where the formula has NaN, each infinity where it has that one, finite elsewhere."""
    got, want = got.detach().cpu().double(), want.double()
    for name, f in (("NaN", torch.isnan), ("inf", torch.isposinf), ("-inf", torch.isneginf)):
        assert torch.equal(f(got), f(want)), f"{what}: {name} at other places than in the formula"
    return got.isfinite()


# Each layout: a wave a row (float32), four waves, eight waves by 32 lanes (float32, bfloat16) and by 16, and
# tiles chained in two widths.
INFINITE = [(20, 700, 130), (100, 20, 701), (300, 20, 300), (150, 20, 601), (300, 2, 40), (1300, 1, 40), (1200, 8, 140)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", INFINITE, ids=str)
def test_infinite_candidates_and_states(dev, shape, dtype):
    """(1 - z) n is infinite with n, and a state that is infinite stays so, also over spans of steps whose z
    multiply to less than the smallest float."""
    T, B, H = shape
    gi, h0, _, dout, dh = scan._inputs(T, B, H, dtype, seed=T)
    inf = float("inf")
    gi[3, 0, H], gi[5, 0, H + 1], gi[T - 4, 0, H + 2], h0[1 % B, 0] = inf, -inf, inf, inf
    gi[9, 0, H + 1] = -inf  # the same infinity again
    gi[11, 0, H] = -inf     # the other one: NaN from here on
    x, s = gi.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    out, last = G.gated_linear_scan(x, s, activation="identity")
    dgi, dh0 = torch.autograd.grad((out, last), (x, s), (dout.to(dev), dh.to(dev)))
    (o, e), (hl, _), (dg, _), (d0, _), _, _ = scan._oracle(gi, h0, None, "identity", dout, dh)
    ok = _same_kind(out, o, "out")
    _same_kind(last, hl, "h_T")
    _same_kind(dgi, dg, "dgi")
    _same_kind(dh0, d0, "dh0")
    u = 2.0 ** -8 if dtype == BF16 else 0.0
    assert ((out.detach().cpu().double() - o).abs()[ok] <= (e * (1 + u) + u * o.abs())[ok]).all()


@pytest.mark.parametrize("shape", INFINITE, ids=str)
def test_infinite_gradients(dev, shape):
    T, B, H = shape
    gi, h0, _, dout, dh = scan._inputs(T, B, H, F32, seed=T + 1)
    dout[T - 3, 0, 0], dh[0, 1] = float("inf"), -float("inf")
    x, s = gi.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    out, last = G.gated_linear_scan(x, s)
    dgi, dh0 = torch.autograd.grad((out, last), (x, s), (dout.to(dev), dh.to(dev)))
    _, _, (dg, _), (d0, _), _, _ = scan._oracle(gi, h0, None, "tanh", dout, dh)
    _same_kind(dgi, dg, "dgi")
    _same_kind(dh0, d0, "dh0")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_step_with_infinities(dev, dtype):
    inf = float("inf")
    gi = torch.tensor([[0.5, 0.5, 20.0, 0.5, 0.5, inf, -inf, inf, -inf, 0.25]]).to(dtype)
    state = torch.tensor([[1.0, 2.0, 3.0, inf, inf]])
    want, _ = scan._oracle(gi[None], state, None, "identity")
    cache = state.to(dev)
    out = G.gated_linear_step(gi.to(dev), cache, activation="identity")
    _same_kind(out, want[0][0], "out")
    _same_kind(cache, want[0][0], "state")


def test_an_axis_past_a_launch(dev):
    """2^28 steps and more are walked, not chained: the end, after a reset, is that of the end alone."""
    T, tail = (1 << 28) + 5, 700
    gi, h0, _, _, _ = scan._inputs(tail, 1, 1, F32, seed=3)
    long = torch.zeros(T, 1, 2, device=dev)
    long[-tail:] = gi.to(dev)
    reset = torch.zeros(T, 1, dtype=torch.bool, device=dev)
    reset[-tail] = True
    out, last = G.gated_linear_scan(long, torch.ones(1, 1, device=dev), reset=reset)
    (o, e), (hl, el) = scan._oracle(gi, torch.zeros(1, 1), None, "tanh")
    scan._near(out[-tail:], o, e, "out")
    scan._near(last, hl, el, "h_T")
    assert (out[:30, 0, 0].cpu() == 2.0 ** -torch.arange(1.0, 31)).all() and not out[200:-tail].any()


# Walked layouts over four tiles and more, so that both LDS buffers are written again: four waves (tiles of 32
# steps), eight by 32 lanes (128) and eight by 16 (256); odd channel counts, and even ones that bfloat16 takes in pairs.
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("p", [0.0, 0.03], ids=["", "resets"])
@pytest.mark.parametrize("shape", [(140, 20, 701), (140, 20, 1402), (500, 20, 301), (500, 20, 600), (1000, 10, 301),
                                   (1000, 10, 600)], ids=str)
def test_many_tiles(dev, shape, p, dtype):
    scan._check(dev, *scan._inputs(*shape, dtype, seed=sum(shape), p_reset=p), "tanh")


def _check_linked(dev, gi, h0, reset, dout, dh, nans):
    """scan._check with NaN where the formula has it (and nowhere else), whose bounds a reset ends too."""
    dtype, H = gi.dtype, h0.shape[1]
    for t, b, j in nans["gi"]:
        gi[t, b, j] = float("nan")
    for t, b, j in nans["dout"]:
        dout[t, b, j] = float("nan")
    x, s = gi.to(dev).requires_grad_(True), h0.to(dev).requires_grad_(True)
    out, last = G.gated_linear_scan(x, s, reset=None if reset is None else reset.to(dev))
    dgi, dh0 = torch.autograd.grad((out, last), (x, s), (dout.to(dev), dh.to(dev)))
    (o, eo), (hl, el), (dg, edg), (d0, e0), hp, z = scan._oracle(gi, h0, reset, "tanh", dout, dh)
    if dtype == BF16:
        u, size, run = scan.U16, torch.empty_like(o), dh.double().abs()
        for t in range(o.shape[0] - 1, -1, -1):
            if t + 1 < o.shape[0]:
                run = run * z[t + 1]
                if reset is not None:
                    run = torch.where(reset[t + 1][:, None], 0.0, run)
            size[t] = run = run + dout[t].double().abs()
        edg[..., :H] += u * hp.abs() * size * z * (1 - z)
        eo, edg = eo * (1 + u) + u * o.abs(), edg * (1 + u) + u * dg.abs()
    for got, want, bound, what in ((out, o, eo, "out"), (last, hl, el, "h_T"), (dgi, dg, edg + 1e-38, "dgi"),
                                   (dh0, d0, e0 + 1e-38, "dh0")):
        ok = _same_kind(got, want, what)
        off = (got.detach().cpu().double() - want).abs()
        assert (off[ok] <= bound[ok]).all(), what


# 50 tiles and a part: chained tiles of 16 lanes are 256 steps, of 32 lanes 128, and every 16th publishes its state.
# Few channels take 16 lanes, from 512 on (pairs of them in bfloat16, backwards only) 32.
LINKED = [(50 * 256 + 9, 3, 20, 256), (50 * 256, 3, 21, 256), (50 * 128 + 9, 2, 270, 128), (50 * 128, 4, 270, 128)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("resets", ["none", "at links", "many"])
@pytest.mark.parametrize("shape", LINKED, ids=str)
def test_chains_over_links(dev, shape, resets, dtype):
    """States handed on over three links, and NaN that a reset before or after a link stops, from both ends."""
    T, B, H, tile = shape
    link = 16 * tile
    gi, h0, reset, dout, dh = scan._inputs(T, B, H, dtype, seed=T + H, p_reset=0.002 if resets == "many" else 0.0)
    nans = dict(gi=[], dout=[])
    if resets == "at links":
        reset = torch.zeros(T, B, dtype=torch.bool)
        # row 0: in the last tile before a link, NaN before it; the group of links after that has none
        reset[link - 100, 0] = True
        nans["gi"] += [(link - 110, 0, 3), (link - 110, 0, H + 4)]
        # row 1: in the first tile after a link, the NaN before the link
        reset[2 * link + 10, 1] = True
        nans["gi"] += [(2 * link - 7, 1, 0), (2 * link - 7, 1, H + H - 1)]
        # the same from the end, where the backward's links are
        reset[T - 1 - (link - 100), 1] = True
        nans["dout"] += [(T - 1 - (link - 110), 1, 5)]
        reset[T - 1 - (2 * link + 10), 0] = True
        nans["dout"] += [(T - 1 - (2 * link - 7), 0, 2)]
    _check_linked(dev, gi, h0, reset, dout, dh, nans)
