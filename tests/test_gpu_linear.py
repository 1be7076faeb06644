"""linear_act (gs_linear_fwd / gs_linear_bwd) against its formula in 64 bits.

Tolerances: u is float32's unit roundoff (2^-24), U that of the tensors' type (2^-24 or
2^-8). A sum of K products in float32, in any order, is within 2 (K + 2) u of the sum of
their magnitudes. Activations have slopes of at most 1.2 and second derivatives of at
most 1, and are computed within 16 u of |argument| + 1. Each output rounds to its type
once; the backward reads pre rounded to the type, and dpre is an operand rounded to it.
"""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}
ACTS = ["none", "relu", "gelu", "silu", "tanh", "sigmoid"]
TYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def _act(pre, act):
    """value and slope in float64"""
    if act == "none":
        return pre, torch.ones_like(pre)
    p = pre.clone().requires_grad_(True)
    f = dict(relu=torch.relu, gelu=torch.nn.functional.gelu, silu=torch.nn.functional.silu, tanh=torch.tanh,
             sigmoid=torch.sigmoid)[act]
    with torch.enable_grad():
        y = f(p)
        slope, = torch.autograd.grad(y, p, torch.ones_like(y))
    return y.detach(), slope


def _near(got, want, bound, what):
    assert got.shape == want.shape, what
    off = (got.detach().double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {off.max()} off, {(off / bound).max()} of the bound"


def _check(x, w, bias, res, dy, act, got):
    """got: (y, dx, dw, dbias) of the call (gradients may be missing)."""
    U = UNIT[x.dtype]
    M, K = x.shape
    N = w.shape[0]
    x, w, dy = (t.detach().double() for t in (x, w, dy))
    pre = x @ w.t()
    e = 2 * (K + 2) * U32 * (x.abs() @ w.abs().t())
    if bias is not None:
        pre = pre + bias.detach().double()
        e = e + 2 * U32 * bias.detach().double().abs()
    y, slope = _act(pre, act)
    ey = 1.2 * e + (16 * U32 * (pre.abs() + 1) if act != "none" else 0.0)
    if res is not None:
        y = y + res.detach().double()
        ey = ey + U32 * (y.abs() + res.detach().double().abs())
    _near(got[0], y, ey * (1 + U) + U * y.abs(), "y")
    if len(got) == 1:
        return
    ep = e + U * pre.abs() if act != "none" else torch.zeros_like(pre)
    es = ep + 16 * U32 * (1 + pre.abs()) if act != "none" else ep
    if act == "relu":
        es = (pre.abs() <= e).double() + 2 * U32
    d = dy * slope
    raw = dy.abs() * es
    ed = raw * (1 + U) + (U * d.abs() if act != "none" else 0.0)
    dx, dw, db = d @ w, d.t() @ x, d.sum(0)
    _near(got[1], dx, (ed @ w.abs() + 2 * (N + 2) * U32 * (d.abs() @ w.abs())) * (1 + U) + U * dx.abs() + 1e-38, "dx")
    _near(got[2], dw, (ed.t() @ x.abs() + 2 * (M + 2) * U32 * (d.abs().t() @ x.abs())) * (1 + U) + U * dw.abs() + 1e-38, "dw")
    if bias is not None:
        _near(got[3], db, (raw.sum(0) + 2 * (M + 2) * U32 * d.abs().sum(0)) * (1 + U) + U * db.abs() + 1e-38, "dbias")


def _inputs(dev, M, N, K, dtype, seed, bias=True, res=True):
    g = torch.Generator().manual_seed(seed)

    def new(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)

    return (new(M, K), new(N, K, scale=K ** -0.5), new(N) if bias else None, new(M, N) if res else None, new(M, N))


def _call(x, w, bias, res, dy, act):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, bias) if t is not None]
    y = G.linear_act(leaves[0], leaves[1], leaves[2] if bias is not None else None, activation=act, residual=res)
    grads = torch.autograd.grad(y, leaves, dy)
    plain = G.linear_act(x, w, bias, activation=act, residual=res)
    assert torch.allclose(y, plain, rtol=0, atol=0, equal_nan=True) and y.dtype == plain.dtype == x.dtype
    return (y, *grads)


# around the tiles of 64 and 128, slices of 64 k, 16-byte rows and splits of K
SHAPES = [(1, 1, 1), (1, 5, 3), (3, 17, 8), (8, 64, 64), (16, 130, 33), (65, 64, 65), (64, 128, 128), (129, 136, 127),
          (200, 96, 1000), (31, 47, 1030), (32, 96, 4096), (33, 33, 256), (333, 257, 301), (7, 2048, 1024), (17, 515, 2050), (700, 520, 264), (2100, 40, 24)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(dev, shape, dtype):
    args = _inputs(dev, *shape, dtype, seed=sum(shape))
    act = ACTS[sum(shape) % len(ACTS)]
    _check(*args, act, _call(*args, act))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("res", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("bias", [False, True], ids=["", "bias"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(33, 70, 45), (130, 136, 72), (9, 72, 600)], ids=str)
def test_epilogues(dev, shape, act, bias, res, dtype):
    args = _inputs(dev, *shape, dtype, seed=7, bias=bias, res=res)
    _check(*args, act, _call(*args, act))


@pytest.mark.parametrize("shape", [(3600, 3848, 72), (3600, 72, 3848), (72, 3600, 3848)], ids=str)
@pytest.mark.parametrize("cut", [0, 3])
def test_many_tiles(dev, shape, cut):
    """Enough tiles for the largest tile in the forward, in dx and in dw; and the same with odd sizes."""
    M, N, K = (s - cut for s in shape)
    args = _inputs(dev, M, N, K, torch.bfloat16, seed=8)
    _check(*args, "gelu", _call(*args, "gelu"))


@pytest.mark.parametrize("shape", [(20, 4104, 33), (32, 4096, 40), (5, 8200, 16), (16, 8192, 16), (8, 40, 2056), (8, 40, 2048)],
                         ids=str)
def test_few_rows_of_wide_and_long_layers(dev, shape):
    args = _inputs(dev, *shape, torch.bfloat16, seed=13)
    _check(*args, "silu", _call(*args, "silu"))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_strides_and_alignment(dev, dtype):
    M, N, K = 70, 72, 64
    x, w, bias, res, dy = _inputs(dev, 3 * M, N, 3 * K, dtype, seed=9)
    w = torch.randn(N, 3 * K, generator=torch.Generator().manual_seed(10)).to(dtype).to(dev)
    for views in (
        (x[:M, 5:5 + K], w[:, 3:3 + K], bias, res[:M], dy[:M]),  # rows off 16 bytes; a weight that is no block
        (x[::3, :K], w[:, :K], bias, res[::3], dy[::3]),
        (x[:K, :M].t(), w[:, :K], bias, res[:M].t().contiguous().t(), dy[:M].t().contiguous().t()),
        (x[:1, :K].expand(M, K), w[:, :K], bias, res[:1].expand(M, N), dy[:1, :1].expand(M, N)),
    ):
        _check(*views, "silu", _call(*views, "silu"))


def test_leading_dimensions_and_needed_gradients(dev):
    x, w, bias, _, _ = _inputs(dev, 30, 24, 20, torch.float32, seed=11)
    x3, res = x.view(2, 3, 5, 20), torch.randn(2, 3, 5, 24, device=dev, requires_grad=True)
    dy = torch.randn(2, 3, 5, 24, device=dev)
    y = G.linear_act(x3, w, bias, activation="tanh", residual=res)
    dres, = torch.autograd.grad(y, res, dy)
    assert y.shape == (2, 3, 5, 24) and torch.equal(dres, dy)
    full = _call(x, w, bias, res.detach().view(30, 24), dy.view(30, 24), "tanh")
    for k in range(3):  # each gradient alone is the one of the whole call
        leaves = [x, w, bias]
        leaves[k] = leaves[k].detach().requires_grad_(True)
        got, = torch.autograd.grad(G.linear_act(*leaves, activation="tanh", residual=res.detach().view(30, 24)), leaves[k],
                                   dy.view(30, 24))
        assert torch.equal(got, full[1 + k])


def test_gradient_of_a_broadcast_residual(dev):
    x, w, bias, _, dy = _inputs(dev, 40, 24, 20, torch.float32, seed=12)
    r = torch.randn(1, 24, device=dev, requires_grad=True)
    got, = torch.autograd.grad(G.linear_act(x, w, bias, residual=r.expand(40, 24)), r, dy)
    want = dy.double().sum(0, keepdim=True)
    assert ((got.double() - want).abs() <= 2 * 42 * U32 * dy.double().abs().sum(0)).all()


def test_gradient_against_differences(dev):
    """Central differences with a step of 2^-6 of a sum weighted by about 1: their own error is under
    2^-12 / 6 of the third derivative (at most 2 here, over 5 outputs a weight or input), rounding
    30 u / 2^-6."""
    x, w, bias, res, dy = _inputs(dev, 6, 5, 4, torch.float32, seed=13)
    for act in ("gelu", "silu", "tanh", "sigmoid"):
        _, *grads = _call(x, w, bias, res, dy, act)
        for t, g in zip((x, w, bias), grads):
            for at in range(t.numel()):
                keep = t.view(-1)[at].item()
                sums = []
                for k in (1, -1):
                    t.view(-1)[at] = keep + k * 2.0 ** -6
                    sums.append((G.linear_act(x, w, bias, activation=act, residual=res).double() * dy).sum().item())
                t.view(-1)[at] = keep
                assert abs((sums[0] - sums[1]) * 2.0 ** 5 - g.view(-1)[at].item()) < 2.0 ** -7


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_bad_values_stay_in_their_rows(dev, dtype):
    """NaN and infinities of one row of x, one column of a padded edge, reach that row alone."""
    x, w, bias, res, dy = _inputs(dev, 70, 67, 65, dtype, seed=14)
    clean = _call(x, w, bias, res, dy, "relu")
    x[40, 64], x[41, 0] = float("nan"), float("inf")
    y, dx, dw, db = _call(x, w, bias, res, dy, "relu")
    keep = torch.tensor([i not in (40, 41) for i in range(70)], device=dev)
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert y[40].isnan().all()


def test_same_inputs_same_results(dev):
    args = _inputs(dev, 1000, 264, 520, torch.bfloat16, seed=15)
    a, b = _call(*args, "gelu"), _call(*args, "gelu")
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_second_derivatives_are_refused(dev):
    x, w, bias, res, _ = _inputs(dev, 6, 9, 5, torch.float32, seed=31)
    leaves = [t.requires_grad_(True) for t in (x, w, bias, res)]
    y = G.linear_act(x, w, bias, activation="silu", residual=res)
    plain = torch.autograd.grad(y.sum(), leaves)
    y = G.linear_act(x, w, bias, activation="silu", residual=res)
    graph = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graph))
    with pytest.raises(RuntimeError, match="linear_act: second derivatives"):
        torch.autograd.grad(graph[0].square().sum(), w)
    alone, = torch.autograd.grad(G.linear_act(x, w.detach()).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="linear_act: second derivatives"):
        alone.sum().backward()


def test_refusals(dev):
    x, w, bias, res, _ = _inputs(dev, 6, 5, 4, torch.float32, seed=16)
    f = G.linear_act
    for call in (lambda: f(x.cpu(), w), lambda: f(x, w.cpu()), lambda: f(x, w, bias.cpu()), lambda: f(x.half(), w.half()),
                 lambda: f(x, w.bfloat16()), lambda: f(x, w, bias.bfloat16()), lambda: f(x, w.t()), lambda: f(x, w[0]),
                 lambda: f(x[:0], w), lambda: f(x, w[:0]), lambda: f(x, w, bias[:4]), lambda: f(x, w, residual=res[:5]),
                 lambda: f(x, w, residual=bias), lambda: f(x, w, activation="swish"), lambda: f(x, w, activation=None)):
        with pytest.raises(ValueError):
            call()
