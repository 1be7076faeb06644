"""The operators over sequences of tokens without a GPU: what the C ABI refuses before any device
work, its size queries, the Python entry points' errors, and the plain definitions that the
GPU tests compare with against autograd in 64 bits and torch's own functions."""

from __future__ import annotations

import ctypes

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P
from gru_qat_amd import _lib

FAKE = 4096  # never dereferenced: validation fails before any device access


def _conv(**kw):
    return _set(_lib.GsConvArgs(x=FAKE, w=FAKE, y=FAKE, T=4, B=3, C=8, W=4, sx_t=24, sx_b=8, sy_t=24, sy_b=8), kw)


def _conv_bwd(**kw):
    return _set(_lib.GsConvBwdArgs(x=FAKE, w=FAKE, dy=FAKE, dx=FAKE, T=4, B=3, C=8, W=4, sx_t=24, sx_b=8, sdy_t=24, sdy_b=8,
                                   sdx_t=24, sdx_b=8), kw)


def _conv_step(**kw):
    return _set(_lib.GsConvStepArgs(x=FAKE, w=FAKE, state=FAKE, y=FAKE, B=3, C=8, W=4, S=3, sx=8, ss=24, sy=8), kw)


_SSM = dict(u=FAKE, delta=FAKE, bm=FAKE, cm=FAKE, A=FAKE, T=4, B=3, H=8, N=16, su_t=24, su_b=8, sdl_t=24, sdl_b=8, sb_t=48,
            sb_b=16, sc_t=48, sc_b=16)


def _ssm(**kw):
    return _set(_lib.GsSsmArgs(y=FAKE, sy_t=24, sy_b=8, **_SSM), kw)


def _ssm_bwd(**kw):
    return _set(_lib.GsSsmBwdArgs(saved=FAKE, dy=FAKE, du=FAKE, ddelta=FAKE, sdy_t=24, sdy_b=8, sdu_t=24, sdu_b=8, sdd_t=24,
                                  sdd_b=8, **_SSM), kw)


def _ssm_step(**kw):
    return _set(_lib.GsSsmStepArgs(u=FAKE, delta=FAKE, bm=FAKE, cm=FAKE, A=FAKE, state=FAKE, y=FAKE, B=3, H=8, N=16, S=3, su=8,
                                   sdl=8, sb=16, sc=16, ss=128, sy=8), kw)


def _embedding(**kw):
    return _set(_lib.GsEmbeddingArgs(tokens=FAKE, w=FAKE, out=FAKE, M=4, V=5, K=8, so=8, scale=1.0, token_bits=64), kw)


def _embedding_bwd(**kw):
    return _set(_lib.GsEmbeddingBwdArgs(tokens=FAKE, dout=FAKE, dw=FAKE, M=4, V=5, K=8, sdo=8, scale=1.0, token_bits=64), kw)


def _logprobs(**kw):
    return _set(_lib.GsLogprobsArgs(x=FAKE, tokens=FAKE, logprob=FAKE, entropy=FAKE, M=4, V=50, sx=50, token_bits=64), kw)


def _logprobs_bwd(**kw):
    return _set(_lib.GsLogprobsBwdArgs(x=FAKE, tokens=FAKE, entropy=FAKE, stats=FAKE, dx=FAKE, M=4, V=50, sx=50, sdx=50,
                                       token_bits=64), kw)


def _set(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


STEPS = [dict(T=0), dict(B=0), dict(T=-1), dict(T=2 ** 31), dict(B=2 ** 31), dict(dtype=2), dict(dtype=-1)]
SLOTS = [dict(B=0), dict(S=0), dict(S=2), dict(ss=7), dict(sy=7), dict(B=70000, S=70000), dict(dtype=3), dict(state=0)]
REFUSED = (
    [("gs_conv_fwd", _conv, kw) for kw in STEPS + [dict(C=0), dict(C=2 ** 21), dict(W=1), dict(W=5), dict(x=0), dict(w=0), dict(y=0),
                                                   dict(activation=1), dict(sx_t=-1), dict(sr_t=-1), dict(sy_t=8), dict(sy_b=7)]]
    + [("gs_conv_bwd", _conv_bwd, kw) for kw in STEPS + [dict(C=0), dict(W=1), dict(dy=0), dict(dx=0), dict(activation=2),
                                                         dict(sdy_b=-1), dict(sdx_t=8), dict(sdx_b=7)]]
    + [("gs_conv_step", _conv_step, kw) for kw in SLOTS + [dict(x=0), dict(w=0), dict(y=0), dict(W=5), dict(sx=-1)]]
    + [("gs_ssm_fwd", _ssm, kw) for kw in STEPS + [dict(H=0), dict(N=0), dict(N=33), dict(H=2 ** 21), dict(u=0), dict(delta=0),
                                                   dict(A=0), dict(bm=0), dict(cm=0), dict(y=0), dict(su_t=-1), dict(sdl_b=-1),
                                                   dict(sz_t=-1), dict(sb_t=-1), dict(sc_b=-1), dict(sr_b=-1), dict(sy_t=8),
                                                   dict(B=2 ** 20, H=2 ** 20)]]
    + [("gs_ssm_bwd", _ssm_bwd, kw) for kw in STEPS + [dict(H=0), dict(N=33), dict(saved=0), dict(dy=0), dict(du=0), dict(ddelta=0),
                                                       dict(sdy_t=-1), dict(sdu_t=8), dict(sdd_b=7), dict(z=FAKE, sdz_t=24, sdz_b=8),
                                                       dict(z=FAKE, dz=FAKE, sdz_t=8, sdz_b=8)]]
    + [("gs_ssm_step", _ssm_step, kw) for kw in SLOTS + [dict(H=0), dict(N=0), dict(u=0), dict(A=0), dict(cm=0), dict(y=0),
                                                         dict(ss=127), dict(sb=-1)]]
    + [("gs_embedding_fwd", _embedding, kw) for kw in [dict(M=0), dict(V=0), dict(K=0), dict(M=2 ** 26), dict(V=2 ** 26),
                                                       dict(tokens=0), dict(w=0), dict(out=0), dict(token_bits=16), dict(so=7),
                                                       dict(dtype=2), dict(scale=float("nan")), dict(scale=float("inf"))]]
    + [("gs_embedding_bwd", _embedding_bwd, kw) for kw in [dict(M=0), dict(V=-1), dict(K=0), dict(tokens=0), dict(dout=0), dict(dw=0),
                                                           dict(sdo=7), dict(token_bits=0), dict(dtype=-1)]]
    + [("gs_logprobs_fwd", _logprobs, kw) for kw in [dict(M=0), dict(V=0), dict(M=2 ** 24), dict(V=2 ** 25), dict(x=0), dict(tokens=0),
                                                     dict(logprob=0), dict(entropy=0), dict(top=-1), dict(top=33), dict(top=4, V=3),
                                                     dict(top=4), dict(top=4, V=2 ** 20), dict(top=1, M=2 ** 22, V=2 ** 19),
                                                     dict(sx=-1), dict(token_bits=8), dict(dtype=2)]]
    + [("gs_logprobs_bwd", _logprobs_bwd, kw) for kw in [dict(M=0), dict(V=0), dict(x=0), dict(stats=0), dict(entropy=0), dict(dx=0),
                                                         dict(sdx=49), dict(token_bits=8), dict(dtype=2)]]
)


@pytest.mark.parametrize("fn,make,kw", REFUSED, ids=[f"{f}-{k}" for f, _, k in REFUSED])
def test_refused_before_any_device_work(fn, make, kw):
    lib = _lib.load()
    assert getattr(lib, fn)(ctypes.byref(make(**kw)), None) == _lib.GS_ERR_INVALID
    assert fn.encode() in lib.gs_last_error()


@pytest.mark.parametrize("fn", sorted({f for f, _, _ in REFUSED}))
def test_null_arguments(fn):
    assert getattr(_lib.load(), fn)(None, None) == _lib.GS_ERR_INVALID


@pytest.mark.parametrize("fn,query,args", [
    ("gs_conv_bwd", "gs_conv_bwd_scratch_bytes", _conv_bwd()),
    ("gs_ssm_fwd", "gs_ssm_scratch_bytes", _ssm(T=500)),
    ("gs_ssm_bwd", "gs_ssm_bwd_scratch_bytes", _ssm_bwd()),
    ("gs_embedding_bwd", "gs_embedding_bwd_scratch_bytes", _embedding_bwd()),
    ("gs_logprobs_fwd", "gs_logprobs_scratch_bytes", _logprobs(V=20000, sx=20000)),
    ("gs_logprobs_fwd", "gs_logprobs_scratch_bytes", _logprobs(top=3, top_logprob=FAKE, top_token=FAKE)),
], ids=str)
def test_missing_scratch(fn, query, args):
    lib = _lib.load()
    need = getattr(lib, query)(ctypes.byref(args))
    assert need > 0
    for scratch, nbytes in ((0, 0), (FAKE, 16), (FAKE + 8, need)):
        args.scratch, args.scratch_bytes = scratch, nbytes
        assert getattr(lib, fn)(ctypes.byref(args), None) == _lib.GS_ERR_INVALID
        assert b"scratch" in lib.gs_last_error()


def test_size_queries():
    lib = _lib.load()
    for query, a in (("gs_conv_bwd_scratch_bytes", _conv_bwd(T=0)), ("gs_ssm_scratch_bytes", _ssm(N=0)), ("gs_ssm_saved_bytes", _ssm(H=0)),
                     ("gs_ssm_bwd_scratch_bytes", _ssm_bwd(B=0)), ("gs_embedding_bwd_scratch_bytes", _embedding_bwd(V=0)),
                     ("gs_logprobs_scratch_bytes", _logprobs(top=40))):
        assert getattr(lib, query)(ctypes.byref(a)) == _lib.GS_ERR_INVALID
        assert getattr(lib, query)(None) == _lib.GS_ERR_INVALID
    assert lib.gs_ssm_scratch_bytes(ctypes.byref(_ssm())) == 0  # short axes are not cut
    assert lib.gs_ssm_saved_bytes(ctypes.byref(_ssm(T=33))) == 3 * 3 * 16 * 8 * 4
    assert lib.gs_logprobs_scratch_bytes(ctypes.byref(_logprobs())) == 0


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: G.causal_conv(_t(4, 2, 6), _t(6, 4)),
    lambda: G.causal_conv(None, _t(6, 4)),
    lambda: G.causal_conv(_t(4, 2, 6), _t(6, 4), activation="gelu"),
    lambda: G.causal_conv(_t(4, 2, 6), _t(6, 4), reset=[1]),
    lambda: G.causal_conv_step(_t(2, 6), _t(6, 4), None, _t(2, 3, 6)),
    lambda: G.causal_conv_step(_t(2, 6), _t(6, 4), None, None),
    lambda: G.causal_conv_step(_t(2, 6), _t(6, 4), None, _t(2, 3, 6), activation=3),
    lambda: G.selective_scan(_t(4, 2, 6), _t(4, 2, 6), _t(6, 16), _t(4, 2, 16), _t(4, 2, 16)),
    lambda: G.selective_scan(_t(4, 2, 6), 1.0, _t(6, 16), _t(4, 2, 16), _t(4, 2, 16)),
    lambda: G.selective_step(_t(2, 6), _t(2, 6), _t(6, 16), _t(2, 16), _t(2, 16), _t(2, 6, 16)),
    lambda: G.selective_step(_t(2, 6), _t(2, 6), _t(6, 16), _t(2, 16), _t(2, 16), None),
    lambda: G.embedding(torch.zeros(3, dtype=torch.long), _t(5, 4)),
    lambda: G.embedding([1, 2], _t(5, 4)),
    lambda: G.embedding(torch.zeros(3, dtype=torch.long), _t(5, 4), scale="x"),
    lambda: G.token_logprobs(_t(3, 5), torch.zeros(3, dtype=torch.long)),
    lambda: G.token_logprobs(_t(3, 5), None),
    lambda: G.token_logprobs(_t(3, 5), torch.zeros(3, dtype=torch.long), top=1.5),
    lambda: G.SelectiveLayer(0, 8),
    lambda: G.SelectiveLayer(8, 8, rank=0),
    lambda: G.SelectiveLayer(8, 8, states=33),
    lambda: G.SelectiveLayer(8, 8, taps=1),
], ids=range(21))
def test_python_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_layer_starts_where_it_says():
    torch.manual_seed(0)
    layer = G.SelectiveLayer(12, 40, states=5, dtype=torch.bfloat16)
    step = torch.nn.functional.softplus(layer.bias_d)
    assert (step >= 0.999e-3).all() and (step <= 0.1001).all() and layer.bias_d.dtype == torch.float32
    assert torch.allclose(torch.exp(layer.A_log[7]), torch.arange(1.0, 6.0)) and layer.rank == 3
    state = layer.new_state(4)
    assert state.conv.shape == (4, 3, 40) and state.conv.dtype == torch.bfloat16
    assert state.ssm.shape == (4, 40, 5) and state.ssm.dtype == torch.float32


# ---- the plain definitions ------------------------------------------------------------------


def test_plain_scan_gradients():
    g = torch.Generator().manual_seed(0)
    T, B, H, N = 12, 2, 5, 3

    def r(*s):
        return torch.randn(s, generator=g).double()

    t = dict(u=r(T, B, H), delta=r(T, B, H), A=-r(H, N).exp(), B=r(T, B, N), C=r(T, B, N), D=r(H), z=r(T, B, H), h0=r(B, H, N),
             delta_bias=r(H))
    reset = torch.rand(T, B, generator=g) < 0.2
    dy, dh = r(T, B, H), r(B, H, N)
    leaf = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    h, ys = leaf["h0"], []
    for k in range(T):
        h = torch.where(reset[k][:, None, None], 0.0, h)
        dt = torch.nn.functional.softplus(leaf["delta"][k] + leaf["delta_bias"])
        h = torch.exp(dt[..., None] * leaf["A"]) * h + (dt * leaf["u"][k])[..., None] * leaf["B"][k][:, None]
        ys.append(((h * leaf["C"][k][:, None]).sum(-1) + leaf["D"] * leaf["u"][k]) * torch.nn.functional.silu(leaf["z"][k]))
    want = torch.autograd.grad((torch.stack(ys), h), list(leaf.values()), (dy, dh))
    args = [t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "h0")]
    kw = dict(delta_bias=t["delta_bias"], reset=reset, dy=dy, dh=dh)
    y, last, got = P.selective_scan(*args, **kw)
    assert torch.allclose(y, torch.stack(ys).detach(), atol=1e-12) and torch.allclose(last, h.detach(), atol=1e-12)
    size = P.selective_scan(*args, size=True, **kw)
    for k, w in zip(leaf, want):
        assert torch.allclose(got[k], w, rtol=1e-9, atol=1e-11), k
        assert (size[2][k] >= got[k].abs() - 1e-12).all(), k
    assert (size[0] >= y.abs() - 1e-12).all()


@pytest.mark.parametrize("activation", ["silu", "none"])
@pytest.mark.parametrize("T", [1, 2, 9])
def test_plain_conv_gradients(T, activation):
    g = torch.Generator().manual_seed(1)
    B, C, W = 2, 4, 4
    x, w, b, s, dy, dl = (torch.randn(n, generator=g).double() for n in ((T, B, C), (C, W), (C,), (B, W - 1, C), (T, B, C), (B, W - 1, C)))
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b, s)]
    full = torch.cat([leaves[3].transpose(0, 1), leaves[0]])
    pre = torch.nn.functional.conv1d(full.permute(1, 2, 0), leaves[1][:, None], leaves[2], groups=C).permute(2, 0, 1)
    want_y = torch.nn.functional.silu(pre) if activation == "silu" else pre
    want = torch.autograd.grad((want_y, full[T:].transpose(0, 1)), leaves, (dy, dl))
    y, last, got = P.causal_conv(x, w, b, s, activation=activation, dy=dy, dlast=dl)
    assert torch.allclose(y, want_y.detach()) and torch.equal(last, full[T:].transpose(0, 1).detach())
    for k, v in zip(("x", "weight", "bias", "state"), want):
        assert torch.allclose(got[k], v), k


def test_plain_conv_starts_anew():
    g = torch.Generator().manual_seed(2)
    x, w, s = (torch.randn(n, generator=g).double() for n in ((9, 1, 3), (3, 4), (1, 3, 3)))
    reset = torch.zeros(9, 1, dtype=torch.bool)
    reset[4] = True
    y, last = P.causal_conv(x, w, None, s, reset=reset)
    a, _ = P.causal_conv(x[:4], w, None, s)
    b, end = P.causal_conv(x[4:], w)
    assert torch.allclose(y, torch.cat([a, b])) and torch.equal(last, end)


def test_plain_logprobs():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 40, generator=g).double().requires_grad_(True)
    tokens = torch.randint(0, 40, (5,), generator=g)
    dl, de = torch.randn(5, generator=g).double(), torch.randn(5, generator=g).double()
    logp = torch.log_softmax(x, -1)
    given, h = logp.gather(1, tokens[:, None])[:, 0], -(logp.exp() * logp).sum(-1)
    want, = torch.autograd.grad((given, h), x, (dl, de))
    got = P.token_logprobs(x.detach(), tokens, 3, dl, de)
    assert torch.allclose(got[0], given.detach()) and torch.allclose(got[1], h.detach()) and torch.allclose(got[4], want)
    assert torch.equal(got[3], x.detach().topk(3).indices)


def test_plain_embedding():
    w = torch.randn(6, 4).double().requires_grad_(True)
    tokens = torch.tensor([[1, 5], [1, -1]])
    d = torch.randn(2, 2, 4).double()
    out, dw = P.embedding(tokens, w, 2.0, d)
    want = 2.0 * torch.nn.functional.embedding(tokens.clamp(min=0), w) * (tokens >= 0)[..., None]
    assert torch.allclose(out, want.detach()) and torch.allclose(dw, torch.autograd.grad(want, w, d)[0])
