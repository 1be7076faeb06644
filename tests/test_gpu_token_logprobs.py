"""Token log probabilities, entropy, the likeliest tokens and the gradient against the definition in
64 bits (sequence_plain)."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def _make(M, V, dtype, dev, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, V, generator=g) * scale).to(dtype).to(dev)
    tokens = torch.randint(0, V, (M,), generator=g).to(dev)
    return x, tokens, torch.randn(M, generator=g).to(dev), torch.randn(M, generator=g).to(dev)


def _check(x, tokens, top, dl=None, de=None):
    V = x.shape[-1]
    leaf = x.detach().requires_grad_(dl is not None or de is not None)
    got = G.token_logprobs(leaf, tokens, top=top)
    want = P.token_logprobs(x, tokens, top, dl, de)
    # sums of positive terms: relative errors of V roundings in a chain, exp within 8 units at arguments that are
    # off by 4 units of the range of logits; a term of the entropy is p times a log probability
    spread = 1 + (x.double().cpu().nan_to_num(posinf=0.0, neginf=0.0).abs().amax(-1))
    roundings = V // 64 + 64
    for name, g, w in zip(("logprobs", "entropy"), got, want):
        assert g.dtype == F32
        P.assert_within(g, w, spread, roundings, name)
    P.assert_within(got[2], want[2], spread[..., None].expand_as(want[2]), roundings, "top")
    ok = ~want[0].isnan() if top else None
    assert got[3].dtype == torch.int64
    if top:
        rows = ~x.isnan().any(-1).cpu() & ok
        assert torch.equal(got[3].cpu()[rows], want[3][rows])
    if dl is None and de is None:
        return got
    outs, grads = zip(*[(o, g) for o, g in ((got[0], dl), (got[1], de)) if g is not None])
    dx, = torch.autograd.grad(outs, leaf, grads)
    p = torch.softmax(x.double().cpu(), -1).nan_to_num()
    size = p * ((0 if dl is None else dl.cpu().double().abs()) + (0 if de is None else de.cpu().double().abs() * 2 * spread))[..., None]
    if dl is not None:  # at the token itself the terms are dlogp and dlogp p
        size = size + dl.cpu().double().abs()[..., None] * torch.nn.functional.one_hot(tokens.cpu().long().clamp(0, V - 1), V)
    # p is off by the error of its exponent, which is of the logits' size
    P.assert_within(dx, want[4], size * spread[..., None], roundings, "dx")
    return got


# rows in whole accesses and not, one part and several, the likeliest out of one wave, workgroup and many
@pytest.mark.parametrize("M,V", [(1, 1), (3, 2), (5, 64), (2, 1000), (300, 257), (4, 8192), (3, 8193), (2, 40001), (1, 200000)])
@pytest.mark.parametrize("top", [0, 1, 7, 32])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_forward_and_backward(dev, M, V, top, dtype):
    x, tokens, dl, de = _make(M, V, dtype, dev, seed=V)
    _check(x, tokens, min(top, V), dl, de)


@pytest.mark.parametrize("which", ["logprobs", "entropy"])
def test_one_gradient_alone(dev, which):
    x, tokens, dl, de = _make(20, 300, F32, dev)
    _check(x, tokens, 0, dl if which == "logprobs" else None, de if which == "entropy" else None)


@pytest.mark.parametrize("V", [100, 9000])
def test_masked_logits(dev, V):
    x, tokens, dl, de = _make(6, V, F32, dev, seed=1)
    x[0, ::2] = -INF
    tokens[0] = 1
    tokens[1] = 4
    x[1, 4] = -INF  # the given token cannot come
    x[2] = -INF     # nothing can
    x[3] = -INF
    x[3, V - 1] = 2.0  # one can
    tokens[3] = V - 1
    x[4] = torch.finfo(F32).min  # the lowest value is no mask: all equal
    x[5, :V // 2] = torch.finfo(F32).min
    got = _check(x, tokens, 5, dl, de)
    assert got[0][2] == -INF and got[1][2] == 0 and (got[2][2] == -INF).all() and got[3][2].tolist() == list(range(5))
    assert got[0][3] == 0 and got[1][3] == 0


@pytest.mark.parametrize("top", [0, 3])
def test_nan_and_infinity_make_their_row_nan(dev, top):
    x, tokens, dl, de = _make(5, 300, BF16, dev, seed=2)
    x[1, 77] = float("nan")
    x[3, 12] = INF
    leaf = x.detach().requires_grad_(True)
    lp, h, t, ids = G.token_logprobs(leaf, tokens, top=top)
    dx, = torch.autograd.grad((lp, h), leaf, (dl, de))
    for r in (1, 3):
        assert lp[r].isnan() and h[r].isnan() and t[r].isnan().all() and dx[r].isnan().any()
        assert ((ids[r] >= 0) & (ids[r] < 300)).all()
    keep = [0, 2, 4]
    _check(x[keep].contiguous(), tokens[keep], top, dl[keep], de[keep])
    assert lp[keep].isfinite().all() and dx[keep].isfinite().all()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_tokens_that_do_not_count(dev, kind):
    x, tokens, dl, de = _make(6, 130, F32, dev, seed=3)
    tokens[1], tokens[2], tokens[4] = -1, 130, -5
    tokens = tokens.to(kind)
    _check(x, tokens, 2, dl, de)
    lp, _, _, _ = G.token_logprobs(x, tokens)
    assert lp[1] == 0 and lp[4] == 0 and lp[2].isnan()


@pytest.mark.parametrize("V", [70, 5000, 20000])
def test_ties_go_to_the_lowest(dev, V):
    x = torch.zeros(3, V, device=dev)
    x[0, 10::7] = 1.0
    x[1, ::3] = -0.0
    x[2, V - 1] = x[2, 5] = 2.0
    tokens = torch.zeros(3, dtype=torch.long, device=dev)
    _, _, _, ids = G.token_logprobs(x, tokens, top=6)
    assert ids[0].tolist() == [10 + 7 * k for k in range(6)]
    assert ids[1].tolist() == list(range(6))  # -0 equals 0
    assert ids[2].tolist() == [5, V - 1, 0, 1, 2, 3]


def test_shapes_and_strides(dev):
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(4, 3, 310, generator=g).to(dev)
    for off, V in ((0, 304), (1, 300), (4, 304)):
        x = wide[..., off:off + V]
        tokens = torch.randint(0, V, (3, 4), generator=g).to(dev).t()
        lp, h, t, ids = G.token_logprobs(x, tokens, top=3)
        assert lp.shape == h.shape == (4, 3) and t.shape == ids.shape == (4, 3, 3)
        want = P.token_logprobs(x, tokens, 3)
        assert torch.equal(ids.cpu(), want[3])
        assert torch.allclose(lp.cpu().double(), want[0], atol=1e-5) and torch.allclose(h.cpu().double(), want[1], atol=1e-5)
    one = G.token_logprobs(wide[0, 0], tokens[0, 0], top=2)
    assert one[0].shape == () and one[3].shape == (2,)
    same = wide[0, 0].expand(5, 310)  # rows that share memory
    lp = G.token_logprobs(same, torch.arange(5, device=dev))[0]
    assert torch.allclose(lp.cpu().double(), torch.log_softmax(wide[0, 0].cpu().double(), -1)[:5], atol=1e-5)


def test_differences(dev):
    x, tokens, dl, de = _make(4, 30, F32, dev, seed=5, scale=1.0)
    leaf = x.detach().requires_grad_(True)
    lp, h, _, _ = G.token_logprobs(leaf, tokens)
    dx, = torch.autograd.grad((lp, h), leaf, (dl, de))
    d = torch.randn(4, 30, generator=torch.Generator().manual_seed(6)).double()

    def value(s):
        a, b, _, _ = P.token_logprobs(x.cpu().double() + s * d, tokens)
        return (a * dl.cpu() + b * de.cpu()).sum()

    want = (value(1e-5) - value(-1e-5)) / 2e-5
    assert abs((dx.cpu().double() * d).sum() - want) < 1e-4
