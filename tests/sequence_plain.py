"""The operators over sequences of tokens from their definitions, in 64 bits on the CPU, a step at a
time. `size=True` replaces every term of every sum by its magnitude: the results are then what the
rounding errors of sums in float32 are measured by, as no result is off by more than the number of
roundings on its way times 2^-24 of that.

The tests' bound for a result in type t is thus half(t) |result| + roundings 2^-24 size, with
half(t) = torch.finfo(t).eps / 2 its last rounding.
"""

from __future__ import annotations

import torch


def _d(t):
    return None if t is None else t.detach().cpu().double()


def selective_scan(u, delta, A, B, C, D=None, z=None, h0=None, *, delta_bias=None, reset=None, dy=None, dh=None, size=False):
    """(y, h_T), and with dy the gradients as a dict, of [T, B, ...] tensors."""
    u, delta, A, B, C, D, z, h0, bias, dy, dh = (_d(t) for t in (u, delta, A, B, C, D, z, h0, delta_bias, dy, dh))
    T, nb, H = u.shape
    N = A.shape[1]
    mag = torch.abs if size else (lambda t: t)
    x = delta + (0 if bias is None else bias)
    dt = torch.nn.functional.softplus(x, threshold=1e9)
    a = torch.exp(dt[..., None] * A)
    u, B, C, D_ = mag(u), mag(B), mag(C), mag(torch.zeros(H, dtype=u.dtype) if D is None else D)
    h = torch.zeros(nb, H, N, dtype=u.dtype) if h0 is None else mag(h0)
    starts = torch.zeros(T, nb, dtype=torch.bool) if reset is None else reset.cpu()
    before, after = [], []
    for t in range(T):
        h = torch.where(starts[t][:, None, None], 0.0, h)
        before.append(h)
        h = a[t] * h + (dt[t] * u[t])[..., None] * B[t][:, None]
        after.append(h)
    before, after = torch.stack(before), torch.stack(after)
    ungated = (after * C[:, :, None]).sum(-1) + D_ * u
    gate = torch.ones_like(u) if z is None else mag(z * torch.sigmoid(z))
    y = ungated * gate
    if dy is None and dh is None:
        return y, after[-1]
    dy = torch.zeros_like(u) if dy is None else mag(dy)
    r = {}
    if z is not None:
        s = torch.sigmoid(z)
        r["z"] = dy * ungated * (s * (1 + z.abs() * (1 - s)) if size else s * (1 + z * (1 - s)))
    g = dy * gate
    G = torch.zeros_like(h) if dh is None else mag(dh)
    Gs = []
    for t in range(T - 1, -1, -1):
        G = G + C[t][:, None] * g[t][..., None]
        Gs.append(G)
        G = torch.where(starts[t][:, None, None], 0.0, a[t] * G)
    Gs = torch.stack(Gs[::-1])
    r["h0"] = G
    q = Gs * a * before
    S = (Gs * B[:, :, None]).sum(-1)
    r["B"] = (Gs * (dt * u)[..., None]).sum(2)
    r["C"] = (after * g[..., None]).sum(2)
    r["u"] = dt * S + D_ * g
    r["delta"] = ((q * mag(A)).sum(-1) + u * S) * torch.sigmoid(x)
    r["A"] = (q * dt[..., None]).sum((0, 1))
    r["D"] = (u * g).sum((0, 1))
    r["delta_bias"] = r["delta"].sum((0, 1))
    return y, after[-1], r


def causal_conv(x, w, bias=None, state=None, *, activation="silu", reset=None, dy=None, dlast=None, size=False):
    """(y, last), and with dy or dlast the gradients as a dict, of [T, B, C] tensors."""
    x, w, bias, state, dy, dlast = (_d(t) for t in (x, w, bias, state, dy, dlast))
    T, B, C = x.shape
    W = w.shape[1]
    mag = torch.abs if size else (lambda t: t)
    past = torch.zeros(W - 1, B, C, dtype=x.dtype) if state is None else state.transpose(0, 1)
    full = torch.cat([past, x])
    starts = torch.zeros(T, B, dtype=torch.bool) if reset is None else reset.cpu()

    def seen(t, s):
        """Whether step t sees input s (s < 0: of the state): no start after s up to t."""
        return ~starts[max(s + 1, 0):t + 1].any(0)[:, None]

    pre = torch.zeros_like(x) if bias is None else bias.expand_as(x).clone()
    whole = pre.abs()
    for t in range(T):
        for k in range(W):
            s = t - (W - 1) + k
            term = torch.where(seen(t, s), w[:, k] * full[s + W - 1], 0.0)
            pre[t] += term
            whole[t] += term.abs()
    sig = torch.sigmoid(pre)
    silu = activation == "silu"
    # an error of the argument moves silu by at most 1.1 of it
    y = (1.1 * whole if size else pre * sig) if silu else (whole if size else pre)
    last = torch.stack([torch.where(seen(T - 1, T - (W - 1) + k), full[T + k], 0.0) for k in range(W - 1)], 1)
    if dy is None and dlast is None:
        return y, last
    dy = torch.zeros_like(x) if dy is None else dy
    slope = sig * (1 + pre * (1 - sig)) if silu else torch.ones_like(pre)
    # and silu' (at most 1.1) by at most half of it
    g = dy.abs() * (1.1 + (0.5 * whole if silu else 0)) if size else dy * slope
    dfull, dw = torch.zeros_like(full), torch.zeros_like(w)
    for t in range(T):
        for k in range(W):
            s = t - (W - 1) + k
            ok = seen(t, s)
            dfull[s + W - 1] += torch.where(ok, mag(w[:, k]) * g[t], 0.0)
            dw[:, k] += torch.where(ok, mag(full[s + W - 1]) * g[t], 0.0).sum(0)
    if dlast is not None:
        for k in range(W - 1):
            dfull[T + k] += torch.where(seen(T - 1, T - (W - 1) + k), mag(dlast[:, k]), 0.0)
    return y, last, dict(x=dfull[W - 1:], state=dfull[:W - 1].transpose(0, 1), weight=dw, bias=g.sum((0, 1)))


def embedding(tokens, w, scale=1.0, dout=None, size=False):
    """out, and with dout the weight's gradient."""
    tokens, w, dout = tokens.cpu().long(), _d(w), _d(dout)
    flat = tokens.reshape(-1)
    V, K = w.shape
    out = torch.zeros(flat.numel(), K, dtype=w.dtype)
    some = (flat >= 0) & (flat < V)
    out[some] = scale * w[flat[some]]
    out[flat >= V] = float("nan")
    out = out.view(*tokens.shape, K)
    if dout is None:
        return out
    d = dout.reshape(-1, K)[some]
    return out, torch.zeros_like(w).index_add_(0, flat[some], scale * (d.abs() if size else d))


def token_logprobs(x, tokens, top=0, dlogp=None, dentropy=None):
    """(logprobs, entropy, top_logprobs, top_tokens), and with dlogp or dentropy the logits' gradient."""
    x, dlogp, dentropy = _d(x), _d(dlogp), _d(dentropy)
    tokens = tokens.cpu().long()
    V = x.shape[-1]
    inf = float("inf")
    none = (x == -inf).all(-1)
    logp = torch.where(none[..., None], -inf, torch.log_softmax(x, -1))
    p = torch.where(none[..., None], 0.0, logp.exp())
    entropy = -torch.xlogy(p, p).sum(-1)
    given = logp.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0]
    given = torch.where(tokens < 0, 0.0, torch.where(tokens >= V, float("nan"), given))
    left, ids = torch.where(x.isnan(), inf, x), []
    taken = torch.zeros_like(left, dtype=torch.bool)
    for _ in range(top):
        best = torch.where(taken, -inf, left).amax(-1, keepdim=True)
        first = torch.where((left == best) & ~taken, torch.arange(V), V).amin(-1, keepdim=True)
        ids.append(first)
        taken = taken.scatter(-1, first, True)
    ids = torch.cat(ids, -1) if ids else tokens[..., None][..., :0]
    r = given, entropy, logp.gather(-1, ids), ids
    if dlogp is None and dentropy is None:
        return r
    zero = torch.zeros_like(entropy)
    g = zero if dlogp is None else torch.where((tokens >= 0) & (tokens < V), dlogp, 0.0)
    e = zero if dentropy is None else dentropy
    hot = torch.zeros_like(x).scatter_(-1, tokens.clamp(0, V - 1)[..., None], 1.0)
    plogp = torch.where(p == 0, 0.0, p * logp)
    plogp = torch.where(p.isnan(), p, plogp)
    d = g[..., None] * (hot - p) - e[..., None] * (plogp + p * entropy[..., None])
    return *r, torch.where(none[..., None], 0.0, d)


def assert_within(got, want, size, roundings, what=""):
    """|got - want| <= half(type) |want| + roundings 2^-24 size, NaN and infinities where they are."""
    got_d = got.detach().cpu().double()
    assert got_d.shape == want.shape, (what, got_d.shape, want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(got_d[odd].nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0)), (what, "NaN or infinity")
    room = torch.finfo(got.dtype).eps / 2 * want.abs() + roundings * 2.0 ** -24 * size + 1e-37
    over = torch.where(odd, 0.0, (got_d - want).abs() - room)
    assert not (over > 0).any() and not got_d[~odd].isnan().any(), (
        what, "off by", (got_d - want).abs()[~odd].max().item(), "worst over its bound", over.max().item())
