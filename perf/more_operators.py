"""The operators of a recurrent language model, as timed cases.

Tokens become vectors (``embedding``), each layer mixes a few neighbouring steps
(``causal_conv``; ``causal_conv_step`` for one token of each request) and runs a state
space recurrence whose decay depends on its input (``selective_scan``;
``selective_step``), and the head's logits become log probabilities of given tokens with
the entropy and the likeliest alternatives (``token_logprobs``). A case is one of these
calls with its sizes:

* ``op`` "scan": u, delta, z [T, B, H], B and C [T, B, N], A [H, N]; ``train`` adds the
  backward; ``reset`` starts new sequences inside the rows, as packed documents do.
* ``op`` "step": one token of ``B`` requests and a cache of ``slots`` states [H, N].
* ``op`` "conv": x [T, B, C], ``W`` taps; ``train`` adds the backward. ``slots`` other
  than 0 is the form for one token (T = 1) over a cache of the last W - 1 inputs.
* ``op`` "embed": ``M`` tokens of a vocabulary ``V``, vectors of ``K``, and the backward.
* ``op`` "logprobs": logits [M, V], ``top`` alternatives; ``train`` adds the backward.

``dtype`` is that of activations, their gradients, the convolution's and the embedding's
weights. A, D, the step size's bias, states of the recurrence and sums are float32.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# The largest listed work of each operator, which no drawn case exceeds.
MAX_SCAN = 4096 * 8 * 1024 * 16  # steps x rows x channels x states of a training call
MAX_LONG = 65536 * 1024 * 16  # of a forward alone
MAX_CONV = 8192 * 8 * 2048
MAX_EMBED = (3 * 16384 + 32000) * 1024
MAX_LOGITS = 8192 * 32000


def _scan(T, B, H, N, dtype, train, reset=0):
    return dict(op="scan", T=T, B=B, H=H, N=N, dtype=dtype, train=train, reset=reset)


def _step(B, H, N, slots, dtype):
    return dict(op="step", B=B, H=H, N=N, slots=slots, dtype=dtype)


def _conv(T, B, C, W, dtype, train, reset=0, slots=0):
    return dict(op="conv", T=T, B=B, C=C, W=W, dtype=dtype, train=train, reset=reset, slots=slots)


def _embed(M, V, K, dtype, pad=False):
    return dict(op="embed", M=M, V=V, K=K, dtype=dtype, pad=pad)


def _logprobs(M, V, top, dtype, train):
    return dict(op="logprobs", M=M, V=V, top=top, dtype=dtype, train=train)


def listed():
    named = [
        # one token for each of a few requests while serving: latency alone
        ("step_serve", _step(8, 1024, 16, 64, "bf16")),
        # one for each request of a full server, odd sizes: the states' bytes
        ("step_batch", _step(301, 1002, 16, 400, "f32")),
        # a training step of an ordinary layer
        ("scan_train", _scan(512, 16, 512, 16, "f32", True)),
        # odd sizes, packed sequences of about 40 tokens
        ("scan_train_ragged", _scan(1001, 3, 333, 16, "f32", True, 40)),
        # a long batch in bfloat16: as much as the recurrence works through in one training call
        ("scan_train_large", _scan(4096, 8, 1024, 16, "bf16", True)),
        # prefill of one long document with shorter ones packed in it: few channels, a long axis
        ("scan_long", _scan(65536, 1, 1024, 16, "bf16", False, 9000)),
        # the convolution of a serving step: latency
        ("conv_serve", _conv(1, 8, 1024, 4, "bf16", False, 0, 64)),
        # a long batch in bfloat16: bytes alone
        ("conv_train_large", _conv(8192, 8, 2048, 4, "bf16", True)),
        # a small vocabulary of odd sizes in float32, rows with padding
        ("embed_train_ragged", _embed(1237, 1003, 333, "f32", True)),
        # a long batch over a large vocabulary, tokens as frequent as in text
        ("embed_train_large", _embed(16384, 32000, 1024, "bf16")),
        # scores of a few requests' next tokens, with the eight likeliest
        ("logprobs_serve", _logprobs(8, 32000, 8, "bf16", False)),
        # the loss of a long batch over a large vocabulary: bytes alone
        ("logprobs_train_large", _logprobs(8192, 32000, 0, "bf16", True)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("scan", "scan", "step", "conv", "embed", "logprobs"))
    dtype = rng.choice(("f32", "bf16"))
    half = 1 if dtype == "bf16" else 2
    if op == "scan":
        train, N = rng.random() < 0.6, rng.choice((4, 8, 16, 16, 16, 13, 32))
        most = (MAX_SCAN if train else MAX_LONG) // half
        H = _log(rng, 24, 2048)
        each = H * max(N, 16)
        B = _log(rng, 1, max(1, min(64, most // each)))
        T = _log(rng, 1, max(1, min(65536, most // (B * each))))
        return _scan(T, B, H, N, dtype, train, rng.choice((0, 0, 7, 500)))
    if op == "step":
        B = _log(rng, 1, 301)
        return _step(B, _log(rng, 24, 1002), rng.choice((4, 8, 16, 16)), B + rng.randint(0, 64), dtype)
    if op == "conv":
        W, C = rng.choice((2, 3, 4, 4)), _log(rng, 24, 4096)
        if rng.random() < 0.3:
            B = _log(rng, 1, 512)
            return _conv(1, B, C, W, dtype, False, 0, B + rng.randint(0, 64))
        most = MAX_CONV // half
        B = _log(rng, 1, 64)
        T = _log(rng, 1, max(1, min(65536, most // (B * C))))
        return _conv(T, B, C, W, dtype, rng.random() < 0.6, rng.choice((0, 0, 7, 500)))
    if op == "embed":
        K = _log(rng, 32, 2048)
        most = MAX_EMBED // half // K
        V = _log(rng, 200, min(64000, most * 2 // 3))
        return _embed(_log(rng, 1, min(32768, (most - V) // 3)), V, K, dtype, rng.random() < 0.5)
    V = _log(rng, 100, 200000)
    M = _log(rng, 1, max(1, min(16384, MAX_LOGITS // half // V)))
    return _logprobs(M, V, rng.choice((0, 1, 5, 8, 20)), dtype, rng.random() < 0.5)


def _tokens(shape, V, g):
    """Tokens whose frequency falls with their rank as in text; ranks are shuffled over the vocabulary."""
    rank = torch.exp(torch.rand(shape, device=DEV, generator=g) * math.log(V + 1.0)).long() - 1
    return torch.randperm(V, device=DEV, generator=g)[rank.clamp_(0, V - 1)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op, dtype = case["op"], TYPES[case["dtype"]]

    def noise(*shape, scale=1.0, kind=dtype):
        return (torch.randn(shape, device=DEV, generator=g) * scale).to(kind)

    def leaf(t):
        return t.detach().requires_grad_(case["train"])

    s = dict(case=case)
    if op == "embed":
        M, V, K = case["M"], case["V"], case["K"]
        s["tokens"] = _tokens((M,), V, g)
        if case["pad"]:
            s["tokens"] = torch.where(torch.rand(M, device=DEV, generator=g) < 0.1, -1, s["tokens"])
        s["weight"] = noise(V, K, scale=0.02).requires_grad_(True)
        s["scale"] = math.sqrt(K)
        s["dout"] = noise(M, K)
        return s
    if op == "logprobs":
        M, V = case["M"], case["V"]
        s["logits"] = leaf(noise(M, V, scale=2.0))
        s["tokens"] = _tokens((M,), V, g)
        if case["train"]:
            s["dlogp"] = torch.full((M,), -1.0 / M, device=DEV)  # of the mean loss
            s["dentropy"] = noise(M, scale=0.01 / M, kind=torch.float32)
        return s
    if op == "conv":
        T, B, C, W = case["T"], case["B"], case["C"], case["W"]
        wide = noise(T, B, 2 * C)  # the projection whose first half goes through the convolution
        s["weight"], s["bias"] = leaf(noise(C, W, scale=W ** -0.5)), leaf(noise(C, scale=0.1))
        if case["slots"]:
            s["x"] = wide[0, :, :C]
            s["state"] = noise(case["slots"], W - 1, C)
            s["slots"] = torch.randperm(case["slots"], device=DEV, generator=g)[:B].to(torch.int32)
            return s
        s["x"] = leaf(wide[..., :C])
        s["state"] = None if case["train"] else noise(B, W - 1, C)
        s["reset"] = torch.rand((T, B), device=DEV, generator=g) < 1.0 / case["reset"] if case["reset"] else None
        s["dy"] = noise(T, B, C) if case["train"] else None
        return s
    H, N, B = case["H"], case["N"], case["B"]
    lead = (B,) if op == "step" else (case["T"], B)
    train = op == "scan" and case["train"]
    # decays of 1, 2, ... N times the step size, which is 0.001 to 0.1, as such layers start and train from
    rate = torch.arange(1, N + 1, device=DEV).float() * torch.exp(0.2 * noise(H, N, kind=torch.float32))
    size = torch.exp(torch.rand(H, device=DEV, generator=g) * math.log(100.0)) * 1e-3
    s["A"], s["D"] = -rate, 1 + noise(H, scale=0.1, kind=torch.float32)
    s["delta_bias"] = size + torch.log(-torch.expm1(-size))
    s["u"] = noise(*lead, H)
    s["delta"] = noise(*lead, H)
    low = noise(*lead, 32 + 2 * N)  # the projection that B and C are columns of
    s["B"], s["C"] = low[..., 32:32 + N], low[..., 32 + N:]
    s["z"] = noise(*lead, 2 * H)[..., H:]
    if op == "step":
        s["state"] = noise(case["slots"], H, N, scale=0.3, kind=torch.float32)
        s["slots"] = torch.randperm(case["slots"], device=DEV, generator=g)[:B].to(torch.int32)
        return s
    s["h0"] = noise(B, H, N, scale=0.3, kind=torch.float32)
    s["reset"] = torch.rand(lead, device=DEV, generator=g) < 1.0 / case["reset"] if case["reset"] else None
    if train:
        for key in LEAVES:
            s[key] = leaf(s[key])
        s["dy"], s["dh"] = noise(*lead, H), noise(B, H, N, kind=torch.float32)
    return s


LEAVES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "h0")


# ---- the operators in plain form ------------------------------------------------------


def _f(t):
    return t.detach().float()


def _compose(a, b):
    """h_t = a_t h_{t-1} + b_t with h_{-1} = 0, for every t: spans of 1, 2, 4, ... steps are joined."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain_scan(s):
    case, dtype = s["case"], s["u"].dtype
    u, A, B, C, D, z, h0 = (_f(s[k]) for k in ("u", "A", "B", "C", "D", "z", "h0"))
    x = _f(s["delta"]) + _f(s["delta_bias"])
    dt = _softplus(x)
    a = torch.exp(dt[..., None] * A)
    if s["reset"] is not None:
        a = torch.where(s["reset"][..., None, None], 0.0, a)
    b = (dt * u)[..., None] * B[:, :, None]
    b[0] += a[0] * h0
    h = _compose(a, b)
    del b
    y = (h * C[:, :, None]).sum(-1) + D * u
    gate = torch.sigmoid(z)
    out, last = (y * z * gate).to(dtype), h[-1].clone()
    if not case["train"]:
        return out, last
    dout = s["dy"].float()
    dz = dout * y * gate * (1 + z * (1 - gate))
    dy = dout * z * gate
    d = C[:, :, None] * dy[..., None]
    d[-1] += s["dh"]
    back = torch.cat([torch.zeros_like(a[:1]), a[1:].flip(0)])  # G_t = d_t + a_{t+1} G_{t+1}, from the end
    G = _compose(back, d.flip(0)).flip(0)
    del back, d
    dB, dC = (G * (dt * u)[..., None]).sum(2), (h * dy[..., None]).sum(2)
    GB = (G * B[:, :, None]).sum(-1)
    q = G * a * torch.cat([h0[None], h[:-1]])
    ddelta = ((q * A).sum(-1) + u * GB) * torch.sigmoid(x)
    dA = (q * dt[..., None]).sum((0, 1))
    return (out, last, (dt * GB + D * dy).to(dtype), ddelta.to(dtype), dA, dB.to(dtype), dC.to(dtype),
            (dy * u).sum((0, 1)), dz.to(dtype), ddelta.sum((0, 1)), a[0] * G[0])


def _plain_step(s):
    at = s["slots"].long()
    u, A, B, C, D, z = (_f(s[k]) for k in ("u", "A", "B", "C", "D", "z"))
    dt = _softplus(_f(s["delta"]) + _f(s["delta_bias"]))
    h = torch.exp(dt[..., None] * A) * s["state"][at] + (dt * u)[..., None] * B[:, None]
    s["state"][at] = h
    y = (h * C[:, None]).sum(-1) + D * u
    return (y * z * torch.sigmoid(z)).to(s["u"].dtype), s["state"]


def _plain_conv(s):
    case, dtype = s["case"], s["x"].dtype
    w, bias, x = _f(s["weight"]), _f(s["bias"]), _f(s["x"])
    W = w.shape[1]
    if case["slots"]:
        at = s["slots"].long()
        full = torch.cat([s["state"][at].float(), x[:, None]], 1)
        pre = (full * w.t()).sum(1) + bias
        s["state"][at] = full[:, 1:].to(dtype)
        return (pre * torch.sigmoid(pre)).to(dtype), s["state"]
    T = x.shape[0]
    first = torch.zeros_like(x[:1]).expand(W - 1, -1, -1) if s["state"] is None else _f(s["state"]).transpose(0, 1)
    full = torch.cat([first, x])
    if s["reset"] is None:
        since = None
    else:  # sequences counted along a row; the inputs before it belong to the first
        since = torch.cumsum(s["reset"].int(), 0)
        since = torch.cat([torch.zeros_like(since[:1]).expand(W - 1, -1), since])[..., None]

    def tap(k):
        t = full[k:k + T]
        return t if since is None else torch.where(since[k:k + T] == since[W - 1:], t, 0.0)

    pre = bias + sum(w[:, k] * tap(k) for k in range(W))
    gate = torch.sigmoid(pre)
    last = full[T:] if since is None else torch.where(since[T:] == since[-1:], full[T:], 0.0)
    y, last = (pre * gate).to(dtype), last.transpose(0, 1).to(dtype)
    if not case["train"]:
        return y, last
    dpre = s["dy"].float() * gate * (1 + pre * (1 - gate))
    dfull, dw = torch.zeros_like(full), []
    for k in range(W):
        d = w[:, k] * dpre
        dfull[k:k + T] += d if since is None else torch.where(since[k:k + T] == since[W - 1:], d, 0.0)
        dw.append((dpre * tap(k)).sum((0, 1)))
    return y, last, dfull[W - 1:].to(dtype), torch.stack(dw, 1).to(dtype), dpre.sum((0, 1)).to(dtype)


def _plain_embed(s):
    tokens, w = s["tokens"], _f(s["weight"])
    some = (tokens >= 0)[:, None]
    out = torch.where(some, w[tokens.clamp(min=0)] * s["scale"], 0.0)
    # rows in the order of their tokens: a token's gradient is the difference of two running sums, kept in 64 bits
    order = torch.sort(tokens, stable=True).indices
    total = torch.cumsum(s["dout"][order].double(), 0)
    total = torch.cat([torch.zeros_like(total[:1]), total])
    edges = torch.searchsorted(tokens[order], torch.arange(w.shape[0] + 1, device=DEV))
    dw = (total[edges[1:]] - total[edges[:-1]]) * s["scale"]
    return out.to(s["weight"].dtype), dw.to(s["weight"].dtype)


def _plain_logprobs(s):
    case, x, tokens = s["case"], _f(s["logits"]), s["tokens"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    logp = (x - m) - torch.log(total)
    p = e / total
    entropy = -(p * logp).sum(1)
    given = logp.gather(1, tokens[:, None])[:, 0]
    if case["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    else:
        ids = tokens[:, None][:, :0]
    r = given, entropy, logp.gather(1, ids), ids
    if not case["train"]:
        return r
    d = -p * (s["dlogp"][:, None] + s["dentropy"][:, None] * (logp + entropy[:, None]))
    d.scatter_add_(1, tokens[:, None], s["dlogp"][:, None])
    return *r, d.to(s["logits"].dtype)


# ---- the framework's calls ------------------------------------------------------------

_G = None


def _package():
    """gru_qat_amd, whose folder is not on the path of a program that runs at the root."""
    global _G
    if _G is None:
        import os
        import sys

        at = os.path.join(os.getcwd(), "gru-triton_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import gru_qat_amd as G

        _G = G
    return _G


def _own_scan(s, G):
    out, h = G.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], s["h0"],
                              delta_bias=s["delta_bias"], reset=s["reset"])
    if not s["case"]["train"]:
        return out, h
    return (out.detach(), h.detach(), *torch.autograd.grad((out, h), [s[k] for k in LEAVES], (s["dy"], s["dh"])))


def _own_step(s, G):
    return G.selective_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], s["slots"], D=s["D"], z=s["z"],
                            delta_bias=s["delta_bias"]), s["state"]


def _own_conv(s, G):
    if s["case"]["slots"]:
        return G.causal_conv_step(s["x"], s["weight"], s["bias"], s["state"], s["slots"], activation="silu"), s["state"]
    y, last = G.causal_conv(s["x"], s["weight"], s["bias"], s["state"], activation="silu", reset=s["reset"])
    if not s["case"]["train"]:
        return y, last
    return (y.detach(), last.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"]))


def _own_embed(s, G):
    out = G.embedding(s["tokens"], s["weight"], scale=s["scale"])
    return (out.detach(), *torch.autograd.grad(out, s["weight"], s["dout"]))


def _own_logprobs(s, G):
    given, entropy, top, ids = G.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    if not s["case"]["train"]:
        return given, entropy, top, ids
    return (given.detach(), entropy.detach(), top.detach(), ids,
            *torch.autograd.grad((given, entropy), s["logits"], (s["dlogp"], s["dentropy"])))


def run(state):
    op = state["case"]["op"]
    if own:
        G = _package()
        return dict(scan=_own_scan, step=_own_step, conv=_own_conv, embed=_own_embed, logprobs=_own_logprobs)[op](state, G)
    return dict(scan=_plain_scan, step=_plain_step, conv=_plain_conv, embed=_plain_embed, logprobs=_plain_logprobs)[op](state)


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op == "scan":
        T, B, H, N = (case[k] for k in "TBHN")
        steps, rows, marks = T * B * H, T * B * N, T * B if case["reset"] else 0
        # forward: u, delta, z in, y out; B, C; A, D, the bias; h0 in, h_T out
        n = steps * 4 * size + rows * 2 * size + (H * N + 2 * H) * 4 + 2 * B * H * N * 4 + marks
        if case["train"]:  # u, delta, z, dy in, three gradients out; B, C and theirs; parameters and theirs; dh in, h0, dh0
            n += steps * 7 * size + rows * 4 * size + (H * N + 2 * H) * 8 + 3 * B * H * N * 4 + marks
        return dict(bytes=n, flops=steps * (N * (7 + (18 if case["train"] else 0)) + (40 if case["train"] else 16)))
    if op == "step":
        B, H, N = (case[k] for k in "BHN")
        return dict(bytes=B * (H * (4 * size + 8 * N) + 2 * N * size + 4) + (H * N + 2 * H) * 4, flops=B * H * (7 * N + 16))
    if op == "conv":
        T, B, C, W = (case[k] for k in "TBCW")
        n, marks = T * B * C, T * B if case["reset"] else 0
        if case["slots"]:
            return dict(bytes=(n * 2 + 2 * (W - 1) * n + C * (W + 1)) * size + 4 * B, flops=n * (2 * W + 6))
        per = 5 if case["train"] else 2  # x in, y out; x and dy in, dx out
        ends = B * (W - 1) * C * (1 if case["train"] else 2)
        return dict(bytes=(n * per + ends + C * (W + 1) * (3 if case["train"] else 1)) * size + marks * (2 if case["train"] else 1),
                    flops=n * (2 * W + 6) * (4 if case["train"] else 1))
    if op == "embed":
        M, V, K = (case[k] for k in "MVK")
        # rows in and out, their gradients in, the weight's out
        return dict(bytes=(min(M, V) + 2 * M + V) * K * size + 16 * M, flops=2 * M * K)
    M, V, top = (case[k] for k in ("M", "V", "top"))
    n = M * V * size * (3 if case["train"] else 1) + M * (16 + 12 * top + (16 if case["train"] else 0))
    return dict(bytes=n, flops=M * V * (12 if case["train"] else 5))


# ---- the definitions in 64 bits -------------------------------------------------------


def _d(t):
    return t.detach().double()


def _exact_scan(s):
    train, reset = s["case"]["train"], s["reset"]
    A, D, bias = _d(s["A"]), _d(s["D"]), _d(s["delta_bias"])
    T, B, H = s["u"].shape
    sig, tiny = torch.sigmoid, torch.nn.functional.softplus

    def at(t):
        x = _d(s["delta"][t]) + bias
        dt = tiny(x, threshold=1e9)
        return _d(s["u"][t]), x, dt, _d(s["B"][t])[:, None], _d(s["C"][t])[:, None], _d(s["z"][t])

    h = _d(s["h0"])
    out = torch.empty((T, B, H), dtype=torch.float64, device=h.device)
    ys, kept = torch.empty_like(out), []
    for t in range(T):
        u, x, dt, Bt, Ct, z = at(t)
        if reset is not None:
            h = torch.where(reset[t][:, None, None], 0.0, h)
        if train:
            kept.append(h)
        h = torch.exp(dt[..., None] * A) * h + (dt * u)[..., None] * Bt
        ys[t] = (h * Ct).sum(-1) + D * u
        out[t] = ys[t] * z * sig(z)
    if not train:
        return out, h
    last, G = h, _d(s["dh"])
    du, dd, dz = torch.empty_like(out), torch.empty_like(out), torch.empty_like(out)
    dA, dD, db = torch.zeros_like(A), torch.zeros_like(D), torch.zeros_like(D)
    dB = torch.empty(s["B"].shape, dtype=torch.float64, device=h.device)
    dC = torch.empty_like(dB)
    for t in range(T - 1, -1, -1):
        u, x, dt, Bt, Ct, z = at(t)
        a = torch.exp(dt[..., None] * A)
        g = _d(s["dy"][t])
        dz[t] = g * ys[t] * (sig(z) + z * sig(z) * sig(-z))
        g = g * z * sig(z)
        h = a * kept[t] + (dt * u)[..., None] * Bt
        G = G + g[..., None] * Ct
        dC[t], dB[t] = (h * g[..., None]).sum(1), (G * (dt * u)[..., None]).sum(1)
        down = (G * Bt).sum(-1)
        du[t] = D * g + dt * down
        slope = G * a * kept[t]
        dd[t] = ((slope * A).sum(-1) + u * down) * sig(x)
        dA += (slope * dt[..., None]).sum(0)
        dD += (g * u).sum(0)
        db += dd[t].sum(0)
        G = G * a
        if reset is not None:
            G = torch.where(reset[t][:, None, None], 0.0, G)
    return out, last, du, dd, dA, dB, dC, dD, dz, db, G


def _exact_step(s):
    A, at = _d(s["A"]), s["slots"].long()
    u, z = _d(s["u"]), _d(s["z"])
    dt = torch.nn.functional.softplus(_d(s["delta"]) + _d(s["delta_bias"]), threshold=1e9)
    state = _d(s["state"])
    h = torch.exp(dt[..., None] * A) * state[at] + dt[..., None] * u[..., None] * _d(s["B"])[:, None]
    state[at] = h
    y = (h * _d(s["C"])[:, None]).sum(2) + _d(s["D"]) * u
    return torch.nn.functional.silu(z) * y, state


def _exact_conv(s):
    case, W = s["case"], s["case"]["W"]
    w, bias = _d(s["weight"]), _d(s["bias"])
    silu = torch.nn.functional.silu
    if case["slots"]:
        at, state = s["slots"].long(), _d(s["state"])
        pre = bias + w[:, -1] * _d(s["x"])
        for k in range(W - 1):
            pre = pre + w[:, k] * state[at, k]
        state[at] = torch.cat([state[at, 1:], _d(s["x"])[:, None]], 1)
        return silu(pre), state
    T, B, C = s["x"].shape
    train = case["train"]
    x = _d(s["x"]).requires_grad_(train)
    w, bias = w.requires_grad_(train), bias.requires_grad_(train)
    past = torch.zeros(B, W - 1, C, dtype=torch.float64, device=x.device) if s["state"] is None else _d(s["state"])
    # each tap's inputs; whatever is before the row's last start counts as zero
    shifted = []
    for k in range(W):
        back = W - 1 - k
        rows = torch.cat([past[:, W - 1 - back:].transpose(0, 1), x])[:T]
        if s["reset"] is not None:
            dead = torch.zeros(T, B, dtype=torch.bool, device=x.device)
            for j in range(min(back, T)):
                dead[j:] |= s["reset"][:T - j]
            rows = rows.masked_fill(dead[..., None], 0.0)
        shifted.append(rows)
    y = silu(bias + sum(w[:, k] * shifted[k] for k in range(W)))
    tail = torch.cat([past.transpose(0, 1), x.detach()])[T:].clone()
    if s["reset"] is not None:
        for i in range(W - 1):
            step = T - (W - 1) + i
            gone = s["reset"][max(step + 1, 0):].any(0)
            tail[i][gone] = 0.0
    tail = tail.transpose(0, 1)
    if not train:
        return y, tail
    dx, dw, db = torch.autograd.grad(y, (x, w, bias), _d(s["dy"]))
    return y.detach(), tail, dx, dw, db


def _exact_embed(s):
    tokens, w = s["tokens"], _d(s["weight"])
    some = tokens >= 0
    out = torch.zeros(len(tokens), w.shape[1], dtype=torch.float64, device=w.device)
    out[some] = s["scale"] * w[tokens[some]]
    dw = torch.zeros_like(w).index_add_(0, tokens[some], s["scale"] * _d(s["dout"])[some])
    return out, dw


def _exact_logprobs(s):
    case, tokens = s["case"], s["tokens"]
    M, V = s["logits"].shape
    whole = dict(given=[], entropy=[], top=[], ids=[], d=[])
    for i in range(0, M, 1024):
        logp = torch.log_softmax(_d(s["logits"][i:i + 1024]), 1)
        p, mine = logp.exp(), tokens[i:i + 1024, None]
        H = -torch.xlogy(p, p).sum(1)
        whole["given"].append(logp.gather(1, mine)[:, 0])
        whole["entropy"].append(H)
        # the largest first, of equal ones the lowest index
        left, ids = logp.clone(), []
        for _ in range(case["top"]):
            best = torch.where(left == left.amax(1, keepdim=True), torch.arange(V, device=p.device), V).amin(1, keepdim=True)
            ids.append(best)
            left.scatter_(1, best, -math.inf)
        ids = torch.cat(ids, 1) if ids else mine[:, :0]
        whole["ids"].append(ids)
        whole["top"].append(logp.gather(1, ids))
        if case["train"]:
            g, e = _d(s["dlogp"][i:i + 1024, None]), _d(s["dentropy"][i:i + 1024, None])
            d = torch.zeros_like(p).scatter_(1, mine, 1.0)
            whole["d"].append((d - p) * g - e * p * (logp + H[:, None]))
    r = [torch.cat(whole[k]) for k in ("given", "entropy", "top", "ids")]
    return (*r, torch.cat(whole["d"])) if case["train"] else tuple(r)


def exact(case, seed):
    if case["op"] == "scan" and case["train"] and case["T"] > 20000:
        return None  # a step at a time there and back: half a minute
    s = prepare(case, seed)
    return dict(scan=_exact_scan, step=_exact_step, conv=_exact_conv, embed=_exact_embed, logprobs=_exact_logprobs)[case["op"]](s)
