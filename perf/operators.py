"""The operators of a gated linear recurrent layer, as timed cases.

A layer projects its input to gates (``linear_act``), runs the recurrence over the
sequence (``gated_linear_scan``; ``gated_linear_step`` for one token of each request),
projects back with a residual (``linear_act`` again), and is trained by AdamW
(``adamw_step``). A case is one of these calls with its sizes:

* ``op`` "scan": gi [T, B, 2H] (gates z, n), h0 [B, H]; ``train`` adds the backward;
  ``reset`` starts new sequences inside the rows, as packed documents do.
* ``op`` "step": gi [B, 2H] and a cache of ``slots`` states, updated in place.
* ``op`` "linear": x [M, K], W [N, K]; ``train`` adds the backward.
* ``op`` "adamw": the tensors of ``layers`` such layers (input I, hidden H) in one step.
  ``bits`` is that of the moments. Parameters in bfloat16 keep a float32 master.

``dtype`` is that of activations, weights and gradients. States of the recurrence, moments
and sums are float32.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 256  # elements that share a scale where moments are held in 8 bits
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01

# The largest listed work of each operator, which no drawn case exceeds.
MAX_STATES = 4096 * 8 * 1024
MAX_LONG = 65536 * 1024
MAX_FLOPS = 32768 * 2048 * 1024
MAX_PARAMS = 16 * (3 * 1024 * 1024)


def _scan(T, B, H, dtype, act, train, reset=0):
    return dict(op="scan", T=T, B=B, H=H, dtype=dtype, act=act, train=train, reset=reset)


def _step(B, H, slots, dtype, act):
    return dict(op="step", B=B, H=H, slots=slots, dtype=dtype, act=act)


def _linear(M, N, K, dtype, act, residual, train):
    return dict(op="linear", M=M, N=N, K=K, dtype=dtype, act=act, residual=residual, train=train)


def _adamw(layers, I, H, dtype, bits):
    return dict(op="adamw", layers=layers, I=I, H=H, dtype=dtype, bits=bits)


def listed():
    named = [
        # one token for each of a few requests while serving: latency alone
        ("step_serve", _step(8, 1024, 64, "bf16", "tanh")),
        # a training step of an ordinary layer at the scans' own width
        ("scan_train", _scan(512, 16, 512, "f32", "tanh", True)),
        # odd sizes, packed sequences of about 40 tokens
        ("scan_train_ragged", _scan(1001, 3, 333, "f32", "identity", True, 40)),
        # a long batch in bfloat16: as much as the recurrence moves in one call
        ("scan_train_large", _scan(4096, 8, 1024, "bf16", "tanh", True)),
        # prefill of one long document with shorter ones packed in it: few channels, a long axis
        ("scan_long", _scan(65536, 1, 1024, "bf16", "identity", False, 9000)),
        # the gates' projection of a few tokens while serving: the weight's bytes
        ("linear_serve", _linear(8, 2048, 1024, "bf16", "none", False, False)),
        # an ordinary training step of the output projection
        ("linear_train", _linear(2048, 1024, 512, "bf16", "gelu", True, True)),
        # odd sizes in float32
        ("linear_train_ragged", _linear(1650, 1002, 301, "f32", "silu", True, True)),
        # the gates' projection of a long batch: the matrix units
        ("linear_train_large", _linear(32768, 2048, 1024, "bf16", "none", False, True)),
        # a small model of odd sizes, moments in 8 bits
        ("adamw8_ragged", _adamw(3, 301, 333, "f32", 8)),
        # an ordinary model in float32
        ("adamw32", _adamw(6, 512, 512, "f32", 32)),
        # a large one in bfloat16 with masters, moments in 8 bits
        ("adamw8_large", _adamw(16, 1024, 1024, "bf16", 8)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("scan", "scan", "step", "linear", "linear", "adamw"))
    dtype = rng.choice(("f32", "bf16"))
    act = rng.choice(("tanh", "identity"))
    if op == "scan":
        train = rng.random() < 0.6
        most = MAX_STATES if train else MAX_LONG
        if dtype == "f32":
            most //= 2
        H = _log(rng, 24, 2048)
        B = _log(rng, 1, max(1, min(64, most // H)))
        T = _log(rng, 1, max(1, min(65536, most // (B * H))))
        return _scan(T, B, H, dtype, act, train, rng.choice((0, 0, 7, 500)))
    if op == "step":
        B = _log(rng, 1, 512)
        return _step(B, _log(rng, 24, 2048), B + rng.randint(0, 64), dtype, act)
    if op == "linear":
        train = rng.random() < 0.6
        N, K = _log(rng, 48, 4096), _log(rng, 32, 2048)
        most = MAX_FLOPS // (8 if dtype == "f32" else 1)
        M = _log(rng, 1, max(1, min(32768, most // (N * K))))
        return _linear(M, N, K, dtype, rng.choice(("none", "relu", "gelu", "silu", "tanh", "sigmoid")),
                       rng.random() < 0.5, train)
    I, H = _log(rng, 24, 1024), _log(rng, 24, 1024)
    layers = max(1, min(rng.randint(1, 16), MAX_PARAMS // (3 * I * H + 2 * H + I)))
    return _adamw(layers, I, H, dtype, rng.choice((8, 32)))


def _sizes(case):
    """The tensors of the case's layers: shapes, and where each starts in one buffer (whole blocks)."""
    I, H = case["I"], case["H"]
    shapes = [(2 * H, I), (2 * H,), (I, H), (I,)] * case["layers"]
    starts, at = [], 0
    for s in shapes:
        starts.append(at)
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return shapes, starts, at


def _views(flat, shapes, starts):
    return [flat[a:a + math.prod(s)].view(s) for s, a in zip(shapes, starts)]


def _prepare_adamw(case, g):
    shapes, starts, total = _sizes(case)
    dtype = TYPES[case["dtype"]]
    live = torch.zeros(total, device=DEV)
    for v in _views(live, shapes, starts):
        v.fill_(1.0)

    def noise():
        return torch.randn(total, device=DEV, generator=g) * live

    s = dict(shapes=shapes, starts=starts, step=1000)
    master = noise() * case["I"] ** -0.5
    # gradients whose scale differs from element to element, as those of a trained model do
    spread = torch.exp(1.5 * noise()) * 1e-3
    s["grad"] = (noise() * spread).to(dtype)
    m, v = noise() * spread * 0.3, (spread * (1.0 + 0.2 * noise())).square() * live
    if dtype == torch.float32:
        s["param"], s["master"] = master, None
    else:
        s["param"], s["master"] = master.to(dtype), master
    if case["bits"] == 8:
        mb, vb = m.view(-1, BLOCK), v.view(-1, BLOCK)
        s["m_scale"], s["v_scale"] = mb.abs().amax(1), vb.amax(1)
        some = torch.ones_like(mb)
        s["m"] = (torch.sign(mb) * torch.round(
            torch.sqrt(mb.abs() / torch.where(mb == 0, some, s["m_scale"][:, None])) * 127)).to(torch.int8).view(-1)
        s["v"] = torch.round(
            torch.sqrt(torch.sqrt(vb / torch.where(vb == 0, some, s["v_scale"][:, None]))) * 255).to(torch.uint8).view(-1)
    else:
        s["m"], s["v"] = m, v
    for key in ("param", "grad", "master", "m", "v"):
        s[key + "s"] = None if s[key] is None else _views(s[key], shapes, starts)
    if case["bits"] == 8:
        blocks = [-(-math.prod(x) // BLOCK) for x in shapes]
        for key in ("m_scale", "v_scale"):
            s[key + "s"] = [s[key][a // BLOCK:a // BLOCK + n] for a, n in zip(starts, blocks)]
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op = case["op"]
    if op == "adamw":
        return dict(_prepare_adamw(case, g), case=case)
    dtype = TYPES[case["dtype"]]

    def noise(*shape, scale=1.0, kind=dtype):
        return (torch.randn(shape, device=DEV, generator=g) * scale).to(kind)

    s = dict(case=case)
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"], s["w"] = noise(M, K), noise(N, K, scale=K ** -0.5)
        s["bias"] = noise(N, scale=0.1)
        s["residual"] = noise(M, N) if case["residual"] else None
        s["dy"] = noise(M, N) if case["train"] else None
        for key in ("x", "w", "bias"):
            s[key].requires_grad_(case["train"])
        return s
    H = case["H"]
    # the update gate remembers for tens to hundreds of steps, as a trained one does
    forget = torch.rand(H, device=DEV, generator=g) * 5.0 - 0.5
    forget = torch.cat([forget, torch.zeros(H, device=DEV)])
    if op == "step":
        B = case["B"]
        s["gi"] = (torch.randn((B, 2 * H), device=DEV, generator=g) + forget).to(dtype)
        s["state"] = noise(case["slots"], H, scale=0.5, kind=torch.float32)
        s["slots"] = torch.randperm(case["slots"], device=DEV, generator=g)[:B].to(torch.int32)
        return s
    T, B = case["T"], case["B"]
    s["gi"] = torch.randn((T, B, 2 * H), device=DEV, generator=g).add_(forget).to(dtype)
    s["h0"] = noise(B, H, scale=0.5, kind=torch.float32)
    s["reset"] = torch.rand((T, B), device=DEV, generator=g) < 1.0 / case["reset"] if case["reset"] else None
    if case["train"]:
        s["dout"], s["dh"] = noise(T, B, H), noise(B, H, kind=torch.float32)
        s["gi"].requires_grad_(True)
        s["h0"].requires_grad_(True)
    return s


# ---- the operators in plain form ------------------------------------------------------


def _compose(a, b):
    """h_t = a_t h_{t-1} + b_t with h_{-1} = 0, for every t: spans of 1, 2, 4, ... steps are joined."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _gates(gi, act):
    x = gi.detach().float()
    H = x.shape[-1] // 2
    z, n = torch.sigmoid(x[..., :H]), x[..., H:]
    return z, torch.tanh(n) if act == "tanh" else n


def _plain_scan(s):
    case, dtype, h0 = s["case"], s["gi"].dtype, s["h0"].detach()
    z, n = _gates(s["gi"], case["act"])
    a = z if s["reset"] is None else torch.where(s["reset"][..., None], torch.zeros_like(z), z)
    b = (1 - z) * n
    b[0] += a[0] * h0
    h = _compose(a, b)
    if not case["train"]:
        return h.to(dtype), h[-1].clone()
    d = s["dout"].to(torch.float32, copy=True)
    d[-1] += s["dh"]
    back = torch.cat([torch.zeros_like(a[:1]), a[1:].flip(0)])  # D_t = d_t + a_{t+1} D_{t+1}, from the end
    D = _compose(back, d.flip(0)).flip(0)
    before = torch.cat([h0[None], h[:-1]])
    if s["reset"] is not None:
        before = torch.where(s["reset"][..., None], torch.zeros_like(before), before)
    dn = D * (1 - z)
    if case["act"] == "tanh":
        dn = dn * (1 - n * n)
    dgi = torch.cat([D * (before - n) * z * (1 - z), dn], -1)
    return h.to(dtype), h[-1].clone(), dgi.to(dtype), a[0] * D[0]


def _plain_step(s):
    at = s["slots"].long()
    z, n = _gates(s["gi"], s["case"]["act"])
    h = z * s["state"][at] + (1 - z) * n
    s["state"][at] = h
    return h.to(s["gi"].dtype), s["state"]


def _act(x, act):
    """act(x) and act'(x)"""
    if act == "relu":
        return torch.clamp(x, min=0), (x > 0).float()
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(x * 0.5 ** 0.5))
        return x * p, p + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    if act == "silu":
        p = torch.sigmoid(x)
        return x * p, p * (1 + x * (1 - p))
    if act == "tanh":
        y = torch.tanh(x)
        return y, 1 - y * y
    y = torch.sigmoid(x)
    return y, y * (1 - y)


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    pre = x @ w.t() + s["bias"].detach().float()
    y, slope = (pre, None) if case["act"] == "none" else _act(pre, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not case["train"]:
        return y.to(dtype)
    dy = s["dy"].float()
    dpre = dy if slope is None else dy * slope
    return y.to(dtype), (dpre @ w).to(dtype), (dpre.t() @ x).to(dtype), dpre.sum(0).to(dtype)


# Moments in 8 bits: the codes of a block of 256 stand for A sign(c) (c / 127)^2 (first moment)
# and A (c / 255)^4 (second), with A the block's largest magnitude; codes are the nearest in the
# root. A block whose largest magnitude is under 2^-120 is held as zeros.
TINY = 2.0 ** -120
UNIT_M, UNIT_V = 1.0 / 127 ** 2, 1.0 / 255 ** 4


def _value_m(code, scale):
    c = code.view(-1, BLOCK).float()
    return (c * c.abs() * (scale * UNIT_M)[:, None]).view(-1)


def _value_v(code, scale):
    c = code.view(-1, BLOCK).float()
    return ((c * c) * (c * c) * (scale * UNIT_V)[:, None]).view(-1)


def _code(x, levels, quartic):
    x = x.view(-1, BLOCK)
    size = x.abs()
    most = size.amax(1)
    none = most < TINY
    inv = torch.where(none, torch.zeros_like(most), torch.ones_like(most) / torch.where(none, torch.ones_like(most), most))
    root = torch.sqrt(size * inv[:, None])
    if quartic:
        root = torch.sqrt(root)
    c = torch.clamp(torch.round(root * levels), max=levels)
    if not quartic:
        c = c * torch.sign(x)
    return c.view(-1), torch.where(none, torch.zeros_like(most), most)


def _plain_adamw(s):
    s["step"] += 1
    c1, c2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    bits = s["case"]["bits"]
    g = s["grad"].float()
    m, v = (_value_m(s["m"], s["m_scale"]), _value_v(s["v"], s["v_scale"])) if bits == 8 else (s["m"], s["v"])
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    p = s["param"] if s["master"] is None else s["master"]
    p.copy_(p * (1 - LR * DECAY) - m / (torch.sqrt(v) * c2 ** -0.5 + EPS) * (LR / c1))
    if s["master"] is not None:
        s["param"].copy_(p)
    if bits == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return s["param"], s["master"], s["m"], s["v"]
    for key, x, levels in (("m", m, 127), ("v", v, 255)):
        code, most = _code(x, levels, key == "v")
        s[key].copy_(code)
        s[key + "_scale"].copy_(most)
    return s["param"], s["master"], _value_m(s["m"], s["m_scale"]), _value_v(s["v"], s["v_scale"])


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
    case = s["case"]
    out, h = G.gated_linear_scan(s["gi"], s["h0"], activation=case["act"], reset=s["reset"])
    if not case["train"]:
        return out, h
    return (out.detach(), h.detach(), *torch.autograd.grad((out, h), (s["gi"], s["h0"]), (s["dout"], s["dh"])))


def _own_step(s, G):
    return G.gated_linear_step(s["gi"], s["state"], s["slots"], activation=s["case"]["act"]), s["state"]


def _own_linear(s, G):
    y = G.linear_act(s["x"], s["w"], s["bias"], activation=s["case"]["act"], residual=s["residual"])
    if not s["case"]["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"]))


def _own_adamw(s, G):
    s["step"] += 1
    scales = {}
    if s["case"]["bits"] == 8:
        scales = dict(exp_avg_scales=s["m_scales"], exp_avg_sq_scales=s["v_scales"])
    G.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                 weight_decay=DECAY, masters=s["masters"], **scales)
    if s["case"]["bits"] == 32:
        return s["param"], s["master"], s["m"], s["v"]
    return (s["param"], s["master"], G.adamw_dequantize_state(s["m"], s["m_scale"]),
            G.adamw_dequantize_state(s["v"], s["v_scale"]))


def run(state):
    op = state["case"]["op"]
    if own:
        G = _package()
        return dict(scan=_own_scan, step=_own_step, linear=_own_linear, adamw=_own_adamw)[op](state, G)
    return dict(scan=_plain_scan, step=_plain_step, linear=_plain_linear, adamw=_plain_adamw)[op](state)


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op == "scan":
        n = case["T"] * case["B"] * case["H"]
        per = 9 if case["train"] else 3  # forward gi 2, out 1; backward gi 2, out 1, dout 1, dgi 2
        ends = (4 if case["train"] else 2) * case["B"] * case["H"] * 4
        marks = (2 if case["train"] else 1) * case["T"] * case["B"] if case["reset"] else 0
        return dict(bytes=n * per * size + ends + marks, flops=n * (40 if case["train"] else 14))
    if op == "step":
        n = case["B"] * case["H"]
        return dict(bytes=n * (3 * size + 8) + 4 * case["B"], flops=14 * n)
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        res = M * N if case["residual"] else 0
        if not case["train"]:
            return dict(bytes=(M * K + N * K + N + M * N + res) * size, flops=2 * M * N * K)
        return dict(bytes=(3 * M * K + 3 * N * K + 2 * N + 2 * M * N + res) * size, flops=6 * M * N * K)
    n = sum(math.prod(s) for s in _sizes(case)[0])
    per = size + (8 if case["dtype"] == "f32" else 8 + 2)  # the gradient; the parameter or master, and its copy
    # moments in 32 bits: read and written; in 8 bits: the codes, and the values that are returned
    per += 16 if case["bits"] == 32 else 4 + 8 + 16 / BLOCK
    return dict(bytes=n * per, flops=n * 20)


# ---- the definitions in 64 bits -------------------------------------------------------


def _exact_scan(s):
    case = s["case"]
    H, T = case["H"], s["gi"].shape[0]
    reset = s["reset"]

    def gates(t):
        x = s["gi"][t].detach().double()
        n = x[:, H:]
        return 1 / (1 + torch.exp(-x[:, :H])), torch.tanh(n) if case["act"] == "tanh" else n

    h = s["h0"].detach().double()
    out = torch.empty((T, *h.shape), dtype=torch.float64, device=h.device)
    for t in range(T):
        z, n = gates(t)
        if reset is not None:
            h = torch.where(reset[t][:, None], 0.0, h)
        h = n + z * (h - n)
        out[t] = h
    if not case["train"]:
        return out, out[-1].clone()
    D = s["dh"].double()
    dgi = torch.empty((T, h.shape[0], 2 * H), dtype=torch.float64, device=h.device)
    for t in range(T - 1, -1, -1):
        z, n = gates(t)
        D = D + s["dout"][t].double()
        hp = out[t - 1] if t else s["h0"].detach().double()
        if reset is not None:
            hp = torch.where(reset[t][:, None], 0.0, hp)
        dgi[t, :, :H] = D * (hp - n) * z * (1 - z)
        dgi[t, :, H:] = D * (1 - z) * (1 - n * n if case["act"] == "tanh" else 1)
        D = D * z
        if reset is not None:
            D = torch.where(reset[t][:, None], 0.0, D)
    return out, out[-1].clone(), dgi, D


def _exact_step(s):
    H = s["case"]["H"]
    x, at = s["gi"].double(), s["slots"].long()
    z, n = 1 / (1 + torch.exp(-x[:, :H])), x[:, H:]
    n = torch.tanh(n) if s["case"]["act"] == "tanh" else n
    state = s["state"].double()
    h = n + z * (state[at] - n)
    state[at] = h
    return h, state


def _exact_linear(s):
    case = s["case"]
    x, w, bias = (s[k].detach().double() for k in ("x", "w", "bias"))
    pre = torch.addmm(bias, x, w.t()).requires_grad_(case["train"])
    f = dict(none=lambda u: 1 * u, relu=torch.relu, gelu=torch.nn.functional.gelu, silu=torch.nn.functional.silu,
             tanh=torch.tanh, sigmoid=torch.sigmoid)[case["act"]]
    y = f(pre)
    full = y.detach() if s["residual"] is None else y.detach() + s["residual"].double()
    if not case["train"]:
        return full
    dpre, = torch.autograd.grad(y, pre, s["dy"].double())
    return full, dpre @ w, dpre.t() @ x, dpre.sum(0)


def _exact_adamw(s):
    t = s["step"] + 1
    g = s["grad"].double()
    p = (s["param"] if s["master"] is None else s["master"]).double()
    if s["case"]["bits"] == 8:
        A, B = (s[k].double().repeat_interleave(BLOCK) for k in ("m_scale", "v_scale"))
        c, d = s["m"].double(), s["v"].double()
        m, v = A * torch.sign(c) * (c / 127) ** 2, B * (d / 255) ** 4
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    if s["case"]["bits"] == 8:
        A, B = (u.abs().view(-1, BLOCK).amax(1).clamp(min=TINY).repeat_interleave(BLOCK) for u in (m, v))
        m = A * torch.sign(m) * (torch.round(127 * (m.abs() / A) ** 0.5) / 127) ** 2
        v = B * (torch.round(255 * (v / B) ** 0.25) / 255) ** 4
    return p, None if s["master"] is None else p, m, v


def exact(case, seed):
    s = prepare(case, seed)
    return dict(scan=_exact_scan, step=_exact_step, linear=_exact_linear, adamw=_exact_adamw)[case["op"]](s)
