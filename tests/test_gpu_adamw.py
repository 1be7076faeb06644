"""AdamW over many tensors (gs_adamw_step) against its formula in 64 bits.

Tolerances: u = 2^-24. A moment is two products and a sum (the second one product
more): within 4 u of the sum of its terms' magnitudes. The update m / (sqrt(v) r + eps)
rate carries the moments' errors (m's relative to its terms, half of v's) and under 10
roundings; p' is one product and one difference of it. Codes are the nearest ones in
the root, up to the root's own rounding: 255 (8 u) of a code beyond one half.
"""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
from gru_qat_amd import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HYPER = dict(lr=0.02, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 2, 3, 5, 255, 256, 257, 0, 1023, 2047, 2048, 2049, 6001]
F32, BF16 = torch.float32, torch.bfloat16


def _make(sizes, seed, pd=F32, gd=F32, bits=32, master=False, dev="cuda", shift=0):
    """Tensors of each size (starting `shift` elements into their storage) and moments of a running average."""
    gen = torch.Generator().manual_seed(seed)

    def new(n, dtype, values):
        t = torch.zeros(n + shift, dtype=dtype, device=dev)[shift:]
        t.copy_(values)
        return t

    s = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], masters=[], exp_avg_scales=[], exp_avg_sq_scales=[])
    for n in sizes:
        p, g = torch.randn(n, generator=gen), torch.randn(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen))
        m, v = torch.randn(n, generator=gen) * 0.3, torch.rand(n, generator=gen) * 2
        s["masters"].append(new(n, F32, p))
        s["params"].append(new(n, pd, p))
        s["grads"].append(new(n, gd, g))
        if bits == 8:
            k = -(-n // 256)
            s["exp_avgs"].append(new(n, torch.int8, torch.randint(-127, 128, (n,), generator=gen)))
            s["exp_avg_sqs"].append(new(n, torch.uint8, torch.randint(0, 256, (n,), generator=gen)))
            s["exp_avg_scales"].append(new(k, F32, torch.rand(k, generator=gen) + 0.1))
            s["exp_avg_sq_scales"].append(new(k, F32, torch.rand(k, generator=gen) + 0.1))
        else:
            s["exp_avgs"].append(new(n, F32, m))
            s["exp_avg_sqs"].append(new(n, F32, v))
    if not master:
        s["masters"] = None
    if bits == 32:
        s["exp_avg_scales"] = s["exp_avg_sq_scales"] = None
    return s


def _clone(s):
    return {k: None if v is None else [t.clone() for t in v] for k, v in s.items()}


def _moments(s, i):
    m, v = s["exp_avgs"][i].cpu().double(), s["exp_avg_sqs"][i].cpu().double()
    if s["exp_avg_scales"] is None:
        return m, v
    n = m.numel()
    A, B = (s[k][i].cpu().double().repeat_interleave(256)[:n] for k in ("exp_avg_scales", "exp_avg_sq_scales"))
    return A * m.sign() * (m / 127) ** 2, B * (v / 255) ** 4


def _check(before, after, step, scale=1.0, lr=0.02, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1):
    b1, b2 = betas
    c1, c2 = 1 - b1 ** step, 1 - b2 ** step
    for i in range(len(before["params"])):
        g = before["grads"][i].cpu().double() * scale
        m0, v0 = _moments(before, i)
        src = before["masters"] or before["params"]
        p0 = src[i].cpu().double()
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        # a stored value of 8 bits is a product of up to three roundings; scaling the gradient is one more, twice in g^2
        em, ev = 8 * U * (b1 * m0.abs() + (1 - b1) * g.abs()), 10 * U * v
        den = (v / c2).sqrt() + eps
        upd = lr / c1 * m / den
        p = (1 - lr * weight_decay) * p0 - upd
        ep = lr / c1 * em / den + 20 * U * upd.abs() + 3 * U * p0.abs()
        got = (after["masters"] or after["params"])[i].cpu().double()
        if before["masters"] is None and before["params"][i].dtype == BF16:
            ep = ep + 2.0 ** -8 * p.abs()
        assert ((got - p).abs() <= ep + 1e-38).all(), (i, (got - p).abs().max())
        if before["masters"] is not None:
            assert torch.equal(after["params"][i], after["masters"][i].to(BF16))
        if before["exp_avg_scales"] is None:
            gm, gv = _moments(after, i)
            assert ((gm - m).abs() <= em + 1e-38).all() and ((gv - v).abs() <= ev + 1e-38).all()
            continue
        for x, e, key, levels, root in ((m, em, "exp_avg", 127, 2), (v, ev, "exp_avg_sq", 255, 4)):
            n = x.numel()
            pad = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
            pad[:n] = x.abs()
            A = pad.view(-1, 256).amax(1)
            pad[:n] = e
            eA = pad.view(-1, 256).amax(1)
            got_A = after[key + "_scales"][i].cpu().double()
            assert ((got_A - A).abs() <= eA + 1e-38).all()
            A, code = A.repeat_interleave(256)[:n], after[key + "s"][i].cpu().double()
            r = (x.abs() / A) ** (1 / root)
            # a value's error moves its root by e / (root r^(root-1) A), and no further than e^(1/root) where r is 0
            slack = levels * (8 * U + torch.minimum(2 * e / A / r.clamp(min=1e-30) ** (root - 1), 2 * (e / A) ** (1 / root)))
            assert ((code.abs() - levels * r).abs() <= 0.5 + slack).all(), (key, i)
            assert ((code == 0) | (code.sign() == x.sign())).all()


def _run(s, step, **kw):
    G.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=step, masters=s["masters"],
                 exp_avg_scales=s["exp_avg_scales"], exp_avg_sq_scales=s["exp_avg_sq_scales"], **{**HYPER, **kw})


KINDS = [(F32, F32, False), (F32, BF16, False), (BF16, BF16, True), (BF16, F32, True), (BF16, BF16, False),
         (BF16, F32, False)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", KINDS, ids=lambda k: f"{k[0]}-{k[1]}-{k[2]}".replace("torch.", ""))
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("step", [1, 1000])
def test_step(dev, step, shift, kind, bits):
    s = _make(SIZES, step + shift, *kind[:2], bits=bits, master=kind[2], shift=shift)
    before = _clone(s)
    _run(s, step)
    _check(before, s, step)
    assert all(torch.equal(a, b) for a, b in zip(before["grads"], s["grads"]))


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_steps(dev, bits):
    s = _make([7 * i % 611 for i in range(131)], 3, bits=bits)
    for step in (1, 2, 3):
        before = _clone(s)
        _run(s, step)
        _check(before, s, step)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_is_a_modification_in_place(dev, bits):
    s = _make([300, 5], 6, pd=BF16, gd=BF16, bits=bits, master=True)
    before = {k: [t._version for t in v] for k, v in s.items() if v is not None}
    _run(s, 1)
    for k, v in before.items():
        assert all((t._version > was) == (k != "grads") for t, was in zip(s[k], v)), k

    w = torch.nn.Parameter(torch.randn(4, 4, device=dev))
    w.grad = torch.ones_like(w)
    y = (w * w).sum()
    G.AdamW([w], state_bits=bits).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_codes_of_a_weight_are_found_again_after_a_step(dev):
    codes = torch.randint(-127, 128, (48, 16), device=dev)
    codes[:, 0] = 127
    w = torch.nn.Parameter(codes * (1 / 128))
    first = _lib.weight_codes(w)
    assert first is not None and torch.equal(first[0].float() * first[1][:, None], w.detach())
    w.grad = torch.randn_like(w)
    G.AdamW([w], lr=0.1).step()
    after = _lib.weight_codes(w)
    assert after is None or torch.equal(after[0].float() * after[1][:, None], w.detach())


@pytest.mark.parametrize("bits", [32, 8])
def test_same_inputs_same_results(dev, bits):
    a = _make([5000, 300], 5, bits=bits)
    b = _clone(a)
    _run(a, 4)
    _run(b, 4)
    for k, v in a.items():
        assert v is None or all(torch.equal(x, y) for x, y in zip(v, b[k]))


@pytest.mark.parametrize("bits", [32, 8])
def test_grad_scale(dev, bits):
    s = _make(SIZES, 6, bits=bits)
    before = _clone(s)
    _run(s, 2, grad_scale=torch.tensor(0.25, device=dev))
    _check(before, s, 2, scale=0.25)
    for bad in (float("inf"), float("nan")):
        before = _clone(s)
        _run(s, 3, grad_scale=torch.tensor([bad], device=dev))
        for k, v in s.items():
            assert v is None or all(torch.equal(x, y) for x, y in zip(v, before[k]))


def test_blocks_of_zeros_and_tiny_values(dev):
    s = _make([600], 7, bits=8)
    for k in ("grads", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales"):
        s[k][0].zero_()
    s["grads"][0][300] = 1e-37  # its moments are under 2^-120
    before = _clone(s)
    _run(s, 1)
    assert (s["exp_avgs"][0] == 0).all() and (s["exp_avg_sqs"][0] == 0).all()
    assert (s["exp_avg_scales"][0] == 0).all() and (s["exp_avg_sq_scales"][0] == 0).all()
    want = before["params"][0].double() * (1 - 0.02 * 0.1)
    assert ((s["params"][0].double() - want).abs() <= 2 * U * want.abs() + 0.02 * 1e-29 / 1e-8).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_bad_gradient_stays_in_its_block(dev, bad):
    for bits in (32, 8):
        s = _make([1000], 8, bits=bits)
        s["grads"][0][300] = bad
        _run(s, 2)
        m, v = _moments(s, 0)
        hit = torch.zeros(1000, dtype=torch.bool)
        hit[256:512] = True
        if bits == 32:
            hit = torch.arange(1000) == 300
        assert not m[hit].isfinite().any() and not v[hit].isfinite().any()
        assert m[~hit].isfinite().all() and v[~hit].isfinite().all()
        assert not s["params"][0][300].isfinite() and s["params"][0][301:].isfinite().all()


def test_dequantized_state(dev):
    s = _make([3, 256, 1001], 9, bits=8, shift=1)
    for i in range(3):
        m, v = _moments(s, i)
        gm = G.adamw_dequantize_state(s["exp_avgs"][i], s["exp_avg_scales"][i]).cpu().double()
        gv = G.adamw_dequantize_state(s["exp_avg_sqs"][i], s["exp_avg_sq_scales"][i]).cpu().double()
        assert ((gm - m).abs() <= 4 * U * m.abs()).all() and ((gv - v).abs() <= 5 * U * v.abs()).all()
    none = torch.zeros(0, dtype=torch.int8, device=dev)
    assert G.adamw_dequantize_state(none, torch.zeros(0, device=dev)).shape == (0,)


def test_optimizer_follows_torch(dev):
    """Ten steps beside torch's own AdamW in float64: each step's rounding (about 20 u of the update
    and 3 u of the parameter) adds up, and the update moves with the moments' errors (10 u)."""
    gen = torch.Generator().manual_seed(10)
    shapes = [(33, 7), (5,), (), (300,)]
    start = [torch.randn(s, generator=gen) for s in shapes]
    mine = [torch.nn.Parameter(t.to(dev)) for t in start]
    ref = [torch.nn.Parameter(t.double()) for t in start]
    idle = torch.nn.Parameter(torch.ones(3, device=dev))
    a = G.AdamW([{"params": mine[:2] + [idle]}, {"params": mine[2:], "lr": 0.05}], **HYPER)
    b = torch.optim.AdamW([{"params": ref[:2]}, {"params": ref[2:], "lr": 0.05}], **HYPER)
    for _ in range(10):
        for x, y in zip(mine, ref):
            g = torch.randn(x.shape, generator=gen)
            x.grad, y.grad = g.to(dev), g.double()
        mine[0].grad = mine[0].grad.t().contiguous().t()  # same values, other strides
        a.step()
        b.step()
    for x, y in zip(mine, ref):
        assert ((x.detach().cpu().double() - y.detach()).abs() <= 10 * (40 * U * 0.05 + 3 * U * 6)).all()
    assert torch.equal(idle.detach().cpu(), torch.ones(3)) and not a.state[idle]


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_state_travels(dev, bits):
    def make():
        gen = torch.Generator().manual_seed(11)
        p = [torch.nn.Parameter(torch.randn(700, generator=gen).to(dev, d)) for d in (F32, BF16)]
        return p, G.AdamW(p, lr=0.01, state_bits=bits)

    def go(p, opt, seed):
        for x in p:
            x.grad = torch.randn(700, generator=torch.Generator().manual_seed(seed)).to(dev, x.dtype)
        opt.step()

    p, opt = make()
    for k in range(3):
        go(p, opt, k)
    q, other = make()
    with torch.no_grad():
        for x, y in zip(q, p):
            x.copy_(y)
    other.load_state_dict(opt.state_dict())
    go(p, opt, 9)
    go(q, other, 9)
    for x, y in zip(p, q):
        assert torch.equal(x, y) and opt.state[x]["step"] == other.state[y]["step"] == 4
        for k, v in opt.state[x].items():
            w = other.state[y][k]
            assert not isinstance(v, torch.Tensor) or (v.dtype == w.dtype and torch.equal(v, w) and v.data_ptr() != w.data_ptr())


def test_training_in_8_bits_solves_a_regression(dev):
    """A linear regression without noise, 1024 weights from N(0, 1): the learning rates sum to 30, several times
    the way any weight has to go, and fall to 0, so that what is left of the loss says whether the moments' 8 bits
    let the iteration settle."""
    gen = torch.Generator().manual_seed(12)
    x = torch.randn(512, 64, generator=gen).to(dev)
    y = x @ torch.randn(64, 16, generator=gen).to(dev)
    w = torch.nn.Parameter(torch.zeros(64, 16, device=dev))
    opt = G.AdamW([w], state_bits=8, weight_decay=0.0)
    for k in range(600):
        loss = (x @ w - y).square().mean()
        w.grad, = torch.autograd.grad(loss, [w])
        opt.param_groups[0]["lr"] = 0.1 * (1 - k / 600)
        opt.step()
    assert loss.item() < 0.01 * y.square().mean().item()


def test_refusals(dev):
    s = _make([4, 300], 1)
    e = _make([4, 300], 1, bits=8)

    def call(**kw):
        kw = {**dict(params=s["params"], grads=s["grads"], exp_avgs=s["exp_avgs"], exp_avg_sqs=s["exp_avg_sqs"], step=1,
                     lr=1e-3), **kw}
        G.adamw_step(kw.pop("params"), kw.pop("grads"), kw.pop("exp_avgs"), kw.pop("exp_avg_sqs"), **kw)

    call(lr=0.0)
    bad = [dict(step=0), dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
           dict(eps=-1.0), dict(weight_decay=float("inf")), dict(params=[t.cpu() for t in s["params"]]),
           dict(grads=[t.cpu() for t in s["grads"]]), dict(grads=s["grads"][:1]), dict(grads=s["grads"][::-1]),
           dict(params=[t.half() for t in s["params"]]), dict(grads=[t.half() for t in s["grads"]]),
           dict(params=[s["params"][0].bfloat16(), s["params"][1]]), dict(exp_avgs=[t.bfloat16() for t in s["exp_avgs"]]),
           dict(exp_avgs=e["exp_avgs"], exp_avg_sqs=e["exp_avg_sqs"]),
           dict(exp_avg_scales=e["exp_avg_scales"], exp_avg_sq_scales=e["exp_avg_sq_scales"]),
           dict(exp_avgs=e["exp_avgs"], exp_avg_sqs=e["exp_avg_sqs"], exp_avg_scales=e["exp_avg_scales"]),
           dict(masters=s["masters"] or [t.clone() for t in s["params"]]),
           dict(grad_scale=torch.ones(2, device=dev)), dict(grad_scale=torch.ones(1)),
           dict(params=[torch.zeros(8, device=dev)[::2], s["params"][1]])]
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        G.AdamW([torch.nn.Parameter(s["params"][0])], state_bits=16)
    with pytest.raises(ValueError):
        G.adamw_dequantize_state(e["exp_avgs"][0].float(), e["exp_avg_scales"][0])
    with pytest.raises(ValueError):
        G.adamw_dequantize_state(e["exp_avgs"][1], e["exp_avg_scales"][0])
