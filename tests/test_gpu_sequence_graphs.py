"""The operators over sequences of tokens in captured graphs (every replay, on inputs that have changed
since, equals the eager call bit for bit), on other streams, and two at a time."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
from test_gpu_operator_graphs import _replays

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _gen(i):
    return torch.Generator().manual_seed(i)


# one chunk, several, and waves that share nothing
@pytest.mark.parametrize("T,B,H", [(30, 2, 33), (400, 1, 70), (700, 24, 260)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_scan(dev, T, B, H, dtype):
    N = 8
    shapes = dict(u=(T, B, H), delta=(T, B, H), B=(T, B, N), C=(T, B, N), z=(T, B, H))
    t = {k: torch.zeros(s, device=dev, dtype=dtype, requires_grad=True) for k, s in shapes.items()}
    A = -torch.rand(H, N, generator=_gen(9)).to(dev) - 0.1
    h0 = torch.zeros(B, H, N, device=dev, requires_grad=True)
    reset = torch.zeros(T, B, device=dev, dtype=torch.bool)
    dy = torch.ones(T, B, H, device=dev, dtype=dtype)

    def fresh(i):
        g = _gen(i)
        return (*(torch.randn(s, generator=g).to(dtype) for s in shapes.values()), torch.randn(h0.shape, generator=g),
                torch.rand(T, B, generator=g) < 0.03)

    def call():
        y, h = G.selective_scan(t["u"], t["delta"], A, t["B"], t["C"], None, t["z"], h0, reset=reset)
        return (y, h, *torch.autograd.grad((y, h), (*t.values(), h0), (dy, torch.ones_like(h))))

    _replays((*t.values(), h0, reset), call, fresh)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_conv(dev, dtype):
    T, B, C, W = 50, 2, 140, 4
    x, w, b, s = (torch.zeros(n, device=dev, dtype=dtype, requires_grad=True) for n in ((T, B, C), (C, W), (C,), (B, W - 1, C)))
    dy = torch.ones(T, B, C, device=dev, dtype=dtype)

    def call():
        y, last = G.causal_conv(x, w, b, s)
        return (y, last, *torch.autograd.grad(y, (x, w, b, s), dy))

    _replays((x, w, b, s), call, lambda i: tuple(torch.randn(t.shape, generator=_gen(i)).to(dtype) for t in (x, w, b, s)))


@pytest.mark.parametrize("M,V", [(300, 50), (9000, 6000)])
def test_embedding(dev, M, V):
    K = 40
    tokens = torch.zeros(M, device=dev, dtype=torch.int64)
    w = torch.zeros(V, K, device=dev, requires_grad=True)
    dy = torch.randn(M, K, device=dev)

    def call():
        y = G.embedding(tokens, w, scale=2.0)
        return (y, *torch.autograd.grad(y, w, dy))

    def fresh(i):
        g = _gen(i)
        return (V * torch.rand(M, generator=g) ** 4).long() - (torch.rand(M, generator=g) < 0.1).long(), torch.randn(V, K, generator=g)

    _replays((tokens, w), call, fresh)


@pytest.mark.parametrize("M,V,top", [(5, 3000, 4), (600, 100, 0)])
def test_logprobs(dev, M, V, top):
    x = torch.zeros(M, V, device=dev, requires_grad=True)
    tokens = torch.zeros(M, device=dev, dtype=torch.int32)
    ones = torch.ones(M, device=dev)

    def call():
        r = G.token_logprobs(x, tokens, top=top)
        return (*r, *torch.autograd.grad(r[:2], x, (ones, ones)))

    _replays((x, tokens), call, lambda i: (torch.randn(M, V, generator=_gen(i)), torch.randint(-1, V, (M,), generator=_gen(i)).int()))


def test_steps(dev):
    """A whole serving step captured: the caches are what changes."""
    torch.manual_seed(0)
    model = G.TokenModel(60, 16, [G.SelectiveLayer(16, 24, device=dev), G.GatedLinearLayer(16, 20, device=dev)], device=dev)
    states = model.new_states(6)
    caches = (states[0].conv, states[0].ssm, states[1])
    tokens = torch.zeros(3, device=dev, dtype=torch.int64)
    slots = torch.tensor([4, 0, 2], device=dev, dtype=torch.int32)

    def call():
        lp, best = model.step(tokens, states, slots, top=3)
        return (lp, best, *caches)

    def fresh(i):
        g = _gen(i)
        return (torch.randint(0, 60, (3,), generator=g), *(torch.randn(c.shape, generator=g) for c in caches))

    _replays((tokens, *caches), call, fresh)


def test_two_streams_at_once(dev):
    """Calls on two streams have workspaces of their own."""
    g = _gen(3)
    T, B, H, N = 300, 3, 200, 16
    one = [torch.randn(s, generator=g).to(dev) for s in ((T, B, H), (T, B, H), (T, B, N), (T, B, N))]
    two = [torch.randn(s, generator=g).to(dev) for s in ((T, B, H), (T, B, H), (T, B, N), (T, B, N))]
    A = -torch.rand(H, N, generator=g).to(dev) - 0.1
    tokens = torch.randint(0, 500, (6000,), generator=g).to(dev)
    w = torch.randn(500, 96, generator=g).to(dev)
    d = torch.randn(6000, 96, generator=g).to(dev)

    def run(t):
        leaves = [x.detach().requires_grad_(True) for x in t]
        y, _ = G.selective_scan(leaves[0], leaves[1], A, leaves[2], leaves[3])
        leaf = w.detach().requires_grad_(True)
        out = G.embedding(tokens, leaf)
        lp = G.token_logprobs(out, tokens % 96, top=2)
        return [y, *torch.autograd.grad(y, leaves, torch.ones_like(y)), *torch.autograd.grad(out, leaf, d), lp[0], lp[2]]

    want = [run(one), run(two)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[k] = run((one, two)[k])
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))
