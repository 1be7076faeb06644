"""The scan, the step and the linear operator captured in a graph: every replay, on inputs
that have changed since, equals the eager call bit for bit."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu


def _replays(inputs, call, fresh):
    """call() -> tensors; fresh(i) -> new values of the inputs, eagerly."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for i in range(4):
        with torch.no_grad():
            for t, v in zip(inputs, fresh(i)):
                t.copy_(v)
        start = [t.detach().clone() for t in inputs]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in captured]
        with torch.no_grad():
            for t, v in zip(inputs, start):  # the step advances its state
                t.copy_(v)
        for k, (a, b) in enumerate(zip(got, call())):
            assert torch.equal(a, b.detach()), (i, k)


# one workgroup a row, and tiles chained through memory
@pytest.mark.parametrize("shape", [(40, 3, 33), (1500, 1, 40)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_scan(dev, shape, dtype):
    T, B, H = shape
    gi = torch.zeros(T, B, 2 * H, device=dev, dtype=dtype, requires_grad=True)
    h0 = torch.zeros(B, H, device=dev, requires_grad=True)
    reset = torch.zeros(T, B, device=dev, dtype=torch.bool)
    dy = torch.ones(T, B, H, device=dev, dtype=dtype)

    def fresh(i):
        g = torch.Generator().manual_seed(i)
        return (torch.randn(gi.shape, generator=g).to(dtype), torch.randn(h0.shape, generator=g),
                torch.rand(reset.shape, generator=g) < 0.05)

    def call():
        out, last = G.gated_linear_scan(gi, h0, reset=reset)
        return (out, last, *torch.autograd.grad(out, (gi, h0), dy))

    _replays((gi, h0, reset), call, fresh)


def test_step(dev):
    B, H, S = 5, 70, 9
    gi = torch.zeros(B, 2 * H, device=dev)
    state = torch.zeros(S, H, device=dev)
    slots = torch.zeros(B, device=dev, dtype=torch.int32)

    def fresh(i):
        g = torch.Generator().manual_seed(i)
        rows = torch.randperm(S, generator=g)[:B].int()
        rows[i % B] = -1
        return torch.randn(gi.shape, generator=g), torch.randn(state.shape, generator=g), rows

    slots.copy_(fresh(0)[2])
    _replays((gi, state, slots), lambda: (G.gated_linear_step(gi, state, slots), state), fresh)


# few rows; a split K; small products side by side; rows that are copied to padded ones
@pytest.mark.parametrize("shape", [(4, 96, 64), (64, 64, 4096), (300, 128, 96), (601, 501, 333)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_linear(dev, shape, dtype):
    M, N, K = shape
    x = torch.zeros(M, K, device=dev, dtype=dtype, requires_grad=True)
    w = torch.zeros(N, K, device=dev, dtype=dtype, requires_grad=True)
    b = torch.zeros(N, device=dev, dtype=dtype, requires_grad=True)
    dy = torch.ones(M, N, device=dev, dtype=dtype)

    def fresh(i):
        g = torch.Generator().manual_seed(i)
        return (torch.randn(M, K, generator=g).to(dtype), (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype),
                torch.randn(N, generator=g).to(dtype))

    def call():
        y = G.linear_act(x, w, b, activation="silu")
        return (y, *torch.autograd.grad(y, (x, w, b), dy))

    _replays((x, w, b), call, fresh)
