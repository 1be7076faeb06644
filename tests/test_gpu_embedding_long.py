"""The embedding's gradient over many positions: lists in several windows of 2^17, and the work of a frequent token."""

from __future__ import annotations

import time

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _grad(tokens, V, dout, scale=1.0):
    w = torch.zeros(V, dout.shape[-1], device=dout.device, dtype=dout.dtype, requires_grad=True)
    return torch.autograd.grad(G.embedding(tokens, w, scale=scale), w, dout)[0]


def _tokens(M, dev):
    """One of nearly all positions, one of every 4001st (chunks over many windows), short lists of 12, one that
    occurs in two windows alone, at their ends, and padding."""
    t = torch.zeros(M, dtype=torch.int64)
    t[::4001] = 1
    t[7::80021] = torch.arange(len(t[7::80021])) // 12 + 4
    if M > 1 << 18:
        t[(1 << 17) - 300:(1 << 17)] = 2
        t[(1 << 18) - 500:1 << 18] = 2
    t[3::977] = -1
    return t.to(dev)


# a window exactly, one position more, and several with a last one of few
@pytest.mark.parametrize("M", [1 << 17, (1 << 17) + 1, (1 << 18) + 40, (1 << 20) + 77])
def test_lists_over_windows(dev, M):
    """Whole numbers, whose sums are exact in any order, and others, which are the same from run to run and near."""
    V, K = 10, 3
    tokens = _tokens(M, dev)
    g = torch.Generator().manual_seed(M)
    whole = torch.randint(-3, 4, (M, K), generator=g)
    some = tokens.cpu() >= 0
    want = torch.zeros(V, K, dtype=torch.int64).index_add_(0, tokens.cpu()[some], whole[some])
    assert torch.equal(_grad(tokens, V, whole.float().to(dev)).cpu(), want.float())
    noise = torch.randn(M, K, generator=g)
    got = _grad(tokens, V, noise.to(dev))
    for _ in range(2):
        assert torch.equal(got, _grad(tokens, V, noise.to(dev)))
    d = noise.double()[some]
    want = torch.zeros(V, K, dtype=torch.float64).index_add_(0, tokens.cpu()[some], d)
    size = torch.zeros(V, K, dtype=torch.float64).index_add_(0, tokens.cpu()[some], d.abs())
    # a wave adds a quarter of a chunk of 2048 at most, then chunks are added
    assert ((got.cpu() - want).abs() <= (512 + 3 + M / 256 + 2) * 2.0 ** -24 * size).all()


def test_order_does_not_depend_on_where_a_list_lies(dev):
    """The same rows at positions in other windows, and beside other lists, are summed in the same order."""
    M, n, K = (1 << 20) + 9, 1500, 4
    rows = torch.randn(n, K, generator=torch.Generator().manual_seed(5))
    got = []
    for first, step in ((3, 699), ((1 << 17) - 600, 1), (0, 1)):
        tokens, dout = torch.ones(M, dtype=torch.int64), torch.zeros(M, K)
        at = first + step * torch.arange(n)  # on the CPU, where an index past the end is an error
        tokens[at], dout[at] = 0, rows
        got.append(_grad(tokens.to(dev), 2, dout.to(dev))[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_the_work_of_one_token_everywhere(dev):
    """2^23 positions of one token: a list's entries are read some 64 times each, which with everything else takes
    milliseconds. Once for every chunk and window, as many as 4.5 TB, they would take half a second at 10 TB/s."""
    M, K = 1 << 23, 8
    tokens = torch.zeros(M, dtype=torch.int32, device=dev)
    dout = torch.ones(M, K, device=dev, dtype=BF16)
    took = []
    for _ in range(2):
        torch.cuda.synchronize()
        t = time.perf_counter()
        dw = _grad(tokens, 2, dout, scale=2.0 ** -20)
        torch.cuda.synchronize()
        took.append(time.perf_counter() - t)
    assert (dw[0] == 8).all() and (dw[1] == 0).all()
    assert min(took) < 0.2, took
