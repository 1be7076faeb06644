"""Scratch of the embedding's gradient: lists, and rows of sums for the lists of several chunks alone. No GPU needed."""

from __future__ import annotations

import ctypes

import pytest

from gru_qat_amd import _lib


def _bytes(M, V, K):
    a = _lib.GsEmbeddingBwdArgs(tokens=4096, dout=4096, dw=4096, M=M, V=V, K=K, sdo=K, scale=1.0, token_bits=64)
    return _lib.load().gs_embedding_bwd_scratch_bytes(ctypes.byref(a))


def _lists(M, V):
    """Counts, starts, places and positions, a chunk's 16 bytes for every list of 17 or more, and padding."""
    return 8 * V + 8 * M + 16 * (min(V, M // 17) + M // 64) + 8 * 256


# many long lists, of one chunk each for the most part; a vocabulary of one; fewer positions than a chunk
@pytest.mark.parametrize("M,V,K", [(1 << 20, 128_000, 4096), (16384, 32000, 1024), (1 << 20, 1, 64), (64, 10, 4096), (1 << 25, 50_000, 512)])
def test_rows_of_sums(M, V, K):
    chunk = 2048 if M >= 1 << 20 else 64
    rows = 2 * M // chunk if M > chunk else 0
    assert 0 < _bytes(M, V, K) <= _lists(M, V) + 4 * K * rows


def test_a_large_batch_of_a_large_vocabulary():
    """2^20 tokens of 128 000 x 4096: tens of megabytes, where a row for every list of 17 or more would be a gigabyte."""
    assert _bytes(1 << 20, 128_000, 4096) < 40e6
