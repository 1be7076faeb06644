"""Where a language model begins and ends: vectors of tokens, and log probabilities of them.

The kernels are ``gs_embedding_fwd`` / ``_bwd`` and ``gs_logprobs_fwd`` / ``_bwd`` of libgruscan.so,
their checks and autograd in csrc/torch_sequence_ops.cpp. No counterpart in the reference.
"""

from __future__ import annotations

from typing import Tuple

import torch

from . import _lib


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[tokens]`` [..., K] for ``tokens`` [...] (int32 or int64) and ``weight`` [V, K]
    (float32 or bfloat16). A negative token marks padding: a row of zeros that sends no gradient; one
    of V or more gives NaN and sends none. Differentiable in weight (once): the gradient is dense,
    its sums are float32, and it is the same from run to run. At most 2^25 tokens and 2^25 rows of
    2^20 elements."""
    try:
        return (_lib._ops or _lib.ops()).embedding(tokens, weight, scale)
    except TypeError as e:
        raise ValueError(f"embedding: tokens and weight must be tensors and scale a number ({e})") from None


def token_logprobs(
    logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(logprobs, entropy, top_logprobs, top_tokens)`` of ``logits`` [..., V] (float32 or bfloat16) and
    ``tokens`` [...] (int32 or int64): ``log softmax(logits)`` at the tokens [...], the entropy
    ``-sum p log p`` [...], and the ``top`` (0 to 32) likeliest tokens [..., top] (int64) in falling
    order, of equal ones the lowest first, with their log probabilities. Results are float32.

    A logit of -infinity is a token that cannot come; a row of those alone has log probabilities
    -infinity, entropy 0 and no gradient. A NaN or +infinity makes a row's results NaN. A negative
    token does not count: its log probability is 0 and sends no gradient (its row's entropy does);
    one of V or more gives NaN. The logits of a row to which no gradient comes get zeros, also NaN
    ones. At most 2^23 rows of 2^24 logits, 2^19 with ``top``. Differentiable in logits
    through logprobs and entropy (once): ``-logprobs.sum() / (tokens >= 0).sum()`` is the
    cross entropy over the tokens that count."""
    try:
        return (_lib._ops or _lib.ops()).token_logprobs(logits, tokens, top)
    except TypeError as e:
        raise ValueError(f"token_logprobs: logits and tokens must be tensors and top a number ({e})") from None
