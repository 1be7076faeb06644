"""A language model out of the package's residual layers: vectors of tokens (``embedding``), a
stack of ``GatedLinearLayer`` and ``SelectiveLayer``, and log probabilities of given tokens
(``token_logprobs``) from logits whose weight is the embedding's. Trainable and servable. No
counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Any, Iterable, List, Optional, Tuple

import torch

from .linear import linear_act
from .tokens import embedding, token_logprobs


class TokenModel(torch.nn.Module):
    """``layers``: residual layers of ``size`` features in the model's type, all with the same
    ``batch_first``. The embedding is scaled by sqrt(size), so that one weight serves both ends. A
    negative token is padding: its vector is zero, and as a target it does not count."""

    def __init__(self, vocabulary: int, size: int, layers: Iterable[torch.nn.Module], *, device: Any = None,
                 dtype: Any = None) -> None:
        super().__init__()
        if vocabulary < 1 or size < 1:
            raise ValueError(f"TokenModel: vocabulary and size must be > 0; got {vocabulary} and {size}")
        self.weight = torch.nn.Parameter(torch.empty(vocabulary, size, device=device, dtype=dtype))
        self.layers = torch.nn.ModuleList(layers)
        self.scale = math.sqrt(size)
        with torch.no_grad():
            self.weight.normal_(std=1 / math.sqrt(size))

    def hidden(self, tokens: torch.Tensor, states: Optional[List[Any]] = None,
               reset: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, List[Any]]:
        """``(y, states)`` for tokens [T, B] ([B, T] where the layers are ``batch_first``): y [..., size],
        and the layers' states, with which a following call continues."""
        y = embedding(tokens, self.weight, scale=self.scale)
        last = []
        for k, layer in enumerate(self.layers):
            y, state = layer(y, states[k] if states is not None else None, reset)
            last.append(state)
        return y, last

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor, *, states: Optional[List[Any]] = None,
                reset: Optional[torch.Tensor] = None, top: int = 0) -> Tuple[torch.Tensor, ...]:
        """``(logprobs, entropy, top_logprobs, top_tokens)`` of the targets [T, B] that follow the
        tokens, as ``token_logprobs`` returns them. The training loss is
        ``-logprobs.sum() / (targets >= 0).sum()``: padded targets add 0, and a mean would count them."""
        y, _ = self.hidden(tokens, states, reset)
        return token_logprobs(linear_act(y, self.weight), targets, top=top)

    def new_states(self, rows: int) -> List[Any]:
        """Caches of ``rows`` requests that have seen nothing yet, one for each layer."""
        return [layer.new_state(rows) for layer in self.layers]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, states: List[Any], slots: Optional[torch.Tensor] = None, *,
             top: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(top_logprobs, top_tokens)`` [B, top] of what follows one token [B] of each request; the
        rows ``slots`` of the layers' caches are advanced in place."""
        y = embedding(tokens, self.weight, scale=self.scale)
        for layer, state in zip(self.layers, states):
            y = layer.step(y, state, slots)
        _, _, logprobs, best = token_logprobs(linear_act(y, self.weight), tokens, top=top)
        return logprobs, best
