"""A residual layer around the gated linear recurrence, trainable and servable.

``gi = x W_g^T + b_g`` (``linear_act``), ``out = scan(gi)`` (``gated_linear_scan``; one
token: ``gated_linear_step``), ``y = out W_o^T + b_o + x`` (``linear_act`` with the
residual in its epilogue). No counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Any, Optional, Tuple

import torch

from .gated_linear import gated_linear_scan, gated_linear_step
from .linear import linear_act


class GatedLinearLayer(torch.nn.Module):
    """``size``: features of x and y; ``hidden``: channels of the recurrence. Parameters
    (and x) are float32 or bfloat16; states are float32. The update gate's bias starts
    where channels remember for 1 / (1 - z) = 3 to 50 steps."""

    def __init__(self, size: int, hidden: int, *, activation: str = "tanh", batch_first: bool = False,
                 device: Any = None, dtype: Any = None) -> None:
        super().__init__()
        if size < 1 or hidden < 1:
            raise ValueError(f"GatedLinearLayer: size and hidden must be > 0; got {size} and {hidden}")
        if activation not in ("tanh", "identity"):
            raise ValueError(f"GatedLinearLayer: activation must be 'tanh' or 'identity'; got {activation!r}")
        kw = dict(device=device, dtype=dtype)
        self.hidden, self.activation, self.batch_first = hidden, activation, batch_first
        self.weight_g = torch.nn.Parameter(torch.empty(2 * hidden, size, **kw))
        self.bias_g = torch.nn.Parameter(torch.empty(2 * hidden, **kw))
        self.weight_o = torch.nn.Parameter(torch.empty(size, hidden, **kw))
        self.bias_o = torch.nn.Parameter(torch.zeros(size, **kw))
        with torch.no_grad():
            self.weight_g.uniform_(-1 / math.sqrt(size), 1 / math.sqrt(size))
            self.weight_o.uniform_(-1 / math.sqrt(hidden), 1 / math.sqrt(hidden))
            self.bias_g[:hidden].uniform_(0.7, 3.9)
            self.bias_g[hidden:].zero_()

    def forward(self, x: torch.Tensor, h0: Optional[torch.Tensor] = None,
                reset: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(y, h_T)`` for x [T, B, size] ([B, T, size] when ``batch_first``)."""
        gi = linear_act(x, self.weight_g, self.bias_g)
        out, h = gated_linear_scan(gi, h0, activation=self.activation, reset=reset, batch_first=self.batch_first)
        return linear_act(out, self.weight_o, self.bias_o, residual=x), h

    def new_state(self, rows: int) -> torch.Tensor:
        """A cache of ``rows`` requests that have seen nothing yet."""
        return torch.zeros(rows, self.hidden, device=self.weight_g.device)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y [B, size] for one token x [B, size] of each request; ``state`` [S, hidden] float32
        is advanced in place (``gated_linear_step``)."""
        out = gated_linear_step(linear_act(x, self.weight_g, self.bias_g), state, slots, activation=self.activation)
        return linear_act(out, self.weight_o, self.bias_o, residual=x)
