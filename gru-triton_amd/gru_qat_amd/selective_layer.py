"""A residual layer around the selective state space scan, trainable and servable.

``x, z = split(x W_i^T)`` (``linear_act``), ``u = silu(conv(x))`` (``causal_conv``),
``d, B, C = split(u W_x^T)``, ``delta = d W_d^T``, ``y = scan(u, delta, ...) silu(z)``
(``selective_scan``), ``x + y W_o^T`` (``linear_act`` with the residual in its epilogue); one token:
``causal_conv_step`` and ``selective_step``. No counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Any, NamedTuple, Optional, Tuple

import torch

from .conv import causal_conv, causal_conv_step
from .linear import linear_act
from .selective import selective_scan, selective_step


class SelectiveState(NamedTuple):
    """What a layer carries from one call to the next: the last inputs of the convolution
    [rows, taps - 1, hidden] in the layer's type, and the states [rows, hidden, states] in float32."""

    conv: torch.Tensor
    ssm: torch.Tensor


class SelectiveLayer(torch.nn.Module):
    """``size``: features of x and y; ``hidden``: channels of the recurrence, with ``states`` states
    each; ``rank``: of the projection to step sizes (hidden / 16 rounded up when None). Projections and the
    convolution (and x) are float32 or bfloat16; A, D, the step sizes' bias and states are float32. States decay at
    1 to ``states`` times a step size that starts between 0.001 and 0.1."""

    def __init__(self, size: int, hidden: int, *, states: int = 16, taps: int = 4, rank: Optional[int] = None,
                 batch_first: bool = False, device: Any = None, dtype: Any = None) -> None:
        super().__init__()
        if rank is None:
            rank = -(-hidden // 16)
        if size < 1 or hidden < 1 or rank < 1:
            raise ValueError(f"SelectiveLayer: size, hidden and rank must be > 0; got {size}, {hidden} and {rank}")
        if not 1 <= states <= 32 or not 2 <= taps <= 4:
            raise ValueError(f"SelectiveLayer: states must be 1 to 32 and taps 2 to 4; got {states} and {taps}")
        self.hidden, self.states, self.taps, self.rank, self.batch_first = hidden, states, taps, rank, batch_first

        def uniform(rows: int, cols: int) -> torch.nn.Parameter:
            w = torch.empty(rows, cols, device=device, dtype=dtype)
            return torch.nn.Parameter(w.uniform_(-1 / math.sqrt(cols), 1 / math.sqrt(cols)))

        self.weight_i = uniform(2 * hidden, size)
        self.weight_c = uniform(hidden, taps)
        self.bias_c = torch.nn.Parameter(torch.zeros(hidden, device=device, dtype=dtype))
        self.weight_x = uniform(rank + 2 * states, hidden)
        self.weight_d = uniform(hidden, rank)
        self.weight_o = uniform(size, hidden)
        kw = dict(device=device, dtype=torch.float32)
        step = torch.exp(torch.rand(hidden, **kw) * math.log(100.0)) * 1e-3
        self.bias_d = torch.nn.Parameter(step + torch.log(-torch.expm1(-step)))  # softplus(bias_d) = step
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1, states + 1, **kw)).repeat(hidden, 1))
        self.D = torch.nn.Parameter(torch.ones(hidden, **kw))

    def _projected(self, u: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        d, b, c = linear_act(u, self.weight_x).split([self.rank, self.states, self.states], -1)
        return linear_act(d, self.weight_d), b, c

    def forward(self, x: torch.Tensor, state: Optional[SelectiveState] = None,
                reset: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, SelectiveState]:
        """``(y, state)`` for x [T, B, size] ([B, T, size] when ``batch_first``); ``state`` of B rows
        continues a sequence, ``reset`` [T, B] bool starts new ones inside the rows."""
        h, z = linear_act(x, self.weight_i).chunk(2, -1)
        u, last = causal_conv(h, self.weight_c, self.bias_c, state.conv if state else None, reset=reset,
                              batch_first=self.batch_first)
        delta, b, c = self._projected(u)
        y, ssm = selective_scan(u, delta, -torch.exp(self.A_log), b, c, self.D, z, state.ssm if state else None,
                                delta_bias=self.bias_d, reset=reset, batch_first=self.batch_first)
        return linear_act(y, self.weight_o, residual=x), SelectiveState(last, ssm)

    def new_state(self, rows: int) -> SelectiveState:
        """A cache of ``rows`` requests that have seen nothing yet."""
        return SelectiveState(self.weight_c.new_zeros(rows, self.taps - 1, self.hidden),
                              self.D.new_zeros(rows, self.hidden, self.states))

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: SelectiveState, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y [B, size] for one token x [B, size] of each request; the rows ``slots`` of ``state`` are
        advanced in place."""
        h, z = linear_act(x, self.weight_i).chunk(2, -1)
        u = causal_conv_step(h, self.weight_c, self.bias_c, state.conv, slots)
        delta, b, c = self._projected(u)
        y = selective_step(u, delta, -torch.exp(self.A_log), b, c, state.ssm, slots, D=self.D, z=z, delta_bias=self.bias_d)
        return linear_act(y, self.weight_o, residual=x)
