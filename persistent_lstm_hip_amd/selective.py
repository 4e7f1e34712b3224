"""The forecaster of gated.py with a selective state space scan in the place of the gated recurrence, on the operators of
ops.py:

* SelectiveScanBlock      -- u, z = W_in layer_norm(x); u = causal_conv(u); dt, B, C from u;
                             y = x + dropout(W_out selective_scan(u, dt, A, B, C, D, z)), over a sequence or one step of it.
* SelectiveScanRegressor  -- GatedScanRegressor with such blocks: trained over whole sequences, served token by token.

The gated recurrence keeps one number per channel and forgets by its gates; here a channel keeps `states` numbers that decay
at rates of their own, and what is written to them and read from them is chosen by the input.

`python -m persistent_lstm_hip_amd.gated_demo --block selective` trains one on synthetic series, then serves it.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple, Union

import torch
import torch.nn as nn

from .gated import GatedScanRegressor, _draw
from .ops import causal_conv, causal_conv_step, dropout_add, layer_norm, selective_scan, selective_scan_step

State = Tuple[torch.Tensor, torch.Tensor]  # the convolution's last inputs, the scan's states


class SelectiveScanBlock(nn.Module):
    """One residual block of width dim, expand * dim channels wide inside.  Its state is a pair: the convolution's
    [batch, width - 1, channels], the scan's [batch, channels, states] float32.  The convolution's is of the activations'
    type, under autocast the lower one; forward takes one of any type, step one of the activations' type or float32."""

    def __init__(self, dim: int, dropout: float = 0.0, *, states: int = 16, width: int = 4, expand: int = 2):
        super().__init__()
        channels, self.rank, self.states, self.dropout = expand * dim, max(1, dim // 16), states, dropout
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.norm_bias = nn.Parameter(torch.zeros(dim))
        self.inner = nn.Linear(dim, 2 * channels, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(channels, width).uniform_(-1.0, 1.0) / math.sqrt(width))
        self.conv_bias = nn.Parameter(torch.zeros(channels))
        self.coefs = nn.Linear(channels, self.rank + 2 * states, bias=False)
        self.steps = nn.Linear(self.rank, channels, bias=False)
        # step sizes from 0.001 to 0.1, channel by channel, and decays of 1 to `states`
        step = torch.exp(torch.linspace(math.log(0.001), math.log(0.1), channels))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1.0, states + 1)).repeat(channels, 1))
        self.D = nn.Parameter(torch.ones(channels))
        self.out = nn.Linear(channels, dim, bias=False)

    def _inner(self, x: torch.Tensor):
        return self.inner(layer_norm(x, self.norm_weight, self.norm_bias)).chunk(2, -1)

    def _filter(self, u: torch.Tensor):
        """The convolution's weight and bias for u, in 32 bits where u is of another 16-bit type (under autocast)."""
        w, b = self.conv_weight, self.conv_bias
        return (w, b) if w.dtype in (u.dtype, torch.float32) else (w.float(), b.float())

    def _coefs(self, u: torch.Tensor):
        """What the scan of u takes beside it: dt, A, B, C, D."""
        dt, B, C = self.coefs(u).split([self.rank, self.states, self.states], -1)
        return self.steps(dt), -torch.exp(self.A_log.float()), B, C, self.D.float()

    def forward(self, x: torch.Tensor, state: Optional[State] = None, *, lengths=None, seed: int = 0,
                offset: Union[int, torch.Tensor, None] = None):
        """x [batch, time, dim] -> (y, the state after it).  (seed, offset) pick the dropout mask in training mode, as in
        GatedScanBlock."""
        before, h0 = state if state is not None else (None, None)
        u, z = self._inner(x)
        if before is not None:
            before = before.to(u.dtype)
        u, before = causal_conv(u, *self._filter(u), before, lengths=lengths)
        h, h_n = selective_scan(u, *self._coefs(u), z, h0, dt_bias=self.dt_bias.float(), lengths=lengths)
        p = self.dropout if self.training else 0.0
        if offset is None:
            offset = _draw(x.device) if p > 0.0 else 0
        return dropout_add(self.out(h).to(x.dtype), x, p=p, seed=seed, offset=offset), (before, h_n)

    def step(self, x: torch.Tensor, state: State) -> torch.Tensor:
        """One token x [batch, dim] -> y; both parts of the state are updated in place.  For inference."""
        u, z = self._inner(x)
        if state[0].dtype == torch.float32 and u.dtype != torch.float32:  # under autocast: it holds 16-bit inputs exactly
            u, last = causal_conv_step(u, state[0].to(u.dtype), *self._filter(u))
            state[0].copy_(last)
        else:
            u, _ = causal_conv_step(u, state[0], *self._filter(u), inplace=True)
        dt, A, B, C, D = self._coefs(u)
        h, _ = selective_scan_step(u, dt, A, B, C, state[1], D, z, dt_bias=self.dt_bias.float(), inplace=True)
        return x + self.out(h)

    def initial_state(self, batch: int) -> State:
        w = self.conv_weight
        kind = self.inner.weight.dtype
        if kind != torch.float32 and torch.is_autocast_enabled(w.device.type):  # (float32 holds either 16-bit type)
            kind = torch.get_autocast_dtype(w.device.type)
        return (torch.zeros(batch, w.size(1) - 1, w.size(0), dtype=kind, device=w.device),
                torch.zeros(batch, w.size(0), self.states, dtype=torch.float32, device=w.device))


class SelectiveScanRegressor(GatedScanRegressor):
    """GatedScanRegressor, its dropout masks included, with SelectiveScanBlocks."""

    def __init__(self, input_dim: int, hidden_dim: int, output_dim: int, n_layers: int, dropout: float = 0.2, *,
                 states: int = 16, width: int = 4, expand: int = 2):
        self._options = dict(states=states, width=width, expand=expand)
        super().__init__(input_dim, hidden_dim, output_dim, n_layers, dropout)

    def _block(self, dim: int, dropout: float) -> nn.Module:
        return SelectiveScanBlock(dim, dropout, **self._options)

    def initial_state(self, batch: int) -> List[State]:
        return [block.initial_state(batch) for block in self.blocks]
