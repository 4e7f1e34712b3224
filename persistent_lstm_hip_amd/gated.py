"""A recurrent forecaster that trains in parallel over time, on the block operators (ops.py):

* GatedScanBlock      -- y = x + dropout(W_o scan(W_g layer_norm(x))), over a sequence or one step of it.
* GatedScanRegressor  -- StandardLSTMRegressor's shape (x [B, T, I] -> [B, O] from a row's last step) with such blocks
                         in the place of the stacked LSTM: trained over whole sequences, served token by token.

The recurrence keeps an LSTM's forget and output gate and drops its recurrent weights, so that a sequence is one scan
instead of a chain of matrix products.  The matrix products themselves are torch's.

`python -m persistent_lstm_hip_amd.gated_demo` trains one on synthetic series, then serves it step by step.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Union

import torch
import torch.nn as nn

from .ops import dropout_add, gated_scan, gated_scan_step, layer_norm


def _draw(device: torch.device) -> Union[int, torch.Tensor]:
    """62 bits of torch's host generator, which activation checkpointing restores for its recomputation.  While a graph is
    captured, which would keep them for all its replays, of the device's, in a tensor that every replay draws again."""
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        return torch.randint(1 << 62, (1,), device=device)
    return int(torch.randint(1 << 62, (), device="cpu"))


class GatedScanBlock(nn.Module):
    """One residual block of width dim.  Its state is the scan's, [batch, dim] float32."""

    def __init__(self, dim: int, dropout: float = 0.0):
        super().__init__()
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.norm_bias = nn.Parameter(torch.zeros(dim))
        self.gates = nn.Linear(dim, 3 * dim)
        self.out = nn.Linear(dim, dim)
        self.dropout = dropout
        with torch.no_grad():  # memories from two steps to some hundred, channel by channel
            self.gates.bias[:dim] = torch.linspace(0.5, 6.0, dim)

    def forward(self, x: torch.Tensor, c0: Optional[torch.Tensor] = None, *, lengths=None, seed: int = 0,
                offset: Union[int, torch.Tensor, None] = None):
        """x [batch, time, dim] -> (y, c_n).  (seed, offset) pick the dropout mask in training mode, as in dropout_add.
        Without an offset one is drawn from torch's generator, so that every call (and every replay of a captured
        one) has a mask of its own."""
        gates = self.gates(layer_norm(x, self.norm_weight, self.norm_bias))
        h, c_n = gated_scan(gates, c0, lengths=lengths)
        p = self.dropout if self.training else 0.0
        if offset is None:
            offset = _draw(x.device) if p > 0.0 else 0
        # (under autocast a product is of the lower type; the residual stream keeps its own)
        return dropout_add(self.out(h).to(x.dtype), x, p=p, seed=seed, offset=offset), c_n

    def step(self, x: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
        """One token x [batch, dim] -> y; c is updated in place.  For inference."""
        gates = self.gates(layer_norm(x, self.norm_weight, self.norm_bias))
        h, _ = gated_scan_step(gates, c, inplace=True)
        return x + self.out(h)


class GatedScanRegressor(nn.Module):
    """x [batch, time, input_dim] -> [batch, output_dim], read off at every row's last step.

    In training mode every layer of every pass draws a dropout mask of its own under `seed` (torch.initial_seed() unless
    set).  The passes are counted from the model's construction on and are not in its state_dict: a resumed run, a
    second model of a process, or the ranks of a data-parallel job that share a manual seed set other seeds.  A pass
    that finds torch's host generator where an earlier one found it is that pass once more, with its masks: activation
    checkpointing, which restores the generator, recomputes what it computed.  forward's `offset` gives the pass its
    number in the place of the count: an int, or a one-element int64 tensor on the device, which a captured graph may
    advance.  A captured pass without one draws its number on the device in every replay."""

    _REMEMBERED = 4096  # passes that a recomputation may go back

    def __init__(self, input_dim: int, hidden_dim: int, output_dim: int, n_layers: int, dropout: float = 0.2):
        super().__init__()
        self.stem = nn.Linear(input_dim, hidden_dim)
        self.blocks = nn.ModuleList(GatedScanBlock(hidden_dim, dropout) for _ in range(n_layers))
        self.norm_weight = nn.Parameter(torch.ones(hidden_dim))
        self.norm_bias = nn.Parameter(torch.zeros(hidden_dim))
        self.linear = nn.Linear(hidden_dim, output_dim)
        self.seed = int(torch.initial_seed())
        self._passes = 0  # training passes so far: every layer of every pass has a mask of its own
        self._numbers = {}  # of the last passes, by what they drew from torch's generator

    def _pass_number(self, device: torch.device) -> Union[int, torch.Tensor]:
        drawn = _draw(device)
        if isinstance(drawn, torch.Tensor):
            return drawn
        if drawn not in self._numbers:
            if len(self._numbers) == self._REMEMBERED:
                del self._numbers[next(iter(self._numbers))]  # (the oldest)
            self._numbers[drawn] = self._passes
            self._passes += 1
        return self._numbers[drawn]

    def _head(self, x: torch.Tensor) -> torch.Tensor:
        return self.linear(layer_norm(x, self.norm_weight, self.norm_bias))

    def _offsets(self, offset, device) -> Sequence[Union[int, torch.Tensor]]:
        """The layers' offsets in dropout_add of pass number `offset`."""
        n = len(self.blocks)
        if not isinstance(offset, torch.Tensor):
            return range(offset * n, (offset + 1) * n)
        if offset.numel() != 1 or offset.dtype != torch.int64 or offset.device != device:
            raise ValueError(f"a tensor offset must be one int64 on {device}")
        return (offset.reshape(1, 1) * n + torch.arange(n, device=device).unsqueeze(1)).unbind()

    def forward(self, x: torch.Tensor, lengths=None, offset: Union[int, torch.Tensor, None] = None) -> torch.Tensor:
        if x.dim() != 3 or x.size(1) == 0:
            raise ValueError("x must be a [batch, seq_len, input_size] tensor of at least one step")
        if lengths is not None:
            lengths = torch.as_tensor(lengths)
        drops = self.training and any(block.dropout > 0.0 for block in self.blocks)
        if not drops:
            offset = 0
        elif offset is None:
            offset = self._pass_number(x.device)
        y = self.stem(x)
        for block, mask in zip(self.blocks, self._offsets(offset, x.device)):
            y, _ = block(y, lengths=lengths, seed=self.seed, offset=mask)
        if lengths is None:
            return self._head(y[:, -1])
        last = (lengths.to(y.device, torch.int64) - 1).clamp(0, y.size(1) - 1)  # (an empty row: its first step)
        return self._head(y[torch.arange(y.size(0), device=y.device), last])

    def initial_state(self, batch: int) -> List[torch.Tensor]:
        w = self.norm_weight
        return [torch.zeros(batch, w.numel(), dtype=torch.float32, device=w.device) for _ in self.blocks]

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: List[torch.Tensor]) -> torch.Tensor:
        """One token x [batch, input_dim] -> the forecast after it; state (initial_state) is updated in place."""
        y = self.stem(x)
        for block, c in zip(self.blocks, state):
            y = block.step(y, c)
        return self._head(y)
