"""Operators of a residual block around a recurrence that is parallel over time, for training and serving:

    y = x + dropout(W_o scan(W_g layer_norm(x)))

* gated_scan       -- gated linear recurrence over a whole sequence (an LSTM's gates without its recurrent weights).
* gated_scan_step  -- one token of it, from and to a state.
* layer_norm       -- over the last dimension.
* dropout_add      -- dropout from a counter-based generator, with the residual added in the same pass.

All take float16, bfloat16 and float32 tensors on a HIP device, keep sums, statistics and states in float32, run on
the device's current stream and are differentiable once, in reverse mode: a second derivative raises RuntimeError, a
tensor with a forward-mode tangent ValueError.  As for the LSTM there is no CPU path: a missing library
raises RuntimeError, an argument that the operators do not take, such as a tensor that is not on a HIP device,
ValueError.  The arguments are checked, the outputs allocated and the kernels called in csrc/plh_torch.cpp.  The
reference has no counterpart.
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence, Tuple, Union

import torch

from .extension import require_torch_ops

_U64 = (1 << 64) - 1


def _tensor(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")


def _u64(v, name: str) -> int:
    """An integer of any type modulo 2^64 (numpy's do not take the mask as one of theirs)."""
    try:
        return operator.index(v) & _U64
    except TypeError:
        raise ValueError(f"{name} must be an integer, not {type(v).__name__}") from None


def gated_scan(gates: torch.Tensor, c0: Optional[torch.Tensor] = None, *,
               lengths: Union[torch.Tensor, Sequence[int], None] = None,
               output_gate: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated linear recurrence over gates [batch, time, 3 * hidden] (f, g, o):

        c_t = sigmoid(f_t) c_{t-1} + (1 - sigmoid(f_t)) g_t        out_t = sigmoid(o_t) c_t

    or, with output_gate=False, over [batch, time, 2 * hidden] (f, g) with out_t = c_t.  Returns (out [batch, time,
    hidden] of gates' type, c_n [batch, hidden] float32).  c0: the state before the first step, [batch, hidden]
    (default: zeros).  lengths: row b runs lengths[b] steps, as in a packed sequence: its c_n is the state after them,
    its outputs are zero from there on and what gates holds there, NaN included, changes nothing.  A list or a host
    tensor is checked; a tensor on the device is not (it would synchronise) but taken as clamped to [0, time].  While a
    graph is captured lengths must be on the device.

    gates may have any batch and time strides, so a time-major projection's transpose runs without a copy.
    Differentiable in gates and c0.
    """
    _tensor(gates, "gates")
    if c0 is not None:
        _tensor(c0, "c0")
    if lengths is not None and not isinstance(lengths, torch.Tensor):
        lengths = torch.as_tensor(lengths)
    return require_torch_ops().gated_scan(gates, c0, lengths, output_gate)


def gated_scan_step(gates: torch.Tensor, c: torch.Tensor, *, output_gate: bool = True,
                    inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of gated_scan for serving: gates [batch, 3 * hidden] (or 2 *), c [batch, hidden] float32.  Returns
    (out [batch, hidden], the new c); with inplace=True c itself is overwritten and returned.  Not differentiable."""
    _tensor(gates, "gates")
    _tensor(c, "c")
    return require_torch_ops().gated_scan_step(gates, c, output_gate, inplace)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over x's last dimension, as torch.nn.functional.layer_norm.
    weight and bias [cols], either may be missing, have x's type or float32 (both the same).  Rows may be strided;
    leading dimensions that do not merge into one row stride are copied.  Differentiable in x, weight and bias."""
    _tensor(x, "x")
    if weight is not None:
        _tensor(weight, "weight")
    if bias is not None:
        _tensor(bias, "bias")
    return require_torch_ops().layer_norm(x, weight, bias, eps)


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, *, p: float, seed: int,
                offset: Union[int, torch.Tensor] = 0) -> torch.Tensor:
    """residual + dropout(x): elements of x are zero with probability p and scaled by 1 / (1 - p) otherwise.

    The mask is a function of (seed, offset, position in the contiguous tensor) alone, by Philox4x32-10; nothing is
    stored for the gradient, which computes it again.  Take another offset for every call under one seed (both are
    taken modulo 2^64).  offset may be a one-element int64 tensor on the device, so that a captured graph draws other
    masks at every replay.  p is rounded to a multiple of 2^-16, and the scale is that of the rounded value.  A dropped
    element does not count, infinity and NaN included.  residual: as x (no broadcasting).  Differentiable in both.
    """
    _tensor(x, "x")
    if residual is not None:
        _tensor(residual, "residual")
    if isinstance(offset, torch.Tensor):
        return require_torch_ops().dropout_add(x, residual, p, _u64(seed, "seed"), 0, offset)
    return require_torch_ops().dropout_add(x, residual, p, _u64(seed, "seed"), _u64(offset, "offset"), None)
