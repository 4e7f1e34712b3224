"""Operators of residual blocks around a recurrence that is parallel over time, for training and serving:

    y = x + dropout(W_o scan(W_g layer_norm(x)))

* gated_scan       -- gated linear recurrence over a whole sequence (an LSTM's gates without its recurrent weights).
* gated_scan_step  -- one token of it, from and to a state.
* layer_norm       -- over the last dimension.
* dropout_add      -- dropout from a counter-based generator, with the residual added in the same pass.

or, with a state wider than its channel and decays that depend on the input,

    u, z = W_in layer_norm(x)    u = causal_conv(u)    dt, B, C = W_x u    y = x + W_out selective_scan(u, dt, A, B, C, D, z)

* causal_conv          -- short causal convolution along time with its activation.
* causal_conv_step     -- one token of it, from and to a state.
* selective_scan       -- selective state space scan over a whole sequence, with its skip and gate.
* selective_scan_step  -- one token of it, from and to a state.

and, between a backward pass and an optimizer's step,

* clip_grad_norm   -- many tensors scaled to a global norm.

All take float16, bfloat16 and float32 tensors on a HIP device, keep sums, statistics and states in float32, run on
the device's current stream and are differentiable once, in reverse mode: a second derivative raises RuntimeError, a
tensor with a forward-mode tangent ValueError.  As for the LSTM there is no CPU path: a missing library
raises RuntimeError, an argument that the operators do not take, such as a tensor that is not on a HIP device,
ValueError.  The arguments are checked, the outputs allocated and the kernels called in csrc/plh_torch.cpp.  The
reference has no counterpart.
"""
from __future__ import annotations

import operator
from typing import Iterable, List, Optional, Sequence, Tuple, Union

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


def _lengths(lengths):
    return lengths if lengths is None or isinstance(lengths, torch.Tensor) else torch.as_tensor(lengths)


def _optional(t, name: str) -> None:
    if t is not None:
        _tensor(t, name)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                state: Optional[torch.Tensor] = None, *,
                lengths: Union[torch.Tensor, Sequence[int], None] = None,
                silu: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """A causal convolution along time with a filter of its own for every channel, over x [batch, time, channels]:

        acc_t = bias + sum_k weight[:, k] x_{t - width + 1 + k}        y_t = silu(acc_t), or acc_t with silu=False

    weight [channels, width] with a width of 1 to 8, bias [channels], of x's type or float32 (both the same).  state: the
    width - 1 inputs before the first step, the oldest first, [batch, width - 1, channels] of x's type (default: zeros).
    Returns (y of x's shape, the state after the last step).  lengths: as for gated_scan; a row's state is that after
    its last step, its outputs are zero from there on.

    x may have any batch and time strides (half of a projection's output, say).  Differentiable in x, weight, bias and
    state, from both results.
    """
    _tensor(x, "x")
    _tensor(weight, "weight")
    _optional(bias, "bias")
    _optional(state, "state")
    return require_torch_ops().causal_conv(x, weight, bias, state, _lengths(lengths), silu)


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     silu: bool = True, inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of causal_conv for serving: x [batch, channels], state [batch, width - 1, channels].  Returns (y, the new
    state); with inplace=True state itself is overwritten and returned.  Not differentiable."""
    _tensor(x, "x")
    _tensor(state, "state")
    _tensor(weight, "weight")
    _optional(bias, "bias")
    return require_torch_ops().causal_conv_step(x, state, weight, bias, silu, inplace)


def selective_scan(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   h0: Optional[torch.Tensor] = None, *, dt_bias: Optional[torch.Tensor] = None, softplus: bool = True,
                   lengths: Union[torch.Tensor, Sequence[int], None] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The selective state space scan over u and dt [batch, time, channels], B and C [batch, time, states] (shared by all
    channels); for every channel d and state n

        s_t = softplus(dt_t + dt_bias), or dt_t + dt_bias with softplus=False
        h_t = exp(s_t A[d, n]) h_{t-1} + s_t u_t B_t[n]        y_t = sum_n C_t[n] h_t + D[d] u_t

    and out_t = y_t silu(z_t), or y_t without z [batch, time, channels].  A [channels, states] with 1 to 64 states, not
    positive: it is a decay (with softplus=False a step size may lie below zero, and the state grows).  D and dt_bias
    [channels], either may be missing; these three have u's type or float32 (all the same), the others u's type.  Returns
    (out of u's shape and type, h_n [batch, channels, states] float32).  h0: the state before the first step (default:
    zeros).  lengths: as for gated_scan; a row's h_n is the state after its last step, its outputs are zero from there on.

    u, dt, z, B and C may have any batch and time strides (parts of projections' outputs).  Differentiable in all of
    them, A, D, dt_bias and h0, from both results.
    """
    for t, name in ((u, "u"), (dt, "dt"), (A, "A"), (B, "B"), (C, "C")):
        _tensor(t, name)
    for t, name in ((D, "D"), (z, "z"), (h0, "h0"), (dt_bias, "dt_bias")):
        _optional(t, name)
    return require_torch_ops().selective_scan(u, dt, A, B, C, D, z, h0, dt_bias, softplus, _lengths(lengths))


def selective_scan_step(u: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        h: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, *,
                        dt_bias: Optional[torch.Tensor] = None, softplus: bool = True,
                        inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of selective_scan for serving: u, dt and z [batch, channels], B and C [batch, states], h [batch, channels,
    states] float32.  Returns (out, the new h); with inplace=True h itself is overwritten and returned.  Not
    differentiable."""
    for t, name in ((u, "u"), (dt, "dt"), (A, "A"), (B, "B"), (C, "C"), (h, "h")):
        _tensor(t, name)
    for t, name in ((D, "D"), (z, "z"), (dt_bias, "dt_bias")):
        _optional(t, name)
    return require_torch_ops().selective_scan_step(u, dt, A, B, C, h, D, z, dt_bias, softplus, inplace)


def clip_grad_norm(grads: Iterable[Optional[torch.Tensor]], max_norm: float, *,
                   inplace: bool = False) -> Tuple[List[Optional[torch.Tensor]], torch.Tensor]:
    """The tensors scaled by min(1, max_norm / (norm + 1e-6)), where norm is the Euclidean norm of all their elements
    together.  Returns (the scaled tensors, norm): new tensors, or with inplace=True `grads` themselves, overwritten; norm is
    a float32 scalar on the device (nothing waits for it).  Entries that are None stay None, so that

        clip_grad_norm([p.grad for p in model.parameters()], 1.0, inplace=True)

    serves a training step.  The tensors are on one device, of any shapes, strides and mixed types; those that are
    overwritten must lie in ranges of memory that do not overlap.  Squares are summed in 64 bits.  max_norm may be infinite:
    nothing is scaled.  A norm of infinity scales by zero and one of NaN by NaN, as
    torch.nn.utils.clip_grad_norm_ does.  Not differentiable.
    """
    if isinstance(grads, torch.Tensor):
        raise ValueError("grads must be a sequence of tensors, not a tensor")
    grads = list(grads)
    for g in grads:
        _optional(g, "a gradient")
    out, norm = require_torch_ops().clip_grad_norm([g for g in grads if g is not None], float(max_norm), inplace)
    left = iter(out)
    return [None if g is None else next(left) for g in grads], norm
