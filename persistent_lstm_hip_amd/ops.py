"""Operators of a residual block around a recurrence that is parallel over time, for training and serving:

    y = x + dropout(W_o scan(W_g layer_norm(x)))

* gated_scan       -- gated linear recurrence over a whole sequence (an LSTM's gates without its recurrent weights).
* gated_scan_step  -- one token of it, from and to a state.
* layer_norm       -- over the last dimension.
* dropout_add      -- dropout from a counter-based generator, with the residual added in the same pass.

All take float16, bfloat16 and float32 tensors on a HIP device, keep sums, statistics and states in float32, run on
the device's current stream and are differentiable once.  As for the LSTM there is no CPU path: a missing library
raises RuntimeError, a tensor that is not on a HIP device ValueError.  The reference has no counterpart.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from .extension import NativeLibrary, _launch, _ptr, require_extension

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # PLH_F16, PLH_BF16, PLH_F32


def _check_tensor(t, name: str, dims: Optional[int] = None) -> int:
    """The library's code of t's type, after the checks that every operand shares."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a HIP device: this library has no CPU path")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float16, bfloat16 or float32, not {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, not {t.dim()}")
    return code


def _check_like(t, name: str, shape, device, dtype=None) -> None:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be a tensor of shape {list(shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")


def _tracks(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- gated linear recurrence --------------------------------------------------------------------


def _scan_shape(gates, output_gate: bool) -> int:
    parts = 3 if output_gate else 2
    if gates.size(-1) == 0 or gates.size(-1) % parts:
        raise ValueError(f"gates needs {parts} * hidden columns (f, g{', o' if output_gate else ''}), "
                         f"not {gates.size(-1)}")
    return gates.size(-1) // parts


def _rows(gates: torch.Tensor) -> torch.Tensor:
    """gates itself where its last dimension is dense (any batch and time strides), else a copy."""
    return gates if gates.stride(-1) == 1 or gates.size(-1) == 1 else gates.contiguous()


def _lengths(lengths, batch: int, seq_len: int, device: torch.device) -> Optional[torch.Tensor]:
    """int32 on the device.  Host lengths are checked; lengths on the device are not (that would synchronise the
    stream): the kernels take them as if clamped to [0, seq_len]."""
    if lengths is None:
        return None
    n = torch.as_tensor(lengths)
    if n.numel() == 0:  # (an empty list has no integer type)
        n = n.to(torch.int32)
    if n.dim() != 1 or n.numel() != batch or n.is_floating_point() or n.is_complex() or n.dtype is torch.bool:
        raise ValueError("lengths must be a 1-D integer tensor with one entry per batch row")
    if n.device.type == "cpu":
        if batch and (int(n.min()) < 0 or int(n.max()) > seq_len):
            raise ValueError(f"lengths must lie in [0, {seq_len}]")
        return n.to(torch.int32).contiguous().pin_memory().to(device, non_blocking=True)
    if n.device != device:
        raise ValueError(f"lengths must be on the host or on {device}")
    return n.clamp(0, seq_len).to(torch.int32) if n.dtype is torch.int64 else n.to(torch.int32).contiguous()


def _scan_workspace(ext: NativeLibrary, B: int, T: int, H: int, device) -> Optional[torch.Tensor]:
    n = ext.lib.plh_gated_scan_workspace_bytes(B, T, H)
    return torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None


def _scan_forward(gates, c0, lengths, output_gate: bool, keep: bool):
    ext = require_extension()
    code, device = _DTYPES[gates.dtype], gates.device
    B, T = gates.size(0), gates.size(1)
    H = gates.size(2) // (3 if output_gate else 2)
    out = torch.empty((B, T, H), dtype=gates.dtype, device=device)
    c_n = torch.empty((B, H), dtype=torch.float32, device=device)
    states = None
    if keep:
        states = torch.empty((ext.lib.plh_gated_scan_states(T), B, H), dtype=torch.float32, device=device)
    ws = _scan_workspace(ext, B, T, H, device)
    rc = _launch(device, ext.lib.plh_gated_scan_forward, code, int(output_gate), gates.data_ptr(), gates.stride(0),
                 gates.stride(1), B, T, H, _ptr(lengths), _ptr(c0), out.data_ptr(), c_n.data_ptr(), _ptr(states),
                 _ptr(ws), 0 if ws is None else ws.numel())
    if rc:
        ext._check(rc, "gated_scan")
    return out, c_n, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, c0, lengths, output_gate):
        out, c_n, states = _scan_forward(gates, c0, lengths, output_gate, True)
        ctx.save_for_backward(gates, lengths, states)
        ctx.output_gate, ctx.has_c0 = output_gate, c0 is not None
        ctx.set_materialize_grads(False)
        return out, c_n

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_cn):
        gates, lengths, states = ctx.saved_tensors
        ext = require_extension()
        B, T = gates.size(0), gates.size(1)
        H = states.size(2)
        device = gates.device
        if d_out is None:
            d_out = torch.zeros((B, T, H), dtype=gates.dtype, device=device)
        d_out = d_out.contiguous()
        if d_cn is not None:
            d_cn = d_cn.contiguous()
        d_gates = torch.empty(gates.shape, dtype=gates.dtype, device=device)
        d_c0 = torch.empty((B, H), dtype=torch.float32, device=device) if ctx.needs_input_grad[1] else None
        ws = _scan_workspace(ext, B, T, H, device)
        rc = _launch(device, ext.lib.plh_gated_scan_backward, _DTYPES[gates.dtype], int(ctx.output_gate),
                     gates.data_ptr(), gates.stride(0), gates.stride(1), B, T, H, _ptr(lengths), states.data_ptr(),
                     d_out.data_ptr(), _ptr(d_cn), d_gates.data_ptr(), _ptr(d_c0), _ptr(ws),
                     0 if ws is None else ws.numel())
        if rc:
            ext._check(rc, "gated_scan backward")
        return d_gates, d_c0, None, None


def gated_scan(gates: torch.Tensor, c0: Optional[torch.Tensor] = None, *,
               lengths: Union[torch.Tensor, Sequence[int], None] = None,
               output_gate: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated linear recurrence over gates [batch, time, 3 * hidden] (f, g, o):

        c_t = sigmoid(f_t) c_{t-1} + (1 - sigmoid(f_t)) g_t        out_t = sigmoid(o_t) c_t

    or, with output_gate=False, over [batch, time, 2 * hidden] (f, g) with out_t = c_t.  Returns (out [batch, time,
    hidden] of gates' type, c_n [batch, hidden] float32).  c0: the state before the first step, [batch, hidden]
    (default: zeros).  lengths: row b runs lengths[b] steps, as in a packed sequence: its c_n is the state after them,
    its outputs are zero from there on and what gates holds there, NaN included, changes nothing.  A list or a host
    tensor is checked; a tensor on the device is not (it would synchronise) but taken as clamped to [0, time].

    gates may have any batch and time strides, so a time-major projection's transpose runs without a copy.
    Differentiable in gates and c0.
    """
    _check_tensor(gates, "gates", 3)
    H = _scan_shape(gates, output_gate)
    device = gates.device
    if c0 is not None:
        _check_tensor(c0, "c0")
        _check_like(c0, "c0", (gates.size(0), H), device)
        c0 = c0.float().contiguous()
    n = _lengths(lengths, gates.size(0), gates.size(1), device)
    gates = _rows(gates)
    if _tracks(gates, c0):
        return _GatedScan.apply(gates, c0, n, bool(output_gate))
    return _scan_forward(gates, c0, n, output_gate, False)[:2]


def gated_scan_step(gates: torch.Tensor, c: torch.Tensor, *, output_gate: bool = True,
                    inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of gated_scan for serving: gates [batch, 3 * hidden] (or 2 *), c [batch, hidden] float32.  Returns
    (out [batch, hidden], the new c); with inplace=True c itself is overwritten and returned.  Not differentiable."""
    code = _check_tensor(gates, "gates", 2)
    H = _scan_shape(gates, output_gate)
    B, device = gates.size(0), gates.device
    _check_like(c, "c", (B, H), device, torch.float32)
    if not c.is_contiguous():
        if inplace:
            raise ValueError("c must be contiguous to be updated in place")
        c = c.contiguous()
    if _tracks(gates, c):
        raise ValueError("gated_scan_step is not differentiable: call it under torch.no_grad(), or gated_scan")
    ext = require_extension()
    gates = _rows(gates)
    out = torch.empty((B, H), dtype=gates.dtype, device=device)
    c_n = c if inplace else torch.empty_like(c)
    rc = _launch(device, ext.lib.plh_gated_scan_forward, code, int(output_gate), gates.data_ptr(), gates.stride(0), 0,
                 B, 1, H, None, c.data_ptr(), out.data_ptr(), c_n.data_ptr(), None, None, 0)
    if rc:
        ext._check(rc, "gated_scan_step")
    return out, c_n


# ---- layer norm ---------------------------------------------------------------------------------


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, cols] with dense rows: a view where one row stride serves, else a copy."""
    cols = x.size(-1)
    if x.dim() == 2 and (x.stride(1) == 1 or cols == 1):
        return x
    rows = x.numel() // cols
    try:
        m = x.view(rows, cols)
    except RuntimeError:  # leading dimensions that do not merge
        m = x.reshape(rows, cols)
    return m if m.stride(1) == 1 or cols == 1 else m.contiguous()


def _norm_forward(x2, weight, bias, eps: float, keep: bool):
    ext = require_extension()
    rows, cols = x2.shape
    y = torch.empty((rows, cols), dtype=x2.dtype, device=x2.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x2.device) if keep else None
    mean = rstd = None
    if keep:
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    w = weight if weight is not None else bias
    code = _DTYPES[x2.dtype]
    rc = _launch(x2.device, ext.lib.plh_layer_norm_forward, code, code if w is None else _DTYPES[w.dtype],
                 x2.data_ptr(), x2.stride(0), rows, cols, _ptr(weight), _ptr(bias), eps, y.data_ptr(), mean, rstd)
    if rc:
        ext._check(rc, "layer_norm")
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _matrix(x)
        y, stats = _norm_forward(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, stats)
        ctx.shape, ctx.wdtype = x.shape, (weight if weight is not None else bias)
        ctx.wdtype = None if ctx.wdtype is None else ctx.wdtype.dtype
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        x2, weight, stats = ctx.saved_tensors
        ext = require_extension()
        rows, cols = x2.shape
        device = x2.device
        d_y = d_y.contiguous()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        d_x = torch.empty((rows, cols), dtype=x2.dtype, device=device) if need_x else None
        d_w = torch.empty(cols, dtype=ctx.wdtype, device=device) if need_w else None
        d_b = torch.empty(cols, dtype=ctx.wdtype, device=device) if need_b else None
        ws, nws = None, 0
        if need_w or need_b:
            nws = ext.lib.plh_layer_norm_workspace_bytes(rows, cols)
            ws = torch.empty(nws, dtype=torch.uint8, device=device)
        code = _DTYPES[x2.dtype]
        rc = _launch(device, ext.lib.plh_layer_norm_backward, code, code if ctx.wdtype is None else _DTYPES[ctx.wdtype],
                     x2.data_ptr(), x2.stride(0), rows, cols, _ptr(weight), stats.data_ptr(),
                     stats.data_ptr() + 4 * rows, d_y.data_ptr(), _ptr(d_x), _ptr(d_w), _ptr(d_b), _ptr(ws), nws)
        if rc:
            ext._check(rc, "layer_norm backward")
        return (None if d_x is None else d_x.view(ctx.shape)), d_w, d_b, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over x's last dimension, as torch.nn.functional.layer_norm.
    weight and bias [cols], either may be missing, have x's type or float32 (both the same).  Rows may be strided;
    leading dimensions that do not merge into one row stride are copied.  Differentiable in x, weight and bias."""
    _check_tensor(x, "x")
    if x.dim() < 1 or x.size(-1) == 0:
        raise ValueError("x needs a last dimension of at least one element")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check_like(t, name, (x.size(-1),), x.device)
            if t.dtype is not x.dtype and t.dtype is not torch.float32:
                raise ValueError(f"{name} must be {x.dtype} or float32, not {t.dtype}")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise ValueError("weight and bias must have the same type")
    if not eps >= 0.0:
        raise ValueError("eps must be non-negative")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _tracks(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_forward(_matrix(x), weight, bias, eps, False)[0].view(x.shape)


# ---- dropout ------------------------------------------------------------------------------------


def _dropout(x, residual, threshold: int, seed: int, offset: int, offset_dev) -> torch.Tensor:
    ext = require_extension()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rc = _launch(x.device, ext.lib.plh_dropout_add, _DTYPES[x.dtype], x.data_ptr(), _ptr(residual), out.data_ptr(),
                 x.numel(), threshold, seed, offset, _ptr(offset_dev))
    if rc:
        ext._check(rc, "dropout_add")
    return out


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, offset, offset_dev):
        if offset_dev is not None:  # the mask is that of the offset as it is now
            offset_dev = offset_dev.clone()
        ctx.mask = (threshold, seed, offset)
        ctx.save_for_backward(offset_dev)
        return _dropout(x, residual, threshold, seed, offset, offset_dev)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        need_x, need_r = ctx.needs_input_grad[:2]
        offset_dev, = ctx.saved_tensors
        d_x = _dropout(d_out.contiguous(), None, *ctx.mask, offset_dev) if need_x else None
        return d_x, (d_out if need_r else None), None, None, None, None


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, *, p: float, seed: int,
                offset: Union[int, torch.Tensor] = 0) -> torch.Tensor:
    """residual + dropout(x): elements of x are zero with probability p and scaled by 1 / (1 - p) otherwise.

    The mask is a function of (seed, offset, position in the contiguous tensor) alone, by Philox4x32-10; nothing is
    stored for the gradient, which computes it again.  Take another offset for every call under one seed (both are
    taken modulo 2^64).  offset may be a one-element int64 tensor on the device, so that a captured graph draws other
    masks at every replay.  p is rounded to a multiple of 2^-16, and the scale is that of the rounded value.  A dropped
    element does not count, infinity and NaN included.  residual: as x (no broadcasting).  Differentiable in both.
    """
    _check_tensor(x, "x")
    if residual is not None:
        _check_like(residual, "residual", x.shape, x.device, x.dtype)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must lie in [0, 1]")
    offset_dev = None
    if isinstance(offset, torch.Tensor):
        if offset.numel() != 1 or offset.dtype is not torch.int64 or offset.device != x.device:
            raise ValueError(f"a tensor offset must be one int64 on {x.device}")
        offset, offset_dev = 0, offset.detach()
    threshold = int(math.floor(p * 65536.0 + 0.5))
    seed, offset = int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFFFFFFFFFF
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    if _tracks(x, residual):
        return _DropoutAdd.apply(x, residual, threshold, seed, offset, offset_dev)
    return _dropout(x, residual, threshold, seed, offset, offset_dev)
