"""Loader of the native library and its torch-facing front end.

The native boundary is the C ABI in include/persistent_lstm_hip.h (library
persistent_lstm_hip_amd/lib/libpersistent_lstm_hip.so), bound here with ctypes.  torch only supplies
device memory and the current HIP stream.  `load_extension()` keeps the contract of the reference's
loader (persistent_lstm_hip/extension.py:7-12): it returns the extension object, or None when the
library cannot be loaded (the reason is kept in `load_error()`).  The model classes turn None into a
loud RuntimeError; nothing falls back to a CPU path.

The extension object also exposes the reference extension's function names
(persistent_lstm_hip/csrc/bindings.cpp:154-165) with their tensor signatures, so code written
against `persistent_lstm_hip_ext` keeps working.
"""
from __future__ import annotations

import contextlib
import ctypes
import importlib.util
import os
from functools import lru_cache
from typing import Dict, List, Optional, Sequence

import torch

# Built by persistent_lstm_hip_amd/build.py.
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libpersistent_lstm_hip.so")
TORCH_PATH = os.path.join(os.path.dirname(LIB_PATH), "plh_torch.so")  # the block operators' torch front end

PLH_OK = 0
PLH_ERR_INVALID = 1
PLH_ERR_UNSUPPORTED = 2
PLH_ERR_HIP = 3
PLH_ERR_DEVICE = 4
PLH_STATUS_TIMEOUT = 1

_load_error: Optional[str] = None

_vp = ctypes.c_void_p
_i32 = ctypes.c_int
_i64 = ctypes.c_int64


def _declare(lib: ctypes.CDLL) -> None:
    lib.plh_abi_version.restype = _i32
    lib.plh_abi_version.argtypes = []
    lib.plh_last_error.restype = ctypes.c_char_p
    lib.plh_last_error.argtypes = []
    lib.plh_supports.restype = _i32
    lib.plh_supports.argtypes = [_i32] * 4
    lib.plh_packed_bytes.restype = _i64
    lib.plh_packed_bytes.argtypes = [_i32] * 4
    lib.plh_pack_regressor.restype = _i32
    lib.plh_pack_regressor.argtypes = [_i32] * 4 + [ctypes.POINTER(_vp)] * 4 + [_vp, _vp, _vp, _i64, _vp]
    lib.plh_workspace_bytes.restype = _i64
    lib.plh_workspace_bytes.argtypes = [_i32] * 6
    lib.plh_forward.restype = _i32
    lib.plh_forward.argtypes = (
        [_vp] + [_i32] * 4 + [_vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _vp, _vp, _vp, _i64, _vp]
    )
    lib.plh_detects_uniform.restype = _i32
    lib.plh_detects_uniform.argtypes = [_i32] * 6
    lib.plh_forward_detect.restype = _i32
    lib.plh_forward_detect.argtypes = [_vp] + [_i32] * 4 + [_vp, _i32, _i32, _vp, _vp, _i64, _vp]
    lib.plh_status.restype = _i32
    lib.plh_status.argtypes = [_vp, ctypes.POINTER(ctypes.c_uint32), _vp]
    lib.plh_kernel_timing.restype = _i32
    lib.plh_kernel_timing.argtypes = [_i32]
    lib.plh_kernel_timing_read.restype = _i32
    lib.plh_kernel_timing_read.argtypes = [ctypes.POINTER(ctypes.c_double), ctypes.POINTER(_i32)]
    lib.plh_repeat_first_row.restype = _i32
    lib.plh_repeat_first_row.argtypes = [_vp, _vp, _i32, _i32, _vp]
    lib.plh_set_wait_limit_us.restype = _i32
    lib.plh_set_wait_limit_us.argtypes = [_i64]
    lib.plh_inject_wait_failure.restype = _i32
    lib.plh_inject_wait_failure.argtypes = [_i32]
    lib.plh_forward_noalloc.restype = _i32
    lib.plh_forward_noalloc.argtypes = (
        [_vp] + [_i32] * 4 + [_vp, _i32, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _vp, _vp, _vp]
    )
    lib.plh_noalloc_scratch_bytes.restype = _i64
    lib.plh_noalloc_scratch_bytes.argtypes = []
    lib.plh_noalloc_status.restype = _i32
    lib.plh_noalloc_status.argtypes = [ctypes.POINTER(ctypes.c_uint32), _vp]
    lib.plh_probe_mfma_f16.restype = _i32
    lib.plh_probe_mfma_f16.argtypes = [ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
    lib.plh_input_projection.restype = _i32
    lib.plh_input_projection.argtypes = [_vp, _i64, _vp, _i32, _vp, _i64, _i64, _i32, _i32, _vp]
    lib.plh_gated_scan_states.restype = _i64
    lib.plh_gated_scan_states.argtypes = [_i64]
    lib.plh_gated_scan_workspace_bytes.restype = _i64
    lib.plh_gated_scan_workspace_bytes.argtypes = [_i64, _i64, _i32]
    scan = [_i32, _i32, _vp, _i64, _i64, _i64, _i64, _i32, _vp]
    lib.plh_gated_scan_forward.restype = _i32
    lib.plh_gated_scan_forward.argtypes = scan + [_vp, _vp, _vp, _vp, _vp, _i64, _vp]
    lib.plh_gated_scan_backward.restype = _i32
    lib.plh_gated_scan_backward.argtypes = scan + [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp]
    norm = [_i32, _i32, _vp, _i64, _i64, _i64, _vp]
    lib.plh_layer_norm_forward.restype = _i32
    lib.plh_layer_norm_forward.argtypes = norm + [_vp, ctypes.c_float, _vp, _vp, _vp, _vp]
    lib.plh_layer_norm_workspace_bytes.restype = _i64
    lib.plh_layer_norm_workspace_bytes.argtypes = [_i64, _i64]
    lib.plh_layer_norm_backward.restype = _i32
    lib.plh_layer_norm_backward.argtypes = norm + [_vp] * 7 + [_i64, _vp]
    lib.plh_dropout_add.restype = _i32
    lib.plh_dropout_add.argtypes = [_i32, _vp, _vp, _vp, _i64, _i32, ctypes.c_uint64, ctypes.c_uint64, _vp, _vp]


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def _stream(device: torch.device) -> int:
    """The handle of the device's current stream (without the Stream object around it)."""
    return torch._C._cuda_getCurrentRawStream(_index(device))


def _device_key(device: torch.device) -> tuple:
    """(type, index, current stream) with the index resolved, so "cuda" and "cuda:0" name one device."""
    device = torch.device(device)
    index = _index(device)
    return (device.type, index, torch._C._cuda_getCurrentRawStream(index))


_CURRENT = contextlib.nullcontext()


def _on_device(device: torch.device):
    """torch.cuda.device(device), or nothing when it is already the current device."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _CURRENT
    return torch.cuda.device(device.index)


def _launch(device: torch.device, fn, *args) -> int:
    """fn(*args, the device's current stream) with the device current."""
    current = torch.cuda.current_device()
    index = current if device.index is None else device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == current:
        return fn(*args, stream)
    with torch.cuda.device(index):
        return fn(*args, stream)


class NativeLibrary:
    """Torch-facing wrapper of the C ABI.  All tensors live on one HIP device."""

    ABI_VERSION = 1

    def __init__(self, lib: ctypes.CDLL):
        self.lib = lib
        self.path = LIB_PATH
        self._workspaces: Dict[tuple, torch.Tensor] = {}

    # ---- errors -------------------------------------------------------------------------------
    def _check(self, rc: int, what: str) -> None:
        if rc == PLH_OK:
            return
        msg = f"{what}: {self.lib.plh_last_error().decode(errors='replace')}"
        if rc in (PLH_ERR_INVALID, PLH_ERR_UNSUPPORTED):
            raise ValueError(msg)
        raise RuntimeError(msg)

    def last_error(self) -> str:
        return self.lib.plh_last_error().decode(errors="replace")

    # ---- geometry -----------------------------------------------------------------------------
    def supports(self, input_size: int, hidden_size: int, num_layers: int, output_size: int) -> bool:
        return bool(self.lib.plh_supports(input_size, hidden_size, num_layers, output_size))

    def packed_bytes(self, input_size: int, hidden_size: int, num_layers: int, output_size: int) -> int:
        n = self.lib.plh_packed_bytes(input_size, hidden_size, num_layers, output_size)
        if n < 0:
            raise ValueError(self.last_error())
        return int(n)

    def workspace_bytes(self, input_size, hidden_size, num_layers, output_size, batch, seq_len) -> int:
        n = self.lib.plh_workspace_bytes(input_size, hidden_size, num_layers, output_size, batch, seq_len)
        if n < 0:
            raise ValueError(self.last_error())
        return int(n)

    # ---- packing ------------------------------------------------------------------------------
    def pack(
        self,
        w_ih: Sequence[torch.Tensor],
        w_hh: Sequence[torch.Tensor],
        b_ih: Sequence[Optional[torch.Tensor]],
        b_hh: Optional[Sequence[Optional[torch.Tensor]]],
        lin_w: Optional[torch.Tensor],
        lin_b: Optional[torch.Tensor],
    ) -> torch.Tensor:
        """Pack torch-layout parameters (any float dtype, one device) into the kernel's blob."""
        L = len(w_ih)
        if L == 0 or len(w_hh) != L or len(b_ih) != L:
            raise ValueError("w_ih, w_hh and b_ih need one tensor per layer")
        device = w_hh[0].device
        if device.type != "cuda":
            raise ValueError("weights must be on a HIP device")
        H = int(w_hh[0].shape[1])
        I = int(w_ih[0].shape[1])
        O = 0 if lin_w is None else int(lin_w.shape[0])
        half = lambda t: None if t is None else t.detach().to(device=device, dtype=torch.float16).contiguous()  # noqa: E731
        for l in range(L):
            k = I if l == 0 else H
            if tuple(w_ih[l].shape) != (4 * H, k) or tuple(w_hh[l].shape) != (4 * H, H):
                raise ValueError(f"layer {l}: expected weight_ih [{4 * H}, {k}] and weight_hh [{4 * H}, {H}]")
            for b in (b_ih[l], None if b_hh is None else b_hh[l]):
                if b is not None and tuple(b.shape) != (4 * H,):
                    raise ValueError(f"layer {l}: expected biases of shape [{4 * H}]")
        if lin_w is not None and tuple(lin_w.shape) != (O, H):
            raise ValueError(f"linear weight must be [{O}, {H}]")
        keep: List[torch.Tensor] = []

        def arr(ts):
            a = (_vp * L)()
            for i, t in enumerate(ts):
                h = half(t)
                if h is not None:
                    keep.append(h)
                    a[i] = h.data_ptr()
            return a

        a_wih, a_whh, a_bih = arr(w_ih), arr(w_hh), arr(b_ih)
        a_bhh = arr(b_hh) if b_hh is not None else None
        lw, lb = half(lin_w), half(lin_b)
        nbytes = self.packed_bytes(I, H, L, O)
        packed = torch.empty(nbytes, dtype=torch.uint8, device=device)
        rc = _launch(device, self.lib.plh_pack_regressor, I, H, L, O, a_wih, a_whh, a_bih, a_bhh, _ptr(lw), _ptr(lb),
                     packed.data_ptr(), nbytes)
        self._check(rc, "plh_pack_regressor")
        # The fp16 copies in `keep` are read asynchronously; the caching allocator only hands their
        # blocks to later work on the same stream, which runs after the pack kernels.
        return packed

    # ---- forward ------------------------------------------------------------------------------
    def workspace(self, device: torch.device, nbytes: int) -> torch.Tensor:
        """A cached workspace of at least nbytes per (device, stream): calls on one stream are
        ordered by it; calls on different streams get different workspaces."""
        key = _device_key(device)
        ws = self._workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
            if ws.data_ptr() % 256:
                ws = torch.empty(max(nbytes, 256) + 256, dtype=torch.uint8, device=device)
                off = (-ws.data_ptr()) % 256
                ws = ws[off:]
            self._workspaces[key] = ws
        return ws

    def forward(
        self,
        packed: torch.Tensor,
        dims: Sequence[int],
        x: torch.Tensor,
        *,
        lengths: Optional[torch.Tensor] = None,
        h0: Optional[torch.Tensor] = None,
        c0: Optional[torch.Tensor] = None,
        want_out: bool = True,
        want_seq: bool = False,
        want_state: bool = False,
        probe_steps: Optional[Sequence[int]] = None,
        check_status: bool = False,
        outputs: Optional[Dict[str, torch.Tensor]] = None,
    ) -> Dict[str, torch.Tensor]:
        """Run plh_forward.  dims = (I, H, L, O).  x: [B, T, I] on a HIP device (cast to fp16).

        Returns a dict with "out" [B, O], "out_seq" [B, T, H], "h_n"/"c_n" [L, B, H] (fp16) and
        "probe_h"/"probe_c" [P, L, B, H] (fp32), as requested.  `outputs` may supply any of these
        tensors (contiguous, right shape, dtype and device) to be written instead of new ones.
        """
        I, H, L, O = (int(d) for d in dims)
        if not isinstance(x, torch.Tensor) or x.dim() != 3:
            raise ValueError("x must be a [batch, seq_len, input_size] tensor")
        if x.device.type != "cuda":
            raise ValueError("x must be on a HIP device: this library has no CPU path")
        if int(x.size(2)) != I:
            raise ValueError(f"x has input size {int(x.size(2))}, the model expects {I}")
        if not x.is_floating_point():
            raise ValueError("x must be a floating-point tensor")
        device = x.device
        B, T = int(x.size(0)), int(x.size(1))
        xh = (x if x.dtype is torch.float16 else x.to(torch.float16)).contiguous()
        given = dict(outputs) if outputs else {}

        def buf(name, shape, dtype=torch.float16):
            t = given.pop(name, None)
            if t is None:
                return torch.empty(shape, device=device, dtype=dtype)
            if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device or not t.is_contiguous():
                raise ValueError(f"outputs[{name!r}] must be a contiguous {dtype} tensor of shape {tuple(shape)} "
                                 f"on {device}")
            return t

        out = buf("out", (B, O)) if (want_out and O > 0) else None
        out_seq = buf("out_seq", (B, T, H)) if want_seq else None
        h_n = buf("h_n", (L, B, H)) if want_state else None
        c_n = buf("c_n", (L, B, H)) if want_state else None
        lens_dev = None
        if lengths is not None:
            # Host lengths (a list or CPU tensor, as torch.nn.utils.rnn.pack_padded_sequence takes
            # them) are checked on the host and reach the device through pinned memory without a
            # stream synchronisation; device-resident lengths are copied back for the check, which
            # synchronises the stream.
            lens = torch.as_tensor(lengths)
            if lens.dim() != 1 or int(lens.numel()) != B:
                raise ValueError("lengths must be a 1-D tensor with one entry per batch row")
            lc = lens.detach().to("cpu", torch.int64)
            if B and (int(lc.min()) < 0 or int(lc.max()) > T):
                raise ValueError(f"lengths must lie in [0, {T}]")
            if lens.device.type == "cpu":
                lens_dev = lc.to(torch.int32).contiguous().pin_memory().to(device, non_blocking=True)
            else:
                lens_dev = lens.to(device=device, dtype=torch.int32).contiguous()
        states = []
        for s in (h0, c0):
            if s is None:
                states.append(None)
                continue
            if tuple(s.shape) != (L, B, H):
                raise ValueError(f"initial states must be [{L}, {B}, {H}]")
            states.append(s.to(device=device, dtype=torch.float16).contiguous())
        probes = sorted(set(int(p) for p in probe_steps)) if probe_steps is not None else []
        if probes and (probes[0] < 1 or probes[-1] > T):
            raise ValueError(f"probe steps must lie in [1, {T}]")
        P = len(probes)
        probe_dev = torch.tensor(probes, dtype=torch.int32, device=device) if P else None
        probe_h = buf("probe_h", (P, L, B, H), torch.float32) if P else None
        probe_c = buf("probe_c", (P, L, B, H), torch.float32) if P else None
        if given:
            raise ValueError(f"outputs given for ones not requested: {sorted(given)}")
        if packed.device != device:
            raise ValueError("packed weights and x must be on the same device")
        with _on_device(device):
            nws = self.workspace_bytes(I, H, L, O, B, T)
            ws = self.workspace(device, nws)
            rc = self.lib.plh_forward(
                packed.data_ptr(), I, H, L, O, _ptr(xh), B, T, _ptr(lens_dev), _ptr(states[0]), _ptr(states[1]),
                _ptr(out), _ptr(out_seq), _ptr(h_n), _ptr(c_n), _ptr(probe_dev), P, _ptr(probe_h), _ptr(probe_c),
                ws.data_ptr(), ws.numel(), _stream(device),
            )
            self._check(rc, "plh_forward")
            if check_status:
                self.check_status(device)
        res: Dict[str, torch.Tensor] = {}
        if out is not None:
            res["out"] = out
        if out_seq is not None:
            res["out_seq"] = out_seq
        if want_state:
            res["h_n"], res["c_n"] = h_n, c_n
        if P:
            res["probe_h"], res["probe_c"] = probe_h, probe_c
        return res

    def detects_uniform(self, dims: Sequence[int], batch: int, seq_len: int, device: torch.device) -> bool:
        """True if forward_detect finds a batch of equal rows on the device at no cost to other batches."""
        with _on_device(device):
            return bool(self.lib.plh_detects_uniform(*dims, batch, seq_len))

    def forward_detect(self, packed: torch.Tensor, dims: Sequence[int], x: torch.Tensor) -> torch.Tensor:
        """plh_forward_detect: the head outputs [B, O] of full-length rows x [B, T, I] on a HIP device."""
        I, H, L, O = dims
        if not isinstance(x, torch.Tensor) or x.dim() != 3:
            raise ValueError("x must be a [batch, seq_len, input_size] tensor")
        device = x.device
        if device.type != "cuda":
            raise ValueError("x must be on a HIP device: this library has no CPU path")
        if int(x.size(2)) != I:
            raise ValueError(f"x has input size {int(x.size(2))}, the model expects {I}")
        if not x.is_floating_point():
            raise ValueError("x must be a floating-point tensor")
        if packed.device != device:
            raise ValueError("packed weights and x must be on the same device")
        B, T = int(x.size(0)), int(x.size(1))
        xh = (x if x.dtype is torch.float16 else x.to(torch.float16)).contiguous()
        out = torch.empty((B, O), device=device, dtype=torch.float16)
        with _on_device(device):
            ws = self.workspace(device, self.workspace_bytes(I, H, L, O, B, T))
            rc = self.lib.plh_forward_detect(packed.data_ptr(), I, H, L, O, xh.data_ptr(), B, T, out.data_ptr(),
                                             ws.data_ptr(), ws.numel(), _stream(device))
        self._check(rc, "plh_forward_detect")
        return out

    def status(self, device: torch.device) -> int:
        """Synchronise the current stream and return the device status word of the last forward."""
        device = torch.device(device)
        ws = self._workspaces.get(_device_key(device))
        if ws is None:
            return 0
        st = ctypes.c_uint32(0)
        self._check(_launch(device, self.lib.plh_status, ws.data_ptr(), ctypes.byref(st)), "plh_status")
        return int(st.value)

    def check_status(self, device: torch.device) -> None:
        st = self.status(device)
        if st & PLH_STATUS_TIMEOUT:
            raise RuntimeError("persistent LSTM kernel: a layer hand-off wait timed out (outputs are invalid)")
        if st:
            raise RuntimeError(f"persistent LSTM kernel reported status {st:#x}")

    def set_wait_limit(self, seconds: Optional[float]) -> None:
        """Bound on inter-workgroup waits of this thread's later forwards (None: the 2 s default)."""
        us = 0 if seconds is None else max(1, int(round(seconds * 1e6)))
        self._check(self.lib.plh_set_wait_limit_us(us), "plh_set_wait_limit_us")

    def inject_wait_failure(self, step: Optional[int]) -> None:
        """Failure injection for tests (this thread): layer-sequential forwards fail one workgroup's
        wait at `step` (None: off)."""
        self._check(self.lib.plh_inject_wait_failure(-1 if step is None else int(step)), "plh_inject_wait_failure")

    # ---- timing of the persistent kernel alone ----------------------------------------------
    def kernel_timing(self, max_forwards: int) -> None:
        """Arm HIP events around the persistent launch of the next max_forwards forwards (this thread)."""
        self._check(self.lib.plh_kernel_timing(int(max_forwards)), "plh_kernel_timing")

    def kernel_timing_read(self):
        """(summed kernel milliseconds, number of timed forwards); synchronises on the events."""
        ms = ctypes.c_double(0.0)
        n = _i32(0)
        self._check(self.lib.plh_kernel_timing_read(ctypes.byref(ms), ctypes.byref(n)), "plh_kernel_timing_read")
        return float(ms.value), int(n.value)

    def probe_mfma_f16(self):
        """(TFLOP/s, shader GHz): dense fp16 MFMA rate of the current device (v_mfma_f32_16x16x32_f16 on
        every CU) and the clock during that run.  Synchronous, about 30 ms."""
        tf = ctypes.c_double(0.0)
        ghz = ctypes.c_double(0.0)
        self._check(self.lib.plh_probe_mfma_f16(ctypes.byref(tf), ctypes.byref(ghz)), "plh_probe_mfma_f16")
        return float(tf.value), float(ghz.value)

    # ---- the time-parallel input projection GEMM ---------------------------------------------
    def input_projection(self, x: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None, *,
                         blocked: bool = False) -> torch.Tensor:
        """out[m, n] = sum_k x[m, k] w[n, k] (fp16 MFMA GEMM, fp32 accumulation, fp16 result).

        Row-major (blocked=False): x [rows, K] fp16 with unit column stride (its row stride may exceed
        K), out [rows, cols].  Fragment-blocked (blocked=True): x is a contiguous [rows, ldx] tensor
        in the layout of `to_blocked` (the first K columns are used), out likewise [rows, cols]
        blocked.  w: [cols, K] fp16; K % 128 == 0, K <= 65536, cols % 128 == 0.  Replaces the
        reference's torch::matmul input projection (persistent_lstm_hip.cu:2988-2994).  Launched on
        the current stream."""
        for name, t in (("x", x), ("w", w)):
            if t.dim() != 2 or t.dtype != torch.float16 or t.device.type != "cuda":
                raise ValueError(f"{name} must be a 2-D float16 HIP tensor")
        w = w.contiguous()
        cols, k = int(w.size(0)), int(w.size(1))
        rows = int(x.size(0))
        if blocked:
            if not x.is_contiguous():
                raise ValueError("a blocked x must be contiguous")
            ldx = int(x.size(1))
        else:
            if x.stride(1) != 1 or (rows > 1 and x.stride(0) < x.size(1)):
                raise ValueError("x must have unit column stride and row stride >= its width")
            if int(x.size(1)) != k:
                raise ValueError("x and w must have the same K")
            ldx = int(x.stride(0)) if rows > 1 else k
        if out is None:
            out = torch.empty((rows, cols), dtype=torch.float16, device=x.device)
        elif (tuple(out.shape) != (rows, cols) or out.dtype != torch.float16 or out.stride(1) != 1
              or (blocked and not out.is_contiguous())):
            raise ValueError("out must be a float16 [rows, cols] tensor with unit column stride (blocked: contiguous)")
        ldo = cols if (blocked or rows <= 1) else int(out.stride(0))
        rc = _launch(x.device, self.lib.plh_input_projection, x.data_ptr(), ldx, w.data_ptr(), k, out.data_ptr(), ldo,
                     rows, cols, 1 if blocked else 0)
        self._check(rc, "plh_input_projection")
        return out

    @staticmethod
    def to_blocked(t: torch.Tensor) -> torch.Tensor:
        """[rows, ld] (rows % 16 == 0, ld % 32 == 0) -> the fragment-blocked layout of the same shape:
        element (r, c) at (((r / 16) (ld / 32) + c / 32) 64 + ((c % 32) / 8) 16 + r % 16) 8 + c % 8."""
        rows, ld = int(t.size(0)), int(t.size(1))
        if rows % 16 or ld % 32:
            raise ValueError("blocked layouts need rows % 16 == 0 and columns % 32 == 0")
        return t.reshape(rows // 16, 16, ld // 32, 4, 8).permute(0, 2, 3, 1, 4).reshape(rows, ld).contiguous()

    @staticmethod
    def from_blocked(t: torch.Tensor) -> torch.Tensor:
        """Inverse of to_blocked."""
        rows, ld = int(t.size(0)), int(t.size(1))
        return t.reshape(rows // 16, ld // 32, 4, 16, 8).permute(0, 3, 1, 2, 4).reshape(rows, ld).contiguous()

    # ---- reference extension surface (bindings.cpp:154-165) ----------------------------------
    def repeat_first_row(self, inp: torch.Tensor, output_batch_size: int) -> torch.Tensor:
        """bindings.cpp:164: out[r] = inp[0] for r < output_batch_size (fp16, HIP tensor)."""
        if inp.dim() != 2 or inp.dtype != torch.float16 or inp.device.type != "cuda":
            raise ValueError("repeat_first_row expects a 2-D float16 HIP tensor")
        inp = inp.contiguous()
        cols = int(inp.size(1))
        out = torch.empty((int(output_batch_size), cols), dtype=inp.dtype, device=inp.device)
        rc = _launch(inp.device, self.lib.plh_repeat_first_row, inp.data_ptr(), out.data_ptr(), int(output_batch_size),
                     cols)
        self._check(rc, "plh_repeat_first_row")
        return out

    def _packed_for(self, source: tuple, make_weights) -> tuple:
        """(packed blob, dims) for reference-format arguments, cached on the identity and version of
        the tensors the caller passed (`source`): the reference's dispatcher passes the same cached
        tensors to every forward (model.py:542-582), so they are converted and packed once per weight
        version.  make_weights() -> (w_ih list, w_hh list, fused bias list, linear weight, linear
        bias) in torch layout; it runs only on a cache miss, so a hit launches nothing but the
        forward."""
        from .model import _TensorSetKey  # noqa: PLC0415 (model imports this module)

        key = getattr(self, "_compat_key", None)
        if key is None or not key.matches(source):
            w_ih, w_hh, bias, linear_weight, linear_bias = make_weights()
            if not (len(w_ih) == len(w_hh) == len(bias)) or not w_ih:
                raise ValueError("weight_ih, weight_hh and bias need one tensor per layer")
            self._compat_blob = self.pack(w_ih, w_hh, bias, None, linear_weight, linear_bias)
            self._compat_dims = (int(w_ih[0].shape[1]), int(w_hh[0].shape[1]), len(w_ih),
                                 int(linear_weight.shape[0]))
            self._compat_key = _TensorSetKey(source)
        return self._compat_blob, self._compat_dims

    def persistent_lstm_regressor_forward_generic_projected(
        self, x, weight_ih: List[torch.Tensor], weight_hh: List[torch.Tensor], bias: List[torch.Tensor],
        linear_weight: torch.Tensor, linear_bias: torch.Tensor,
    ) -> torch.Tensor:
        """bindings.cpp:163: (x, [W_ih], [W_hh], [b_ih + b_hh], W_lin, b_lin) -> [B, O]."""
        source = tuple(weight_ih) + tuple(weight_hh) + tuple(bias) + (linear_weight, linear_bias)
        return self._forward_reference_format(
            x, source, lambda: (list(weight_ih), list(weight_hh), list(bias), linear_weight, linear_bias))

    def _forward_reference_format(self, x, source: tuple, make_weights) -> torch.Tensor:
        if not isinstance(x, torch.Tensor) or x.dim() != 3:
            raise ValueError("x must be a [batch, seq_len, input_size] tensor")
        packed, dims = self._packed_for(source, make_weights)
        return self.forward(packed, dims, x)["out"]

    @staticmethod
    def unpack_kpairs(packed: torch.Tensor, k: int) -> torch.Tensor:
        """Invert the reference's kpairs layout P[p, c, j] = W[c, 2p + j] (model.py:20-27), as its CPU
        branch does (persistent_lstm_op.cpp:161-168): returns W [4H, k]."""
        if packed.dim() != 3 or packed.size(2) != 2:
            raise ValueError("kpairs-packed weight must be [ceil(K/2), 4H, 2]")
        pairs, out = int(packed.size(0)), int(packed.size(1))
        full = packed.permute(0, 2, 1).reshape(pairs * 2, out)
        return full[:k].t().contiguous()

    @staticmethod
    def _four_layers(args) -> None:
        if len(args) != 14:
            raise ValueError("expected 12 per-layer tensors (weight_ih, weight_hh, bias for 4 layers) plus the "
                             "linear weight and bias")

    def persistent_lstm4_forward(self, x, *args) -> torch.Tensor:
        """bindings.cpp:155: torch-layout weights [4H, K] and fused biases, 4 layers."""
        self._four_layers(args)
        return self._forward_reference_format(
            x, args, lambda: ([args[3 * l] for l in range(4)], [args[3 * l + 1] for l in range(4)],
                              [args[3 * l + 2] for l in range(4)], args[12], args[13]))

    def persistent_lstm4_forward_packed(self, x, *args) -> torch.Tensor:
        """bindings.cpp:156: transposed weights W^T [K, 4H] (persistent_lstm_hip.cu:2005-2018) and fused
        biases, 4 layers."""
        self._four_layers(args)
        return self._forward_reference_format(
            x, args, lambda: ([args[3 * l].t() for l in range(4)], [args[3 * l + 1].t() for l in range(4)],
                              [args[3 * l + 2] for l in range(4)], args[12], args[13]))

    def persistent_lstm4_forward_interleaved(self, x, *args) -> torch.Tensor:
        """bindings.cpp:157: kpairs-packed W_ih and W_hh (model.py:562-578) and fused biases."""
        self._four_layers(args)
        H = int(args[1].size(1)) // 4
        I = int(x.size(2)) if isinstance(x, torch.Tensor) and x.dim() == 3 else 0
        return self._forward_reference_format(
            x, args, lambda: ([self.unpack_kpairs(args[3 * l], I if l == 0 else H) for l in range(4)],
                              [self.unpack_kpairs(args[3 * l + 1], H) for l in range(4)],
                              [args[3 * l + 2] for l in range(4)], args[12], args[13]))

    def persistent_lstm4_forward_monolithic(self, x, *args) -> torch.Tensor:
        """bindings.cpp:162: the interleaved arguments (the reference's all-layers-in-one-kernel variant,
        persistent_lstm_hip.cu:2823-2921); here the same single path as every other entry point."""
        return self.persistent_lstm4_forward_interleaved(x, *args)

    def persistent_lstm4_forward_projected(self, x, *args) -> torch.Tensor:
        """bindings.cpp:158: native W_ih [4H, K] with kpairs-packed W_hh (model.py:548-560)."""
        self._four_layers(args)
        H = int(args[0].size(0)) // 4
        return self._forward_reference_format(
            x, args, lambda: ([args[3 * l] for l in range(4)],
                              [self.unpack_kpairs(args[3 * l + 1], H) for l in range(4)],
                              [args[3 * l + 2] for l in range(4)], args[12], args[13]))

    def persistent_lstm4_forward_projected_uniform(self, x, virtual_batch_size: int, *args) -> torch.Tensor:
        """bindings.cpp:159: the projected arguments for ONE sequence x [1, T, I] -> [1, O] (the caller
        broadcasts it with repeat_first_row).  The reference runs `virtual_batch_size` redundant copies
        of that sequence (persistent_lstm_hip.cu:2399-2549); they change nothing in the result, so one
        row is computed.  Like the reference, any other x (or virtual_batch_size <= 0) takes the
        ordinary projected forward of every row (cu:2416-2433)."""
        return self.persistent_lstm4_forward_projected(x, *args)

    def persistent_lstm4_forward_projected_uniform_p4(self, x, virtual_batch_size: int, *args) -> torch.Tensor:
        """bindings.cpp:160: as persistent_lstm4_forward_projected_uniform (the reference's 4-way K
        partition of the same recurrence, persistent_lstm_hip.cu:2551-2685)."""
        return self.persistent_lstm4_forward_projected_uniform(x, virtual_batch_size, *args)

    def persistent_lstm4_forward_projected_uniform_p8(self, x, virtual_batch_size: int, *args) -> torch.Tensor:
        """bindings.cpp:161: as persistent_lstm4_forward_projected_uniform (8-way K partition there,
        persistent_lstm_hip.cu:2687-2821)."""
        return self.persistent_lstm4_forward_projected_uniform(x, virtual_batch_size, *args)


# The reference extension's exported names (bindings.cpp:154-165), in its order.
REFERENCE_ENTRY_POINTS = (
    "persistent_lstm4_forward",
    "persistent_lstm4_forward_packed",
    "persistent_lstm4_forward_interleaved",
    "persistent_lstm4_forward_projected",
    "persistent_lstm4_forward_projected_uniform",
    "persistent_lstm4_forward_projected_uniform_p4",
    "persistent_lstm4_forward_projected_uniform_p8",
    "persistent_lstm4_forward_monolithic",
    "persistent_lstm_regressor_forward_generic_projected",
    "repeat_first_row",
)


def library_path() -> str:
    return LIB_PATH


@lru_cache(maxsize=1)
def load_extension() -> Optional[NativeLibrary]:
    """The native library, or None if it cannot be loaded (see load_error())."""
    global _load_error
    if not os.path.exists(LIB_PATH):
        _load_error = f"{LIB_PATH} is missing: run `python -m persistent_lstm_hip_amd.build`"
        return None
    try:
        # torch ships the HIP runtime; loading it first lets the library bind to the same copy.
        import torch.cuda  # noqa: F401

        lib = ctypes.CDLL(LIB_PATH)
        _declare(lib)
        if lib.plh_abi_version() != NativeLibrary.ABI_VERSION:
            _load_error = "ABI version mismatch between the library and its Python front end"
            return None
        return NativeLibrary(lib)
    except OSError as exc:
        _load_error = f"cannot load {LIB_PATH}: {exc}"
        return None
    except AttributeError as exc:  # built before a function this front end binds was added
        _load_error = f"{LIB_PATH} is out of date ({exc}): run `python -m persistent_lstm_hip_amd.build`"
        return None


def load_error() -> Optional[str]:
    return _load_error


def require_extension() -> NativeLibrary:
    """The native library; RuntimeError (never a fallback) if it is unavailable."""
    ext = load_extension()
    if ext is None:
        raise RuntimeError(f"persistent_lstm_hip_amd native library unavailable: {_load_error}")
    return ext


@lru_cache(maxsize=1)
def require_torch_ops():
    """The module plh_torch (csrc/plh_torch.cpp), the torch front end of the block operators; RuntimeError (never a
    fallback) if it or the library under it is unavailable."""
    require_extension()
    try:
        spec = importlib.util.spec_from_file_location("plh_torch", TORCH_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except (ImportError, OSError) as exc:
        raise RuntimeError(f"persistent_lstm_hip_amd: cannot load {TORCH_PATH} ({exc}): run "
                           "`python -m persistent_lstm_hip_amd.build`") from exc
    return module
