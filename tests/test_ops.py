"""The block operators' host side: their generator against published vectors, their formulas' gradients against
differences, and everything that they refuse (no kernel is launched)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import ops_plain as plain
import persistent_lstm_hip_amd as P
from persistent_lstm_hip_amd import ops
from persistent_lstm_hip_amd.extension import PLH_ERR_INVALID, PLH_ERR_UNSUPPORTED, PLH_OK, require_extension


@pytest.mark.parametrize("counter,key,want", [
    # the published known answers of Philox4x32-10
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_the_plain_generator_gives_the_published_vectors(counter, key, want):
    got = plain.philox(np.array([counter], dtype=np.uint64), key)[0]
    assert tuple(int(v) for v in got) == want


def _directional(f, x, d, step=1e-6):
    return (f(x + step * d) - f(x - step * d)) / (2 * step)


@pytest.mark.parametrize("gated", [True, False])
def test_the_scan_formulas_gradient_is_that_of_differences(gated):
    g = torch.Generator().manual_seed(3)
    B, T, H = 3, 9, 4
    z = torch.randn(B, T, (3 if gated else 2) * H, generator=g, dtype=torch.float64)
    c0, dc = torch.randn(B, H, generator=g, dtype=torch.float64), torch.randn(B, H, generator=g, dtype=torch.float64)
    dh, n = torch.randn(B, T, H, generator=g, dtype=torch.float64), [9, 0, 5]

    def loss(z, c0):
        out, c_n = plain.scan(z, c0, n, gated)
        return ((out * dh).sum() + (c_n * dc).sum()).item()

    _, _, dz, d0, _ = plain.scan(z, c0, n, gated, dh, dc)
    way, way0 = torch.randn(z.shape, generator=g, dtype=torch.float64), torch.randn(B, H, generator=g, dtype=torch.float64)
    assert abs(_directional(lambda v: loss(v, c0), z, way) - (dz * way).sum().item()) < 1e-7
    assert abs(_directional(lambda v: loss(z, v), c0, way0) - (d0 * way0).sum().item()) < 1e-7


def test_the_norm_formulas_gradient_is_that_of_differences():
    g = torch.Generator().manual_seed(4)
    x, dy, way = (torch.randn(5, 7, generator=g, dtype=torch.float64) for _ in range(3))
    w, b, ww = (torch.randn(7, generator=g, dtype=torch.float64) for _ in range(3))

    def loss(x, w, b):
        return (plain.norm(x, w, b, 1e-5) * dy).sum().item()

    _, dx, dw, db = plain.norm(x, w, b, 1e-5, dy)
    assert abs(_directional(lambda v: loss(v, w, b), x, way) - (dx * way).sum().item()) < 1e-7
    assert abs(_directional(lambda v: loss(x, v, b), w, ww) - (dw * ww).sum().item()) < 1e-7
    assert abs(_directional(lambda v: loss(x, w, v), b, ww) - (db * ww).sum().item()) < 1e-7


def test_public_names():
    for name in ("gated_scan", "gated_scan_step", "layer_norm", "dropout_add"):
        assert name in P.__all__ and getattr(P, name) is getattr(ops, name)


@pytest.mark.parametrize("call", [
    lambda t: P.gated_scan(t(2, 3, 12)),
    lambda t: P.gated_scan_step(t(2, 12), t(2, 4)),
    lambda t: P.layer_norm(t(2, 8)),
    lambda t: P.dropout_add(t(2, 8), p=0.1, seed=1),
    lambda t: P.dropout_add(t(2, 8), p=0.1, seed=-1, offset=torch.zeros(1, dtype=torch.int64)),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="HIP device"):
        call(torch.zeros)
    with pytest.raises(ValueError, match="must be a tensor"):
        call(lambda *shape: [0.0])


def test_a_missing_front_end_is_an_error_that_names_it(tmp_path, monkeypatch):
    from persistent_lstm_hip_amd import extension

    monkeypatch.setattr(extension, "TORCH_PATH", str(tmp_path / "plh_torch.so"))
    with pytest.raises(RuntimeError, match="plh_torch.so.*persistent_lstm_hip_amd.build"):
        extension.require_torch_ops.__wrapped__()
    (tmp_path / "plh_torch.so").write_bytes(b"not a library")
    with pytest.raises(RuntimeError, match="plh_torch.so"):
        extension.require_torch_ops.__wrapped__()


# ---- the C ABI refuses before it touches a device ------------------------------------------------

ANY = ctypes.c_void_p(256)  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return require_extension().lib


def _scan(lib, *, dtype=0, gates=ANY, sb=36, st=12, B=2, T=3, H=4, out=ANY, ws=None, nws=0):
    return lib.plh_gated_scan_forward(dtype, 1, gates, sb, st, B, T, H, None, None, out, None, None, ws, nws, None)


def _scan_back(lib, *, dtype=0, gates=ANY, states=ANY, d_out=ANY, d_gates=ANY, B=2, T=3, H=4, ws=None, nws=0):
    return lib.plh_gated_scan_backward(dtype, 1, gates, 36, 12, B, T, H, None, states, d_out, None, d_gates, None, ws,
                                       nws, None)


@pytest.mark.parametrize("call", [_scan, _scan_back])
def test_scan_refusals(lib, call):
    assert call(lib, dtype=3) == PLH_ERR_INVALID and b"dtype" in lib.plh_last_error()
    assert call(lib, B=-1) == PLH_ERR_INVALID
    assert call(lib, T=-1) == PLH_ERR_INVALID
    assert call(lib, H=0) == PLH_ERR_UNSUPPORTED and b"hidden" in lib.plh_last_error()
    assert call(lib, H=1 << 24, B=64) == PLH_ERR_UNSUPPORTED
    assert call(lib, T=(1 << 30) + 1) == PLH_ERR_UNSUPPORTED
    assert call(lib, gates=None) == PLH_ERR_INVALID and b"gates" in lib.plh_last_error()
    # two rows of 100000 steps are split over the time axis: a workspace is needed
    need = lib.plh_gated_scan_workspace_bytes(2, 100000, 4)
    assert need > 0
    assert call(lib, T=100000) == PLH_ERR_INVALID and b"workspace" in lib.plh_last_error()
    assert call(lib, T=100000, ws=ANY, nws=need - 1) == PLH_ERR_INVALID
    assert call(lib, T=100000, ws=ctypes.c_void_p(260), nws=need) == PLH_ERR_INVALID
    assert call(lib, B=0) == PLH_OK


def test_scan_refuses_missing_outputs(lib):
    assert _scan(lib, out=None) == PLH_ERR_INVALID and b"out" in lib.plh_last_error()
    assert _scan(lib, sb=-1) == PLH_ERR_INVALID and b"strides" in lib.plh_last_error()
    for name in ("states", "d_out", "d_gates"):
        assert _scan_back(lib, **{name: None}) == PLH_ERR_INVALID and name.encode() in lib.plh_last_error()


def test_scan_sizes(lib):
    assert lib.plh_gated_scan_states(0) == 0 and lib.plh_gated_scan_states(1) == 1
    assert lib.plh_gated_scan_states(-1) == -1
    # one state per row, channel and tile; ragged sizes round up
    n = lib.plh_gated_scan_states(1000)
    assert lib.plh_gated_scan_states(1001) >= n > 0
    assert lib.plh_gated_scan_workspace_bytes(100000, 1000, 128) == 0  # enough rows: the time axis is not split
    assert lib.plh_gated_scan_workspace_bytes(-1, 1, 1) == -1 == lib.plh_gated_scan_workspace_bytes(1, 1, 0)
    assert lib.plh_gated_scan_workspace_bytes(0, 5, 5) >= 0


def test_norm_refusals(lib):
    def fwd(dtype=0, wdtype=0, x=ANY, stride=8, rows=2, cols=8, y=ANY):
        return lib.plh_layer_norm_forward(dtype, wdtype, x, stride, rows, cols, None, None, 1e-5, y, None, None, None)

    def back(x=ANY, rows=2, cols=8, mean=ANY, dy=ANY, dw=None, ws=None, nws=0):
        return lib.plh_layer_norm_backward(0, 0, x, 8, rows, cols, None, mean, ANY, dy, ANY, dw, None, ws, nws, None)

    assert fwd(dtype=-1) == PLH_ERR_INVALID and fwd(dtype=0, wdtype=1) == PLH_ERR_INVALID
    assert b"wdtype" in lib.plh_last_error()
    assert fwd(rows=-1) == PLH_ERR_INVALID and fwd(cols=0) == PLH_ERR_UNSUPPORTED
    assert fwd(cols=(1 << 24) + 1) == PLH_ERR_UNSUPPORTED
    assert fwd(x=None) == PLH_ERR_INVALID and fwd(y=None) == PLH_ERR_INVALID and fwd(stride=-8) == PLH_ERR_INVALID
    assert fwd(rows=0) == PLH_OK
    assert back(mean=None) == PLH_ERR_INVALID and back(dy=None) == PLH_ERR_INVALID
    assert back(dw=ANY) == PLH_ERR_INVALID and b"workspace" in lib.plh_last_error()
    assert back(dw=ANY, ws=ANY, nws=lib.plh_layer_norm_workspace_bytes(2, 8) - 1) == PLH_ERR_INVALID
    assert lib.plh_layer_norm_workspace_bytes(-1, 8) == -1 == lib.plh_layer_norm_workspace_bytes(1, 0)


def test_dropout_refusals(lib):
    def call(dtype=0, x=ANY, out=ANY, n=8, threshold=1):
        return lib.plh_dropout_add(dtype, x, None, out, n, threshold, 1, 0, None, None)

    assert call(dtype=7) == PLH_ERR_INVALID and call(n=-1) == PLH_ERR_INVALID
    assert call(threshold=-1) == PLH_ERR_INVALID and call(threshold=65537) == PLH_ERR_INVALID
    assert call(x=None) == PLH_ERR_INVALID and call(out=None) == PLH_ERR_INVALID
    assert call(n=0) == PLH_OK


def test_a_planted_mistake_is_seen():
    """The comparison that the GPU tests rest on fails for a result that is off by two roundings in one element."""
    want = torch.linspace(-2, 2, 64, dtype=torch.float64)
    for dtype in plain.ROUNDING:
        plain.assert_within(want.to(dtype), want, 0.0, dtype, "rounded")
        bad = want.to(dtype).double()
        bad[17] *= 1 + 4 * plain.ROUNDING[dtype][0]
        with pytest.raises(AssertionError, match="element 17"):
            plain.assert_within(bad, want, 0.0, dtype, "planted")
