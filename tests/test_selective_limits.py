"""The sizes that the selective scan takes and refuses, at their borders.  What it takes is called without an output, which it
asks for after the sizes: no kernel is launched."""
from __future__ import annotations

import ctypes

import pytest

from persistent_lstm_hip_amd.extension import (
    PLH_ERR_INVALID,
    PLH_ERR_UNSUPPORTED,
    SelectiveScanArgs,
    SelectiveScanGrads,
    require_extension,
)

ANY = ctypes.c_void_p(256)  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return require_extension().lib


def _args(batch, seq_len, channels, states):
    a = SelectiveScanArgs()
    a.batch, a.seq_len, a.channels, a.states, a.softplus = batch, seq_len, channels, states, 1
    a.u = a.dt = a.B = a.C = a.A = 256
    return ctypes.byref(a)


# lanes per channel, four states each
@pytest.mark.parametrize("states,lanes", [(1, 1), (4, 1), (5, 2), (8, 2), (9, 4), (16, 4), (17, 8), (32, 8), (33, 16),
                                          (64, 16)])
def test_a_step_has_fewer_threads_than_a_launch_holds(lib, states, lanes):
    def step(batch, channels):
        rc = lib.plh_selective_scan_step(_args(batch, 1, channels, states), ANY, None, ANY, None)
        return rc, lib.plh_last_error()

    most = ((1 << 32) - 256) // lanes
    for batch, channels in ((most, 1), (most // 7, 7), (most // (1 << 20), 1 << 20)):
        rc, msg = step(batch, channels)
        assert rc == PLH_ERR_INVALID and b"out" in msg, (batch, channels)
    for batch, channels in ((most + 1, 1), ((1 << 32) // lanes, 1), ((1 << 12) // lanes + 1, 1 << 20), (1 << 62, 1 << 20)):
        assert step(batch, channels)[0] == PLH_ERR_UNSUPPORTED, (batch, channels)


@pytest.mark.parametrize("states", [1, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("backward", [False, True])
def test_rows_and_channels_that_a_launch_holds(lib, states, backward):
    def call(batch, channels):
        a = _args(batch, 2, channels, states)
        if backward:  # (without the forward pass's states)
            rc = lib.plh_selective_scan_backward(a, None, ANY, None, ctypes.byref(SelectiveScanGrads()), ANY, 1 << 62, None)
        else:
            rc = lib.plh_selective_scan_forward(a, None, None, None, None, None, 0, None)
        return rc, lib.plh_last_error()

    for batch, channels in ((16385, 1024), (65535, 1024), ((1 << 21) - 1, 24), (7, 1 << 20), (63, 1 << 20), (1 << 21, 8),
                            ((1 << 21) - 1, 9)):
        rc, msg = call(batch, channels)
        if batch * 2 * states > 1 << 30:
            continue
        # the workgroups of either direction, each with its threads
        per, side = (16, 1) if states <= 16 else (8, 2) if states <= 32 else (4, 2)
        groups = (channels + per - 1) // per
        assert batch * groups * 256 < 1 << 32
        assert ((batch + side - 1) // side if groups == 1 else batch * ((groups + side - 1) // side)) * side * 256 < 1 << 32
        assert rc == PLH_ERR_INVALID and (b"required" in msg), (batch, channels, msg)
    for batch, channels in ((65536, 1024), (1 << 21, 9), ((1 << 21) + 1, 1), (64, 1 << 20), ((1 << 21) - 1, 33), (1 << 40, 1),
                            (1 << 62, 1 << 20)):
        rc, msg = call(batch, channels)
        assert rc == PLH_ERR_UNSUPPORTED and b"2^2" in msg, (batch, channels, msg)
