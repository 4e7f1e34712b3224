"""The sizes that the selective scan takes and refuses, at their borders.  What it takes is called without an output, which it
asks for after the sizes: no kernel is launched."""
from __future__ import annotations

import ctypes

import pytest

from persistent_lstm_hip_amd.extension import PLH_ERR_INVALID, PLH_ERR_UNSUPPORTED, SelectiveScanArgs, require_extension

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
@pytest.mark.parametrize("states,lanes", [(1, 1), (4, 1), (5, 2), (8, 2), (9, 4), (16, 4), (17, 8), (32, 8), (33, 16), (64, 16)])
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
