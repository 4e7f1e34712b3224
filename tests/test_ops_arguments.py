"""Arguments of the block operators as callers have them (no kernel is launched)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import persistent_lstm_hip_amd as P
from persistent_lstm_hip_amd import ops


class _Recorder:
    def dropout_add(self, x, residual, p, seed, offset, offset_dev):
        return seed, offset, offset_dev


@pytest.fixture
def calls(monkeypatch):
    monkeypatch.setattr(ops, "require_torch_ops", lambda: _Recorder())


@pytest.mark.parametrize("kind", [int, np.int64, np.int32, np.uint8, np.uint64, torch.tensor])
def test_seed_and_offset_are_integers_of_any_type(calls, kind):
    x = torch.zeros(2)
    assert P.dropout_add(x, p=0.1, seed=kind(7), offset=3)[:2] == (7, 3)
    if kind is not torch.tensor:  # (a tensor offset is the device's)
        assert P.dropout_add(x, p=0.1, seed=1, offset=kind(7))[:2] == (1, 7)


def test_seed_and_offset_are_taken_modulo_2_64(calls):
    x = torch.zeros(2)
    assert P.dropout_add(x, p=0.1, seed=-1, offset=2**64 + 5)[:2] == (2**64 - 1, 5)
    assert P.dropout_add(x, p=0.1, seed=np.int64(-2), offset=np.int32(-1))[:2] == (2**64 - 2, 2**64 - 1)


@pytest.mark.parametrize("bad", [1.0, "1", None, [1], np.float32(1)])
def test_what_is_no_integer_is_refused(calls, bad):
    x = torch.zeros(2)
    with pytest.raises(ValueError, match="seed must be an integer"):
        P.dropout_add(x, p=0.1, seed=bad)
    with pytest.raises(ValueError, match="offset must be an integer"):
        P.dropout_add(x, p=0.1, seed=1, offset=bad)
