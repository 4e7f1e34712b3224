"""The forecaster's dropout masks on the GPU where a pass runs more than once: activation checkpointing."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from persistent_lstm_hip_amd import GatedScanRegressor

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _model():
    torch.manual_seed(11)
    return GatedScanRegressor(2, 32, 3, 2, 0.5).cuda()


def test_checkpointed_gradients_are_the_passes_own(gpu):
    """Two outstanding passes against the same without checkpointing."""
    _say("checkpoint")
    xs = [torch.randn(4, 70, 2, generator=torch.Generator().manual_seed(s)).cuda() for s in (1, 2)]

    def gradients(run):
        m = _model()
        sum(run(m, x).square().sum() for x in xs).backward()
        return [p.grad for p in m.parameters()]

    want = gradients(lambda m, x: m(x))
    got = gradients(lambda m, x: checkpoint(m, x, use_reentrant=False))
    for a, b in zip(got, want):  # (torch's weight gradients may sum in another order)
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4 * max(1.0, b.abs().max().item()))
