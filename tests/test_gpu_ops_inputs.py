"""Block operators on the GPU: tensors that hold something else than their storage says, or that may not be written."""
from __future__ import annotations

import pytest
import torch

import persistent_lstm_hip_amd as P

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _x(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_an_inference_tensor_is_refused_before_it_is_overwritten(gpu):
    """As torch does: outside inference mode it may not be updated in place, and then it is as it was."""
    _say("inference state")
    z = _x(2, 12)
    with torch.inference_mode():
        c = _x(2, 4, seed=1)
    before = c.tolist()
    with torch.no_grad():
        with pytest.raises(ValueError, match="inference"):
            P.gated_scan_step(z, c, inplace=True)
        assert c.tolist() == before
        want = P.gated_scan_step(z, c)[1]  # (not in place: fine)
    with torch.inference_mode():
        assert P.gated_scan_step(z, c, inplace=True)[1] is c
    assert torch.equal(c.clone(), want.clone())
    plain = _x(2, 4, seed=1)
    with torch.inference_mode():  # an ordinary tensor in inference mode
        P.gated_scan_step(z, plain, inplace=True)
    assert torch.equal(plain, want.clone())


def test_a_models_states_of_inference_mode(gpu):
    """No block's state moves on where the first one's is refused."""
    _say("inference model states")
    torch.manual_seed(0)
    m = P.GatedScanRegressor(2, 8, 3, 2, 0.0).cuda().eval()
    with torch.inference_mode():
        state = m.initial_state(3)
    with pytest.raises(ValueError, match="inference"):
        m.step(_x(3, 2), state)
    assert not any(s.any() for s in state)
    with torch.inference_mode():
        m.step(_x(3, 2), state)
    assert all(s.any() for s in state)
