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


def test_lazily_negated_tensors(gpu):
    """A real tensor may stand for the negative of its storage, as the imaginary part of a conjugate does."""
    _say("negated views")
    neg = torch._neg_view
    x, r, w, z, c = _x(3, 8), _x(3, 8, seed=1), _x(8, seed=2), _x(3, 5, 12, seed=3), _x(3, 4, seed=4)
    for got, want in (
            (P.layer_norm(neg(x), neg(w), neg(w)), P.layer_norm(-x, -w, -w)),
            (P.layer_norm(neg(x.view(3, 2, 4))), P.layer_norm(-x.view(3, 2, 4))),
            (P.dropout_add(neg(x), neg(r), p=0.3, seed=1), P.dropout_add(-x, -r, p=0.3, seed=1)),
            (P.gated_scan(neg(z), neg(c))[0], P.gated_scan(-z, -c)[0]),
            (P.gated_scan(neg(z).transpose(0, 1).contiguous().transpose(0, 1), neg(c))[1], P.gated_scan(-z, -c)[1]),
            (P.gated_scan_step(neg(z[:, 0]), neg(c))[1], P.gated_scan_step(-z[:, 0], -c)[1])):
        assert torch.equal(got, want)
    with pytest.raises(ValueError, match="negated"):
        P.gated_scan_step(z[:, 0], neg(c), inplace=True)
    one = torch.complex(_x(1), _x(1, seed=1)).conj().imag
    assert torch.equal(P.dropout_add(one, p=0.0, seed=1), one.clone())
    leaf = x.clone().requires_grad_(True)
    d = _x(3, 8, seed=5)
    for f in (lambda t: P.layer_norm(neg(t)), lambda t: P.dropout_add(neg(t), p=0.3, seed=1),
              lambda t: P.gated_scan(neg(t).view(1, 3, 8), output_gate=False)[0].view(3, 4)):
        y = f(leaf)
        dy = d[:, :y.shape[1]]
        got, = torch.autograd.grad(y, leaf, neg(dy.contiguous()), retain_graph=True)
        assert torch.equal(got, torch.autograd.grad(y, leaf, -dy)[0])
