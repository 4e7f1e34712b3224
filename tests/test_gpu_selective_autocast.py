"""The forecaster on the selective scan, served under autocast from the state that it is documented to start from, and handed
on between what runs under autocast and what does not."""
from __future__ import annotations

import pytest
import torch

from persistent_lstm_hip_amd import SelectiveScanBlock, SelectiveScanRegressor

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _model():
    torch.manual_seed(12)
    m = SelectiveScanRegressor(3, 64, 6, 2, 0.2).cuda().eval()
    return m, torch.randn(5, 40, 3, generator=torch.Generator().manual_seed(1)).cuda()


def _close(a, b, dtype):
    """8 stages per layer and 3 more, each rounded to dtype once, amplified by at most a few by the norms behind it (the
    same bound as a forward pass under autocast has)."""
    eps = torch.finfo(dtype).eps / 2
    assert (a.float() - b.float()).abs().max() <= 96 * eps * max(1.0, b.abs().max().item())


@pytest.mark.parametrize("dtype", HALVES)
def test_token_by_token(gpu, dtype):
    _say(f"selective autocast tokens {dtype}")
    m, x = _model()
    with torch.no_grad():
        whole = m(x)
    state = m.initial_state(5)
    places = [t.data_ptr() for pair in state for t in pair]
    with torch.autocast("cuda", dtype=dtype):
        for t in range(40):
            out = m.step(x[:, t], state)
    assert out.dtype == dtype
    _close(out, whole, dtype)
    assert [t.data_ptr() for pair in state for t in pair] == places  # in place, as without autocast


@pytest.mark.parametrize("dtype", HALVES)
def test_a_prompt_then_tokens(gpu, dtype):
    """A block from its initial state over a prompt under autocast, a second part from what that returned, then tokens."""
    _say(f"selective autocast prompt {dtype}")
    torch.manual_seed(5)
    block = SelectiveScanBlock(32).cuda().eval()
    x = torch.randn(3, 30, 32, device="cuda")
    with torch.no_grad():
        whole, _ = block(x)
        with torch.autocast("cuda", dtype=dtype):
            y, state = block(x[:, :17], block.initial_state(3))
            assert state[0].dtype == dtype and state[1].dtype == torch.float32
            ys = [y]
            y, state = block(x[:, 17:20], state)
            ys.append(y)
            for t in range(20, 30):
                ys.append(block.step(x[:, t], state).unsqueeze(1))
    _close(torch.cat(ys, 1), whole, dtype)


@pytest.mark.parametrize("dtype", HALVES)
def test_a_state_that_leaves_and_enters_autocast(gpu, dtype):
    """float32 states hold what a step under autocast puts in, and a sequence takes a state of either type; tokens in 32 bits
    into a 16-bit state would lose bits of it unseen, and are refused."""
    _say(f"selective autocast mixed {dtype}")
    torch.manual_seed(6)
    block = SelectiveScanBlock(32).cuda().eval()
    x = torch.randn(2, 24, 32, device="cuda")
    with torch.no_grad():
        whole, _ = block(x)
        y, state = block(x[:, :8])
        ys = [y]
        with torch.autocast("cuda", dtype=dtype):
            for t in range(8, 12):
                ys.append(block.step(x[:, t], state).unsqueeze(1))
            y, low = block(x[:, 12:16], state)
            ys.append(y)
        with pytest.raises(ValueError, match="state must be"):
            block.step(x[:, 16], low)
        y, state = block(x[:, 16:20], low)
        assert state[0].dtype == torch.float32
        ys.append(y)
        for t in range(20, 24):
            ys.append(block.step(x[:, t], state).unsqueeze(1))
    _close(torch.cat(ys, 1), whole, dtype)


def test_a_captured_step(gpu):
    _say("selective autocast graph")
    m, x = _model()
    eager, state = m.initial_state(5), m.initial_state(5)
    token = x[:, 0].clone()
    with torch.autocast("cuda", dtype=torch.float16, cache_enabled=False):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(token, m.initial_state(5))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.step(token, state)
        for t in range(4):
            token.copy_(x[:, t])
            want = m.step(token, eager)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), f"replay {t}"
            assert all(torch.equal(a, b) for p, q in zip(state, eager) for a, b in zip(p, q))


def test_gradients_through_a_given_state(gpu):
    _say("selective autocast state gradient")
    torch.manual_seed(7)
    block = SelectiveScanBlock(16).cuda().eval()
    x = torch.randn(2, 9, 16, device="cuda")
    conv, h = (t.normal_().requires_grad_(True) for t in block.initial_state(2))
    want = torch.autograd.grad(block(x, (conv, h))[0].sum(), (conv, h))
    with torch.autocast("cuda", dtype=torch.float16):
        got = torch.autograd.grad(block(x, (conv, h))[0].float().sum(), (conv, h))
    for a, b in zip(got, want):
        assert a.dtype == torch.float32
        _close(a, b, torch.float16)


@pytest.mark.parametrize("dtype,other", [(torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
def test_a_model_of_the_other_16_bit_type(gpu, dtype, other):
    _say(f"selective autocast {dtype} in {other}")
    torch.manual_seed(8)
    block = SelectiveScanBlock(32).cuda().eval()
    x = torch.randn(2, 12, 32, device="cuda")
    with torch.no_grad():
        whole, _ = block(x)
        block, x = block.to(dtype), x.to(dtype)
        with torch.autocast("cuda", dtype=other):
            state = block.initial_state(2)
            assert state[0].dtype == other
            y, handed = block(x[:, :8])
            ys = [y]
            for t in range(8, 12):
                ys.append(block.step(x[:, t], handed).unsqueeze(1).to(dtype))
            _close(torch.cat(ys, 1), whole, torch.bfloat16)
            for t in range(12):
                out = block.step(x[:, t], state)
            _close(out, whole[:, -1], torch.bfloat16)
