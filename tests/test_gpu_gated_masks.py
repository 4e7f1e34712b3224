"""The forecaster's dropout masks on the GPU where a pass runs more than once: activation checkpointing,
captured graphs."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from persistent_lstm_hip_amd import GatedScanBlock, GatedScanRegressor, gated

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


def test_every_replay_of_a_captured_step_draws_masks_of_its_own(gpu):
    """Forward pass and gradient in one graph whose pass number is on the device, replayed with eager work in between,
    each replay against the eager pass of that number."""
    _say("captured step")
    m = _model()
    x = torch.randn(4, 70, 2, device="cuda", requires_grad=True)
    d = torch.randn(4, 3, device="cuda")
    number = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step(offset):
        y = m(x, None, offset)
        return y.detach(), torch.autograd.grad(y, x, d)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(number)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(number)
        number.add_(1)
    number.fill_(5)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(4, 70, 2, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        assert int(number) == 6 + i
        want = step(5 + i)
        for a, b in zip(got, want):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-5), f"replay {i}"
        if i:
            assert not torch.allclose(got[0], step(4 + i)[0], rtol=1e-3, atol=1e-3), f"replay {i} has the mask before"


@pytest.mark.parametrize("kind", ["model", "block"])
def test_replays_draw_masks_by_themselves(gpu, kind, monkeypatch):
    """Without an offset: what every replay drew on the device, given to an eager pass, gives the replay's results."""
    _say(f"captured {kind} without offset")
    if kind == "model":
        m, x, pick = _model(), torch.randn(4, 70, 2, device="cuda", requires_grad=True), (lambda y: y)
    else:
        torch.manual_seed(11)
        m, x, pick = GatedScanBlock(8, 0.5).cuda(), torch.randn(4, 70, 8, device="cuda", requires_grad=True), (lambda y: y[0])
    drawn, draw = [], gated._draw
    monkeypatch.setattr(gated, "_draw", lambda device: drawn.append(draw(device)) or drawn[-1])

    def step(**offset):
        y = pick(m(x, **offset))
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(), step(offset=torch.zeros(1, dtype=torch.int64, device="cuda"))
    torch.cuda.current_stream().wait_stream(s)
    assert isinstance(drawn.pop(), int)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    numbers = set()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        numbers.add(int(drawn[0]))
        for given in (drawn[0], int(drawn[0])):
            for a, b in zip(got, step(offset=given)):
                assert torch.allclose(a, b, rtol=1e-5, atol=1e-5), f"replay {i}"
    assert len(numbers) == 4 and len(drawn) == 1


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_pass_in_a_captured_step(gpu, reentrant, monkeypatch):
    """The recomputation draws the pass' own number in every replay."""
    _say(f"captured checkpoint reentrant={reentrant}")
    m, x = _model(), torch.randn(4, 70, 2, device="cuda", requires_grad=True)
    drawn, draw = [], gated._draw
    monkeypatch.setattr(gated, "_draw", lambda device: drawn.append(draw(device)) or drawn[-1])

    def step():
        y = checkpoint(m, x, use_reentrant=reentrant)
        y.sum().backward()
        return y

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    del drawn[:]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    seen = set()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        first, again = (int(v) for v in drawn)
        assert first == again
        seen.add(first)
        m(x, offset=0)
    assert len(seen) == 3
