"""Which dropout masks the block and the forecaster draw: their offsets, with the operators' formulas in torch on the CPU."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import ops_plain as plain
from persistent_lstm_hip_amd import GatedScanBlock, GatedScanRegressor, gated


def _scan(gates, c0=None, *, lengths=None):
    f, g, o = gates.chunk(3, -1)
    a = torch.sigmoid(f)
    c, hs = torch.zeros_like(f[:, 0]) if c0 is None else c0, []
    for t in range(gates.shape[1]):
        c = a[:, t] * c + (1 - a[:, t]) * g[:, t]
        hs.append(torch.sigmoid(o[:, t]) * c)
    return torch.stack(hs, 1), c


@pytest.fixture
def masks(monkeypatch):
    """The (seed, offset) of every mask with anything dropped, in the order of the calls."""
    seen = []

    def dropout_add(x, residual, *, p, seed, offset):
        offset = int(offset)
        k = int(p * 65536 + 0.5)
        if k:
            seen.append((seed, offset))
        keep = plain.keep(0, x.numel(), k, seed, offset).view(x.shape)
        return residual + torch.where(keep, x * (65536 / (65536 - k)), torch.zeros(()))

    monkeypatch.setattr(gated, "dropout_add", dropout_add)
    monkeypatch.setattr(gated, "gated_scan", _scan)
    monkeypatch.setattr(gated, "layer_norm", lambda x, w, b: torch.nn.functional.layer_norm(x, w.shape, w, b))
    return seen


def _block(p):
    torch.manual_seed(1)
    return GatedScanBlock(8, p)


def test_a_block_called_without_an_offset_draws_a_mask_of_its_own(masks):
    block, other, x = _block(0.5), _block(0.5), torch.randn(2, 6, 8)
    a, b = block(x)[0], block(x)[0]
    other(x)
    assert len(set(masks)) == 3 and not torch.equal(a, b)
    # the same state of torch's generator, the same mask: as torch's own dropout
    torch.manual_seed(5)
    a = block(x)[0]
    torch.manual_seed(5)
    assert torch.equal(block(x)[0], a)


def test_a_block_takes_the_offset_that_it_is_given(masks):
    block, x = _block(0.5), torch.randn(2, 6, 8)
    state = torch.get_rng_state()
    block(x, seed=3, offset=0)
    block(x, seed=3, offset=7)
    assert masks == [(3, 0), (3, 7)]
    assert torch.equal(torch.get_rng_state(), state)


def test_a_block_without_dropout_leaves_torchs_generator_alone(masks):
    x, state = torch.randn(2, 6, 8), None
    for block in (_block(0.0), _block(0.5).eval()):
        state = torch.get_rng_state()
        block(x)
        assert torch.equal(torch.get_rng_state(), state)
    assert masks == []


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_block_recomputes_its_own_mask(masks, reentrant):
    block, x = _block(0.5), torch.randn(2, 6, 8, requires_grad=True)
    y, _ = checkpoint(block, x, use_reentrant=reentrant)
    block(x)  # (another pass before the recomputation)
    got = torch.autograd.grad(y.square().sum(), x) if not reentrant else None
    if reentrant:
        y.square().sum().backward()
        got = (x.grad,)
    first = masks[0]
    assert masks[2] == first != masks[1]
    want = torch.autograd.grad(block(x, offset=first[1])[0].square().sum(), x)
    assert torch.allclose(got[0], want[0])


def _model(p=0.5, layers=2):
    torch.manual_seed(1)
    return GatedScanRegressor(3, 8, 2, layers, p)


def test_the_forecasters_passes_are_numbered(masks):
    m, x = _model(), torch.randn(2, 6, 3)
    m(x), m(x)
    assert masks == [(m.seed, i) for i in range(4)]
    m.eval()
    m(x)
    assert len(masks) == 4
    m.train()
    m(x)
    assert masks[4:] == [(m.seed, 4), (m.seed, 5)]


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_forecaster_recomputes_its_own_masks(masks, reentrant):
    """Two passes are outstanding when the first is recomputed; their gradients are those without checkpointing."""
    m = _model()
    xs = [torch.randn(2, 6, 3, requires_grad=True) for _ in range(2)]
    ys = [checkpoint(m, x, use_reentrant=reentrant) for x in xs]
    for p in m.parameters():
        p.grad = None
    sum(y.square().sum() for y in ys).backward()
    assert sorted(masks[:4]) == sorted(masks[4:]) == [(m.seed, i) for i in range(4)]
    got = [p.grad.clone() for p in m.parameters()]
    fresh = _model()
    sum(fresh(x).square().sum() for x in xs).backward()
    for a, b in zip(got, fresh.parameters()):
        assert torch.allclose(a, b.grad, atol=1e-6)
    del masks[:]
    m(xs[0])
    assert masks == [(m.seed, 4), (m.seed, 5)]  # (the recomputations are no passes of their own)


def test_a_forecaster_without_dropout_leaves_torchs_generator_alone(masks):
    m, x = _model(0.0), torch.randn(2, 6, 3)
    state = torch.get_rng_state()
    m(x)
    assert torch.equal(torch.get_rng_state(), state) and masks == []


def test_what_a_forecaster_remembers_is_bounded(masks, monkeypatch):
    monkeypatch.setattr(GatedScanRegressor, "_REMEMBERED", 3)
    m, x = _model(layers=1), torch.randn(2, 2, 3)
    for _ in range(7):
        m(x)
    assert len(m._numbers) == 3 and masks == [(m.seed, i) for i in range(7)]


@pytest.mark.parametrize("kind", [int, lambda v: torch.tensor([v]), torch.tensor])
def test_a_forecaster_takes_the_pass_number_that_it_is_given(masks, kind):
    m, x = _model(), torch.randn(2, 6, 3)
    state = torch.get_rng_state()
    a = m(x, None, kind(7))
    assert masks == [(m.seed, 14), (m.seed, 15)]
    assert torch.equal(torch.get_rng_state(), state) and m._passes == 0
    assert torch.equal(m(x, offset=7), a)
    y = checkpoint(m, x.requires_grad_(True), None, kind(7), use_reentrant=False)
    y.sum().backward()
    assert masks[4:] == [(m.seed, 14), (m.seed, 15)] * 2


def test_pass_numbers_that_are_refused(masks):
    m, x = _model(), torch.randn(2, 6, 3)
    for bad in (torch.tensor([1, 2]), torch.tensor([1.0]), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError, match="one int64"):
            m(x, offset=bad)
