"""Infinite states and gradients of the gated linear recurrence: every step's factor is positive, so that they stay what
they are however many steps a map is composed of."""
from __future__ import annotations

import pytest
import torch

import ops_plain as plain
import persistent_lstm_hip_amd as P

pytestmark = pytest.mark.gpu

INF = float("inf")


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _gates(B, T, H, dtype, seed=0):
    """Forget gates from -9 to 6: products of a few factors underflow in the first channels, of many in none of the last."""
    z = _rand(B, T, 3 * H, seed=seed)
    z[..., :H] += torch.linspace(-9.0, 6.0, H)
    return z.to(dtype)


def _same_infinities(got, want, what):
    """NaN where the formulas give one, infinities of the same sign, and finite elsewhere."""
    got = got.detach().cpu().double()
    for name, f in (("NaN", torch.isnan), ("+inf", torch.isposinf), ("-inf", torch.isneginf)):
        a, b = f(got), f(want)
        assert torch.equal(a, b), f"{what}: {name} at {a.sum().item()} places, expected at {b.sum().item()}"


# (B, T, H): a few steps; one tile of each size; several tiles; split; slabs of either width; one channel per thread
SHAPES = [(2, 5, 24), (2, 9, 24), (2, 30, 24), (2, 64, 24), (2, 65, 24), (2, 700, 24), (2, 3000, 40), (45, 200, 264),
          (33, 130, 1000), (2, 300, 3)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H", SHAPES)
def test_infinite_states(gpu, B, T, H, dtype):
    _say(f"infinite states {B} {T} {H} {dtype}")
    z, c0 = _gates(B, T, H, dtype), _rand(B, H, seed=1)
    c0[0, ::3] = INF
    c0[1, ::4] = -INF
    z[1, T // 3, H + 1::5] = INF  # a candidate (in some channels onto -inf: NaN from there on)
    z[0, T - 2, H + 2::5] = -INF
    out, c_n = P.gated_scan(z.cuda(), c0.cuda())
    want, want_c = plain.scan(z, c0, None, True)
    _same_infinities(out, want, "out")
    _same_infinities(c_n, want_c, "c_n")
    n = torch.full((B,), T)
    n[0], n[1] = (T + 1) // 2, T - 1
    out, c_n = P.gated_scan(z.cuda(), c0.cuda(), lengths=n)
    want, want_c = plain.scan(z, c0, n, True)
    _same_infinities(out, want, "ragged out")
    _same_infinities(c_n, want_c, "ragged c_n")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H", SHAPES)
def test_infinite_gradients(gpu, B, T, H, dtype):
    _say(f"infinite gradients {B} {T} {H} {dtype}")
    z, c0 = _gates(B, T, H, dtype), _rand(B, H, seed=1)
    dh, dc = _rand(B, T, H, seed=5).to(dtype), _rand(B, H, seed=6)
    dc[0, ::3] = INF
    dc[1, ::4] = -INF
    dh[1, T // 2, 1::5] = INF
    zd, cd = z.cuda().requires_grad_(True), c0.cuda().requires_grad_(True)
    got = torch.autograd.grad(P.gated_scan(zd, cd), (zd, cd), (dh.cuda(), dc.cuda()))
    _, _, dz, d0, _ = plain.scan(z, c0, None, True, dh, dc)
    big = torch.finfo(dtype).max
    assert dz[dz.isfinite()].abs().max() < big
    _same_infinities(got[0], dz, "d_gates")
    _same_infinities(got[1], d0, "d_c0")
