"""The selective scan with step sizes below zero, whose states grow: they follow the formulas as long as fp32 holds the states,
over runs, tiles and segments of steps, and a state of zero stays zero however fast it would grow."""
from __future__ import annotations

import pytest
import torch

import ops_plain
import persistent_lstm_hip_amd as P
import selective_plain as plain

pytestmark = pytest.mark.gpu

F32 = torch.float32
LEAVES = ("u", "dt", "A", "B", "C", "D", "z", "h0", "dt_bias")


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _check(d, d_out=None, d_hn=None, lengths=None):
    want = plain.scan(*(d[n] for n in LEAVES), softplus=False, lengths=lengths, d_out=d_out, d_hn=d_hn)
    dev = {n: None if t is None else t.cuda().requires_grad_(True) for n, t in d.items()}
    out, h_n = P.selective_scan(*(dev[n] for n in LEAVES[:-1]), dt_bias=dev["dt_bias"], softplus=False, lengths=lengths)
    got = {"out": out, "h_n": h_n}
    if d_out is not None:
        given = [n for n in LEAVES if dev[n] is not None]
        grads = torch.autograd.grad((out, h_n), [dev[n] for n in given], (d_out.cuda(), d_hn.cuda()))
        got.update({"d_" + n: t for n, t in zip(given, grads)})
    # selective_plain bounds d_u and d_A for step sizes that are not negative; here all terms of their sums have one sign,
    # so that their relative errors are those of the states and of E over all steps, and of the sums over states and time
    T = d["u"].shape[1]
    x = (d["dt"].double().abs().sum(1).max() * d["A"].double().abs().max()).item()
    rel = (12 * x + 10 * T + 300) * ops_plain.U
    for name, t in got.items():
        value, bound = want[name]
        if name in ("d_u", "d_A"):
            bound = rel * value.abs()
        assert value.abs().max() < 1e38, f"{name}: the test's own values do not fit fp32"
        ops_plain.assert_within(t, value, bound + plain.TINY, F32, name)


def _inputs(T, D, N, step, seed=0):
    """Every state grows by exp(step) per step."""
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return 0.1 + torch.rand(*shape, generator=g)

    return dict(u=rand(1, T, D), dt=torch.full((1, T, D), -0.5), A=torch.full((D, N), -2.0 * step), B=rand(1, T, N),
                C=rand(1, T, N), D=None, z=None, h0=None, dt_bias=None)


@pytest.mark.parametrize("N", [5, 16, 33])
@pytest.mark.parametrize("T", [200, 900, 2000])
def test_zeros_before_a_growing_state(gpu, T, N):
    """Inputs in a row's last 30 steps alone; then no inputs, and an output's gradient in its first 30 alone: the steps before
    them, or after them, are zero times a factor that fp32 does not hold."""
    _say(f"selective growth zeros T={T} N={N}")
    d = _inputs(T, 6, N, 2.0)
    d["u"][:, :T - 30] = 0.0
    _check(d)
    _check(d, lengths=[T - 7])
    d["u"].zero_()
    d_out = torch.zeros(1, T, 6)
    d_out[:, :30] = 1.0
    _check(d, d_out, torch.zeros(1, 6, N))
    _check(d, d_out, torch.zeros(1, 6, N), lengths=[T - 7])


@pytest.mark.parametrize("N", [5, 16, 33])
@pytest.mark.parametrize("T,step", [(10, 13.0), (20, 6.5), (40, 3.6), (70, 2.0), (1000, 0.15)])
def test_a_small_state_that_grows(gpu, T, step, N):
    """From 2^-100 by more than fp32's largest number, within one run of steps, a tile, a segment."""
    _say(f"selective growth T={T} step={step} N={N}")
    d = _inputs(T, 6, N, step)
    d["u"].zero_()
    d["h0"] = torch.full((1, 6, N), 2.0**-100)
    _check(d, torch.zeros(1, T, 6), torch.full((1, 6, N), 2.0**-100))


@pytest.mark.parametrize("N", [5, 16])
@pytest.mark.parametrize("T,shrink,by", [(128, 64, 20.0), (700, 64, 20.0), (100, 8, 80.0)])
def test_steps_of_both_signs(gpu, T, shrink, by, N):
    """Steps that shrink a state by more than fp32 holds, then steps that would grow it back: nothing of it is left."""
    _say(f"selective growth both signs T={T} shrink={shrink} N={N}")
    d = _inputs(T, 6, N, 1.0)
    d["u"].zero_()
    d["h0"] = torch.ones(1, 6, N)
    d["dt"][:, :shrink] = 0.5 * by
    d["dt"][:, shrink + 64:] = 0.0
    _check(d)  # (64 - shrink by is below -500: zero in 64 bits too, but for less than TINY)
