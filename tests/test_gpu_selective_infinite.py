"""Infinite inputs, step sizes and gradients of the selective scan, at every number of states: what they reach is infinite or
NaN where the formulas say so, whether or not the states fill the lanes that hold them."""
from __future__ import annotations

import pytest
import torch

import persistent_lstm_hip_amd as P
import selective_plain as plain

pytestmark = pytest.mark.gpu

INF = float("inf")
LEAVES = ("u", "dt", "A", "B", "C", "D", "z", "h0", "dt_bias")


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _inputs(B, T, D, N, gate):
    """Everything positive but A, so that infinities of both signs meet nowhere but where a test puts them."""
    g = torch.Generator().manual_seed(N)

    def rand(*shape):
        return 0.1 + torch.rand(*shape, generator=g)

    return dict(u=rand(B, T, D), dt=rand(B, T, D) - 2.0, A=-rand(D, N), B=rand(B, T, N), C=rand(B, T, N), D=rand(D),
                z=rand(B, T, D) if gate else None, h0=rand(B, D, N), dt_bias=rand(D))


def _compare(got, want, bound, what):
    """NaN and infinities as the formulas have them, and every finite value within its bound."""
    got = got.detach().cpu().double()
    for name, f in (("NaN", torch.isnan), ("+inf", torch.isposinf), ("-inf", torch.isneginf)):
        a, b = f(got), f(want)
        assert torch.equal(a, b), f"{what}: {name} at {a.sum().item()} places, expected at {b.sum().item()}"
    sure = torch.isfinite(want) & torch.isfinite(bound)
    over = (got - want).abs() - (bound + plain.TINY + 2.0**-24 * want.abs())
    assert not sure.any() or over[sure].max() <= 0, f"{what}: {over[sure].max():.3g} beyond its bound"


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 8, 10, 15, 16, 17, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("gate", [True, False])
def test_infinite_values(gpu, N, gate):
    """One in u, in dt, in the output's gradient and, for all channels, in B and C in turn; one tile and several, the first
    and a later wave's steps, channels that fill no group."""
    for T, at in ((7, 2), (70, 0), (70, 20), (70, 37)):
        for name in ("u", "dt", "d_out", "B", "C"):
            _say(f"selective infinite N={N} gate={gate} T={T} {name}[{at}]")
            d = _inputs(2, T, 11, N, gate)
            d_out = 0.1 + torch.rand(2, T, 11, generator=torch.Generator().manual_seed(5))
            (d_out if name == "d_out" else d[name])[0, at, 0 if name in "BC" else 5] = INF
            want = plain.scan(*(d[n] for n in LEAVES), d_out=d_out)
            dev = {n: None if t is None else t.cuda().requires_grad_(True) for n, t in d.items()}
            out, h_n = P.selective_scan(*(dev[n] for n in LEAVES[:-1]), dt_bias=dev["dt_bias"])
            _compare(out, *want["out"], "out")
            _compare(h_n, *want["h_n"], "h_n")
            given = [n for n in LEAVES if dev[n] is not None]
            for n, t in zip(given, torch.autograd.grad(out, [dev[n] for n in given], d_out.cuda())):
                _compare(t, *want["d_" + n], "d_" + n)


@pytest.mark.parametrize("N", [3, 10, 16, 20, 33])
def test_infinite_values_in_segments(gpu, N):
    """A long row of few channels, whose time axis is split."""
    for name in ("u", "d_out"):
        _say(f"selective infinite segments N={N} {name}")
        d = _inputs(1, 900, 6, N, True)
        d_out = 0.1 + torch.rand(1, 900, 6, generator=torch.Generator().manual_seed(5))
        (d_out if name == "d_out" else d[name])[0, 450, 4] = INF
        want = plain.scan(*(d[n] for n in LEAVES), d_out=d_out)
        dev = {n: t.cuda().requires_grad_(True) for n, t in d.items()}
        out, h_n = P.selective_scan(*(dev[n] for n in LEAVES[:-1]), dt_bias=dev["dt_bias"])
        _compare(out, *want["out"], "out")
        _compare(h_n, *want["h_n"], "h_n")
        for n, t in zip(LEAVES, torch.autograd.grad(out, [dev[n] for n in LEAVES], d_out.cuda())):
            _compare(t, *want["d_" + n], "d_" + n)


@pytest.mark.parametrize("N", [1, 3, 5, 16, 33])
def test_a_step_of_infinite_values(gpu, N):
    for name in ("u", "dt"):
        _say(f"selective infinite step N={N} {name}")
        d = _inputs(2, 1, 12, N, True)
        d[name][0, 0, 5] = INF
        want = plain.scan(*(d[n] for n in LEAVES))
        one = {n: t[:, 0].cuda() if n in ("u", "dt", "B", "C", "z") else t.cuda() for n, t in d.items()}
        out, h = P.selective_scan_step(one["u"], one["dt"], one["A"], one["B"], one["C"], one["h0"], one["D"], one["z"],
                                       dt_bias=one["dt_bias"])
        _compare(out, want["out"][0][:, 0], want["out"][1][:, 0], "out")
        _compare(h, *want["h_n"], "h")
