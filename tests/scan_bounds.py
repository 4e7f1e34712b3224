"""The gated linear recurrence in 64 bits with a bound for every element of its results, for the tests.

U = 2^-24.  A logistic function of z and its complement come from 2^(-z log2 e), whose exponent is one rounded product: they
are within (8 + 1.5 |z|) U of their values, relative.  A state is a sum of terms, each a candidate times the factors of the
steps since.  A term passes, per step, one factor's error and the roundings of one product and one addition, and a share
of those that compose the maps of a tile (at most 16 for 64 steps): together (rho + 3 U) of the term.  Once per call it
passes the maps of the segments and of the tile it ends in, and the backward pass starts again from a saved state: 64 U.
So the error follows the recurrence itself, with the terms' magnitudes in the place of the terms, and is forgotten as
fast as they are.  The gradient that runs backwards likewise.  Steps past a row's length have a = 1, 1 - a = 0 and are exact.
"""
from __future__ import annotations

import torch

import ops_plain as plain
from ops_plain import U, d64

STEP, ONCE = 3 * U, 64 * U


def _rho(z):
    return (8 + 1.5 * z.abs()) * U


def scan(gates, c0, lengths, output_gate, d_out, d_cn):
    """name -> (value, bound) for out, c_n, d_gates and d_c0; without the roundings to the results' types."""
    z = d64(gates)
    B, T, width = z.shape
    H = width // (3 if output_gate else 2)
    n = torch.full((B,), T) if lengths is None else torch.as_tensor(lengths).cpu().long().clamp(0, T)
    live = (torch.arange(T).unsqueeze(0) < n.unsqueeze(1)).unsqueeze(2)
    none = torch.zeros((), dtype=torch.float64)
    z, dh = torch.where(live, z, none), torch.where(live, d64(d_out), none)
    f, g = z[..., :H], z[..., H:2 * H]
    a, na, rho = torch.sigmoid(f), torch.sigmoid(-f), _rho(f)
    if output_gate:
        o = z[..., 2 * H:]
        s, ns, rho_o = torch.sigmoid(o), torch.sigmoid(-o), _rho(o)
    else:
        s, ns, rho_o = torch.ones_like(a), torch.zeros_like(a), torch.zeros_like(a)
    c = torch.zeros(B, H, dtype=torch.float64) if c0 is None else d64(c0)
    size, err = c.abs(), torch.zeros_like(c)  # the terms' magnitudes, the running error
    track = [torch.zeros(B, T, H, dtype=torch.float64) for _ in range(6)]
    for t in range(T):
        track[0][:, t], track[1][:, t], track[2][:, t] = c, size, err
        on = live[:, t]
        c = torch.where(on, a[:, t] * c + na[:, t] * g[:, t], c)
        most = a[:, t] * size + na[:, t] * g[:, t].abs()
        err = torch.where(on, a[:, t] * err + (rho[:, t] + STEP) * most, err)
        size = torch.where(on, most, size)
        track[3][:, t], track[4][:, t], track[5][:, t] = c, size, err
    before, size0, err0, after, size1, err1 = track
    bound1 = err1 + ONCE * size1
    out = torch.where(live, s * after, none)
    out_bound = torch.where(live, s * bound1 + (rho_o + 2 * U) * s * (after.abs() + bound1), none)
    result = {"out": (out, out_bound), "c_n": (c, err + ONCE * size)}

    u = s * dh
    e = torch.zeros(B, H, dtype=torch.float64) if d_cn is None else d64(d_cn)
    size, err = e.abs(), torch.zeros_like(e)
    dz, bz = torch.zeros_like(z), torch.zeros_like(z)
    for t in reversed(range(T)):
        on, at, nt, r = live[:, t], a[:, t], na[:, t], rho[:, t]
        D, most = u[:, t] + e, u[:, t].abs() + size
        err_D = err + (rho_o[:, t] + 2 * U) * u[:, t].abs()
        bound_D = err_D + ONCE * most
        dg = nt * D
        q = before[:, t] - g[:, t]
        bound_q = err0[:, t] + 2 * ONCE * size0[:, t] + U * q.abs()
        dz[:, t, :H] = torch.where(on, at * dg * q, none)
        bz[:, t, :H] = torch.where(on, at * nt * (q.abs() * bound_D + (D.abs() + bound_D) * bound_q)
                                   + (2 * r + 4 * U) * (at * dg * q).abs(), none)
        dz[:, t, H:2 * H] = torch.where(on, dg, none)
        bz[:, t, H:2 * H] = torch.where(on, nt * bound_D + (r + 2 * U) * dg.abs(), none)
        e = torch.where(on, at * D, e)
        err = torch.where(on, at * err_D + (r + STEP) * at * most, err)
        size = torch.where(on, at * most, size)
    if output_gate:
        w = (s * ns * dh).abs()
        dz[..., 2 * H:] = s * ns * dh * after
        bz[..., 2 * H:] = w * (bound1 + ONCE * size1) + (2 * rho_o + 4 * U) * w * after.abs()
    result["d_gates"], result["d_c0"] = (dz, bz), (e, err + ONCE * size)
    return result


def check(got, want, dtype, what=""):
    """got: (out, c_n, d_gates, d_c0) of a call (d_c0 may be None); want: of scan()."""
    for (name, (value, bound)), x in zip(want.items(), got):
        if x is not None:
            plain.assert_within(x, value, bound, torch.float32 if name in ("c_n", "d_c0") else dtype, f"{what} {name}")
