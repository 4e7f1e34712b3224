"""The causal convolution, the selective scan and the gradient norm from their formulas in 64 bits on the CPU, with a bound
for every element of their results, for the tests.

U = 2^-24.  Roundings to the results' types are not in the bounds (ops_plain.assert_within adds them).

sigmoid(v) is within 8 U absolutely and (8 + 1.5 |v|) U relatively; silu(v) = v sigmoid(v) one rounding more; its slope
s (1 + v (1 - s)) within (16 + 12 |v|) U, since 1 - s is within 9 U.

softplus(v) = max(v, 0) + log1p(exp(-|v|)), v = raw + bias rounded once: that moves it by |v| U sigmoid(v) <= |v| U
softplus(v).  The exponential is within (2 |v| + 3) U, the quotient and the series add 6 U, the sum one: relatively
(3 |v| + 12) U.

A decay exp(s A) is 2^x' with x' = s (A log2 e): two roundings and the constant's, and the exponential's own 2 U, so with
x = s A and rho the step size's error it is within |x| (rho + 3 U) + 3 U.  A state is a sum of terms that pass, per step, one
decay and one fused product and sum; once per eight steps the decay of a run, whose exponent is a sum of eight rounded
terms (8 |x| U per step, with the exponential's 3 U shared by its steps), and per tile at most eight folds of two
roundings over 32 steps.  Together |x| (rho + 11 U) + 9 U of the term, per step.  Once per call it passes the segments'
maps and starts again from a saved state: 64 U.  The gradient that runs backwards likewise.

Below 2^-126 errors are absolute: a decay that small is flushed to zero, a run's held at 2^-126, and a product is a multiple of
2^-149.  Each moves a term by up to 2^-126 of what it multiplies, at most three times per step; with fewer than 2^12 steps
and factors below 2^12 that is less than TINY = 2^-100.
"""
from __future__ import annotations

import torch

from ops_plain import U, d64

STEP, ONCE, SUM = 9 * U, 64 * U, 24 * U
TINY = 2.0**-100


def _none():
    return torch.zeros((), dtype=torch.float64)


def live_rows(B, T, lengths):
    n = torch.full((B,), T) if lengths is None else torch.as_tensor(lengths).cpu().long().clamp(0, T)
    return n, torch.arange(T).unsqueeze(0) < n.unsqueeze(1)


def silu(v):
    return v * torch.sigmoid(v)


def slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * torch.sigmoid(-v))


# ---- causal convolution ---------------------------------------------------------------------------


def conv(x, weight, bias, state, lengths, activation, d_y=None, d_state_n=None):
    """name -> (value, bound): y, state_n and with d_y d_x, d_weight, d_bias, d_state."""
    x, w = d64(x), d64(weight)
    B, T, C = x.shape
    W = w.shape[1]
    n, live = live_rows(B, T, lengths)
    live = live.unsqueeze(2)
    x = torch.where(live, x, _none())
    st = torch.zeros(B, W - 1, C, dtype=torch.float64) if state is None else d64(state)
    b = torch.zeros(C, dtype=torch.float64) if bias is None else d64(bias)
    line = torch.cat([st, x], 1)
    acc = b.expand(B, T, C).clone()
    size = b.abs().expand(B, T, C).clone()
    for k in range(W):
        acc += w[:, k] * line[:, k:k + T]
        size += (w[:, k] * line[:, k:k + T]).abs()
    err = (W + 2) * U * size
    y, y_err = (silu(acc), 1.1 * err + (10 + 1.5 * acc.abs()) * U * silu(acc).abs()) if activation else (acc, err)
    at = n.unsqueeze(1) + torch.arange(W - 1)
    rows = torch.arange(B).unsqueeze(1)
    out = {"y": (torch.where(live, y, _none()), torch.where(live, y_err, _none())),
           "state_n": (line[rows, at], torch.zeros(B, W - 1, C, dtype=torch.float64))}
    if d_y is None:
        return out
    dy = torch.where(live, d64(d_y), _none())
    da = dy * slope(acc) if activation else dy
    da_err = dy.abs() * (0.5 * err + (18 + 12 * acc.abs()) * U) if activation else torch.zeros_like(dy)
    d_line, d_err = torch.zeros_like(line), torch.zeros_like(line)
    dw, dw_err = torch.zeros_like(w), torch.zeros_like(w)
    for k in range(W):
        d_line[:, k:k + T] += w[:, k] * da
        d_err[:, k:k + T] += w[:, k].abs() * (da_err + (W + 3) * U * da.abs())
        part = line[:, k:k + T]
        dw[:, k] = (da * part).sum((0, 1))
        dw_err[:, k] = (da_err * part.abs() + 192 * U * (da * part).abs()).sum((0, 1))
    if d_state_n is not None:
        d_line[rows, at] += d64(d_state_n)
        d_err[rows, at] += (W + 3) * U * d64(d_state_n).abs()
    out["d_x"] = (torch.where(live, d_line[:, W - 1:], _none()), torch.where(live, d_err[:, W - 1:], _none()))
    out["d_weight"] = (dw, dw_err)
    out["d_bias"] = (da.sum((0, 1)), (da_err + 192 * U * da.abs()).sum((0, 1)))
    out["d_state"] = (d_line[:, :W - 1], d_err[:, :W - 1])
    return out


# ---- selective scan -------------------------------------------------------------------------------


def scan(u, dt, A, B, C, D=None, z=None, h0=None, dt_bias=None, softplus=True, lengths=None, d_out=None, d_hn=None):
    """name -> (value, bound): out, h_n and with d_out d_u, d_dt, d_A, d_B, d_C, d_D, d_z, d_h0, d_dt_bias."""
    u, A = d64(u), d64(A)
    rows, T, channels = u.shape
    N = A.shape[1]
    _, live = live_rows(rows, T, lengths)
    live = live.unsqueeze(2)
    u, raw, Bm, Cm = (torch.where(live, d64(t), _none()) for t in (u, dt, B, C))
    skip = torch.zeros(channels, dtype=torch.float64) if D is None else d64(D)
    v = raw + (0.0 if dt_bias is None else d64(dt_bias))
    if softplus:
        s, rho = torch.logaddexp(v, _none()), (3 * v.abs() + 12) * U
    else:
        s, rho = v, torch.full_like(v, U)
    s = torch.where(live, s, _none())
    x = s.unsqueeze(3) * A
    a, rho_a = torch.exp(x), x.abs() * (rho.unsqueeze(3) + 11 * U) + STEP
    b = (s * u).unsqueeze(3) * Bm.unsqueeze(2)
    h = torch.zeros(rows, channels, N, dtype=torch.float64) if h0 is None else d64(h0)
    size, err = h.abs(), torch.zeros_like(h)
    shape = (rows, T, channels, N)
    before, size0, err0 = (torch.zeros(shape, dtype=torch.float64) for _ in range(3))
    after, size1, err1 = (torch.zeros(shape, dtype=torch.float64) for _ in range(3))
    for t in range(T):
        before[:, t], size0[:, t], err0[:, t] = h, size, err
        on = live[:, t].unsqueeze(2)
        new = torch.where(on, a[:, t] * h + b[:, t], h)
        most = a[:, t] * size + b[:, t].abs()
        err = torch.where(on, a[:, t] * err + rho_a[:, t] * a[:, t] * size
                          + (rho[:, t].unsqueeze(2) + 4 * U) * b[:, t].abs() + U * most, err)
        h, size = new, torch.where(on, most, size)
        after[:, t], size1[:, t], err1[:, t] = h, size, err
    bound0, bound1 = err0 + ONCE * size0, err1 + ONCE * size1
    Ce = Cm.unsqueeze(2)
    y = (after * Ce).sum(3) + skip * u
    y_size = (size1 * Ce.abs()).sum(3) + (skip * u).abs()
    y_err = (bound1 * Ce.abs()).sum(3) + SUM * y_size
    if z is None:
        gate, gate_rho, out, out_err = torch.ones_like(u), torch.zeros_like(u), y, y_err
    else:
        z = torch.where(live, d64(z), _none())
        gate, gate_rho = silu(z), (10 + 1.5 * z.abs()) * U
        out = y * gate
        out_err = gate.abs() * (y_err + (gate_rho + U) * (y.abs() + y_err))
    result = {"out": (torch.where(live, out, _none()), torch.where(live, out_err, _none())),
              "h_n": (h, err + ONCE * size)}
    if d_out is None:
        return result

    do = torch.where(live, d64(d_out), _none())
    dy, dy_rho = do * gate, gate_rho + U
    e = torch.zeros(rows, channels, N, dtype=torch.float64) if d_hn is None else d64(d_hn)
    size, err = e.abs(), torch.zeros_like(e)
    G, G_err, E, E_err = (torch.zeros(shape, dtype=torch.float64) for _ in range(4))
    for t in reversed(range(T)):
        on = live[:, t].unsqueeze(2)
        term = dy[:, t].unsqueeze(2) * Ce[:, t]
        g, most = term + e, term.abs() + size
        g_err = err + (dy_rho[:, t].unsqueeze(2) + 2 * U) * term.abs() + U * most
        G[:, t], G_err[:, t] = torch.where(on, g, _none()), torch.where(on, g_err + ONCE * most, _none())
        e = torch.where(on, a[:, t] * g, e)
        err = torch.where(on, a[:, t] * g_err + rho_a[:, t] * a[:, t] * most, err)
        size = torch.where(on, a[:, t] * most, size)
        E[:, t], E_err[:, t] = torch.where(on, e, _none()), torch.where(on, err + ONCE * size, _none())
    Be, se, ue, rhoe = Bm.unsqueeze(2), s.unsqueeze(3), u.unsqueeze(3), rho.unsqueeze(3)
    s1 = (G * Be).sum(3)
    s1_err = ((G_err + SUM * G.abs()) * Be.abs()).sum(3)
    m = E * before
    m_err = E_err * (before.abs() + bound0) + E.abs() * bound0 + U * m.abs()
    s2 = (m * A).sum(3)
    s2_err = ((m_err + (SUM + 4 * U) * m.abs()) * A.abs()).sum(3)
    du = s * s1 + dy * skip
    du_err = s * s1_err + (rho + 2 * U) * (s * s1).abs() + (dy_rho + 2 * U) * (dy * skip).abs()
    inner = u * s1 + s2
    inner_err = u.abs() * s1_err + s2_err + 3 * U * ((u * s1).abs() + s2.abs())
    sg, sg_rho = (torch.sigmoid(v), (10 + 2.5 * v.abs()) * U) if softplus else (torch.ones_like(v), torch.zeros_like(v))
    dr = torch.where(live, inner * sg, _none())
    dr_err = torch.where(live, sg * (inner_err + (sg_rho + U) * (inner.abs() + inner_err)), _none())
    chain = (T / 4 + rows / 32 + 72) * U
    result["d_u"], result["d_dt"] = (torch.where(live, du, _none()), torch.where(live, du_err, _none())), (dr, dr_err)
    ms = m * se
    result["d_A"] = (ms.sum((0, 1)), (m_err * se + (rhoe + chain) * ms.abs()).sum((0, 1)))
    gb, hc = G * se * ue, after * dy.unsqueeze(3)
    wide = (channels / 32 + 40) * U
    result["d_B"] = (gb.sum(2), (G_err * (se * ue).abs() + (rhoe + wide) * gb.abs()).sum(2))
    result["d_C"] = (torch.where(live, hc.sum(2), _none()),
                     torch.where(live, (bound1 * dy.abs().unsqueeze(3) + (dy_rho.unsqueeze(3) + wide) * hc.abs()).sum(2),
                                 _none()))
    result["d_D"] = ((dy * u).sum((0, 1)), ((dy_rho + chain) * (dy * u).abs()).sum((0, 1)))
    if z is not None:
        dz = do * y * slope(z)
        dz_err = do.abs() * ((y_err + 3 * U * y.abs()) * slope(z).abs() + (18 + 12 * z.abs()) * U * (y.abs() + y_err))
        result["d_z"] = (torch.where(live, dz, _none()), torch.where(live, dz_err, _none()))
    result["d_h0"] = (e, err + ONCE * size)
    result["d_dt_bias"] = (dr.sum((0, 1)), (dr_err + chain * dr.abs()).sum((0, 1)))
    return result


# ---- gradient norm --------------------------------------------------------------------------------


def clip(grads, max_norm):
    """(the scaled tensors, the norm) in 64 bits."""
    norm = torch.sqrt(sum((d64(g) ** 2).sum() for g in grads))
    factor = max_norm / (norm + 1e-6)
    factor = torch.ones_like(factor) if max_norm == float("inf") or factor > 1 else factor
    return [d64(g) * factor for g in grads], norm
