"""The block operators from their formulas in 64 bits on the CPU, for the tests: the gated linear recurrence and layer
norm step by step in torch.float64 with their written-out gradients, Philox4x32-10 in numpy's unsigned 64-bit
arithmetic."""
from __future__ import annotations

import numpy as np
import torch

# Half a unit in the last place, relative, of what an operator's result is rounded to, and half the spacing of its
# subnormal numbers.
ROUNDING = {torch.float16: (2.0**-11, 2.0**-25), torch.bfloat16: (2.0**-8, 0.0), torch.float32: (2.0**-24, 0.0)}
U = 2.0**-24


def d64(t):
    return None if t is None else t.detach().cpu().double()


def scan(gates, c0, lengths, output_gate, d_out=None, d_cn=None):
    """(out, c_n) and with d_out (d_gates, d_c0, the largest |D|) of the recurrence."""
    z = d64(gates)
    B, T, width = z.shape
    H = width // (3 if output_gate else 2)
    n = torch.full((B,), T) if lengths is None else torch.as_tensor(lengths).cpu().long().clamp(0, T)
    live = torch.arange(T).unsqueeze(0) < n.unsqueeze(1)
    z = torch.where(live.unsqueeze(2), z, torch.zeros((), dtype=torch.float64))  # what a row does not reach, it ignores
    a, g = torch.sigmoid(z[..., :H]), z[..., H:2 * H]
    s = torch.sigmoid(z[..., 2 * H:]) if output_gate else torch.ones_like(a)
    c = torch.zeros(B, H, dtype=torch.float64) if c0 is None else d64(c0)
    before, after = torch.zeros(B, T, H, dtype=torch.float64), torch.zeros(B, T, H, dtype=torch.float64)
    for t in range(T):
        before[:, t] = c
        c = torch.where(live[:, t:t + 1], a[:, t] * c + (1 - a[:, t]) * g[:, t], c)
        after[:, t] = c
    out = torch.where(live.unsqueeze(2), s * after, torch.zeros((), dtype=torch.float64))
    if d_out is None:
        return out, c
    dh = torch.where(live.unsqueeze(2), d64(d_out), torch.zeros((), dtype=torch.float64))
    e = torch.zeros(B, H, dtype=torch.float64) if d_cn is None else d64(d_cn)
    dz, most = torch.zeros_like(z), e.abs().max().item() if e.numel() else 0.0
    for t in reversed(range(T)):
        on = live[:, t:t + 1]
        D = s[:, t] * dh[:, t] + e
        dz[:, t, :H] = on * (a[:, t] * (1 - a[:, t]) * (before[:, t] - g[:, t]) * D)
        dz[:, t, H:2 * H] = on * ((1 - a[:, t]) * D)
        e = torch.where(on, a[:, t] * D, e)
        if D.numel():
            most = max(most, D.abs().max().item())
    if output_gate:
        dz[..., 2 * H:] = dh * after * s * (1 - s)
    return out, c, dz, e, most


def norm(x, weight, bias, eps, d_y=None):
    """y and with d_y (d_x, d_weight, d_bias) of layer norm over the last dimension of [rows, cols]."""
    x = d64(x)
    cols = x.shape[1]
    w = torch.ones(cols, dtype=torch.float64) if weight is None else d64(weight)
    b = torch.zeros(cols, dtype=torch.float64) if bias is None else d64(bias)
    xc = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + eps)
    xh = xc * r
    y = xh * w + b
    if d_y is None:
        return y
    dy = d64(d_y)
    v = dy * w
    dx = r * (v - v.mean(1, keepdim=True) - xh * (v * xh).mean(1, keepdim=True))
    return y, dx, (dy * xh).sum(0), dy.sum(0)


def philox(counter, key):
    """Philox4x32-10 of counter [n, 4] and key [2], 32-bit words held in uint64."""
    u = np.uint64
    c = [np.asarray(counter)[:, i].astype(u) for i in range(4)]
    k = [int(v) for v in key]
    for _ in range(10):
        p0, p1 = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(p1 >> u(32)) ^ c[1] ^ u(k[0]), p1 & u(0xFFFFFFFF), (p0 >> u(32)) ^ c[3] ^ u(k[1]), p0 & u(0xFFFFFFFF)]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def keep(first, n, threshold, seed, offset):
    """Which of the elements first .. first + n - 1 stay."""
    seed, offset = seed % 2**64, offset % 2**64
    q = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    counter = np.stack([q & np.uint64(0xFFFFFFFF), q >> np.uint64(32),
                        np.full_like(q, offset & 0xFFFFFFFF), np.full_like(q, offset >> 32)], 1)
    words = philox(counter, (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)
    return torch.from_numpy(bits[first % 8:first % 8 + n].astype(np.int64) >= threshold)


def assert_within(got, want, tol, dtype, what):
    """|got - want| <= tol + the rounding of want to dtype, everywhere; tol: a number or a tensor."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    assert bool(torch.isfinite(got).all()), f"{what}: non-finite values"
    rel, sub = ROUNDING[dtype]
    over = (got - want).abs() - (tol + rel * (want.abs() + tol) + sub)
    if over.numel():
        i = int(over.argmax())
        assert over.max().item() <= 0.0, (f"{what}: element {i} is {got.flatten()[i].item()!r}, expected "
                                          f"{want.flatten()[i].item()!r}, {over.max().item():.3g} beyond its bound")
