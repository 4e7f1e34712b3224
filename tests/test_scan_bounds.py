"""The bounds that the scan's GPU tests hold its long rows to, on the CPU: an honest result in 32 bits is inside them, and
results with a mistake of the kind that a split time axis can have are not."""
from __future__ import annotations

import pytest
import torch

import ops_plain as plain
import scan_bounds

CASES = [(2, 700, 130), (1, 2500, 24), (2, 4100, 100)]


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _inputs(B, T, H, dtype):
    z = _rand(B, T, 3 * H, seed=0)
    z[..., :H] += torch.linspace(-2.0, 6.0, H)
    return z.to(dtype), _rand(B, H, seed=1), _rand(B, T, H, seed=5).to(dtype), _rand(B, H, seed=6)


def _in_32_bits(z, c0, dh, dc):
    """The recurrence and its gradient step by step in float32."""
    H, T = c0.shape[1], z.shape[1]
    f, g, o = z.float().split(H, -1)
    a, na, s, ns = torch.sigmoid(f), torch.sigmoid(-f), torch.sigmoid(o), torch.sigmoid(-o)
    c, before, after = c0, [], []
    for t in range(T):
        before.append(c)
        c = a[:, t] * c + na[:, t] * g[:, t]
        after.append(c)
    before, after, e = torch.stack(before, 1), torch.stack(after, 1), dc
    dz = torch.zeros_like(z, dtype=torch.float32)
    for t in reversed(range(T)):
        D = s[:, t] * dh[:, t].float() + e
        dz[:, t, :H], dz[:, t, H:2 * H] = a[:, t] * na[:, t] * (before[:, t] - g[:, t]) * D, na[:, t] * D
        e = a[:, t] * D
    dz[..., 2 * H:] = dh.float() * after * s * ns
    return (s * after).to(z.dtype), c, dz.to(z.dtype), e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H", CASES)
def test_bounds(B, T, H, dtype):
    z, c0, dh, dc = _inputs(B, T, H, dtype)
    want = scan_bounds.scan(z, c0, None, True, dh, dc)
    for name, value in zip(want, plain.scan(z, c0, None, True, dh, dc)):
        torch.testing.assert_close(want[name][0], value, rtol=1e-10, atol=1e-12)
    got = _in_32_bits(z, c0, dh, dc)
    scan_bounds.check(got, want, dtype, "32 bits")

    def seen(name, out=None, c_n=None, d_gates=None, d_c0=None):
        mine = [b if a is None else a for a, b in zip((out, c_n, d_gates, d_c0), got)]
        with pytest.raises(AssertionError, match=name):
            scan_bounds.check(mine, want, dtype, "planted")

    # no gradient at all, in any of the gates
    for part in range(3):
        bad = got[2].clone()
        bad[..., part * H:(part + 1) * H] = 0
        seen("d_gates", d_gates=bad)
    # a split time axis whose carry, in either direction, does not arrive at the second part, or at a later tile's start
    for cut in (64, 64 * (T // 128), 64 * (T // 64)):
        first = plain.scan(z[:, :cut], c0, None, True, dh[:, :cut], None)
        last = plain.scan(z[:, cut:], first[1], None, True, dh[:, cut:], dc)
        bad = torch.cat([first[2], last[2]], 1).to(dtype)
        seen("d_gates", d_gates=bad)  # E stops at the cut
        lost = plain.scan(z[:, cut:], None, None, True, dh[:, cut:], dc)
        seen("out", out=torch.cat([first[0], lost[0]], 1).to(dtype))  # c does
        whole = plain.scan(z, c0, None, True, dh, dc)[2]
        seen("d_gates", d_gates=torch.cat([whole[:, :cut], lost[2]], 1).to(dtype))  # the backward pass' saved state does
        # a saved state of the tile before
        stale = plain.scan(z[:, :cut - 64], c0, None, True)[1]
        stale = plain.scan(z[:, cut:], stale, None, True, dh[:, cut:], dc)[2]
        seen("d_gates", d_gates=torch.cat([whole[:, :cut], stale], 1).to(dtype))


def test_a_mistake_past_a_row_is_seen():
    """The gradient of c_n comes through the steps past a row's end as it is."""
    z, c0, dh, dc = _inputs(2, 700, 130, torch.float32)
    n = torch.tensor([321, 700])
    want = scan_bounds.scan(z, c0, n, True, dh, dc)
    out, c_n, dz, d0, _ = plain.scan(z, c0, n, True, dh, dc)
    scan_bounds.check((out.float(), c_n.float(), dz.float(), d0.float()), want, torch.float32, "ragged")
    lost = plain.scan(z, c0, n, True, dh, dc * torch.tensor([[0.0], [1.0]]))
    with pytest.raises(AssertionError, match="d_gates"):
        scan_bounds.check((out.float(), c_n.float(), lost[2].float(), d0.float()), want, torch.float32, "planted")
    bad = dz.float()
    bad[0, 321:] = 1e-20  # (nothing at all past a row's end)
    with pytest.raises(AssertionError, match="d_gates"):
        scan_bounds.check((out.float(), c_n.float(), bad, d0.float()), want, torch.float32, "planted")
