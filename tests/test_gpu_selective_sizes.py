"""The selective scan at sizes near its limits: rows are independent, so that a few of them by themselves give the same."""
from __future__ import annotations

import pytest
import torch

import persistent_lstm_hip_amd as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


@pytest.mark.parametrize("N,T,D", [(4, 2, 1024), (20, 3, 600), (40, 2, 300)])
def test_many_short_rows(gpu, N, T, D):
    _say(f"selective many rows N={N}")
    B = 16385 if D == 1024 else 28001
    g = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    u, dt, z = (rand(B, T, D).to(BF16) for _ in range(3))
    Bm, C = (rand(B, T, N).to(BF16) for _ in range(2))
    A, skip, d_out = -torch.rand(D, N, generator=g, device="cuda"), rand(D), rand(B, T, D).to(BF16)

    def run(rows):
        leaves = [t[rows].clone().requires_grad_(True) for t in (u, dt, Bm, C, z)]
        params = [t.clone().requires_grad_(True) for t in (A, skip)]
        out, h_n = P.selective_scan(leaves[0], leaves[1], params[0], leaves[2], leaves[3], params[1], leaves[4])
        grads = torch.autograd.grad(out, leaves + params, d_out[rows])
        return (out.detach(), h_n.detach(), *grads[:5]), grads[5:]

    rows, sums = run(slice(0, B))
    edge = B - 61
    first, first_sums = run(slice(0, edge))
    last, last_sums = run(slice(edge, B))
    for whole, a, b in zip(rows, first, last):
        assert torch.equal(whole[:edge], a) and torch.equal(whole[edge:], b)
    for whole, a, b in zip(sums, first_sums, last_sums):
        # sums of B T terms in another order: B / 32 additions in a chain, each off by 2^-24 of a sum whose terms have either
        # sign and are of size ten at most
        assert ((whole - a - b).abs() <= B / 32 * 2.0**-24 * 10 * (B * T * N) ** 0.5).all()


def test_the_largest_step(gpu):
    """2^32 - 4096 channels of all rows, a state each; every row has the same inputs."""
    _say("selective largest step")
    B, D = 4096, (1 << 20) - 1
    g = torch.Generator().manual_seed(1)
    u, dt = (torch.randn(1, D, generator=g).cuda().to(BF16) for _ in range(2))
    Bm, C = (torch.randn(1, 1, generator=g).cuda().to(BF16) for _ in range(2))
    A = -torch.rand(D, 1, generator=g).cuda()
    h = torch.zeros(B, D, 1, device="cuda")
    h[-1], h[B // 2] = 1.0, 2.0
    rows = [0, B // 2, B - 1]
    want = P.selective_scan_step(u.expand(3, D), dt.expand(3, D), A, Bm.expand(3, 1), C.expand(3, 1), h[rows])
    out, same = P.selective_scan_step(u.expand(B, D), dt.expand(B, D), A, Bm.expand(B, 1), C.expand(B, 1), h, inplace=True)
    assert same is h and torch.equal(out[rows], want[0]) and torch.equal(h[rows], want[1])
    torch.cuda.empty_cache()
