"""The selective scan at sizes near its limits: rows are independent, so that a few of them by themselves give the same."""
from __future__ import annotations

import pytest
import torch

import persistent_lstm_hip_amd as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


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
