"""Long rows of the gated linear recurrence on the GPU, every element of every result within a bound of its own (derived in
scan_bounds.py, where a test on the CPU shows what it rejects)."""
from __future__ import annotations

import pytest
import torch

import persistent_lstm_hip_amd as P
import scan_bounds

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _check(B, T, H, gated, dtype, lengths, with_c0, what):
    print(f"[gpu-case] scan bounds {B} {T} {H} gated={gated} {dtype} {what}", flush=True)
    z = _rand(B, T, (3 if gated else 2) * H, seed=B + T + H)
    z[..., :H] += torch.linspace(-2.0, 6.0, H)
    z, dh, dc = z.to(dtype), _rand(B, T, H, seed=5).to(dtype), _rand(B, H, seed=6)
    c0 = _rand(B, H, seed=1) if with_c0 else None
    zd = z.cuda().requires_grad_(True)
    cd = None if c0 is None else c0.cuda().requires_grad_(True)
    out, c_n = P.gated_scan(zd, cd, lengths=lengths, output_gate=gated)
    grads = torch.autograd.grad((out, c_n), (zd,) if cd is None else (zd, cd), (dh.cuda(), dc.cuda()))
    want = scan_bounds.scan(z, c0, lengths, gated, dh, dc)
    scan_bounds.check((out, c_n, *grads), want, dtype, what)


# (B, T, H): a few slabs, the time axis in many segments; segments of several tiles, in one direction or in both; wide
# slabs; slabs enough for no split; one channel per thread; tiles' edges
SHAPES = [(1, 2500, 24), (2, 700, 130), (8, 700, 402), (2, 3000, 700), (2, 4100, 1000), (20, 1000, 264), (33, 300, 1000),
          (2, 1300, 3), (3, 129, 61), (5, 64, 130), (5, 65, 130)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("B,T,H", SHAPES)
def test_full_rows(gpu, B, T, H, gated, dtype):
    _check(B, T, H, gated, dtype, None, True, "full")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,T,H", SHAPES)
def test_ragged_rows(gpu, B, T, H, dtype):
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B + T))
    n[0] = T if B < 3 else 0
    _check(B, T, H, True, dtype, n, False, "ragged")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,H", [(2, 3000, 700), (2, 4100, 1000)])
def test_rows_that_end_anywhere_in_a_segment(gpu, B, T, H, dtype):
    """In each tile of a segment, on a tile's edge and one step to either side of it."""
    for i, tiles in enumerate(range(10, 16)):
        n = torch.tensor([64 * tiles + 1, 64 * tiles - i % 2])
        _check(B, T, H, True, dtype, n, True, f"{n.tolist()} steps")
