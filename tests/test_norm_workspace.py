"""The workspace of layer norm's backward pass: no more than its partial sums, and never less."""
from __future__ import annotations

import pytest
import torch

import ops_plain as plain
from persistent_lstm_hip_amd.extension import PLH_OK, require_extension


@pytest.fixture(scope="module")
def lib():
    return require_extension().lib


# (rows, cols, rows of partial sums that any type needs at most)
@pytest.mark.parametrize("rows,cols,most", [
    (1024, 1 << 20, 64),   # rows too long for registers: 64 runs of rows
    (40, 1 << 24, 40),     # no more than there are rows
    (1 << 20, 16384, 256), # a workgroup of 256 threads or more per row: one on each CU, or two
    (1 << 20, 8192, 512),
    (1 << 20, 128, 1024),  # short rows: up to 1024 workgroups
    (3, 128, 3),
    (0, 128, 1),
])
def test_size(lib, rows, cols, most):
    assert 0 < lib.plh_layer_norm_workspace_bytes(rows, cols) <= most * 2 * cols * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(3000, 5), (3000, 24), (3000, 128), (1500, 512), (1100, 1030), (1100, 2048),
                                       (700, 4100), (700, 8192), (600, 16384), (100, 16392), (40, 33000), (3, 33000)])
def test_the_sums_stay_inside_it(gpu, lib, rows, cols, dtype):
    """The C call with a workspace of exactly that size: the bytes behind it stay as they are."""
    print(f"[gpu-case] norm workspace {rows} {cols} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows + cols)
    x, dy = (torch.randn(rows, cols, generator=g).to(dtype) for _ in range(2))
    code = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[dtype]
    need = lib.plh_layer_norm_workspace_bytes(rows, cols)
    room = torch.full((need + 1025 * 2 * cols * 4,), 0x5A, dtype=torch.uint8, device="cuda")  # (more than a call writes)
    stats = torch.empty(2, rows, device="cuda")
    xd, dyd = x.cuda(), dy.cuda()
    y, dx, dw, db = torch.empty_like(xd), torch.empty_like(xd), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    assert lib.plh_layer_norm_forward(code, 2, xd.data_ptr(), cols, rows, cols, None, None, 1e-5, y.data_ptr(),
                                      stats[0].data_ptr(), stats[1].data_ptr(), s) == PLH_OK
    assert lib.plh_layer_norm_backward(code, 2, xd.data_ptr(), cols, rows, cols, None, stats[0].data_ptr(),
                                       stats[1].data_ptr(), dyd.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                       room.data_ptr(), need, s) == PLH_OK
    torch.cuda.synchronize()
    assert bool((room[need:] == 0x5A).all())
    _, _, want_w, want_b = plain.norm(x, None, None, 1e-5, dy)
    x64, dy64 = x.double(), dy.double().abs()
    xh = ((x64 - x64.mean(1, keepdim=True)) / x64.std(1, unbiased=False, keepdim=True)).abs()
    # a normalised value carries the row mean's and deviation's errors, 16 U each of the row's largest (below 8); a sum
    # of R rows goes through R roundings at most, of partial sums that its terms' magnitudes bound
    terms = rows + 256
    plain.assert_within(dw, want_w, plain.U * ((terms * dy64 * xh).sum(0) + (160 * dy64 * (1 + xh)).sum(0)), torch.float32, "dw")
    plain.assert_within(db, want_b, plain.U * terms * dy64.sum(0), torch.float32, "db")
