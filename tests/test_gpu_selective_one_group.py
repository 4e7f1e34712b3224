"""The selective scan of more than 16 states and so few channels that they make one group: the backward pass then takes two
rows per workgroup, whose lengths differ, and the last one of an odd number alone."""
from __future__ import annotations

import pytest
import torch

from test_gpu_selective import _check, _inputs, _lengths, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,D,N", [(1, 40, 8, 17), (2, 33, 5, 32), (5, 70, 3, 33), (4, 65, 4, 64), (3, 700, 6, 20),
                                     (2, 900, 2, 48), (7, 9, 1, 24)])
def test_two_rows_per_workgroup(gpu, B, T, D, N, dtype):
    _say(f"selective scan one group {B} {T} {D} {N} {dtype}")
    _check(_inputs(B, T, D, N, dtype), what="full")
    _check(_inputs(B, T, D, N, dtype, dtype, seed=1), _lengths(B, T), what="ragged")
    _check(_inputs(B, T, D, N, dtype, gate=False, skip=False, state=False, bias=False, seed=2), _lengths(B, T).flip(0),
           what="bare")
