"""The residual block by itself on the GPU: its types under autocast."""
from __future__ import annotations

import pytest
import torch

from persistent_lstm_hip_amd import GatedScanBlock

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


@pytest.mark.parametrize("low", [torch.float16, torch.bfloat16])
def test_a_residual_stream_in_32_bits_under_autocast(gpu, low):
    """The products are of the lower type, the stream stays as it is; forward, backward and step by step."""
    _say(f"block under autocast {low}")
    torch.manual_seed(0)
    block = GatedScanBlock(24).cuda()
    x = torch.randn(3, 40, 24, device="cuda", requires_grad=True)
    want, want_c = block(x)
    d = torch.randn_like(x)
    want_grads = torch.autograd.grad(want, [x, *block.parameters()], d)
    with torch.autocast("cuda", dtype=low):
        y, c_n = block(x)
    assert y.dtype == torch.float32 and c_n.dtype == torch.float32
    grads = torch.autograd.grad(y, [x, *block.parameters()], d)
    # eight stages rounded to the lower type, each amplified a few times: 64 units, and twice as many backwards
    u = torch.finfo(low).eps / 2
    assert (y - want).abs().max() <= 64 * u * max(1.0, want.abs().max().item())
    for a, b in zip(grads, want_grads):
        assert a.dtype == torch.float32
        assert (a - b).abs().max() <= 128 * u * max(1.0, b.abs().max().item())
    c = torch.zeros(3, 24, device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=low):
        for t in range(40):
            one = block.step(x[:, t], c)
    assert one.dtype == torch.float32
    assert (one - y[:, -1]).abs().max() <= 64 * u * max(1.0, y.abs().max().item())
