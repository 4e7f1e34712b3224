"""Trains a GatedScanRegressor on synthetic series, then serves it step by step.

    python -m persistent_lstm_hip_amd.gated_demo [--hidden 128 --layers 4 --batch 128 --seq-len 1000 --steps 100]
"""
from __future__ import annotations

import argparse
import time
from typing import List

import torch
import torch.nn.functional as F

from .gated import GatedScanRegressor


def _series(batch: int, steps: int, ahead: int, device, gen: torch.Generator):
    """Sums of two sines and noise: (x [batch, steps, 1], the next `ahead` values)."""
    t = torch.arange(steps + ahead, device=device)
    f = 0.02 + 0.2 * torch.rand(batch, 2, 1, device=device, generator=gen)
    ph = 6.2832 * torch.rand(batch, 2, 1, device=device, generator=gen)
    clean = torch.sin(f * t + ph).sum(1)
    noisy = clean[:, :steps] + 0.05 * torch.randn(batch, steps, device=device, generator=gen)
    return noisy.unsqueeze(-1), clean[:, steps:]


def train(model: GatedScanRegressor, *, batch: int, seq_len: int, steps: int, lr: float = 2e-3, seed: int = 1,
          report=None) -> List[float]:
    """`steps` optimizer steps on synthetic series; the losses."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    dtype, losses = model.linear.weight.dtype, []
    model.train()
    for i in range(steps):
        x, want = _series(batch, seq_len, model.linear.out_features, "cuda", gen)
        loss = F.mse_loss(model(x.to(dtype)).float(), want)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if report and (i + 1) % report == 0:
            print(f"step {i + 1}: loss {losses[-1].item():.4f}", flush=True)
    return [v.item() for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description="Train a gated-scan forecaster on synthetic series and serve it.")
    ap.add_argument("--hidden", type=int, default=128)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=128)
    ap.add_argument("--seq-len", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=100)
    a = ap.parse_args()
    torch.manual_seed(42)
    model = GatedScanRegressor(1, a.hidden, 24, a.layers, dropout=0.05).to("cuda")
    t0 = time.perf_counter()
    losses = train(model, batch=a.batch, seq_len=a.seq_len, steps=a.steps, report=max(1, a.steps // 5))
    print(f"{a.steps} steps of {a.batch} x {a.seq_len}: {1e3 * (time.perf_counter() - t0) / a.steps:.2f} ms each, "
          f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    model.eval()
    x, _ = _series(4, a.seq_len, 24, "cuda", torch.Generator(device="cuda").manual_seed(7))
    with torch.no_grad():
        whole = model(x)
        state = model.initial_state(4)
        for t in range(a.seq_len):
            out = model.step(x[:, t], state)
    print(f"served step by step: forecasts differ from the whole sequence's by {(out - whole).abs().max().item():.2e}")


if __name__ == "__main__":
    main()
