"""The forecaster on the selective scan: its outputs and every parameter's gradient against the same model in 64 bits on the
CPU, its serving form against its forward pass, a sequence in parts, a clipped training step."""
from __future__ import annotations

import math

import pytest
import torch

import ops_plain as plain
from persistent_lstm_hip_amd import SelectiveScanBlock, SelectiveScanRegressor, clip_grad_norm
from persistent_lstm_hip_amd.gated_demo import train

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _model(I, H, O, L, dropout, dtype=torch.float32, **kw):
    torch.manual_seed(12)
    m = SelectiveScanRegressor(I, H, O, L, dropout, **kw)
    for p in m.parameters():  # (no parameter at a special value)
        p.data += 0.1 * torch.randn_like(p)
    return m.to("cuda", dtype)


def _plain_forward(params, x, lengths, L, p, seed, offset):
    """The model in 64 bits from its definition; params: name -> float64 tensor."""
    def norm(y, w, b):
        c = y - y.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b

    def silu(v):
        return v * torch.sigmoid(v)

    none = torch.zeros((), dtype=torch.float64)
    B, T, _ = x.shape
    n = torch.full((B,), T) if lengths is None else lengths
    on = (torch.arange(T).unsqueeze(0) < n.unsqueeze(1)).unsqueeze(2)
    y = x @ params["stem.weight"].t() + params["stem.bias"]
    k = int(p * 65536 + 0.5)
    for i in range(L):
        w = {name[len(f"blocks.{i}."):]: t for name, t in params.items() if name.startswith(f"blocks.{i}.")}
        u, z = (norm(y, w["norm_weight"], w["norm_bias"]) @ w["inner.weight"].t()).chunk(2, -1)
        E, W = w["conv_weight"].shape
        N = w["A_log"].shape[1]
        line = torch.cat([torch.zeros(B, W - 1, E, dtype=torch.float64), torch.where(on, u, none)], 1)
        u = torch.where(on, silu(w["conv_bias"] + sum(w["conv_weight"][:, j] * line[:, j:j + T] for j in range(W))), none)
        low, Bm, Cm = (u @ w["coefs.weight"].t()).split([w["coefs.weight"].shape[0] - 2 * N, N, N], -1)
        dt = torch.where(on, torch.nn.functional.softplus(low @ w["steps.weight"].t() + w["dt_bias"], threshold=1e9), none)
        A, h, outs = -torch.exp(w["A_log"]), torch.zeros(B, E, N, dtype=torch.float64), []
        for t in range(T):
            h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * Bm[:, t, None]
            outs.append((h * Cm[:, t, None]).sum(-1) + w["D"] * u[:, t])
        h = torch.where(on, torch.stack(outs, 1) * silu(z), none) @ w["out.weight"].t()
        keep = plain.keep(0, h.numel(), k, seed, offset + i).view(h.shape).double() * (65536 / (65536 - k))
        y = y + h * keep
    last = (n - 1).clamp(0, T - 1)
    y = norm(y[torch.arange(B), last], params["norm_weight"], params["norm_bias"])
    return y @ params["linear.weight"].t() + params["linear.bias"]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("H,L,kw", [(24, 2, {}), (33, 1, dict(states=5, width=3, expand=1))])
def test_model_and_its_gradients(gpu, H, L, kw, ragged):
    _say(f"selective model H={H} L={L} ragged={ragged}")
    B, T, I, O, p = 5, 70, 3, 4, 0.25
    m = _model(I, H, O, L, p, **kw)
    g = torch.Generator().manual_seed(1)
    x, d = torch.randn(B, T, I, generator=g), torch.randn(B, O, generator=g)
    lengths = torch.tensor([70, 1, 64, 0, 33]) if ragged else None
    out = m(x.cuda(), lengths)
    grads = torch.autograd.grad(out, list(m.parameters()), d.cuda())
    params = {n: t.detach().cpu().double().requires_grad_(True) for n, t in m.named_parameters()}
    want = _plain_forward(params, x.double(), lengths, L, p, m.seed, 0)
    want_grads = torch.autograd.grad(want, list(params.values()), d.double())
    # float32 throughout: every value is a sum of some hundred terms in a few dependent stages
    tol = 2000 * plain.U
    assert (out.detach().cpu().double() - want.detach()).abs().max() <= tol * max(1.0, want.abs().max().item())
    for name, a, b in zip(params, grads, want_grads):
        assert (a.cpu().double() - b).abs().max() <= tol * max(1.0, b.abs().max().item()), name
    # the gradients clipped together
    norm = math.sqrt(sum((b ** 2).sum().item() for b in want_grads))
    clipped, got = clip_grad_norm(grads, 0.25 * norm)
    assert abs(got.item() - norm) <= tol * norm
    assert abs(clip_grad_norm(clipped, float("inf"))[1].item() - 0.25 * norm) <= 4 * tol * norm


def test_model_under_autocast(gpu):
    _say("selective autocast")
    m = _model(3, 61, 4, 2, 0.25)
    x = torch.randn(5, 70, 3, generator=torch.Generator().manual_seed(1)).cuda()
    lengths = torch.tensor([70, 1, 64, 0, 33])
    whole = m(x, lengths, offset=3)
    with torch.autocast("cuda", dtype=torch.float16):
        out = m(x, lengths, offset=3)
    assert out.dtype == torch.float16
    # 8 L + 3 = 19 stages rounded to 11 bits, weights too, each amplified by at most a few by the norms behind it
    assert (out.float() - whole).abs().max() <= 96 * 2.0**-11 * max(1.0, whole.abs().max().item())
    grads = torch.autograd.grad(out.float().sum(), list(m.parameters()))
    assert all(g.dtype == torch.float32 and bool(torch.isfinite(g).all()) for g in grads)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.float16, 2e-2), (torch.bfloat16, 1.6e-1)])
def test_serving_step_by_step_is_the_forward_pass(gpu, dtype, tol):
    _say(f"selective serve {dtype}")
    m = _model(3, 64, 6, 2, 0.2, dtype).eval()
    x = torch.randn(7, 90, 3, generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    with torch.no_grad():
        whole = m(x)
    state = m.initial_state(7)
    for t in range(90):
        out = m.step(x[:, t], state)
    assert (out.float() - whole.float()).abs().max().item() <= tol * max(1.0, whole.float().abs().max().item())


def test_a_prompt_then_tokens(gpu):
    """A block over a prompt, its state handed on to a second part and then to single tokens."""
    _say("selective prompt")
    torch.manual_seed(5)
    block = SelectiveScanBlock(32).cuda().eval()
    x = torch.randn(3, 60, 32, device="cuda")
    with torch.no_grad():
        whole, last = block(x)
        y1, state = block(x[:, :37])
        y2, state = block(x[:, 37:50], state)
        ys = [y1, y2]
        for t in range(50, 60):
            ys.append(block.step(x[:, t], state).unsqueeze(1))
    assert (torch.cat(ys, 1) - whole).abs().max() < 1e-4
    assert all((a - b).abs().max() < 1e-4 for a, b in zip(state, last))


def test_training_runs_with_clipped_gradients(gpu):
    _say("selective train")
    torch.manual_seed(3)
    m = SelectiveScanRegressor(1, 32, 8, 2, dropout=0.05).to("cuda")
    losses = train(m, batch=8, seq_len=100, steps=3, clip=0.01)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
    norm = clip_grad_norm([p.grad for p in m.parameters()], float("inf"))[1].item()
    assert norm <= 0.01 * (1 + 1e-5)
