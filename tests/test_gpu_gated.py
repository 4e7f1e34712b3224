"""The forecaster on the block operators: its outputs and every parameter's gradient against the same model in 64 bits on
the CPU, its serving form against its forward pass, and a short training run."""
from __future__ import annotations

import pytest
import torch

import ops_plain as plain
from persistent_lstm_hip_amd import GatedScanRegressor
from persistent_lstm_hip_amd.gated_demo import train

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _model(I, H, O, L, dropout, dtype=torch.float32):
    torch.manual_seed(11)
    m = GatedScanRegressor(I, H, O, L, dropout)
    for p in m.parameters():  # (no parameter at a special value)
        p.data += 0.1 * torch.randn_like(p)
    return m.to("cuda", dtype)


def _plain_forward(params, x, lengths, L, p, seed, offset):
    """The model in 64 bits from its definition; params: name -> float64 tensor."""
    def norm(y, w, b):
        c = y - y.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b

    B, T, _ = x.shape
    n = torch.full((B,), T) if lengths is None else lengths
    y = x @ params["stem.weight"].t() + params["stem.bias"]
    k = int(p * 65536 + 0.5)
    for i in range(L):
        w = {name[len(f"blocks.{i}."):]: t for name, t in params.items() if name.startswith(f"blocks.{i}.")}
        H = y.shape[-1]
        z = norm(y, w["norm_weight"], w["norm_bias"]) @ w["gates.weight"].t() + w["gates.bias"]
        c, hs = torch.zeros(B, H, dtype=torch.float64), []
        for t in range(T):
            on = (n > t).unsqueeze(1)
            a = torch.sigmoid(z[:, t, :H])
            c = torch.where(on, a * c + (1 - a) * z[:, t, H:2 * H], c)
            hs.append(torch.where(on, torch.sigmoid(z[:, t, 2 * H:]) * c, torch.zeros((), dtype=torch.float64)))
        h = torch.stack(hs, 1) @ w["out.weight"].t() + w["out.bias"]
        keep = plain.keep(0, h.numel(), k, seed, offset + i).view(h.shape).double() * (65536 / (65536 - k))
        y = y + h * keep
    last = (n - 1).clamp(0, T - 1)
    y = norm(y[torch.arange(B), last], params["norm_weight"], params["norm_bias"])
    return y @ params["linear.weight"].t() + params["linear.bias"]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("H,L", [(24, 2), (61, 1)])
def test_model_and_its_gradients(gpu, H, L, ragged):
    _say(f"model H={H} L={L} ragged={ragged}")
    B, T, I, O, p = 5, 70, 3, 4, 0.25
    m = _model(I, H, O, L, p)
    g = torch.Generator().manual_seed(1)
    x, d = torch.randn(B, T, I, generator=g), torch.randn(B, O, generator=g)
    lengths = torch.tensor([70, 1, 64, 0, 33]) if ragged else None
    m._passes = 3  # (masks of a later pass)
    out = m(x.cuda(), lengths)
    grads = torch.autograd.grad(out, list(m.parameters()), d.cuda())
    params = {n: t.detach().cpu().double().requires_grad_(True) for n, t in m.named_parameters()}
    want = _plain_forward(params, x.double(), lengths, L, p, m.seed, 3 * L)
    want_grads = torch.autograd.grad(want, list(params.values()), d.double())
    # float32 throughout: every value is a sum of some hundred terms in a few dependent stages
    tol = 2000 * plain.U
    assert (out.detach().cpu().double() - want.detach()).abs().max() <= tol * max(1.0, want.abs().max().item())
    for name, a, b in zip(params, grads, want_grads):
        assert (a.cpu().double() - b).abs().max() <= tol * max(1.0, b.abs().max().item()), name


def test_model_under_autocast(gpu):
    """fp32 parameters and fp16 products: the block's operators take a mixture of the two as autocast makes it."""
    _say("autocast")
    B, T, I, H, L, O, p = 5, 70, 3, 61, 2, 4, 0.25
    m = _model(I, H, O, L, p)
    g = torch.Generator().manual_seed(1)
    x, d = torch.randn(B, T, I, generator=g), torch.randn(B, O, generator=g)
    lengths = torch.tensor([70, 1, 64, 0, 33])
    with torch.autocast("cuda", dtype=torch.float16):
        out = m(x.cuda(), lengths)
    assert out.dtype == torch.float16
    grads = torch.autograd.grad(out.float(), list(m.parameters()), d.cuda())
    params = {n: t.detach().cpu().double().requires_grad_(True) for n, t in m.named_parameters()}
    want = _plain_forward(params, x.double(), lengths, L, p, m.seed, 0)
    want_grads = torch.autograd.grad(want, list(params.values()), d.double())
    # 6 L + 3 = 15 stages rounded to 11 bits, weights too, each amplified by at most a few by the norms behind it: 64
    # units; the gradients go through as many again
    u16 = 2.0 ** -11
    assert (out.detach().cpu().double() - want.detach()).abs().max() <= 64 * u16 * max(1.0, want.abs().max().item())
    for name, a, b in zip(params, grads, want_grads):
        assert a.dtype == torch.float32, name
        assert (a.cpu().double() - b).abs().max() <= 128 * u16 * max(1.0, b.abs().max().item()), name


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.float16, 2e-2)])
def test_serving_step_by_step_is_the_forward_pass(gpu, dtype, tol):
    _say(f"serve {dtype}")
    m = _model(3, 128, 6, 3, 0.2, dtype).eval()
    x = torch.randn(7, 90, 3, generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    with torch.no_grad():
        whole = m(x)
    state = m.initial_state(7)
    for t in range(90):
        out = m.step(x[:, t], state)
    assert (out.float() - whole.float()).abs().max().item() <= tol * max(1.0, whole.float().abs().max().item())


def test_training_learns(gpu):
    _say("train")
    torch.manual_seed(3)
    m = GatedScanRegressor(1, 64, 8, 2, dropout=0.05).to("cuda")
    losses = train(m, batch=64, seq_len=150, steps=120)
    first, last = sum(losses[:10]) / 10, sum(losses[-10:]) / 10
    assert last < 0.5 * first, (first, last)


def test_masks_differ_between_passes_and_not_in_evaluation(gpu):
    _say("masks")
    m = _model(2, 32, 3, 2, 0.5)
    x = torch.randn(4, 20, 2, device="cuda")
    with torch.no_grad():
        a, b = m(x), m(x)
        assert not torch.equal(a, b)
        m._passes = 0
        assert torch.equal(m(x), a)
        m.eval()
        assert torch.equal(m(x), m(x))


def test_model_refusals(gpu):
    _say("model refusals")
    m = _model(2, 32, 3, 1, 0.0)
    for bad in (lambda: m(torch.zeros(2, 0, 2, device="cuda")), lambda: m(torch.zeros(2, 2, device="cuda")),
                lambda: m(torch.zeros(2, 5, 2, device="cuda"), [1, 6]), lambda: m(torch.zeros(2, 5, 2, device="cuda"), [1])):
        with pytest.raises(ValueError):
            bad()
