"""What the speed of the selective-scan operators is measured on.

A block around a selective state space scan,

    u, z = W_in norm(x)        u = silu(causal_conv(u))        dt, B, C = W_x u
    y = x + W_out selective_scan(u, dt, A, B, C, D, z)

takes two operators besides its matrix products and norm: a short causal convolution along time
(`causal_conv`, and `causal_conv_step` for one token) and the scan (`selective_scan`,
`selective_scan_step`).  Training such a model clips the gradients by their global norm
(`clip_grad_norm`).  Inference calls the forward alone; a training case is a forward and the
gradients of everything that it was given.

The plain form computes each from elementary torch operations in 32 bits (the norm in 64), rounded
once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"

# Elements of the plain scan's [batch, time, channels, states], and of one activation tensor, of the largest cases.
_MAX_STATES = 1 << 29
_MAX_TENSOR = 1 << 27


def listed():
    return [
        # One token of one series in a live forecaster: the smallest call, all latency.
        dict(name="scan_step_one_series", op="scan_step", B=1, D=256, N=16, gated=True, dtype="float16", wdtype="float32"),
        # One token of every series of the benchmark's batch, in a block of twice its hidden size 512.
        dict(name="scan_step_batch", op="scan_step", B=512, D=1024, N=16, gated=True, dtype="bfloat16", wdtype="float32"),
        # The prompt of one long record: one row, so the time axis has to be split.
        dict(name="scan_prompt_long", op="scan", train=False, B=1, T=16384, D=1280, N=16, gated=True, skip=True,
             state=False, lo=0, dtype="bfloat16", wdtype="float32"),
        # A training step of the demonstration's forecaster (128 series of 1000 steps, hidden 128, expanded twice).
        dict(name="scan_train_forecaster", op="scan", train=True, B=128, T=1000, D=256, N=16, gated=True, skip=True,
             state=False, lo=200, dtype="float16", wdtype="float32"),
        # The largest call: a training batch of a wide block.
        dict(name="scan_train_wide", op="scan", train=True, B=8, T=2048, D=2048, N=16, gated=True, skip=True,
             state=False, lo=0, dtype="bfloat16", wdtype="float32"),
        # A small model over a year of daily values in 32 bits, some rows empty, from a state, no gate and no skip;
        # nothing a multiple of a tile.
        dict(name="scan_train_daily", op="scan", train=True, B=37, T=365, D=123, N=10, gated=False, skip=False,
             state=True, lo=-40, dtype="float32", wdtype="float32"),
        # The convolution in front of one token's scan, for one series and for a batch of them.
        dict(name="conv_step_one_series", op="conv_step", B=1, C=256, W=4, silu=True, dtype="float16", wdtype="float32"),
        dict(name="conv_step_batch", op="conv_step", B=64, C=1024, W=4, silu=True, dtype="bfloat16", wdtype="bfloat16"),
        # Training at the headline's sizes: 512 ragged rows of up to 1000 steps.
        dict(name="conv_train_headline", op="conv", train=True, B=512, T=1000, C=256, W=4, silu=True, state=False, lo=200,
             dtype="float16", wdtype="float32"),
        # An odd width without an activation, continuing from a state: no row but the first is aligned.
        dict(name="conv_train_odd", op="conv", train=True, B=61, T=731, C=333, W=3, silu=False, state=True, lo=0,
             dtype="float32", wdtype="float32"),
        # The gradients of a small forecaster in 32 bits: many tiny tensors.
        dict(name="clip_forecaster", op="clip", layers=4, H=128, inputs=5, limit=0.5, dtype="float32", vdtype="float32"),
        # A few layers of a wide model in bfloat16, as one process of several holds them; vectors in 32 bits.
        dict(name="clip_wide", op="clip", layers=5, H=4096, inputs=64, limit=0.1, dtype="bfloat16", vdtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _width(rng, lo, hi):
    """A row length: often 8 times an odd number or a power of two, sometimes any odd number."""
    kind = rng.random()
    if kind < 0.35:
        return 8 * (_log_int(rng, max(1, lo // 8), max(1, hi // 8 - 1)) | 1)
    if kind < 0.65:
        return 1 << rng.randint(max(3, int(math.log2(lo))), int(math.log2(hi)))
    return _log_int(rng, lo, hi - 1) | 1


def draw(rng):
    """One more case: 1 to 4096 channels, 1 to 64 states, lengths of 1 to 16384 steps, 1 to 8 taps, every type; up to 5
    layers' gradients."""
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    wdtype = rng.choice([dtype, "float32"])
    pick = rng.random()
    train, gated = rng.random() < 0.6, rng.random() < 0.7
    if pick < 0.12:
        N = rng.choice([1, 3, 8, 16, 16, 16, 24, 64])
        D = _width(rng, 1, 4096)
        B = _log_int(rng, 1, max(1, min(1024, (1 << 24) // (D * N)))) | 1
        return dict(op="scan_step", B=B, D=D, N=N, gated=gated, dtype=dtype, wdtype=wdtype)
    if pick < 0.5:
        N = rng.choice([1, 4, 5, 8, 16, 16, 16, 16, 31, 64])
        D = _width(rng, 1, 2048)
        T = _log_int(rng, 1, 16384) | 1
        T = min(T, max(1, _MAX_STATES // (D * N)))
        B = _log_int(rng, 1, max(1, min(512, _MAX_STATES // (T * D * N))))
        lo = rng.choice([0, 0, 1 + T // 5, -(T // 8) - 1])
        return dict(op="scan", train=train, B=B, T=T, D=D, N=N, gated=gated, skip=rng.random() < 0.7,
                    state=rng.random() < 0.4, lo=lo, dtype=dtype, wdtype=wdtype)
    if pick < 0.6:
        return dict(op="conv_step", B=_log_int(rng, 1, 1024) | 1, C=_width(rng, 1, 4096), W=rng.choice([1, 2, 3, 4, 4, 4, 8]),
                    silu=rng.random() < 0.7, dtype=dtype, wdtype=wdtype)
    if pick < 0.8:
        C = _width(rng, 1, 4096)
        T = _log_int(rng, 1, 16384) | 1
        B = _log_int(rng, 1, max(1, min(512, _MAX_TENSOR // (T * C))))
        lo = rng.choice([0, 0, 1 + T // 5, -(T // 8) - 1])
        return dict(op="conv", train=train, B=B, T=T, C=C, W=rng.choice([1, 2, 3, 4, 4, 4, 8]), silu=rng.random() < 0.7,
                    state=rng.random() < 0.4, lo=lo, dtype=dtype, wdtype=wdtype)
    H = _width(rng, 16, 4096)
    most = max(1, min(5, (1 << 29) // (6 * H * H)))
    return dict(op="clip", layers=rng.randint(1, most), H=H, inputs=rng.randint(1, 64), limit=rng.choice([0.01, 0.5, 0.9, 3.0]),
                dtype=dtype, vdtype=rng.choice([dtype, "float32"]))


# ---- inputs ------------------------------------------------------------------------------------


def _lengths(case, gen):
    """lo = 0: rows of full length (none); above: lengths from lo to T; below: the same with 1 - lo of T + 1 - lo rows
    empty in the mean."""
    if case["lo"] == 0:
        return None
    n = torch.randint(min(case["lo"], case["T"]), case["T"] + 1, (case["B"],), device=DEVICE, generator=gen)
    return n.clamp(min=0).to(torch.int32)


def _clip_shapes(case):
    """The parameters of a selective-scan forecaster of width H, expanded twice, with 16 states: a stem, per layer a
    norm, the projections in, to the scan's coefficients and out, the convolution and the scan's own, a head."""
    H, E = case["H"], 2 * case["H"]
    rank = (H + 15) // 16
    shapes = [(H, case["inputs"]), (H,)]
    for _ in range(case["layers"]):
        shapes += [(H,), (H,), (2 * E, H), (E, 4), (E,), (rank + 32, E), (E, rank), (E,), (E, 16), (E,), (H, E)]
    return shapes + [(24, H), (24,)]


def _inputs(case, seed):
    """The tensors of one pass, on the GPU."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def rand(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    d = {}
    if case["op"] == "clip":
        vdtype = getattr(torch, case["vdtype"])
        shapes = _clip_shapes(case)
        d["grads"] = [(0.01 * rand(*s)).to(dtype if len(s) == 2 else vdtype) for s in shapes]
        d["max_norm"] = case["limit"] * 0.01 * math.sqrt(sum(math.prod(s) for s in shapes))
        return d
    wdtype = getattr(torch, case["wdtype"])
    if case["op"] in ("conv", "conv_step"):
        B, C, W = case["B"], case["C"], case["W"]
        d["weight"], d["bias"] = (rand(C, W) / math.sqrt(W)).to(wdtype), (0.1 * rand(C)).to(wdtype)
        if case["op"] == "conv_step":
            # (one half of a projection's output)
            d["x"], d["state"] = rand(B, 2 * C).to(dtype)[:, :C], rand(B, W - 1, C).to(dtype)
            return d
        d["x"] = rand(B, case["T"], 2 * C).to(dtype)[..., :C]
        d["state"] = rand(B, W - 1, C).to(dtype) if case["state"] else None
        d["lengths"] = _lengths(case, gen)
        if case["train"]:
            d["d_y"], d["d_state"] = rand(B, case["T"], C).to(dtype), rand(B, W - 1, C).to(dtype)
        return d
    B, D, N = case["B"], case["D"], case["N"]
    lead = (B,) if case["op"] == "scan_step" else (B, case["T"])
    # Decays of -1, -2, ... and step sizes between 0.001 and 0.1, channel by channel, as such models start from.
    d["A"] = -(torch.arange(1, N + 1, device=DEVICE) * (1.0 + 0.1 * torch.rand(D, N, device=DEVICE, generator=gen)))
    step = torch.exp(torch.rand(D, device=DEVICE, generator=gen) * math.log(100.0) + math.log(0.001))
    d["dt_bias"] = (step + torch.log(-torch.expm1(-step))).to(wdtype)
    d["A"] = d["A"].to(wdtype)
    d["u"], d["dt"] = rand(*lead, D).to(dtype), (0.5 * rand(*lead, D)).to(dtype)
    both = rand(*lead, 2 * N).to(dtype)
    d["Bm"], d["Cm"] = both[..., :N], both[..., N:]
    d["z"] = rand(*lead, 2 * D).to(dtype)[..., D:] if case["gated"] else None
    if case["op"] == "scan_step":
        d["D"], d["h"] = (1.0 + 0.1 * rand(D)).to(wdtype), rand(B, D, N)
        return d
    d["D"] = (1.0 + 0.1 * rand(D)).to(wdtype) if case["skip"] else None
    d["h0"] = rand(B, D, N) if case["state"] else None
    d["lengths"] = _lengths(case, gen)
    if case["train"]:
        d["d_y"], d["d_h"] = rand(B, case["T"], D).to(dtype), rand(B, D, N)
    return d


_LEAVES = {"scan": ("u", "dt", "A", "Bm", "Cm", "D", "z", "h0", "dt_bias"), "conv": ("x", "weight", "bias", "state")}


def _given(case, d):
    """What a training case has gradients of, in the order that they are returned in."""
    return [d[name] for name in _LEAVES[case["op"]] if d[name] is not None]


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if case.get("train"):
        for t in _given(case, d):
            t.requires_grad_(True)
    return d


# ---- the framework's operators -----------------------------------------------------------------


def _run_own(s):
    import persistent_lstm_hip_amd as plh

    case = s["case"]
    if case["op"] == "clip":
        return plh.clip_grad_norm(s["grads"], s["max_norm"])
    if case["op"] == "scan_step":
        with torch.no_grad():
            return plh.selective_scan_step(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], s["h"], s["D"], s["z"],
                                           dt_bias=s["dt_bias"])
    if case["op"] == "conv_step":
        with torch.no_grad():
            return plh.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], silu=case["silu"])
    if case["op"] == "conv":
        def call():
            return plh.causal_conv(s["x"], s["weight"], s["bias"], s["state"], lengths=s["lengths"], silu=case["silu"])
    else:
        def call():
            return plh.selective_scan(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"], s["h0"],
                                      dt_bias=s["dt_bias"], lengths=s["lengths"])
    if not case["train"]:
        with torch.no_grad():
            return call()
    y, state = call()
    d_state = s["d_h"] if case["op"] == "scan" else s["d_state"]
    grads = torch.autograd.grad((y, state), _given(case, s), (s["d_y"], d_state))
    return (y.detach(), state.detach(), *grads)


# ---- the plain forms ---------------------------------------------------------------------------


def _linear_scan(a, b):
    """y_t = a_t y_{t-1} + b_t along dim 1, by doubling; overwrites its arguments."""
    s, T = 1, a.size(1)
    while s < T:
        nb = b[:, s:] + a[:, s:] * b[:, :-s]
        na = a[:, s:] * a[:, :-s]
        b[:, s:], a[:, s:] = nb, na
        s *= 2
    return b


def _softplus(v):
    return v.clamp(min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _live(s, T):
    if s["lengths"] is None:
        return None
    return (torch.arange(T, device=DEVICE) < s["lengths"].unsqueeze(1)).unsqueeze(-1)


def _plain_scan(s):
    case, T = s["case"], s["case"]["T"]
    dtype = s["u"].dtype
    u, A, Bm, Cm = s["u"].float(), s["A"].float(), s["Bm"].float(), s["Cm"].float()
    raw = s["dt"].float() + s["dt_bias"].float()
    dt = _softplus(raw)
    live = _live(s, T)
    if live is not None:
        u, dt, Bm, Cm = (torch.where(live, v, 0.0) for v in (u, dt, Bm, Cm))
    a = torch.exp(dt.unsqueeze(-1) * A)
    b = (dt * u).unsqueeze(-1) * Bm.unsqueeze(2)
    if s["h0"] is not None:
        b[:, 0] += a[:, 0] * s["h0"]
    h = _linear_scan(a.clone(), b)
    y = (h * Cm.unsqueeze(2)).sum(-1)
    if s["D"] is not None:
        y = y + s["D"].float() * u
    out = y
    if s["z"] is not None:
        z = s["z"].float()
        sz = torch.sigmoid(z)
        out = y * (z * sz)
    if live is not None:
        out = torch.where(live, out, 0.0)
    out, h_n = out.to(dtype), h[:, -1].clone()
    if not case["train"]:
        return out, h_n
    dy = s["d_y"].float()
    if live is not None:
        dy = torch.where(live, dy, 0.0)
    grads = {}
    if s["z"] is not None:
        dz = dy * y * (sz * (1.0 + z * (1.0 - sz)))
        grads["z"] = (dz if live is None else torch.where(live, dz, 0.0)).to(dtype)
        dy = dy * (z * sz)
    if s["D"] is not None:
        grads["D"] = (dy * u).sum((0, 1)).to(s["D"].dtype)
    grads["Cm"] = (h * dy.unsqueeze(-1)).sum(2).to(dtype)
    # G_t = dy_t C_t + a_{t+1} G_{t+1}: the same scan over the reversed time axis
    g = dy.unsqueeze(-1) * Cm.unsqueeze(2)
    g[:, -1] += s["d_h"]
    back = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    g = _linear_scan(back, g.flip(1)).flip(1)
    del back
    if s["h0"] is not None:
        grads["h0"] = a[:, 0] * g[:, 0]
    per_u = (g * Bm.unsqueeze(2)).sum(-1)
    grads["Bm"] = (g * (dt * u).unsqueeze(-1)).sum(2).to(dtype)
    du = dt * per_u
    if s["D"] is not None:
        du = du + dy * s["D"].float()
    first = torch.zeros_like(h[:, :1]) if s["h0"] is None else s["h0"].unsqueeze(1)
    m = g * a * torch.cat([first, h[:, :-1]], 1)
    if live is not None:
        m = torch.where(live.unsqueeze(-1), m, 0.0)
    grads["A"] = (m * dt.unsqueeze(-1)).sum((0, 1)).to(s["A"].dtype)
    d_raw = (u * per_u + (m * A).sum(-1)) * torch.sigmoid(raw)
    if live is not None:
        du, d_raw = torch.where(live, du, 0.0), torch.where(live, d_raw, 0.0)
    grads["u"], grads["dt"] = du.to(dtype), d_raw.to(dtype)
    grads["dt_bias"] = d_raw.sum((0, 1)).to(s["dt_bias"].dtype)
    return (out, h_n, *(grads[name] for name in _LEAVES["scan"] if s[name] is not None))


def _plain_scan_step(s):
    u, Bm, Cm = s["u"].float(), s["Bm"].float(), s["Cm"].float()
    dt = _softplus(s["dt"].float() + s["dt_bias"].float())
    h = torch.exp(dt.unsqueeze(-1) * s["A"].float()) * s["h"] + (dt * u).unsqueeze(-1) * Bm.unsqueeze(1)
    y = (h * Cm.unsqueeze(1)).sum(-1) + s["D"].float() * u
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    return y.to(s["u"].dtype), h


def _plain_conv(s):
    case, T, W = s["case"], s["case"]["T"], s["case"]["W"]
    dtype, w = s["x"].dtype, s["weight"].float()
    x, live = s["x"].float(), _live(s, T)
    if live is not None:
        x = torch.where(live, x, 0.0)
    B, C = x.size(0), x.size(2)
    before = torch.zeros(B, W - 1, C, device=DEVICE) if s["state"] is None else s["state"].float()
    xp = torch.cat([before, x], 1)
    acc = s["bias"].float().expand(B, T, C)
    for k in range(W):
        acc = acc + w[:, k] * xp[:, k:k + T]
    sg = torch.sigmoid(acc)
    y = acc * sg if case["silu"] else acc
    if live is not None:
        y = torch.where(live, y, 0.0)
    at = torch.arange(W - 1, device=DEVICE) + (T if live is None else s["lengths"].unsqueeze(1).long())
    at = at.expand(B, W - 1).unsqueeze(2).expand(B, W - 1, C)
    out, state = y.to(dtype), torch.gather(xp, 1, at).to(dtype)
    if not case["train"]:
        return out, state
    da = s["d_y"].float()
    if case["silu"]:
        da = da * (sg * (1.0 + acc * (1.0 - sg)))
    if live is not None:
        da = torch.where(live, da, 0.0)
    dxp, dw = torch.zeros_like(xp), torch.empty_like(w)
    for k in range(W):
        dxp[:, k:k + T] += w[:, k] * da
        dw[:, k] = (da * xp[:, k:k + T]).sum((0, 1))
    dxp.scatter_add_(1, at, s["d_state"].float())
    dx = dxp[:, W - 1:]
    if live is not None:
        dx = torch.where(live, dx, 0.0)
    grads = (dx.to(dtype), dw.to(s["weight"].dtype), da.sum((0, 1)).to(s["bias"].dtype))
    if s["state"] is not None:
        grads += (dxp[:, :W - 1].to(dtype),)
    return (out, state, *grads)


def _plain_conv_step(s):
    xp = torch.cat([s["state"], s["x"].unsqueeze(1)], 1)
    acc = s["bias"].float() + (xp.float() * s["weight"].float().t()).sum(1)
    y = acc * torch.sigmoid(acc) if s["case"]["silu"] else acc
    return y.to(s["x"].dtype), xp[:, 1:].contiguous()


def _plain_clip(s):
    squares = [g.double().square().sum() for g in s["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return [(g.float() * coef).to(g.dtype) for g in s["grads"]], norm.float()


def run(state):
    if own:
        return _run_own(state)
    plain = {"scan": _plain_scan, "scan_step": _plain_scan_step, "conv": _plain_conv, "conv_step": _plain_conv_step,
             "clip": _plain_clip}
    with torch.no_grad():
        return plain[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------


def _size(name):
    return 4 if name == "float32" else 2


def _steps(case):
    """Steps that a row runs, in the mean."""
    lo, T = case["lo"], case["T"]
    return T if lo == 0 else (min(lo, T) + T) / 2 if lo > 0 else T * (T + 1) / 2 / (T + 1 - lo)


def work(case):
    """Each input read once, each output written once; an exponential, a division or a product counts as one."""
    if case["op"] == "clip":
        shapes, s, v = _clip_shapes(case), _size(case["dtype"]), _size(case["vdtype"])
        n = sum(math.prod(q) for q in shapes)
        return {"bytes": 2.0 * sum(math.prod(q) * (s if len(q) == 2 else v) for q in shapes), "flops": 3.0 * n}
    s, w = _size(case["dtype"]), _size(case["wdtype"])
    if case["op"] == "conv_step":
        n = case["B"] * case["C"]
        return {"bytes": n * s * 2.0 * case["W"] + case["C"] * (case["W"] + 1.0) * w, "flops": n * (2.0 * case["W"] + 5.0)}
    if case["op"] == "conv":
        row = _steps(case) * case["C"] * case["B"]  # elements that are read; outputs are written past a row's length too
        full, edge = case["B"] * case["T"] * case["C"], case["B"] * (case["W"] - 1) * case["C"]
        weights = case["C"] * (case["W"] + 1.0) * w
        nbytes, flops = (row + full + edge * (2 if case["state"] else 1)) * s + weights, row * (2.0 * case["W"] + 5.0)
        if case["train"]:
            nbytes += (row + full + edge * (2 if case["state"] else 1)) * s + weights
            flops += row * (4.0 * case["W"] + 10.0)
        return {"bytes": nbytes, "flops": flops}
    B, D, N, gated = case["B"], case["D"], case["N"], case["gated"]
    weights = (D * N + 2.0 * D) * w
    if case["op"] == "scan_step":
        return {"bytes": B * D * ((4.0 if gated else 3.0) * s + 8.0 * N) + 2.0 * B * N * s + weights,
                "flops": B * D * (7.0 * N + 12.0)}
    row, full = B * _steps(case) * D, B * case["T"] * D
    state = 4.0 * B * D * N * (2 if case["state"] else 1)
    reads = 3 if gated else 2
    both = 2.0 * B * N * s
    nbytes = (row * reads + full) * s + both * _steps(case) + weights + state
    flops = row * (7.0 * N + 12.0)
    if case["train"]:
        nbytes += (row + full * reads) * s + both * case["T"] + weights + state
        flops += row * (16.0 * N + 20.0)
    return {"bytes": nbytes, "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_scan(case, d):
    """Step by step in both directions."""
    B, T, D, N = case["B"], case["T"], case["D"], case["N"]
    if T * (B * D * N / 2e10 + 2.5e-4) > 20.0:
        return None
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    n = d["lengths"] if d["lengths"] is not None else torch.full((B,), T, device=DEVICE)
    on = (torch.arange(T, device=DEVICE).unsqueeze(0) < n.unsqueeze(1)).unsqueeze(2)
    A = d["A"].double()
    pre = d["dt"].double() + d["dt_bias"].double()
    dt = torch.where(on, torch.logaddexp(pre, zero), zero)
    u = torch.where(on, d["u"].double(), zero)
    keep = case["train"]
    h = zero.expand(B, D, N) if d["h0"] is None else d["h0"].double()
    before = torch.empty((T, B, D, N) if keep else 0, dtype=torch.float64, device=DEVICE)
    y = torch.empty(B, T, D, dtype=torch.float64, device=DEVICE)
    b, c = torch.where(on, d["Bm"].double(), zero), torch.where(on, d["Cm"].double(), zero)
    for t in range(T):
        if keep:
            before[t] = h
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[:, :, None] * b[:, t, None, :]
        y[:, t] = torch.matmul(h, c[:, t, :, None])[..., 0]
    if d["D"] is not None:
        y = y + d["D"].double() * u
    if d["z"] is None:
        out = torch.where(on, y, zero)
    else:
        z = torch.where(on, d["z"].double(), zero)
        gate = z / (1.0 + torch.exp(-z))
        out = torch.where(on, y * gate, zero)
    if not keep:
        return out, h
    dy = torch.where(on, d["d_y"].double(), zero)
    grads = {}
    if d["z"] is not None:
        s = 1.0 / (1.0 + torch.exp(-z))
        grads["z"] = dy * y * (s + gate * (1.0 - s))
        dy = dy * gate
    if d["D"] is not None:
        grads["D"] = torch.tensordot(dy * u, torch.ones(B, T, dtype=torch.float64, device=DEVICE), ([0, 1], [0, 1]))
    db, dc = torch.zeros(B, T, N, dtype=torch.float64, device=DEVICE), torch.zeros(B, T, N, dtype=torch.float64, device=DEVICE)
    du, ddt = torch.zeros_like(y), torch.zeros_like(y)
    dA = torch.zeros_like(A)
    back = d["d_h"].double()
    h_after = h
    for t in reversed(range(T)):
        decay = torch.exp(dt[:, t, :, None] * A)
        dc[:, t] = torch.matmul(dy[:, t, None, :], h_after)[:, 0]
        g = back + dy[:, t, :, None] * c[:, t, None, :]
        db[:, t] = torch.matmul((dt[:, t] * u[:, t])[:, None, :], g)[:, 0]
        along = torch.matmul(g, b[:, t, :, None])[..., 0]
        du[:, t], back = dt[:, t] * along, g * decay
        through = back * before[t]
        ddt[:, t] = u[:, t] * along + (through * A).sum(-1)
        dA += (through * dt[:, t, :, None]).sum(0)
        h_after = before[t]
    if d["D"] is not None:
        du = du + dy * d["D"].double()
    ddt = torch.where(on, ddt / (1.0 + torch.exp(-pre)), zero)
    grads.update(u=torch.where(on, du, zero), dt=ddt, A=dA, Bm=torch.where(on, db, zero), Cm=torch.where(on, dc, zero), h0=back,
                 dt_bias=ddt.flatten(0, 1).sum(0))
    return (out, h, *(grads[name] for name in _LEAVES["scan"] if d[name] is not None))


def _exact_scan_step(case, d):
    dt = torch.logaddexp(d["dt"].double() + d["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device=DEVICE))
    h = d["h"].double() * torch.exp(dt[:, :, None] * d["A"].double())
    h += torch.matmul((dt * d["u"].double())[:, :, None], d["Bm"].double()[:, None, :])
    y = torch.matmul(h, d["Cm"].double()[:, :, None])[..., 0] + d["u"].double() * d["D"].double()
    if d["z"] is not None:
        z = d["z"].double()
        y = y * z / (1.0 + torch.exp(-z))
    return y, h


def _exact_conv(case, d):
    """A grouped convolution of torch in 64 bits and its derivatives by autograd."""
    B, T, C, W = case["B"], case["T"], case["C"], case["W"]
    x, w, b = d["x"].double(), d["weight"].double(), d["bias"].double()
    st = torch.zeros(B, W - 1, C, dtype=torch.float64, device=DEVICE) if d["state"] is None else d["state"].double()
    leaves = (x, w, b) if d["state"] is None else (x, w, b, st)
    if case["train"]:
        for t in leaves:
            t.requires_grad_(True)
    n = torch.full((B,), T, device=DEVICE) if d["lengths"] is None else d["lengths"].long()
    on = torch.arange(T, device=DEVICE)[None, :, None] < n[:, None, None]
    line = torch.cat([st, x.masked_fill(~on, 0.0)], 1)
    acc = b.expand(B, T, C)
    for k in range(W):
        acc = torch.addcmul(acc, line.narrow(1, k, T), w.select(1, k))
    y = (acc / (1.0 + torch.exp(-acc)) if case["silu"] else acc).masked_fill(~on, 0.0)
    rows = torch.arange(B, device=DEVICE)[:, None]
    state = line[rows, n[:, None] + torch.arange(W - 1, device=DEVICE)]
    if not case["train"]:
        return y, state
    return (y.detach(), state.detach(), *torch.autograd.grad((y, state), leaves, (d["d_y"].double(), d["d_state"].double())))


def _exact_conv_step(case, d):
    line = torch.cat([d["state"], d["x"][:, None]], 1)
    acc = torch.einsum("bkc,ck->bc", line.double(), d["weight"].double()) + d["bias"].double()
    return (acc / (1.0 + torch.exp(-acc)) if case["silu"] else acc), line[:, 1:].double()


def _exact_clip(case, d):
    total = torch.zeros((), dtype=torch.float64, device=DEVICE)
    for g in d["grads"]:
        v = g.double().flatten()
        total = total + torch.dot(v, v)
    norm = torch.sqrt(total)
    factor = torch.minimum(d["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
    return [g.double() * factor for g in d["grads"]], norm


def exact(case, seed):
    d = _inputs(case, seed)
    return {"scan": _exact_scan, "scan_step": _exact_scan_step, "conv": _exact_conv, "conv_step": _exact_conv_step,
            "clip": _exact_clip}[case["op"]](case, d)
