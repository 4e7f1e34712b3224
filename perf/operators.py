"""What the speed of the block operators is measured on.

A residual block around a recurrence that is parallel over time,

    y = x + dropout(W_o scan(W_g layer_norm(x)))

takes three operators besides its matrix products: the gated linear recurrence (`gated_scan`, and
`gated_scan_step` for one token), `layer_norm` and `dropout_add`.  Inference calls the forward
alone; a training case is a forward and the gradients of everything that it was given.

The plain form computes each from elementary torch operations in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"

# Bytes of one activation tensor of the largest cases.
_MAX_TENSOR = 1 << 28


def listed():
    return [
        # One token of one series in a live forecaster: the smallest call, all latency.
        dict(name="step_one_series", op="step", B=1, H=128, gated=True, dtype="float16"),
        # One token of every series of the benchmark's batch, at its hidden size 512.
        dict(name="step_batch_512", op="step", B=512, H=512, gated=True, dtype="bfloat16"),
        # Scoring the headline batch (512 rows of up to 1000 steps, hidden 128) with ragged rows.
        dict(name="scan_ragged_h128", op="scan", train=False, B=512, T=1000, H=128, gated=True, dtype="float16", lo=200),
        # Two long records in one step of training: few rows, so the time axis has to be split.
        dict(name="scan_train_long", op="scan", train=True, B=2, T=16384, H=640, gated=True, dtype="bfloat16", lo=0),
        # The largest call: a full training batch of a wide block.
        dict(name="scan_train_wide", op="scan", train=True, B=16, T=4096, H=2048, gated=True, dtype="bfloat16", lo=0),
        # A small model over a year of daily values in 32 bits, rows of unequal lengths, some of them empty, no output
        # gate; nothing a multiple of a tile.
        dict(name="scan_train_daily_h60", op="scan", train=True, B=200, T=365, H=60, gated=False, dtype="float32", lo=-40),
        # The norm in front of one token's projections.
        dict(name="norm_one_token", op="norm", train=False, rows=1, D=512, dtype="float16", wdtype="float16"),
        # Training at the headline's sizes: very many short rows.
        dict(name="norm_train_headline", op="norm", train=True, rows=512000, D=128, dtype="float16", wdtype="float16"),
        # Training a wide model in bfloat16 with master weights in 32 bits.
        dict(name="norm_train_wide", op="norm", train=True, rows=16384, D=8192, dtype="bfloat16", wdtype="float32"),
        # An odd width: no row but the first is aligned.
        dict(name="norm_train_odd", op="norm", train=True, rows=7301, D=1001, dtype="float16", wdtype="float16"),
        # The end of a block at the headline's sizes: dropout and the residual.
        dict(name="dropout_train_headline", op="dropout", train=True, shape="512x1000x128", residual=True, p=0.2, dtype="float16"),
        # Dropout on the inputs of a small model, an odd number of elements, no residual.
        dict(name="dropout_train_odd", op="dropout", train=True, shape="200x365x61", residual=False, p=0.1, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, hi):
    """A row length: often 8 times an odd number or a power of two, sometimes any odd number."""
    kind = rng.random()
    if kind < 0.35:
        return 8 * (_log_int(rng, 1, hi // 8 - 1) | 1)
    if kind < 0.65:
        return 1 << rng.randint(5, int(math.log2(hi)))
    return _log_int(rng, 1, hi - 1) | 1


def draw(rng):
    """One more case: rows of 1 to 8192 elements, lengths of 1 to 16384 steps, tensors of up to 256 MiB, every type."""
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    most = _MAX_TENSOR // (4 if dtype == "float32" else 2)
    pick = rng.random()
    train = rng.random() < 0.6
    if pick < 0.15:
        H = _width(rng, 2048)
        if H == 1024:
            H = 1000
        return dict(op="step", B=_log_int(rng, 1, 4096) | 1, H=H, gated=rng.random() < 0.7, dtype=dtype)
    if pick < 0.55:
        H = _width(rng, 2048)
        if H == 1024:
            H = 1000
        T = _log_int(rng, 1, 16384) | 1
        B = _log_int(rng, 1, max(1, min(512, most // (T * H))))
        lo = rng.choice([0, 0, 1 + T // 5, -(T // 8) - 1])
        return dict(op="scan", train=train, B=B, T=T, H=H, gated=rng.random() < 0.7, dtype=dtype, lo=lo)
    if pick < 0.82:
        D = _width(rng, 8192)
        wdtype = rng.choice([dtype, "float32"])
        return dict(op="norm", train=train, rows=_log_int(rng, 1, min(400000, most // D)) | 1, D=D, dtype=dtype,
                    wdtype=wdtype)
    D = _width(rng, 8192)
    shape = f"{_log_int(rng, 1, min(400000, most // D)) | 1}x{D}"
    return dict(op="dropout", train=train, shape=shape, residual=rng.random() < 0.6, p=round(rng.uniform(0.02, 0.6), 3),
                dtype=dtype)


# ---- inputs ------------------------------------------------------------------------------------


def _gates(case, T, rand):
    """[B, T, 3H] (or 2H) logits as a projection gives them: forget gates with a bias per channel from 0 to 6 (memories
    of two to some hundred steps), candidates and output gates around zero."""
    B, H = case["B"], case["H"]
    t = rand(B, T, (3 if case["gated"] else 2) * H)
    t[..., :H] += torch.linspace(0.0, 6.0, H, device=DEVICE)
    return t


def _inputs(case, seed):
    """The tensors of one pass, on the GPU."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def rand(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    d = {}
    if case["op"] == "step":
        d["gates"] = _gates(case, 1, rand)[:, 0].to(dtype).contiguous()
        d["c"] = rand(case["B"], case["H"])
    elif case["op"] == "scan":
        B, T, H = case["B"], case["T"], case["H"]
        d["gates"] = _gates(case, T, rand).to(dtype)
        d["c0"] = rand(B, H)
        # lo = 0: rows of full length; above: lengths from lo to T; below: the same with 1 - lo of T + 1 - lo rows
        # empty in the mean.
        d["lengths"] = None
        if case["lo"] != 0:
            n = torch.randint(min(case["lo"], T), T + 1, (B,), device=DEVICE, generator=gen)
            d["lengths"] = n.clamp(min=0).to(torch.int32)
        if case["train"]:
            d["d_out"], d["d_cn"] = rand(B, T, H).to(dtype), rand(B, H)
    elif case["op"] == "norm":
        rows, D = case["rows"], case["D"]
        wdtype = getattr(torch, case["wdtype"])
        x = rand(rows, D) * (0.5 + torch.rand(D, device=DEVICE, generator=gen)) + 0.5 * rand(D)
        x[:, :: max(1, D // 4)] *= 8.0  # a few columns of a trained model's stream are far larger than the rest
        d["x"] = x.to(dtype)
        d["weight"], d["bias"] = (1.0 + 0.1 * rand(D)).to(wdtype), (0.1 * rand(D)).to(wdtype)
        if case["train"]:
            d["d_y"] = rand(rows, D).to(dtype)
    else:
        shape = [int(n) for n in case["shape"].split("x")]
        d["x"] = rand(*shape).to(dtype)
        d["residual"] = rand(*shape).to(dtype) if case["residual"] else None
        d["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63)
        d["offset"] = seed % 1000003
        if case["train"]:
            d["d_out"] = rand(*shape).to(dtype)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = case
    if case.get("train"):
        for name in ("gates", "c0", "x", "residual", "weight", "bias"):
            if d.get(name) is not None:
                d[name].requires_grad_(True)
    return d


# ---- the framework's operators -----------------------------------------------------------------


def _run_own(s):
    import persistent_lstm_hip_amd as plh

    case = s["case"]
    if case["op"] == "step":
        with torch.no_grad():
            return plh.gated_scan_step(s["gates"], s["c"], output_gate=case["gated"])
    if case["op"] == "scan":
        if not case["train"]:
            with torch.no_grad():
                return plh.gated_scan(s["gates"], s["c0"], lengths=s["lengths"], output_gate=case["gated"])
        out, c_n = plh.gated_scan(s["gates"], s["c0"], lengths=s["lengths"], output_gate=case["gated"])
        grads = torch.autograd.grad((out, c_n), (s["gates"], s["c0"]), (s["d_out"], s["d_cn"]))
        return (out.detach(), c_n.detach(), *grads)
    if case["op"] == "norm":
        if not case["train"]:
            with torch.no_grad():
                return plh.layer_norm(s["x"], s["weight"], s["bias"])
        y = plh.layer_norm(s["x"], s["weight"], s["bias"])
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["d_y"]))
    if not case["train"]:
        with torch.no_grad():
            return plh.dropout_add(s["x"], s["residual"], p=case["p"], seed=s["seed"], offset=s["offset"])
    out = plh.dropout_add(s["x"], s["residual"], p=case["p"], seed=s["seed"], offset=s["offset"])
    wrt = (s["x"],) if s["residual"] is None else (s["x"], s["residual"])
    return (out.detach(), *torch.autograd.grad(out, wrt, s["d_out"]))


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


def _plain_scan(s):
    case, H = s["case"], s["case"]["H"]
    dtype, T = s["gates"].dtype, s["case"]["T"]
    z = s["gates"].float()
    a, r, g = torch.sigmoid(z[..., :H]), torch.sigmoid(-z[..., :H]), z[..., H:2 * H]
    o = torch.sigmoid(z[..., 2 * H:]) if case["gated"] else None
    live = None
    b = r * g
    if s["lengths"] is not None:
        live = (torch.arange(T, device=DEVICE) < s["lengths"].unsqueeze(1)).unsqueeze(-1)
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    b[:, 0] += a[:, 0] * s["c0"]
    c = _linear_scan(a.clone(), b)
    h = c * o if case["gated"] else c
    if live is not None:
        h = torch.where(live, h, 0.0)
    out, c_n = h.to(dtype), c[:, -1].clone()
    if not case["train"]:
        return out, c_n
    dh = s["d_out"].float()
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    dd = dh * o if case["gated"] else dh.clone()
    dd[:, -1] += s["d_cn"]
    # D_t = dd_t + a_{t+1} D_{t+1}: the same scan over the reversed time axis
    back = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    dd = _linear_scan(back, dd.flip(1)).flip(1)
    prev = torch.cat([s["c0"].unsqueeze(1), c[:, :-1]], 1)
    parts = [dd * (prev - g) * a * r, dd * r]
    if case["gated"]:
        parts.append(dh * c * o * (1.0 - o))
    dz = torch.cat(parts, -1)
    if live is not None:
        dz = torch.where(live, dz, 0.0)
    return out, c_n, dz.to(dtype), a[:, 0] * dd[:, 0]


def _plain_step(s):
    H = s["case"]["H"]
    z = s["gates"].float()
    c = torch.sigmoid(z[:, :H]) * s["c"] + torch.sigmoid(-z[:, :H]) * z[:, H:2 * H]
    h = torch.sigmoid(z[:, 2 * H:]) * c if s["case"]["gated"] else c
    return h.to(s["gates"].dtype), c


def _plain_norm(s):
    x, w = s["x"].float(), s["weight"].float()
    xc = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh = xc * r
    y = (xh * w + s["bias"].float()).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y
    dy = s["d_y"].float()
    dw, db = (dy * xh).sum(0), dy.sum(0)
    dxh = dy * w
    dx = r * (dxh - dxh.mean(-1, keepdim=True) - xh * (dxh * xh).mean(-1, keepdim=True))
    return y, dx.to(s["x"].dtype), dw.to(s["weight"].dtype), db.to(s["bias"].dtype)


def _philox_words(groups, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) of the counters (group, offset) under the key `seed`, as four
    int64 tensors of 32-bit values."""
    m32 = 0xFFFFFFFF
    c0, c1 = groups & m32, groups >> 32
    c2, c3 = torch.full_like(groups, offset & m32), torch.full_like(groups, offset >> 32)
    k0, k1 = seed & m32, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (mod 2^64: the high word's bits survive the sign)
        c0, c1, c2, c3 = ((p1 >> 32) & m32) ^ c1 ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c3 ^ k1, p0 & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return c0, c1, c2, c3


def _plain_keep(shape, k, seed, offset):
    """Which elements stay: element e of the flattened tensor has the 16 bits e % 8 of group e / 8's four words."""
    n = math.prod(shape)
    words = _philox_words(torch.arange((n + 7) // 8, device=DEVICE), seed, offset)
    halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
    return (torch.stack(halves, 1).flatten()[:n] >= k).view(shape)


def _plain_dropout(s):
    x = s["x"].float()
    k = int(math.floor(s["case"]["p"] * 65536 + 0.5))
    keep, scale = _plain_keep(x.shape, k, s["seed"], s["offset"]), 65536.0 / (65536 - k)
    out = torch.where(keep, x * scale, 0.0)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = out.to(s["x"].dtype)
    if not s["case"]["train"]:
        return out
    keep = _plain_keep(x.shape, k, s["seed"], s["offset"])
    dx = torch.where(keep, s["d_out"].float() * scale, 0.0).to(s["x"].dtype)
    return (out, dx) if s["residual"] is None else (out, dx, s["d_out"])


def run(state):
    if own:
        return _run_own(state)
    plain = {"scan": _plain_scan, "step": _plain_step, "norm": _plain_norm, "dropout": _plain_dropout}
    with torch.no_grad():
        return plain[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------


def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    """Each input read once, each output written once; an exponential, a division or a product counts as one."""
    s = _size(case["dtype"])
    if case["op"] == "step":
        n, parts = case["B"] * case["H"], 3 if case["gated"] else 2
        return {"bytes": n * ((parts + 1) * s + 8.0), "flops": 10.0 * n}
    if case["op"] == "scan":
        B, T, H, parts = case["B"], case["T"], case["H"], 3 if case["gated"] else 2
        lo = case["lo"]
        steps = T if lo == 0 else (lo + T) / 2 if lo > 0 else T * (T + 1) / 2 / (T + 1 - lo)
        n = B * steps * H  # elements that are read; outputs are written past a row's length too
        full = B * T * H
        nbytes, flops = (n * parts + full) * s + 8.0 * B * H, 10.0 * n
        if case["train"]:
            nbytes += (n + full * parts) * s + 8.0 * B * H
            flops += 20.0 * n
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "norm":
        n, w = case["rows"] * case["D"], _size(case["wdtype"])
        if not case["train"]:
            return {"bytes": 2.0 * n * s + 2.0 * case["D"] * w, "flops": 8.0 * n}
        return {"bytes": 4.0 * n * s + 4.0 * case["D"] * w, "flops": 20.0 * n}
    n = math.prod(int(v) for v in case["shape"].split("x"))
    tensors = (3 if case["residual"] else 2) + (2 if case["train"] else 0)
    return {"bytes": float(tensors * n * s), "flops": (30.0 if case["train"] else 15.0) * n}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _exact_scan(case, d):
    """Step by step in both directions."""
    B, T, H = case["B"], case["T"], case["H"]
    z = d["gates"].double()
    a, g = 1.0 / (1.0 + torch.exp(-z[..., :H])), z[..., H:2 * H]
    s = 1.0 / (1.0 + torch.exp(-z[..., 2 * H:])) if case["gated"] else torch.ones_like(a)
    n = d["lengths"] if d["lengths"] is not None else torch.full((B,), T, device=DEVICE)
    c = d["c0"].double()
    seq = torch.empty(T, B, H, dtype=torch.float64, device=DEVICE)
    for t in range(T):
        on = (n > t).unsqueeze(1)
        c = torch.where(on, g[:, t] + a[:, t] * (c - g[:, t]), c)
        seq[t] = c
    seq = seq.transpose(0, 1)
    on = (torch.arange(T, device=DEVICE).unsqueeze(0) < n.unsqueeze(1)).unsqueeze(2)
    out = torch.where(on, s * seq, 0.0)
    if not case["train"]:
        return out, c
    dh, back = d["d_out"].double(), d["d_cn"].double()
    dz = torch.zeros_like(z)
    for t in reversed(range(T)):
        live = on[:, t]
        dc = back + torch.where(live, s[:, t] * dh[:, t], 0.0)
        before = seq[:, t - 1] if t else d["c0"].double()
        at = a[:, t]
        dz[:, t, :H] = torch.where(live, dc * (before - g[:, t]) * at * (1.0 - at), 0.0)
        dz[:, t, H:2 * H] = torch.where(live, dc * (1.0 - at), 0.0)
        back = torch.where(live, dc * at, back)
    if case["gated"]:
        dz[..., 2 * H:] = torch.where(on, dh * seq * s * (1.0 - s), 0.0)
    return out, c, dz, back


def _exact_norm(case, d):
    x, w, b = d["x"].double(), d["weight"].double(), d["bias"].double()
    if not case["train"]:
        var, mu = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        return (x - mu) / torch.sqrt(var + 1e-5) * w + b
    for t in (x, w, b):
        t.requires_grad_(True)
    var, mu = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    y = (x - mu) / torch.sqrt(var + 1e-5) * w + b
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), d["d_y"].double()))


def _exact_keep(n, k, seed, offset):
    """The generator again, on the host in unsigned 64-bit arithmetic."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    i = np.arange((n + 7) // 8, dtype=u)
    ctr = [i & low, i >> u(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        left, right = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(right >> u(32)) ^ ctr[1] ^ u(key[0]), right & low, (left >> u(32)) ^ ctr[3] ^ u(key[1]), left & low]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    bits = np.empty((i.size, 8), dtype=np.uint16)
    for j in range(8):
        bits[:, j] = (ctr[j // 2] >> u(16 * (j % 2))).astype(np.uint16)
    return torch.from_numpy(bits.reshape(-1)[:n] >= k).to(DEVICE)


def _exact_dropout(case, d):
    x = d["x"].double()
    k = int(math.floor(case["p"] * 65536 + 0.5))
    gain = _exact_keep(x.numel(), k, d["seed"], d["offset"]).view(x.shape).double() / (1.0 - k / 65536)
    out = x * gain
    if d["residual"] is not None:
        out = out + d["residual"].double()
    if not case["train"]:
        return out
    dx = d["d_out"].double() * gain
    return (out, dx) if d["residual"] is None else (out, dx, d["d_out"].double())


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "step":
        H = case["H"]
        z, c = d["gates"].double(), d["c"].double()
        g = z[:, H:2 * H]
        c = g + (c - g) / (1.0 + torch.exp(-z[:, :H]))
        return (c / (1.0 + torch.exp(-z[:, 2 * H:])) if case["gated"] else c), c
    return {"scan": _exact_scan, "norm": _exact_norm, "dropout": _exact_dropout}[case["op"]](case, d)
