"""The block operators on the GPU against their formulas in 64 bits.

Bounds.  U = 2^-24.  A logistic function and its complement are within 8 U of their values, relative.  A state is a
sum over the steps that it still remembers, each with a few such factors, so after t steps it is within
16 U (t + 8) of the largest state or input; the gradient that runs backwards through the states likewise, and a gate's
gradient is a product of the two.  A normalised value carries the row mean's error, 16 U times the ratio of the row's
largest value to its deviation.  Everything is rounded once more to the activations' type.
"""
from __future__ import annotations

import pytest
import torch

import ops_plain as plain
import persistent_lstm_hip_amd as P
from ops_plain import U, assert_within

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = [F16, BF16, F32]


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _gates(B, T, H, gated, dtype, seed=0):
    z = _rand(B, T, (3 if gated else 2) * H, seed=seed)
    z[..., :H] += torch.linspace(-2.0, 6.0, H)
    return z.to(dtype)


# (B, T, H): one of everything; no steps; odd; one and several tiles; a time axis that is split; many rows; a few steps;
# rows of few channels; as many rows as it takes for slabs of either width, split in both directions, in one, or not;
# one tile of each size
SCAN_SHAPES = [(1, 1, 1), (3, 0, 5), (0, 4, 3), (2, 64, 64), (2, 65, 60), (5, 129, 7), (1, 2500, 24), (2, 700, 130),
               (70, 33, 61), (300, 5, 200), (9, 8, 51), (9, 9, 51), (40, 2, 2), (2, 300, 3),
               (33, 70, 1000), (24, 130, 1000), (8, 700, 402), (45, 200, 264), (75, 70, 512),
               (3, 16, 260), (30, 12, 70), (5, 17, 130), (2, 32, 517), (1, 63, 1030)]


def _lengths(kind, B, T):
    if kind is None:
        return None
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B + T))
    n[: max(1, B // 4)] = 0
    if B > 1:
        n[-1] = T
    return n


def _check_scan(gates, c0, lengths, gated, dev_gates=None, dev_lengths=None, what=""):
    """Forward and gradients of the device's gates (default: a copy of `gates`) against the formulas."""
    B, T, width = gates.shape
    H = width // (3 if gated else 2)
    dtype = gates.dtype
    dh, dc = _rand(B, T, H, seed=5).to(dtype), _rand(B, H, seed=6)
    want = plain.scan(gates, c0, lengths, gated, dh, dc)
    z = (gates.cuda() if dev_gates is None else dev_gates).requires_grad_(True)
    c = None if c0 is None else c0.cuda().requires_grad_(True)
    n = lengths if dev_lengths is None else dev_lengths
    with torch.no_grad():
        out0, cn0 = P.gated_scan(z, c, lengths=n, output_gate=gated)
    out, c_n = P.gated_scan(z, c, lengths=n, output_gate=gated)
    assert torch.equal(out, out0) and torch.equal(c_n, cn0), f"{what}: inference and training differ"
    wrt = (z,) if c is None else (z, c)
    grads = torch.autograd.grad((out, c_n), wrt, (dh.cuda(), dc.cuda()))
    g64 = plain.d64(gates)[..., H:2 * H]
    g64 = g64[g64.abs() < 100]  # (what lies past a row may be anything)
    top = max([1.0, g64.abs().max().item() if g64.numel() else 0.0] + ([] if c0 is None or not c0.numel()
                                                                       else [c0.abs().max().item()]))
    tol = 16 * U * (T + 8) * top
    most = want[4]
    assert out.dtype == dtype and c_n.dtype == F32 and grads[0].dtype == dtype
    assert_within(out, want[0], tol, dtype, f"{what} out")
    assert_within(c_n, want[1], tol, F32, f"{what} c_n")
    assert_within(grads[0], want[2], 2 * tol * (1 + most) * 2, dtype, f"{what} d_gates")
    if c0 is not None:
        assert_within(grads[1], want[3], 16 * U * (T + 8) * max(1.0, most), F32, f"{what} d_c0")
    return out, c_n, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("B,T,H", SCAN_SHAPES)
def test_scan(gpu, B, T, H, gated, dtype):
    _say(f"scan {B} {T} {H} gated={gated} {dtype}")
    _check_scan(_gates(B, T, H, gated, dtype), _rand(B, H, seed=1), None, gated, what="full")
    _check_scan(_gates(B, T, H, gated, dtype, 7), None, _lengths("ragged", B, T), gated, what="ragged")


@pytest.mark.parametrize("B,T,H", [(2, 3000, 700), (2, 4100, 1000)])
def test_scan_rows_that_end_anywhere_in_a_segment(gpu, B, T, H):
    """A time axis that is split into segments of three tiles, or of five: all rows end in each tile of a segment in
    turn, and the gradient of c_n comes through the steps past them as it is."""
    _say(f"scan segments' ends {B} {T} {H}")
    z, c0 = _gates(B, T, H, True, BF16), _rand(B, H, seed=1)
    for tiles in range(10, 16):
        _check_scan(z, c0, torch.full((B,), 64 * tiles + 1), True, what=f"{64 * tiles + 1} steps")


@pytest.mark.parametrize("place", ["list", "int32 on the device", "int64 on the device"])
def test_scan_lengths_from_anywhere(gpu, place):
    _say(f"scan lengths {place}")
    B, T, H = 4, 70, 24
    n = torch.tensor([0, 70, 1, 64])
    dev = {"list": n.tolist(), "int32 on the device": n.int().cuda(), "int64 on the device": n.cuda()}[place]
    _check_scan(_gates(B, T, H, True, F16), _rand(B, H, seed=1), n, True, dev_lengths=dev, what=place)


def test_scan_clamps_lengths_on_the_device(gpu):
    _say("scan clamped lengths")
    z = _gates(3, 20, 8, True, F32).cuda()
    got = P.gated_scan(z, lengths=torch.tensor([-5, 1 << 30, 7], device="cuda"))
    want = P.gated_scan(z, lengths=[0, 20, 7])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = P.gated_scan(z, lengths=torch.tensor([-5, 1 << 30, 7], device="cuda", dtype=torch.int32))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), torch.finfo(F16).min])
def test_scan_ignores_what_lies_past_a_row(gpu, junk):
    _say(f"scan padding {junk}")
    B, T, H = 5, 130, 20
    n = torch.tensor([0, 130, 64, 65, 3])
    z = _gates(B, T, H, True, F16)
    past = torch.arange(T).unsqueeze(0) >= n.unsqueeze(1)
    z[past] = junk
    out, _, grads = _check_scan(z, _rand(B, H, seed=1), n, True, what="padding")
    assert (out.cpu()[past] == 0).all() and (grads[0].cpu()[past] == 0).all()
    # nor does the gradient of an output that is not there
    z2 = z.cuda().requires_grad_(True)
    d = _rand(B, T, H, seed=5).to(F16)
    d[past] = float("nan")
    got, = torch.autograd.grad(P.gated_scan(z2, lengths=n)[0], z2, d.cuda())
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_gates_at_their_limits(gpu, dtype):
    """A forget gate of +inf keeps the state, of -inf or the type's lowest value takes the candidate, exactly."""
    _say(f"scan limits {dtype}")
    H = 8
    z = torch.zeros(1, 4, 3 * H)
    low = torch.finfo(dtype).min
    z[0, :, :H] = torch.tensor([[float("inf")], [float("-inf")], [low], [torch.finfo(dtype).max]])
    z[0, :, H:2 * H] = torch.tensor([[1.0], [2.0], [3.0], [4.0]])
    z[0, :, 2 * H:] = float("inf")
    out, c_n = P.gated_scan(z.to(dtype).cuda(), torch.full((1, H), 5.0, device="cuda"))
    assert out[0, :, 0].tolist() == [5.0, 2.0, 3.0, 3.0] and c_n[0, 0].item() == 3.0


def test_scan_nan_stays_in_its_channel(gpu):
    _say("scan nan")
    z = _gates(2, 200, 16, True, F32)
    z[1, 70, 3] = float("nan")
    out, c_n = P.gated_scan(z.cuda())
    bad = torch.isnan(out.cpu())
    want = torch.zeros(2, 200, 16, dtype=torch.bool)
    want[1, 70:, 3] = True
    assert torch.equal(bad, want) and torch.isnan(c_n.cpu())[1, 3] and int(torch.isnan(c_n).sum()) == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [8, 12, 10, 9])
@pytest.mark.parametrize("layout", ["time-major", "slice of columns", "every second step", "odd start", "one row for all"])
def test_scan_strides(gpu, layout, H, dtype):
    _say(f"scan strides {layout} H={H} {dtype}")
    B, T, W = 3, 67, 3 * H
    z = _gates(B, T, H, True, dtype)
    if layout == "time-major":
        dev = z.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    elif layout == "slice of columns":
        wide = torch.zeros(B, T, W + 7, dtype=dtype)
        wide[..., 4:4 + W] = z
        dev = wide.cuda()[..., 4:4 + W]
    elif layout == "every second step":
        wide = torch.zeros(B, 2 * T, W, dtype=dtype)
        wide[:, ::2] = z
        dev = wide.cuda()[:, ::2]
    elif layout == "odd start":
        flat = torch.zeros(1 + z.numel(), dtype=dtype)
        flat[1:] = z.flatten()
        dev = flat.cuda()[1:].view(B, T, W)
    else:
        z = z[:1].expand(B, T, W)
        dev = z[:1].cuda().expand(B, T, W)
    assert torch.equal(dev.cpu(), z)
    _check_scan(z, _rand(B, H, seed=1), None, True, dev_gates=dev.detach(), what=layout)


def test_scan_columns_that_are_not_dense(gpu):
    _say("scan non-dense columns")
    z = _gates(2, 9, 4, True, F32)
    dev = z.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    assert torch.equal(P.gated_scan(dev)[0], P.gated_scan(z.cuda())[0])


def test_scan_is_the_same_from_call_to_call_and_on_other_streams(gpu):
    _say("scan repeat, stream")
    z, c0 = _gates(2, 3000, 96, True, BF16).cuda(), _rand(2, 96, seed=1).cuda()
    want = P.gated_scan(z, c0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = P.gated_scan(z, c0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        with torch.cuda.stream(s):
            other = P.gated_scan(z, c0)
        s.synchronize()
        assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])


def test_scan_gradients_of_one_output_alone(gpu):
    _say("scan partial gradients")
    z = _gates(2, 70, 12, True, F32)
    c0, dh, dc = _rand(2, 12, seed=1), _rand(2, 70, 12, seed=5), _rand(2, 12, seed=6)
    zd, cd = z.cuda().requires_grad_(True), c0.cuda().requires_grad_(True)
    tol = 16 * U * 78 * 40
    for a, b in ((dh, None), (None, dc)):
        out, c_n = P.gated_scan(zd, cd)
        outs, ds = ((out,), (a.cuda(),)) if b is None else ((c_n,), (b.cuda(),))
        got = torch.autograd.grad(outs, (zd, cd), ds)
        want = plain.scan(z, c0, None, True, torch.zeros_like(dh) if a is None else a, b)
        assert_within(got[0], want[2], tol, F32, "d_gates")
        assert_within(got[1], want[3], tol, F32, "d_c0")
    # a gradient with strides of its own, and a state that needs none
    out, _ = P.gated_scan(zd, cd.detach())
    got, = torch.autograd.grad(out, zd, dh.transpose(0, 1).contiguous().cuda().transpose(0, 1))
    assert_within(got, plain.scan(z, c0, None, True, dh, None)[2], tol, F32, "strided d_out")


def test_scan_state_in_half_precision(gpu):
    _say("scan fp16 state")
    z, c0 = _gates(2, 10, 8, True, F16).cuda(), _rand(2, 8, seed=1).half()
    c = c0.cuda().requires_grad_(True)
    _, c_n = P.gated_scan(z, c)
    assert c_n.dtype == F32
    g, = torch.autograd.grad(c_n.sum(), c)
    assert g.dtype == F16
    assert torch.equal(c_n, P.gated_scan(z, c0.float().cuda())[1])


def test_scan_in_pieces_is_the_scan(gpu):
    _say("scan pieces")
    z, c = _gates(3, 200, 20, True, F32).cuda(), None
    whole = P.gated_scan(z)
    outs = []
    for lo, hi in ((0, 1), (1, 65), (65, 65), (65, 200)):
        out, c = P.gated_scan(z[:, lo:hi], c)
        outs.append(out)
    tol = 16 * U * 208 * 6
    assert_within(torch.cat(outs, 1), whole[0].cpu().double(), tol, F32, "pieces")
    assert_within(c, whole[1].cpu().double(), tol, F32, "pieces' state")


def test_scan_beyond_32_bits(gpu):
    """More than 2^31 elements of gates: the last row against itself alone."""
    _say("scan beyond 32 bits")
    B, T, H = 3, 400001, 600
    row = torch.randn(1, 20000, 3 * H, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    z = torch.zeros(B, T, 3 * H, dtype=F16, device="cuda")
    z[2, -20000:] = row[0]
    z[2, :-20000, :H] = 60000.0  # keeps the state: c0 arrives at the row's end
    c0 = torch.randn(B, H, device="cuda")
    out, c_n = P.gated_scan(z, c0)
    want, want_c = P.gated_scan(row, c0[2:])
    tol = 16 * U * 400 * 6  # (what a state of these gates still remembers)
    want = want.double().cpu()
    assert_within(out[2:, -20000:], want, tol + 2.0**-11 * want.abs(), F16, "tail")
    assert_within(c_n[2:], want_c.double().cpu(), tol, F32, "c_n")
    del out
    z.requires_grad_(True)
    row.requires_grad_(True)
    d = torch.randn(1, 20000, H, device="cuda").half()
    dz, = torch.autograd.grad(P.gated_scan(z, c0)[0][2:, -20000:], z, d)
    dr, = torch.autograd.grad(P.gated_scan(row, c0[2:])[0], row, d)
    dr = dr.double().cpu()
    assert_within(dz[2:, -20000:], dr, tol * 40 + 2.0**-11 * dr.abs(), F16, "d_gates tail")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,gated", [(1, 1, True), (1, 128, True), (3, 7, False), (512, 60, True), (5, 514, False),
                                       (0, 4, True)])
def test_scan_step(gpu, B, H, gated, dtype):
    _say(f"step {B} {H} {gated} {dtype}")
    z, c0 = _gates(B, 1, H, gated, dtype)[:, 0], _rand(B, H, seed=1)
    want, want_c = plain.scan(z.unsqueeze(1), c0, None, gated)
    c = c0.cuda()
    out, c1 = P.gated_scan_step(z.cuda(), c, output_gate=gated)
    assert torch.equal(c.cpu(), c0)
    tol = 16 * U * 9 * 6
    assert_within(out, want[:, 0], tol, dtype, "out")
    assert_within(c1, want_c, tol, F32, "c")
    wide = torch.zeros(B, z.shape[1] + 3, dtype=dtype, device="cuda")
    wide[:, 1:-2] = z.cuda()
    out2, c2 = P.gated_scan_step(wide[:, 1:-2], c, output_gate=gated, inplace=True)
    assert c2 is c and torch.equal(c2, c1) and torch.equal(out2, out)


# ---- layer norm -----------------------------------------------------------------------------------

# (rows, cols): one element; odd; every way to share a row; rows too long for registers; no rows; many rows
NORM_SHAPES = [(1, 1), (3, 7), (5, 60), (4, 64), (33, 128), (9, 250), (7, 1001), (3, 1024), (3, 2056), (2, 4096),
               (2, 4100), (2, 8192), (2, 16384), (2, 16392), (2, 5001), (3, 33000), (0, 16), (5000, 24), (4099, 8)]


def _check_norm(x, weight, bias, eps=1e-5, dev=None, what=""):
    rows, cols = x.shape
    dtype = x.dtype
    dy = _rand(rows, cols, seed=8).to(dtype)
    want = plain.norm(x, weight, bias, eps, dy)
    leaves = [(x.cuda() if dev is None else dev).requires_grad_(True)]
    params = [None if t is None else t.cuda().requires_grad_(True) for t in (weight, bias)]
    with torch.no_grad():
        y0 = P.layer_norm(leaves[0], *params, eps=eps)
    y = P.layer_norm(leaves[0], *params, eps=eps)
    assert torch.equal(y, y0), f"{what}: inference and training differ"
    wrt = leaves + [t for t in params if t is not None]
    grads = list(torch.autograd.grad(y, wrt, dy.cuda()))
    if not rows:
        assert y.shape == x.shape and all(not g.any() for g in grads)
        return
    x64 = plain.d64(x)
    std = (x64.var(1, unbiased=False, keepdim=True) + eps).sqrt()
    w64 = torch.ones(cols, dtype=torch.float64) if weight is None else plain.d64(weight)
    xh = (x64 - x64.mean(1, keepdim=True)) / std
    err = 16 * U * (x64.abs().amax(1, keepdim=True) / std + xh.abs() + 1)  # of a normalised value
    assert_within(y, want[0], err * w64.abs() + 2 * U * want[0].abs(), dtype, f"{what} y")
    v = plain.d64(dy) * w64
    top, worst = v.abs().amax(1, keepdim=True), err.amax(1, keepdim=True)
    tol = (16 * U * top * (1 + xh.abs().amax(1, keepdim=True)) ** 2 + worst * top * (2 + xh.abs())) / std
    assert_within(grads[0], want[1], tol, dtype, f"{what} d_x")
    dy64 = plain.d64(dy)
    if weight is not None:
        tol = (dy64.abs() * (128 * U * xh.abs() + err)).sum(0)
        assert_within(grads[1], want[2], tol, weight.dtype, f"{what} d_weight")
    if bias is not None:
        assert_within(grads[-1], want[3], 128 * U * dy64.abs().sum(0), bias.dtype, f"{what} d_bias")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_norm(gpu, rows, cols, dtype):
    _say(f"norm {rows} {cols} {dtype}")
    x = (2.0 * _rand(rows, cols, seed=2) + 0.5).to(dtype)
    w, b = (1 + 0.3 * _rand(cols, seed=3)), _rand(cols, seed=4)
    _check_norm(x, w.to(dtype), b.to(dtype), what="all")
    _check_norm(x, w, None, what="fp32 weight, no bias")
    _check_norm(x, None, b, what="fp32 bias, no weight")
    _check_norm(x, None, None, what="neither")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 72, 100, 101, 5001])
@pytest.mark.parametrize("layout", ["slice", "odd start", "one row for all", "transposed"])
def test_norm_strides(gpu, layout, cols, dtype):
    _say(f"norm strides {layout} {cols} {dtype}")
    rows = 6
    x = _rand(rows, cols, seed=2).to(dtype)
    if layout == "slice":
        wide = torch.zeros(rows, cols + 8, dtype=dtype)
        wide[:, 3:3 + cols] = x
        dev = wide.cuda()[:, 3:3 + cols]
    elif layout == "odd start":
        flat = torch.zeros(1 + x.numel(), dtype=dtype)
        flat[1:] = x.flatten()
        dev = flat.cuda()[1:].view(rows, cols)
    elif layout == "transposed":
        dev = x.t().contiguous().cuda().t()
    else:
        x = x[:1].expand(rows, cols)
        dev = x[:1].cuda().expand(rows, cols)
    _check_norm(x, _rand(cols, seed=3), _rand(cols, seed=4), dev=dev.detach(), what=layout)


def test_norm_of_more_dimensions(gpu):
    _say("norm dimensions")
    x = _rand(4, 5, 24, seed=2).cuda()
    w = _rand(24, seed=3).cuda()
    want = P.layer_norm(x.reshape(20, 24), w).view(4, 5, 24)
    assert torch.equal(P.layer_norm(x, w), want)
    swapped = x.transpose(0, 1).requires_grad_(True)
    y = P.layer_norm(swapped, w)
    assert torch.equal(y, want.transpose(0, 1))
    g, = torch.autograd.grad(y.sum(), swapped)
    assert g.shape == swapped.shape
    one = _rand(24, seed=5).cuda()
    assert torch.equal(P.layer_norm(one, w), P.layer_norm(one.unsqueeze(0), w)[0])


def test_norm_reads_rows_where_they_are(gpu):
    """Of what it may read in place the operator makes no copy: one allocation, the output's."""
    _say("norm copies")
    big = torch.randn(600, 1100, device="cuda")
    cube = torch.randn(30, 20, 1000, device="cuda")
    for x, copies in ((big[:, 50:1050], 0), (big[::2, :1000], 0), (cube, 0), (cube[:, :10], 1), (big.t(), 1)):
        y = P.layer_norm(x)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = P.layer_norm(x, eps=1e-5)
        peak = torch.cuda.max_memory_allocated() - before
        assert y.nelement() * 4 * (1 + copies) <= peak < y.nelement() * 4 * (2 + copies), (x.shape, x.stride())


@pytest.mark.parametrize("dtype,mean", [(F32, 1000.0), (F16, 1000.0), (BF16, 100.0)])
def test_norm_of_a_large_mean(gpu, dtype, mean):
    _say(f"norm mean {mean} {dtype}")
    for cols in (96, 1000, 9001):
        _check_norm((_rand(5, cols, seed=2) + mean).to(dtype), _rand(cols, seed=3), None, what=f"mean {mean}")


def test_norm_of_rows_that_do_not_vary(gpu):
    """Constant rows normalise to the bias, rows with an infinity or a NaN to NaN, and no other row is touched."""
    _say("norm special rows")
    x = _rand(6, 40, seed=2)
    x[1] = 3.0
    x[3, 7] = float("inf")
    x[4, 0] = float("nan")
    b = _rand(40, seed=4).cuda()
    y = P.layer_norm(x.cuda(), None, b)
    assert torch.equal(y[1], b)
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all() and torch.isfinite(y[[0, 1, 2, 5]]).all()
    assert torch.equal(y[[0, 2, 5]], P.layer_norm(x[[0, 2, 5]].cuda(), None, b))


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("cols", [64, 33000])
def test_norm_gradients_of_some(gpu, need, cols):
    _say(f"norm gradients {need} {cols}")
    ts = [_rand(9, cols, seed=2).cuda(), _rand(cols, seed=3).cuda(), _rand(cols, seed=4).cuda()]
    dy = _rand(9, cols, seed=8).cuda()
    whole = torch.autograd.grad(P.layer_norm(*[t.requires_grad_(True) for t in ts]), ts, dy)
    some = [t.detach().requires_grad_(bool(n)) for t, n in zip(ts, need)]
    wrt = [t for t, n in zip(some, need) if n]
    got = torch.autograd.grad(P.layer_norm(*some), wrt, dy)
    for g, w in zip(got, [w for w, n in zip(whole, need) if n]):
        assert torch.equal(g, w)


def test_norm_beyond_32_bits(gpu):
    _say("norm beyond 32 bits")
    rows, cols = 1 << 16, 33288  # 2.18e9 elements
    x = torch.zeros(rows, cols, dtype=F16, device="cuda")
    tail = torch.randn(8, cols, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    x[-8:] = tail
    w = torch.rand(cols, device="cuda")
    x.requires_grad_(True)
    y = P.layer_norm(x, w)
    t = tail.clone().requires_grad_(True)
    yt = P.layer_norm(t, w)
    assert torch.equal(y[-8:], yt)
    gx, = torch.autograd.grad(y, x, y.detach())
    gt, = torch.autograd.grad(yt, t, yt.detach())
    assert torch.equal(gx[-8:], gt)


# ---- dropout --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 4100])
@pytest.mark.parametrize("p,seed,offset", [(0.0, 1, 0), (0.5, 0, 0), (0.1, 2**64 - 3, 2**40 + 5), (0.999, -7, 3), (1.0, 5, 1)])
def test_dropout(gpu, n, p, seed, offset, dtype):
    _say(f"dropout {n} {p} {dtype}")
    x, res, d = (_rand(n, seed=i).to(dtype) for i in (1, 2, 3))
    k = int(p * 65536 + 0.5)
    stay = plain.keep(0, n, k, seed, offset)
    scale = 0.0 if k == 65536 else 65536 / (65536 - k)
    for r in (None, res):
        xd = x.cuda().requires_grad_(True)
        rd = None if r is None else r.cuda().requires_grad_(True)
        out = P.dropout_add(xd, rd, p=p, seed=seed, offset=offset)
        want = torch.where(stay, plain.d64(x) * scale, 0.0) + (0.0 if r is None else plain.d64(r))
        assert_within(out, want, 4 * U * (plain.d64(x).abs() * scale + 4), dtype, "out")
        gone = torch.zeros(n, dtype=dtype) if r is None else r
        assert torch.equal(out.detach().cpu()[~stay], gone[~stay])
        grads = torch.autograd.grad(out, (xd,) if rd is None else (xd, rd), d.cuda())
        assert_within(grads[0], torch.where(stay, plain.d64(d) * scale, 0.0), 4 * U * plain.d64(d).abs() * scale, dtype,
                      "d_x")
        assert (grads[0].cpu()[~stay] == 0).all()
        if rd is not None:
            assert torch.equal(grads[1].cpu(), d)


def test_dropout_drops_infinity_and_nan(gpu):
    _say("dropout inf nan")
    x = torch.full((4096,), float("nan"))
    x[::2] = float("inf")
    stay = plain.keep(0, 4096, 32768, 9, 2)
    out = P.dropout_add(x.cuda(), p=0.5, seed=9, offset=2).cpu()
    assert (out[~stay] == 0).all() and not torch.isfinite(out[stay]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_masks_do_not_depend_on_strides(gpu, dtype):
    _say(f"dropout strides {dtype}")
    x = _rand(37, 51, seed=1).to(dtype)
    want = P.dropout_add(x.cuda(), p=0.3, seed=4)
    assert torch.equal(P.dropout_add(x.t().contiguous().cuda().t(), p=0.3, seed=4), want)
    flat = torch.zeros(1 + x.numel(), dtype=dtype, device="cuda")
    flat[1:] = x.flatten().cuda()
    odd = flat[1:].view(37, 51)
    assert torch.equal(P.dropout_add(odd, p=0.3, seed=4), want)
    res = _rand(37, 51, seed=2).to(dtype).cuda()
    assert torch.equal(P.dropout_add(odd, res, p=0.3, seed=4), P.dropout_add(x.cuda(), res.t().contiguous().t(), p=0.3, seed=4))


def test_dropout_share_and_independence(gpu):
    """Of 2^20 elements a share p is dropped, within five standard deviations; masks of other seeds, offsets and places
    agree as often as independent ones."""
    _say("dropout share")
    n, p = 1 << 20, 0.25
    x = torch.ones(n, device="cuda")
    masks = [P.dropout_add(x, p=p, seed=s, offset=o) == 0 for s, o in ((1, 0), (2, 0), (1, 1))]
    masks.append(masks[0].roll(1))
    for m in masks:
        assert abs(m.sum().item() - n * p) < 5 * (n * p * (1 - p)) ** 0.5
    q = p * p + (1 - p) * (1 - p)
    for m in masks[1:]:
        assert abs((m == masks[0]).sum().item() - n * q) < 5 * (n * q * (1 - q)) ** 0.5


def test_dropout_offset_on_the_device(gpu):
    _say("dropout device offset")
    x = _rand(1000, seed=1).cuda().requires_grad_(True)
    off = torch.tensor([12], device="cuda")
    out = P.dropout_add(x, p=0.4, seed=3, offset=off)
    want = P.dropout_add(x, p=0.4, seed=3, offset=12)
    assert torch.equal(out, want)
    off += 1  # the gradient keeps the mask of the forward pass
    d = _rand(1000, seed=2).cuda()
    assert torch.equal(torch.autograd.grad(out, x, d)[0], torch.autograd.grad(want, x, d)[0])
    assert not torch.equal(P.dropout_add(x, p=0.4, seed=3, offset=off), want)


def test_dropout_beyond_32_bits(gpu):
    _say("dropout beyond 32 bits")
    n = (1 << 32) + 11
    x = torch.ones(n, dtype=F16, device="cuda")
    out = P.dropout_add(x, p=0.5, seed=3)
    first = n - 4096 - 11
    assert torch.equal(out[first:].cpu() != 0, plain.keep(first, n - first, 32768, 3, 0))


# ---- together -------------------------------------------------------------------------------------


def test_lengths_on_the_host_are_refused_in_a_capture(gpu):
    """Their copy's source would be freed before a replay."""
    _say("graph, host lengths")
    z = _gates(2, 70, 8, True, F16).cuda()
    n = torch.tensor([70, 3], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        want = P.gated_scan(z, lengths=n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for host in ([70, 3], torch.tensor([70, 3])):
                with pytest.raises(ValueError, match="captured"):
                    P.gated_scan(z, lengths=host)
            got = P.gated_scan(z, lengths=n)
        for _ in range(3):
            got[0].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_operators_in_a_captured_graph(gpu):
    """Every forward in one graph, replayed several times with eager work between the replays, against eager calls;
    the dropout's offset advances on the device."""
    _say("graph")
    B, T, H = 3, 2000, 40
    z, c0 = _gates(B, T, H, True, F16).cuda(), _rand(B, H, seed=1).cuda()
    w, res, off = _rand(H, seed=3).cuda(), _rand(B, T, H, seed=4).half().cuda(), torch.zeros(1, dtype=torch.int64, device="cuda")
    n = torch.tensor([T, 0, 77], dtype=torch.int32, device="cuda")

    def block():
        h, c = P.gated_scan(z, c0, lengths=n)
        return P.dropout_add(P.layer_norm(h, w), res, p=0.2, seed=8, offset=off), c

    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            block()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = block()
            off.add_(1)
        off.zero_()
        seen = []
        for i in range(4):
            z.copy_(_gates(B, T, H, True, F16, seed=20 + i))
            keep = off.clone()
            graph.replay()
            torch.cuda.synchronize()
            assert int(off) == i + 1
            off.copy_(keep)
            want = block()
            off.add_(1)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), f"replay {i}"
            seen.append((got[0] == res).clone())
        assert not torch.equal(seen[0], seen[1])


def test_operators_refuse_on_the_device(gpu):
    _say("refusals")
    z, c = torch.zeros(2, 3, 12, device="cuda"), torch.zeros(2, 4, device="cuda")
    for bad in (lambda: P.gated_scan(z.double()), lambda: P.gated_scan(z[0]), lambda: P.gated_scan(z[..., :11]),
                lambda: P.gated_scan(z, c[:1]), lambda: P.gated_scan(z, c.cpu()), lambda: P.gated_scan(z, lengths=[1]),
                lambda: P.gated_scan(z, lengths=[1, 4]), lambda: P.gated_scan(z, lengths=[-1, 2]),
                lambda: P.gated_scan(z, lengths=[1.5, 2.0]), lambda: P.gated_scan(z, lengths=[True, False]),
                lambda: P.gated_scan(z, lengths=torch.ones(2, 1, dtype=torch.int32)), lambda: P.gated_scan(z[..., :0]),
                lambda: P.gated_scan(z[..., :9], output_gate=False), lambda: P.gated_scan_step(z[:, 0], c.half()),
                lambda: P.gated_scan_step(z, c), lambda: P.gated_scan_step(z[:, 0], c.t().contiguous().t(), inplace=True),
                lambda: P.gated_scan_step(z[:, 0].requires_grad_(True), c),
                lambda: P.layer_norm(c, torch.ones(5, device="cuda")), lambda: P.layer_norm(c, torch.ones(4)),
                lambda: P.layer_norm(c, torch.ones(4, device="cuda").half()), lambda: P.layer_norm(c, eps=-1.0),
                lambda: P.layer_norm(c.half(), torch.ones(4, device="cuda"), torch.ones(4, device="cuda").half()),
                lambda: P.layer_norm(c[0, 0]), lambda: P.layer_norm(c[:, :0]),
                lambda: P.dropout_add(c, p=1.5, seed=1), lambda: P.dropout_add(c, p=float("nan"), seed=1),
                lambda: P.dropout_add(c, c[:1], p=0.1, seed=1), lambda: P.dropout_add(c, c.half(), p=0.1, seed=1),
                lambda: P.dropout_add(c, p=0.1, seed=1, offset=torch.zeros(1)),
                lambda: P.dropout_add(c.to(torch.complex64), p=0.1, seed=1)):
        with pytest.raises(ValueError):
            bad()


def test_hidden_beyond_an_int_is_refused(gpu):
    _say("hidden beyond an int")  # 2^32 + 4 would be 4 in 32 bits; expanded, so that nothing of the size exists
    z, c = torch.zeros(1, 1, 1, device="cuda"), torch.zeros(1, 1, device="cuda")
    for hidden in ((1 << 24) + 1, 1 << 31, (1 << 32) + 4):
        with pytest.raises(ValueError, match="hidden"):
            P.gated_scan(z.expand(1, 1, 3 * hidden))
        with pytest.raises(ValueError, match="hidden"):
            P.gated_scan_step(z[0].expand(1, 3 * hidden), c.expand(1, hidden))


def test_gradients_of_another_type_are_converted(gpu):
    _say("gradient types")
    x = torch.randn(4, 24, device="cuda").half().requires_grad_(True)
    d = torch.randn(4, 24, device="cuda")
    for f in (lambda: P.layer_norm(x), lambda: P.dropout_add(x, p=0.1, seed=1),
              lambda: P.gated_scan(x.view(2, 2, 24), output_gate=False)[0]):
        y = f()
        dy = d.view(-1)[:y.numel()].view(y.shape)
        assert torch.equal(torch.autograd.grad(f(), x, dy)[0], torch.autograd.grad(f(), x, dy.half())[0])
    z = x.detach().float().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(P.layer_norm(z), z, d.half())[0],
                       torch.autograd.grad(P.layer_norm(z), z, d.half().float())[0])


def test_gradients_are_once_differentiable(gpu):
    _say("double backward")
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    for y in (P.layer_norm(x), P.dropout_add(x, p=0.1, seed=1), P.gated_scan(x.view(1, 3, 8), output_gate=False)[0]):
        g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
