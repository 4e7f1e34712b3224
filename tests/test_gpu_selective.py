"""The selective scan on the GPU against its formulas in 64 bits (selective_plain.py, which derives the bounds)."""
from __future__ import annotations

import pytest
import torch

import ops_plain
import persistent_lstm_hip_amd as P
import selective_plain as plain

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = [F16, BF16, F32]
LEAVES = ("u", "dt", "A", "B", "C", "D", "z", "h0", "dt_bias")


def assert_within(got, want, bound, dtype, what):
    ops_plain.assert_within(got, want, bound + plain.TINY, dtype, what)


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _inputs(B, T, D, N, dtype, wdtype=F32, *, gate=True, skip=True, state=True, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    return dict(u=rand(B, T, D).to(dtype), dt=rand(B, T, D).to(dtype),
                A=-(0.2 + torch.arange(1, N + 1) * torch.rand(D, N, generator=g)).to(wdtype),
                B=rand(B, T, N).to(dtype), C=rand(B, T, N).to(dtype), D=rand(D).to(wdtype) if skip else None,
                z=rand(B, T, D).to(dtype) if gate else None, h0=rand(B, D, N) if state else None,
                dt_bias=(rand(D) - 2.0).to(wdtype) if bias else None)


def _call(d, **kw):
    return P.selective_scan(d["u"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["h0"], dt_bias=d["dt_bias"], **kw)


def _check(d, lengths=None, softplus=True, dev=None, dev_lengths=None, grads=True, what=""):
    """Forward and gradients on the device (dev: the device's tensors, default copies) against the formulas."""
    B, T, D = d["u"].shape
    N, dtype, wdtype = d["A"].shape[1], d["u"].dtype, d["A"].dtype
    g = torch.Generator().manual_seed(99)
    d_out, d_hn = torch.randn(B, T, D, generator=g).to(dtype), torch.randn(B, D, N, generator=g)
    want = plain.scan(*(d[n] for n in LEAVES), softplus=softplus, lengths=lengths, d_out=d_out if grads else None, d_hn=d_hn)
    dev = dev or {n: None if t is None else t.cuda() for n, t in d.items()}
    n = lengths if dev_lengths is None else dev_lengths
    with torch.no_grad():
        out0, h0 = _call(dev, softplus=softplus, lengths=n)
    assert out0.dtype == dtype and h0.dtype == F32 and out0.is_contiguous()
    assert_within(out0, *want["out"], dtype, f"{what} out")
    assert_within(h0, *want["h_n"], F32, f"{what} h_n")
    if not grads:
        return out0, h0, None
    given = [name for name in LEAVES if dev[name] is not None]
    for name in given:
        dev[name].requires_grad_(True)
    out, h_n = _call(dev, softplus=softplus, lengths=n)
    assert torch.equal(out, out0) and torch.equal(h_n, h0), f"{what}: inference and training differ"
    got = dict(zip(given, torch.autograd.grad((out, h_n), [dev[name] for name in given], (d_out.cuda(), d_hn.cuda()))))
    types = {"A": wdtype, "D": wdtype, "dt_bias": wdtype, "h0": F32}
    for name, grad in got.items():
        assert grad.dtype == types.get(name, dtype)
        assert_within(grad, *want["d_" + name], types.get(name, dtype), f"{what} d_{name}")
    return out0, h0, got


def _lengths(B, T):
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B + T))
    n[: max(1, B // 4)] = 0
    if B > 1:
        n[-1] = T
    return n


# (B, T, D, N): one of everything; no steps; no rows; every number of lanes per channel, full and padded; runs, tiles and
# their edges; one group of channels and several, full and not, an odd number of them; many rows of few channels
SHAPES = [(1, 1, 1, 1), (2, 0, 5, 3), (0, 4, 3, 2), (2, 3, 4, 4), (3, 8, 7, 5), (2, 9, 40, 8), (2, 31, 33, 10),
          (1, 32, 32, 16), (2, 33, 64, 16), (1, 65, 97, 16), (3, 100, 70, 15), (2, 40, 31, 17), (1, 70, 16, 32),
          (2, 37, 9, 33), (1, 96, 17, 64), (5, 64, 3, 16), (7, 35, 130, 4), (2, 50, 257, 2),
          (4, 33, 129, 1), (1, 300, 20, 16), (9, 5, 24, 31)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N", SHAPES)
def test_scan(gpu, B, T, D, N, dtype):
    _say(f"selective scan {B} {T} {D} {N} {dtype}")
    _check(_inputs(B, T, D, N, dtype), what="full")
    _check(_inputs(B, T, D, N, dtype, dtype, seed=1), _lengths(B, T) if B else None, what="ragged")
    _check(_inputs(B, T, D, N, dtype, gate=False, skip=False, state=False, bias=False, seed=2), what="bare")


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("skip", [True, False])
@pytest.mark.parametrize("bias", [True, False])
def test_every_combination_of_what_may_be_missing(gpu, gate, skip, bias):
    _say(f"selective scan gate={gate} skip={skip} bias={bias}")
    for state in (True, False):
        _check(_inputs(2, 41, 37, 16, BF16, gate=gate, skip=skip, state=state, bias=bias), _lengths(2, 41), what=f"{state}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_sizes_as_they_are(gpu, dtype):
    _say(f"selective scan without softplus {dtype}")
    d = _inputs(2, 45, 20, 16, dtype)
    d["dt"], d["dt_bias"] = (0.1 * d["dt"].float().abs()).to(dtype), 0.01 + 0.1 * d["dt_bias"].abs()
    _check(d, [45, 20], softplus=False)


# few rows and channels over a long time (its axis split into segments), rows that end in each of them
@pytest.mark.parametrize("B,T,D,N,lengths", [(1, 2000, 8, 16, None), (2, 1500, 24, 4, [1500, 0]),
                                             (3, 700, 5, 33, [700, 64, 65]), (2, 1025, 40, 8, [1, 1024]),
                                             (4, 513, 12, 16, [31, 32, 33, 513])])
def test_long_rows(gpu, B, T, D, N, lengths):
    _say(f"selective scan long {B} {T} {D} {N} {lengths}")
    for dtype in (F32, BF16):
        _check(_inputs(B, T, D, N, dtype), lengths, what=str(dtype))


@pytest.mark.parametrize("place", ["list", "int32 on the device", "int64 on the device", "clamped"])
def test_lengths_from_anywhere(gpu, place):
    _say(f"selective scan lengths {place}")
    n = torch.tensor([0, 70, 1, 64])
    dev = {"list": n.tolist(), "int32 on the device": n.int().cuda(), "int64 on the device": n.cuda(),
           "clamped": torch.tensor([-7, 1 << 40, 1, 64], device="cuda")}[place]
    _check(_inputs(4, 70, 24, 16, F16), n, dev_lengths=dev, what=place)


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), torch.finfo(F16).min])
def test_what_lies_past_a_row_changes_nothing(gpu, junk):
    _say(f"selective scan padding {junk}")
    B, T = 5, 70
    n = torch.tensor([0, 70, 32, 33, 3])
    d = _inputs(B, T, 20, 16, F16)
    past = torch.arange(T).unsqueeze(0) >= n.unsqueeze(1)
    clean = {name: None if t is None else t.clone() for name, t in d.items()}
    for name in ("u", "dt", "B", "C", "z"):
        clean[name][past] = 0
        d[name][past] = junk
    dev = {name: None if t is None else t.cuda() for name, t in d.items()}
    out, _, grads = _check(clean, n, dev=dev, what="padding")
    assert (out.cpu()[past] == 0).all()
    for name in ("u", "dt", "B", "C", "z"):
        assert (grads[name].cpu()[past] == 0).all(), name
    # nor does the gradient of an output that is not there
    d_out = torch.randn(B, T, 20).to(F16)
    d_out[past] = junk
    leaves = [dev[name] for name in LEAVES]
    again = torch.autograd.grad(_call(dev, lengths=n)[0], leaves, d_out.cuda())
    assert all(bool(torch.isfinite(t).all()) for t in again)


def test_infinite_states_and_gradients_stay_in_their_channel(gpu):
    _say("selective scan inf")
    d = _inputs(2, 70, 12, 16, F32)
    d["h0"][0, 3, 5] = float("inf")
    dev = {name: t.cuda().requires_grad_(True) for name, t in d.items()}
    out, h_n = _call(dev, lengths=[50, 70])
    assert h_n[0, 3, 5].item() == float("inf") and not torch.isfinite(out[0, :50, 3]).any()
    keep = torch.ones(12, dtype=torch.bool)
    keep[3] = False
    assert torch.isfinite(out[0][:, keep]).all() and torch.isfinite(out[1]).all()
    # an infinite gradient of the last state: steps past the row's end pass it on, and add nothing to what they are not in
    d["h0"][0, 3, 5] = 0.0
    dev = {name: t.cuda().requires_grad_(True) for name, t in d.items()}
    out, h_n = _call(dev, lengths=[0, 70])
    d_hn = torch.zeros(2, 12, 16, device="cuda")
    d_hn[0, 3, 5] = float("inf")
    d_A, d_h0 = torch.autograd.grad(h_n, (dev["A"], dev["h0"]), d_hn)
    assert d_h0[0, 3, 5].item() == float("inf") and torch.isfinite(d_A).all()
    out, h_n = _call(dev, lengths=[3, 70])
    d_A, d_h0 = torch.autograd.grad(h_n, (dev["A"], dev["h0"]), d_hn)
    # (d_A of the state itself holds infinity times h0 = 0: NaN by the formula)
    assert d_h0[0, 3, 5].item() == float("inf") and torch.isfinite(d_A[keep.cuda()]).all()


def test_nan_stays_in_its_row(gpu):
    _say("selective scan nan")
    d = _inputs(3, 40, 70, 16, F32)
    d["B"][1, 7, 2] = float("nan")
    d["u"][2, 9, 5] = float("nan")
    out, h_n = _call({name: t.cuda() for name, t in d.items()})
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, :7]).all() and torch.isnan(out[1, 7:]).all()
    clean = torch.ones(70, dtype=torch.bool)
    clean[5] = False
    assert torch.isfinite(out[2][:, clean]).all() and torch.isnan(out[2, 9:, 5]).all()


@pytest.mark.parametrize("low", [float("-inf"), "lowest", -200.0])
def test_a_closed_gate_and_step(gpu, low):
    """A gate or a step size of minus infinity, or of the type's lowest value, closes: nothing but zeros, no NaN."""
    _say(f"selective scan closed {low}")
    for dtype in DTYPES:
        v = torch.finfo(dtype).min if low == "lowest" else low
        d = {name: t.cuda() for name, t in _inputs(2, 20, 9, 5, dtype).items()}
        z = d["z"].clone()
        z[:, 4:] = v
        out, _ = _call({**d, "z": z})
        assert (out[:, 4:] == 0).all() and torch.isfinite(out).all()
        dt = d["dt"].clone()
        dt[:, 4:] = v
        _, h_n = _call({**d, "dt": dt})
        _, h4 = _call({name: t[:, :4] if name in ("u", "dt", "B", "C", "z") else t for name, t in d.items()})
        assert torch.equal(h_n, h4)


def test_a_state_that_decays_at_once(gpu):
    """A rate of minus infinity: a state of the last input alone, kept past a row's end; no NaN, gradients included."""
    _say("selective scan rate")
    d = _inputs(2, 40, 9, 16, F32)
    d["A"][4, 3] = float("-inf")
    dev = {name: t.cuda().requires_grad_(True) for name, t in d.items()}
    out, h_n = _call(dev, lengths=[40, 13])
    grads = torch.autograd.grad((out, h_n), [dev[n] for n in LEAVES], (torch.ones_like(out), torch.ones_like(h_n)))
    assert all(bool(torch.isfinite(t).all()) for t in (out, h_n, *grads))
    e = {**d, "A": d["A"].clamp(min=-1e6)}  # (decays within one step of any size that occurs here)
    want = plain.scan(*(e[n] for n in LEAVES), lengths=[40, 13])
    assert_within(out, *want["out"], F32, "out")
    assert_within(h_n, *want["h_n"], F32, "h_n")
    one = {n: t.detach()[:, 0] if n in ("u", "dt", "B", "C", "z") else t.detach() for n, t in dev.items()}
    out, h = P.selective_scan_step(one["u"], one["dt"], one["A"], one["B"], one["C"], one["h0"], one["D"], one["z"],
                                   dt_bias=one["dt_bias"])
    first = {n: t.detach()[:, :1] if n in ("u", "dt", "B", "C", "z") else t.detach() for n, t in dev.items()}
    want = _call(first)
    assert (out - want[0][:, 0]).abs().max() < 1e-4 and (h - want[1]).abs().max() < 1e-4


def test_strides_and_alignments(gpu):
    """Parts of one projection's output, a time-major one, an odd offset, an expanded row, a channel-strided tensor."""
    _say("selective scan strides")
    B, T, D, N = 3, 37, 41, 6
    d = _inputs(B, T, D, N, BF16)
    wide = torch.zeros(B, T, 2 * D + 2 * N + 1, dtype=BF16, device="cuda")
    parts = {"u": wide[..., 1:1 + D], "z": wide[..., 1 + D:1 + 2 * D], "B": wide[..., 1 + 2 * D:1 + 2 * D + N],
             "C": wide[..., 1 + 2 * D + N:]}
    for name, t in parts.items():
        t.copy_(d[name])
    dev = {name: None if t is None else t.cuda() for name, t in d.items()}
    _check(d, [37, 5, 0], dev={**dev, **{n: t.detach() for n, t in parts.items()}}, what="parts")
    major = {n: d[n].transpose(0, 1).contiguous().cuda().transpose(0, 1) for n in ("u", "dt", "B", "C", "z")}
    _check(d, dev={**dev, **major}, what="time-major")
    across = {n: d[n].transpose(1, 2).contiguous().cuda().transpose(1, 2) for n in ("u", "dt", "B", "C", "z")}
    _check(d, dev={**dev, **across}, what="channel-strided")
    same = {n: d[n][:1].expand(B, T, -1).contiguous() for n in ("u", "B")}
    e = {**d, **same}
    dev = {n: t.cuda() for n, t in e.items()}
    for n in same:
        dev[n] = d[n][:1].cuda().expand(B, T, -1)
    with torch.no_grad():
        out, h_n = _call(dev)
    want = plain.scan(*(e[n] for n in LEAVES))
    assert_within(out, *want["out"], BF16, "expanded")
    # lazily negated tensors are read as the values they stand for
    neg = {n: torch.complex(torch.zeros(t.shape, device="cuda"), -t.float().cuda()).conj().imag for n, t in d.items()
           if n in ("u", "z", "D")}
    assert all(t.is_neg() for t in neg.values())
    f = {n: t.float() for n, t in d.items()}
    want = plain.scan(*(f[n] for n in LEAVES))
    out, _ = _call({**{n: t.cuda() for n, t in f.items()}, **neg})
    assert_within(out, *want["out"], F32, "negated")


def test_gradients_of_one_result_alone(gpu):
    _say("selective scan one result")
    d = _inputs(2, 40, 20, 16, F32)
    dev = {n: t.cuda().requires_grad_(True) for n, t in d.items()}
    g = torch.Generator().manual_seed(3)
    d_out, d_hn = torch.randn(2, 40, 20, generator=g), torch.randn(2, 20, 16, generator=g)
    leaves = [dev[n] for n in LEAVES]
    got = torch.autograd.grad(_call(dev)[0], leaves, d_out.cuda())
    want = plain.scan(*(d[n] for n in LEAVES), d_out=d_out)
    for n, t in zip(LEAVES, got):
        assert_within(t, *want["d_" + n], F32, n)
    got = torch.autograd.grad(_call(dev)[1], leaves, d_hn.cuda(), allow_unused=True)
    want = plain.scan(*(d[n] for n in LEAVES), d_out=torch.zeros(2, 40, 20), d_hn=d_hn)
    for n, t in zip(LEAVES, got):
        assert_within(t, *want["d_" + n], F32, n)
    # every input by itself
    whole = torch.autograd.grad(_call(dev), leaves, (d_out.cuda(), d_hn.cuda()))
    for n, t in zip(LEAVES, whole):
        alone = {m: (v if m == n else v.detach()) for m, v in dev.items()}
        assert torch.equal(torch.autograd.grad(_call(alone), alone[n], (d_out.cuda(), d_hn.cuda()))[0], t), n


def test_a_sequence_in_parts_is_the_sequence(gpu):
    _say("selective scan in parts")
    d = {n: t.cuda() for n, t in _inputs(2, 90, 33, 16, F32).items()}
    cut = {n: (lambda a, b, t=t, n=n: t[:, a:b] if n in ("u", "dt", "B", "C", "z") else t) for n, t in d.items()}
    want, h_n = _call(d)
    h, outs = d["h0"], []
    for a, b in ((0, 1), (1, 33), (33, 64), (64, 90)):
        out, h = _call({**{n: f(a, b) for n, f in cut.items()}, "h0": h})
        outs.append(out)
    # (the same recurrence with other roundings: 90 steps of 16 states of size about 10, 2^-24 each)
    assert (torch.cat(outs, 1) - want).abs().max() < 1e-4 and (h - h_n).abs().max() < 1e-4


# ---- one token ----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,N", [(1, 1, 1), (3, 7, 5), (2, 300, 16), (65, 33, 16), (1, 129, 64), (5, 20, 33), (4, 50, 4),
                                   (0, 3, 2), (3000, 11, 8), (300, 1000, 16)])
def test_step(gpu, B, D, N, dtype):
    _say(f"selective scan step {B} {D} {N} {dtype}")
    for wdtype, kw in ((F32, {}), (dtype, dict(gate=False, skip=False, bias=False))):
        d = _inputs(B, 1, D, N, dtype, wdtype, **kw)
        want = plain.scan(*(d[n] for n in LEAVES))
        dev = {n: None if t is None else t.cuda() for n, t in d.items()}
        one = {n: t[:, 0] if n in ("u", "dt", "B", "C", "z") and t is not None else t for n, t in dev.items()}

        def step(h, **more):
            return P.selective_scan_step(one["u"], one["dt"], one["A"], one["B"], one["C"], h, one["D"], one["z"],
                                         dt_bias=one["dt_bias"], **more)

        before = one["h0"].clone()
        out, h = step(one["h0"])
        assert torch.equal(one["h0"], before) and out.shape == (B, D) and out.dtype == dtype
        assert_within(out, want["out"][0][:, 0], want["out"][1][:, 0], dtype, "out")
        assert_within(h, *want["h_n"], F32, "h")
        out2, same = step(before, inplace=True)
        assert same is before and torch.equal(out2, out) and torch.equal(before, h)


def test_steps_follow_the_sequence(gpu):
    _say("selective scan steps")
    d = _inputs(3, 20, 24, 16, F32)
    want = plain.scan(*(d[n] for n in LEAVES))
    dev = {n: t.cuda() for n, t in d.items()}
    h = dev["h0"].clone()
    for t in range(20):
        out, _ = P.selective_scan_step(dev["u"][:, t], dev["dt"][:, t], dev["A"], dev["B"][:, t], dev["C"][:, t], h,
                                       dev["D"], dev["z"][:, t], dt_bias=dev["dt_bias"], inplace=True)
        assert_within(out, want["out"][0][:, t], want["out"][1][:, t], F32, f"step {t}")
    assert_within(h, *want["h_n"], F32, "h_n")


# ---- streams, graphs, derivatives, refusals -------------------------------------------------------


def test_another_stream(gpu):
    _say("selective scan stream")
    d = {n: t.cuda() for n, t in _inputs(2, 200, 70, 16, F16).items()}
    want = _call(d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _call(d)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_calls_at_once(gpu):
    """Calls that overlap on two streams, each with segments and so with a workspace."""
    _say("selective scan two streams")
    cases = []
    for seed in (1, 2):
        d = {n: t.cuda().requires_grad_(True) for n, t in _inputs(1, 1500, 20, 16, F32, seed=seed).items()}
        g = torch.randn(1, 1500, 20, device="cuda")

        def run(d=d, g=g):
            out, h = _call(d)
            return (out.detach(), h.detach(), *torch.autograd.grad(out, [d[n] for n in LEAVES], g))

        cases.append((run, run(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for run, _, s in cases:
            with torch.cuda.stream(s):
                got.append(run())
        torch.cuda.synchronize()
        for (_, want, _), have in zip(cases, got):
            assert all(torch.equal(a, b) for a, b in zip(have, want))


def test_inference_mode(gpu):
    _say("selective scan inference")
    d = {n: t.cuda() for n, t in _inputs(2, 20, 24, 16, F16).items()}
    want = _call(d)
    with torch.inference_mode():
        got = _call(d)
        h = d["h0"].clone()
        P.selective_scan_step(d["u"][:, 0], d["dt"][:, 0], d["A"], d["B"][:, 0], d["C"][:, 0], h, d["D"], d["z"][:, 0],
                              dt_bias=d["dt_bias"], inplace=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not torch.equal(h, d["h0"])


def test_a_captured_training_step_replays(gpu):
    """Two graphs and eager work between their replays; every replay gives the eager result of its inputs."""
    _say("selective scan graph")
    cases = []
    for shape, seed in (((2, 100, 70, 16), 1), ((1, 700, 9, 8), 2)):
        d = {n: t.cuda().requires_grad_(True) for n, t in _inputs(*shape, BF16, seed=seed).items()}
        B, T, D, N = shape
        lengths = torch.full((B,), T - 3, device="cuda", dtype=torch.int32)
        grads = (torch.randn(B, T, D, device="cuda").to(BF16), torch.randn(B, D, N, device="cuda"))

        def run(d=d, lengths=lengths, grads=grads):
            # (leaves of its own: a graph's backward pass must not meet an eager graph of the same ones)
            own = {n: t.detach().requires_grad_(True) for n, t in d.items()}
            out = _call(own, lengths=lengths)
            return (*[t.detach() for t in out], *torch.autograd.grad(out, [own[n] for n in LEAVES], grads))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = run()
        cases.append((graph, static, run, d))
    for k in range(4):
        for graph, static, run, d in cases:
            with torch.no_grad():
                d["u"].copy_(torch.randn(d["u"].shape, device="cuda"))
                d["B"].add_(0.125)
            graph.replay()
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(static, run())):
                assert torch.equal(a, b), f"replay {k}, result {i}"


def test_results_are_the_same_from_call_to_call(gpu):
    _say("selective scan repeat")
    d = {n: t.cuda().requires_grad_(True) for n, t in _inputs(3, 150, 200, 16, BF16).items()}
    g = torch.randn(3, 150, 200, device="cuda").to(BF16)
    first = None
    for _ in range(3):
        out, _ = _call(d, lengths=[150, 77, 0])
        now = torch.autograd.grad(out, [d[n] for n in LEAVES], g)
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_a_second_derivative_raises(gpu):
    _say("selective scan second derivative")
    d = {n: t.cuda().requires_grad_(True) for n, t in _inputs(1, 9, 5, 3, F32).items()}
    out, _ = _call(d)
    grads = torch.autograd.grad(out.sum(), [d[n] for n in LEAVES], create_graph=True)
    for g in grads:
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum(), d["u"], retain_graph=True)
    # what is linear has constants for gradients: u alone, C alone, h0 and D together
    for names in (("u",), ("C",), ("B",), ("h0", "D")):
        alone = {m: (v if m in names else v.detach()) for m, v in d.items()}
        grads = torch.autograd.grad(_call(alone)[0].sum(), [alone[n] for n in names], create_graph=True)
        assert not any(g.requires_grad for g in grads), names
    for names in (("dt",), ("A",), ("z",), ("dt_bias",), ("B", "u"), ("C", "h0"), ("u", "D"), ("C", "B")):
        alone = {m: (v if m in names else v.detach()) for m, v in d.items()}
        grads = torch.autograd.grad(_call(alone)[0].sum(), [alone[n] for n in names], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(sum(g.sum() for g in grads), [alone[n] for n in names])


def test_refusals(gpu):
    _say("selective scan refusals")
    d = {n: t.cuda() for n, t in _inputs(2, 6, 8, 4, F16).items()}

    def bad(match, lengths=None, **changed):
        with pytest.raises(ValueError, match=match):
            _call({**d, **changed}, lengths=lengths)

    bad("u must be float16", u=d["u"].double())
    bad("3 dimensions", u=d["u"][0])
    bad("dt must be a tensor of shape", dt=d["dt"][:, :5])
    bad("dt must be", dt=d["dt"].float())
    bad("B must be a tensor of shape", B=d["B"][..., :3])
    bad("A must be", A=d["A"][:5])
    bad("A must be", A=-torch.ones(8, 65, device="cuda"))
    bad("A must be", A=d["A"].to(BF16))
    bad("D must have A's type", D=d["D"].half())
    bad("z must be", z=d["z"].float())
    bad("h0 must be a tensor of shape", h0=d["h0"][:1])
    bad("dt_bias must be a tensor of shape", dt_bias=d["dt_bias"][:3])
    bad("lengths", lengths=[1])
    bad("lengths", lengths=[1, 7])
    bad("u must be on a HIP device", u=d["u"].cpu())
    bad("C must be on cuda", C=d["C"].cpu())
    one = {n: t[:, 0] if n in ("u", "dt", "B", "C", "z") else t for n, t in d.items()}

    def step(**changed):
        a = {**one, **changed}
        return P.selective_scan_step(a["u"], a["dt"], a["A"], a["B"], a["C"], a["h0"], a["D"], a["z"], dt_bias=a["dt_bias"],
                                     inplace=True)

    for match, changed in (("h must be float32", dict(h0=d["h0"].half())),
                           ("contiguous", dict(h0=d["h0"].transpose(1, 2).contiguous().transpose(1, 2))),
                           ("2 dimensions", dict(u=d["u"])),
                           ("not differentiable", dict(u=one["u"].clone().requires_grad_(True)))):
        with pytest.raises(ValueError, match=match):
            step(**changed)
    with torch.inference_mode():
        h = d["h0"].clone()
    with pytest.raises(ValueError, match="inference tensor"):
        step(h0=h)
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        for name in ("u", "A", "z", "h0"):
            bad("forward-mode", **{name: fwad.make_dual(d[name], torch.ones_like(d[name]))})


def test_positions_beyond_32_bits(gpu):
    """More than 2^31 elements in front of the last row."""
    _say("selective scan large")
    B, T, D, N = 3, 400, 2, 2
    d = _inputs(B, T, D, N, F16)
    stride = (1 << 30) + 8
    big = torch.empty(2 * stride + T * D, dtype=F16, device="cuda")
    u = big.as_strided((B, T, D), (stride, D, 1))
    u.copy_(d["u"])
    _check(d, dev={**{n: t.cuda() for n, t in d.items()}, "u": u}, what="large")
