"""The causal convolution on the GPU against its formulas in 64 bits (selective_plain.py, which derives the bounds)."""
from __future__ import annotations

import pytest
import torch

import persistent_lstm_hip_amd as P
import selective_plain as plain
from ops_plain import assert_within

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DTYPES = [F16, BF16, F32]


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _inputs(B, T, C, W, dtype, wdtype, *, bias=True, state=True, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    return (rand(B, T, C).to(dtype), rand(C, W).to(wdtype), rand(C).to(wdtype) if bias else None,
            rand(B, W - 1, C).to(dtype) if state else None)


def _check(given, lengths=None, silu=True, dev=None, dev_lengths=None, what=""):
    x, w, b, st = given
    B, T, C = x.shape
    dtype, wdtype, W = x.dtype, w.dtype, w.shape[1]
    g = torch.Generator().manual_seed(77)
    d_y, d_s = torch.randn(B, T, C, generator=g).to(dtype), torch.randn(B, W - 1, C, generator=g).to(dtype)
    want = plain.conv(x, w, b, st, lengths, silu, d_y, d_s)
    dev = dev or [None if t is None else t.cuda() for t in given]
    n = lengths if dev_lengths is None else dev_lengths
    with torch.no_grad():
        y0, s0 = P.causal_conv(*dev, lengths=n, silu=silu)
    assert y0.dtype == s0.dtype == dtype and y0.is_contiguous()
    assert_within(y0, *want["y"], dtype, f"{what} y")
    assert torch.equal(s0.cpu().double(), want["state_n"][0]), f"{what} state_n"
    leaves = [t.requires_grad_(True) for t in dev if t is not None]
    y, s = P.causal_conv(*dev, lengths=n, silu=silu)
    assert torch.equal(y, y0) and torch.equal(s, s0)
    got = torch.autograd.grad((y, s), leaves, (d_y.cuda(), d_s.cuda()))
    names = [k for k, t in zip(("d_x", "d_weight", "d_bias", "d_state"), dev) if t is not None]
    for name, t in zip(names, got):
        kind = wdtype if name in ("d_weight", "d_bias") else dtype
        assert t.dtype == kind
        assert_within(t, *want[name], kind, f"{what} {name}")
    return y0, s0, got


def _lengths(B, T):
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B + T))
    n[: max(1, B // 4)] = 0
    if B > 2:
        n[1], n[-1] = min(T, 2), T
    return n


# (B, T, C): one of everything; no steps, no rows; fewer channels than a vector; odd; vectors' edges; long rows and a
# stretch's edges; more channels than a slab
SHAPES = [(1, 1, 1), (2, 0, 5), (0, 4, 3), (3, 2, 3), (4, 5, 7), (2, 33, 8), (3, 64, 9), (2, 65, 60), (5, 130, 129),
          (1, 700, 24), (40, 3, 333), (1, 3000, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 6, 7, 8])
def test_conv(gpu, W, dtype):
    for B, T, C in SHAPES:
        _say(f"conv {B} {T} {C} {W} {dtype}")
        _check(_inputs(B, T, C, W, dtype, F32), what=f"{B} {T} {C}")
        _check(_inputs(B, T, C, W, dtype, dtype, bias=False, state=False, seed=1), _lengths(B, T) if B else None, silu=False,
               what=f"{B} {T} {C} ragged")
        _check(_inputs(B, T, C, W, dtype, dtype, seed=2), _lengths(B, T) if B else None, what=f"{B} {T} {C} ragged silu")


def test_many_rows(gpu):
    """Enough stretches that a workgroup takes several, and long ones."""
    _say("conv many rows")
    for B, T, C, dtype in ((300, 200, 520, BF16), (64, 1000, 100, F32)):
        given = _inputs(B, T, C, 4, dtype, F32)
        x, w, b, st = (t.cuda() for t in given)
        got = _run_grad(x, w, b, st)
        # in 64 bits on the device, by autograd
        x64, w64, b64, st64 = (t.detach().double().requires_grad_(True) for t in (x, w, b, st))
        line = torch.cat([st64, x64], 1)
        acc = b64 + sum(w64[:, k] * line[:, k:k + T] for k in range(4))
        want = torch.autograd.grad(acc * torch.sigmoid(acc), (x64, w64, b64, st64), _d_y(x).double())
        for name, t, v in zip("xwbs", got, want):
            # sums of B T terms of size about one, whose errors of 18 + 12 |acc| units add like random ones
            size = 1.0 if name in "xs" else (B * T) ** 0.5
            rel = torch.finfo(t.dtype).eps / 2
            assert ((t.double() - v).abs() <= rel * v.abs() + 300 * 2.0**-24 * size * 10).all(), name


def _d_y(x):
    return torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(x.dtype).cuda()


def _run_grad(x, w, b, st):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, st)]
    return torch.autograd.grad(P.causal_conv(*leaves)[0], leaves, _d_y(x))


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), torch.finfo(F16).min])
def test_what_lies_past_a_row_changes_nothing(gpu, junk):
    _say(f"conv padding {junk}")
    n = torch.tensor([0, 70, 32, 33, 2])
    x, w, b, st = _inputs(5, 70, 20, 4, F16, F32)
    past = torch.arange(70).unsqueeze(0) >= n.unsqueeze(1)
    dirty = x.clone()
    dirty[past] = junk
    for silu in (True, False):
        dev = [dirty.cuda(), w.cuda(), b.cuda(), st.cuda()]
        y, _, grads = _check((x, w, b, st), n, silu, dev=dev)
        assert (y.cpu()[past] == 0).all() and (grads[0].cpu()[past] == 0).all()
        d_y = torch.randn(5, 70, 20).to(F16)
        d_y[past] = junk
        got = torch.autograd.grad(P.causal_conv(*dev, lengths=n, silu=silu)[0], dev, d_y.cuda())
        assert all(bool(torch.isfinite(t).all()) for t in got)


def test_an_infinite_input_stays_where_it_is_used(gpu):
    """Without an activation: in the outputs of its four steps, and as an infinity, not NaN, in the filter's gradient."""
    _say("conv inf")
    x, w, b, st = _inputs(1, 140, 8, 4, F32, F32)
    x[0, 63, 2] = float("inf")
    dev = [t.cuda().requires_grad_(True) for t in (x, w, b, st)]
    y, _ = P.causal_conv(*dev, silu=False)
    bad = torch.zeros(140, 8, dtype=torch.bool)
    bad[63:67, 2] = True
    assert torch.equal(~torch.isfinite(y[0].detach()).cpu(), bad)
    d_y = torch.ones(1, 140, 8, device="cuda")
    d_x, d_w, _, _ = torch.autograd.grad(y, dev, d_y)
    assert torch.isfinite(d_x).all() and (d_w[2] == float("inf")).all() and torch.isfinite(d_w[3]).all()
    x[0, 63, 2] = float("-inf")
    w = w.abs()
    y, _ = P.causal_conv(x.cuda(), w.cuda(), b.cuda(), st.cuda())
    assert (y[0, 63:67, 2] == 0).all()


def test_strides(gpu):
    _say("conv strides")
    given = _inputs(3, 37, 41, 4, BF16, F32)
    x = given[0]
    wide = torch.zeros(3, 37, 90, dtype=BF16, device="cuda")
    wide[..., 1:42] = x.cuda()
    rest = [t.cuda() for t in given[1:]]
    _check(given, [37, 4, 0], dev=[wide[..., 1:42].detach(), *[t.clone() for t in rest]], what="part")
    _check(given, dev=[x.transpose(0, 1).contiguous().cuda().transpose(0, 1), *[t.clone() for t in rest]], what="time-major")
    _check(given, dev=[x.transpose(1, 2).contiguous().cuda().transpose(1, 2), *[t.clone() for t in rest]], what="across")
    w, s = rest[0], rest[2]
    _check(given, dev=[x.cuda(), w.t().contiguous().t(), rest[1].clone(), s.transpose(0, 1).contiguous().transpose(0, 1)],
           what="weights and state")
    one = x[:1].expand(3, 37, 41)
    y, _ = P.causal_conv(x[:1].cuda().expand(3, 37, 41), *rest)
    assert torch.equal(y, P.causal_conv(one.contiguous().cuda(), *rest)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 6, 7, 8])
def test_step(gpu, W, dtype):
    for B, C, wdtype, silu in ((1, 1, F32, True), (3, 7, dtype, False), (65, 129, F32, True),
                               (2, 64, dtype, True), (0, 3, F32, True)):
        _say(f"conv step {B} {C} {W} {dtype}")
        x, w, b, st = _inputs(B, 1, C, W, dtype, wdtype)
        want = plain.conv(x, w, b, st, None, silu)
        dx, dw, db, ds = x.cuda()[:, 0], w.cuda(), b.cuda(), st.cuda()
        y, s = P.causal_conv_step(dx, ds, dw, db, silu=silu)
        assert_within(y, want["y"][0][:, 0], want["y"][1][:, 0], dtype, "y")
        assert torch.equal(s.cpu().double(), want["state_n"][0]) and torch.equal(ds.cpu(), st)
        y2, same = P.causal_conv_step(dx, ds, dw, db, silu=silu, inplace=True)
        assert same is ds and torch.equal(ds, s) and torch.equal(y2, y)


def test_steps_and_parts_follow_the_sequence(gpu):
    _say("conv steps")
    x, w, b, st = (t.cuda() for t in _inputs(3, 20, 24, 4, F16, F32))
    want, last = P.causal_conv(x, w, b, st)
    state, ys = st.clone(), []
    for t in range(20):
        ys.append(P.causal_conv_step(x[:, t], state, w, b, inplace=True)[0])
    assert torch.equal(torch.stack(ys, 1), want) and torch.equal(state, last)
    state, ys = st, []
    for a, e in ((0, 1), (1, 3), (3, 12), (12, 20)):
        y, state = P.causal_conv(x[:, a:e], w, b, state)
        ys.append(y)
    assert torch.equal(torch.cat(ys, 1), want) and torch.equal(state, last)


def test_streams_and_graphs(gpu):
    _say("conv graph")
    x, w, b, st = (t.cuda() for t in _inputs(3, 200, 70, 4, F16, F32))
    lengths = torch.tensor([200, 3, 77], device="cuda", dtype=torch.int32)
    d_y = _d_y(x)

    def run():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, st)]
        out = P.causal_conv(*leaves, lengths=lengths)
        return (*[t.detach() for t in out], *torch.autograd.grad(out[0], leaves, d_y))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        aside = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(aside, run()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run()
    for k in range(4):
        x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(static, run())), f"replay {k}"


def test_derivatives(gpu):
    _say("conv derivatives")
    x, w, b, st = (t.cuda().requires_grad_(True) for t in _inputs(1, 9, 5, 3, F32, F32))
    for names, silu, raises in ((("x",), True, True), (("w",), True, True), (("b",), True, True), (("x", "w"), False, True),
                                (("w", "s"), False, True), (("x", "s", "b"), False, False), (("w", "b"), False, False)):
        t = {k: (v if k in names else v.detach()) for k, v in zip("xwbs", (x, w, b, st))}
        y, _ = P.causal_conv(t["x"], t["w"], t["b"], t["s"], silu=silu)
        leaves = [t[k] for k in names]
        grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
        if raises:
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(sum(g.sum() for g in grads), leaves)
        else:
            assert not any(g.requires_grad for g in grads), names
    # the new state's gradient alone
    _, s = P.causal_conv(x, w, b, st)
    d_x, d_w, d_b, d_s = torch.autograd.grad(s, (x, w, b, st), torch.ones_like(s))
    assert d_x[0, -2:].eq(1).all() and d_x[0, :-2].eq(0).all() and not d_w.any() and not d_b.any() and not d_s.any()


def test_refusals(gpu):
    _say("conv refusals")
    x, w, b, st = (t.cuda() for t in _inputs(2, 6, 8, 4, F16, F32))

    def bad(match, x=x, w=w, b=b, st=st, call=P.causal_conv, **kw):
        with pytest.raises(ValueError, match=match):
            call(x, w, b, st, **kw)

    bad("3 dimensions", x=x[0])
    bad("weight must be \\[channels, width\\]", w=w[:5])
    bad("width of 1 to 8", w=torch.ones(8, 9, device="cuda"))
    bad("weight must be", w=w.to(BF16))
    bad("same type", b=b.half())
    bad("bias must be a tensor of shape", b=b[:3])
    bad("state must be a tensor of shape", st=st[:, :2])
    bad("state must be", st=st.float())
    bad("lengths", lengths=[1, 7])
    bad("HIP device", x=x.cpu())
    bad("weight must be on", w=w.cpu())

    def step(x, w, b, st, **kw):
        return P.causal_conv_step(x, st, w, b, inplace=True)

    bad("2 dimensions", call=step)
    bad("contiguous", x=x[:, 0], st=st.transpose(1, 2).contiguous().transpose(1, 2), call=step)
    bad("not differentiable", x=x[:, 0].clone().requires_grad_(True), call=step)
    with torch.inference_mode():
        frozen = st.clone()
    bad("inference tensor", x=x[:, 0], st=frozen, call=step)


def test_positions_beyond_32_bits(gpu):
    _say("conv large")
    given = _inputs(3, 40, 16, 4, F16, F32)
    stride = (1 << 30) + 8
    big = torch.empty(2 * stride + 40 * 16, dtype=F16, device="cuda")
    x = big.as_strided((3, 40, 16), (stride, 16, 1))
    x.copy_(given[0])
    _check(given, dev=[x, *[t.cuda() for t in given[1:]]], what="large")
