"""The gradient norm on the GPU.  Bounds: the norm is summed in 64 bits and rounded once, to 2^-24; an element is its
product with the factor, rounded to 32 bits as the factor is (2^-23 together), then to its type.  Below the smallest normal
number, 2^-126, numbers are a fixed distance apart, 2^-149 in 32 bits and 2^-133 in bfloat16, and a rounding is off by up
to half of it: 2^-150 for the product and 2^-134 for its bfloat16."""
from __future__ import annotations

import math

import pytest
import torch

import persistent_lstm_hip_amd as P
import selective_plain as plain
from ops_plain import U, assert_within

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


SUBNORMAL = {F16: 0.0, BF16: 2.0**-134 + 2.0**-150, F32: 2.0**-150}  # (float16's is in ops_plain.ROUNDING)


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _check(host, max_norm, what="", dev=None):
    want, norm = plain.clip(host, max_norm)
    dev = [t.cuda() for t in host] if dev is None else dev
    before = [t.clone() for t in dev]
    out, got = P.clip_grad_norm(dev, max_norm)
    assert got.dtype == F32 and got.shape == () and got.device.type == "cuda"
    assert abs(got.item() - norm.item()) <= 2 * U * norm.item(), f"{what} norm"
    for i, (t, v) in enumerate(zip(out, want)):
        assert t.dtype == host[i].dtype and torch.equal(dev[i], before[i])
        assert_within(t, v, 2 * U * v.abs() + SUBNORMAL[t.dtype], t.dtype, f"{what} {i}")
    again, norm2 = P.clip_grad_norm(dev, max_norm, inplace=True)
    assert torch.equal(norm2, got)
    for i, (t, d) in enumerate(zip(again, dev)):
        assert t is d and torch.equal(t, out[i]), f"{what} {i} in place"
    return out, got


SETS = [[(1,)], [(0,)], [(7,), (0,), (3, 5)], [(16384,), (16385,), (16383,)], [(300, 77), (1,), (513, 129)],
        [(5,)] * 99, [(5,)] * 100, [(5,)] * 101, [(33, 3)] * 350, [(3000001,)], [(0,), (100000,), (0,), (0,), (17,), (0,)]]


@pytest.mark.parametrize("k", range(len(SETS)))
@pytest.mark.parametrize("dtype", [F16, BF16, F32, "mixed"])
def test_clip(gpu, k, dtype):
    _say(f"clip set {k} {dtype}")
    kinds = [F16, F32, BF16]
    host = [_rand(*s, seed=i).to(kinds[i % 3] if dtype == "mixed" else dtype) for i, s in enumerate(SETS[k])]
    size = math.sqrt(max(1, sum(t.numel() for t in host)))
    for share in (0.5, 2.0, 0.0, 1e-3, float("inf")):
        _check(host, share * size if share < 1e9 else share, f"{share}")


def test_views_and_orders(gpu):
    """Transposed and sliced tensors, an odd alignment, entries that are None; a row of a larger tensor is left as it is."""
    _say("clip views")
    base = _rand(70, 90).cuda()
    whole = base.clone()
    views = [base[:20].t(), base[20:40, ::2], base[41, 1:88], base[50:60, 5:9], base[61]]
    host = [v.cpu() for v in views]
    want, norm = plain.clip(host, 3.0)
    out, got = P.clip_grad_norm([views[0], None, *views[1:], None], 3.0, inplace=True)
    assert out[1] is None and out[-1] is None and out[0] is views[0]
    for v, w in zip(views, want):
        assert_within(v, w, 2 * U * w.abs(), F32, "view")
    mask = torch.ones(70, 90, dtype=torch.bool)
    mask[:20] = mask[20:40, ::2] = mask[41, 1:88] = mask[50:60, 5:9] = mask[61] = False
    assert torch.equal(base.cpu()[mask], whole.cpu()[mask])
    # not in place any tensor may be an expanded, negated or repeated one
    t = _rand(5, 1).cuda().expand(5, 40)
    n = torch.complex(torch.zeros(6, device="cuda"), -_rand(6).cuda()).conj().imag
    host = [t.cpu(), t.cpu(), n.resolve_neg().cpu()]
    want, _ = plain.clip(host, 1.0)
    for a, b in zip(P.clip_grad_norm([t, t, n], 1.0)[0], want):
        assert_within(a, b, 2 * U * b.abs(), F32, "expanded")
    # a negated view's memory is scaled in place
    want, _ = plain.clip([n.resolve_neg().cpu()], 1.0)
    P.clip_grad_norm([n], 1.0, inplace=True)
    assert_within(n.resolve_neg(), want[0], 2 * U * want[0].abs(), F32, "negated")


@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e18, 3e37])
def test_no_square_overflows_or_vanishes(gpu, scale):
    _say(f"clip scale {scale}")
    for dtype in (BF16, F32):
        host = [(_rand(1000, seed=1).clamp(-3, 3) * scale).to(dtype)]
        _, norm = plain.clip(host, 1.0)
        got = P.clip_grad_norm([host[0].cuda()], float("inf"))[1].item()
        assert abs(got - norm.item()) <= 2 * U * norm.item() if norm < 3.4e38 else got == float("inf")
        _check(host, 1.0 if scale > 1 else scale, str(dtype)) if norm < 3.4e38 else None


def test_infinite_and_nan_norms(gpu):
    """As torch.nn.utils.clip_grad_norm_: infinity scales by zero (itself to NaN), NaN makes NaN."""
    _say("clip inf nan")
    for value in (float("inf"), float("nan")):
        t = _rand(100).cuda()
        t[7] = value
        mine, other = [t.clone(), torch.ones(5, device="cuda")], [t.clone(), torch.ones(5, device="cuda")]
        params = [torch.nn.Parameter(v.clone()) for v in other]
        for p, v in zip(params, other):
            p.grad = v
        theirs = torch.nn.utils.clip_grad_norm_(params, 1.0)
        _, norm = P.clip_grad_norm(mine, 1.0, inplace=True)
        assert torch.equal(torch.nan_to_num(norm, nan=-1.0), torch.nan_to_num(theirs, nan=-1.0))
        for a, p in zip(mine, params):
            assert torch.equal(torch.isnan(a), torch.isnan(p.grad))
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(p.grad))
        same, _ = P.clip_grad_norm([t], float("inf"), inplace=True)  # no limit: nothing is touched
        assert torch.equal(torch.isnan(same[0]), torch.isnan(t))


def test_streams_graphs_and_versions(gpu):
    _say("clip graph")
    grads = [_rand(300, 40, seed=i).cuda() for i in range(130)]
    stash = [g.clone() for g in grads]
    versions = [g._version for g in grads]
    P.clip_grad_norm(grads, 1.0, inplace=True)
    assert all(g._version > v for g, v in zip(grads, versions))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.clip_grad_norm(stash, 1.0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = P.clip_grad_norm(grads, 1.0, inplace=True)
    for k in range(4):
        for g, v in zip(grads, stash):
            g.copy_(v * (k + 1))
        want, wnorm = P.clip_grad_norm(grads, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, wnorm) and all(torch.equal(a, b) for a, b in zip(grads, want)), f"replay {k}"


def test_refusals(gpu):
    _say("clip refusals")
    t = torch.ones(8, device="cuda")

    def bad(match, grads, inplace=True):
        with pytest.raises(ValueError, match=match):
            P.clip_grad_norm(grads, 1.0, inplace=inplace)
        assert (t == 1).all()

    bad("share memory", [t, t])
    bad("share memory", [t[:5], t[4:]])
    bad("share memory", [t.view(2, 4).t(), t])
    bad("expanded", [torch.ones(1, device="cuda").expand(8)])
    bad("must be float16", [t.double()])
    bad("HIP device", [t, torch.ones(3)])
    bad("not differentiable", [t.clone().requires_grad_(True)])
    bad("not differentiable", [t.clone().requires_grad_(True)], inplace=False)
    with torch.inference_mode():
        frozen = torch.ones(3, device="cuda")
    bad("inference tensor", [frozen])
    P.clip_grad_norm([t[:4], t[4:]], 1.0, inplace=True)  # neighbours do not overlap
    with torch.no_grad():
        P.clip_grad_norm([torch.ones(3, device="cuda", requires_grad=True)], 1.0, inplace=True)


def test_inference_mode(gpu):
    _say("clip inference")
    with torch.inference_mode():
        t = torch.full((5,), 2.0, device="cuda")
        out, norm = P.clip_grad_norm([t], 1.0)
        P.clip_grad_norm([t], 1.0, inplace=True)
    assert torch.equal(out[0], t) and abs(norm.item() - math.sqrt(20.0)) < 1e-5


def test_more_than_32_bits_of_elements(gpu):
    _say("clip large")
    n = (1 << 31) + 12345
    g = torch.full((n,), 0.5, dtype=F16, device="cuda")
    g[-1] = 3.0
    out, norm = P.clip_grad_norm([g], 1.0, inplace=True)
    want = math.sqrt(0.25 * (n - 1) + 9.0)
    assert abs(norm.item() - want) <= 2 * U * want
    factor = 1.0 / (want + 1e-6)
    ends = torch.stack([g[0], g[1 << 31], g[-1]]).double().cpu()
    for a, v in zip(ends.tolist(), (0.5 * factor, 0.5 * factor, 3.0 * factor)):
        assert abs(a - v) <= 2.0**-11 * v + 2.0**-25
