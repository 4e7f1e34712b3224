"""The host side of the causal convolution, the selective scan and the gradient norm: their formulas' gradients against
differences, the comparison that the GPU tests rest on, and everything that they refuse (no kernel is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import ops_plain
import persistent_lstm_hip_amd as P
import selective_plain as plain
from persistent_lstm_hip_amd import ops
from persistent_lstm_hip_amd.extension import (
    PLH_ERR_INVALID,
    PLH_ERR_UNSUPPORTED,
    PLH_OK,
    SelectiveScanArgs,
    SelectiveScanGrads,
    require_extension,
)

F64 = torch.float64


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=F64)


def _directional(f, at, way, step=1e-6):
    def moved(sign):
        return f([t if d is None else t + sign * step * d for t, d in zip(at, way)])
    return (moved(1) - moved(-1)) / (2 * step)


@pytest.mark.parametrize("activation", [True, False])
@pytest.mark.parametrize("lengths", [None, [7, 0, 1]])
def test_the_convolutions_gradient_is_that_of_differences(activation, lengths):
    g = torch.Generator().manual_seed(5)
    at = [_rand(g, 3, 7, 4), _rand(g, 4, 4), _rand(g, 4), _rand(g, 3, 3, 4)]
    d_y, d_s = _rand(g, 3, 7, 4), _rand(g, 3, 3, 4)

    def loss(v):
        r = plain.conv(*v, lengths, activation)
        return ((r["y"][0] * d_y).sum() + (r["state_n"][0] * d_s).sum()).item()

    r = plain.conv(*at, lengths, activation, d_y, d_s)
    for i, name in enumerate(("d_x", "d_weight", "d_bias", "d_state")):
        way = [None] * 4
        way[i] = _rand(g, *at[i].shape)
        assert abs(_directional(loss, at, way) - (r[name][0] * way[i]).sum().item()) < 1e-7, name


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("lengths", [None, [6, 0, 3]])
def test_the_scans_gradient_is_that_of_differences(softplus, lengths):
    g = torch.Generator().manual_seed(6)
    R, T, D, N = 3, 6, 4, 3
    names = ("u", "dt", "A", "B", "C", "D", "z", "h0", "dt_bias")
    at = [_rand(g, R, T, D), 0.3 * _rand(g, R, T, D).abs(), -_rand(g, D, N).abs(), _rand(g, R, T, N), _rand(g, R, T, N),
          _rand(g, D), _rand(g, R, T, D), _rand(g, R, D, N), 0.1 * _rand(g, D).abs()]
    d_out, d_hn = _rand(g, R, T, D), _rand(g, R, D, N)

    def loss(v):
        r = plain.scan(*v, softplus=softplus, lengths=lengths)
        return ((r["out"][0] * d_out).sum() + (r["h_n"][0] * d_hn).sum()).item()

    r = plain.scan(*at, softplus=softplus, lengths=lengths, d_out=d_out, d_hn=d_hn)
    for i, name in enumerate(names):
        way = [None] * len(names)
        way[i] = _rand(g, *at[i].shape)
        assert abs(_directional(loss, at, way) - (r["d_" + name][0] * way[i]).sum().item()) < 1e-7, name


def test_planted_mistakes_are_seen():
    """A lost carry, a gradient of one channel too few, a step that is not skipped: each is outside the bounds."""
    g = torch.Generator().manual_seed(7)
    R, T, D, N = 2, 40, 5, 4
    args = (_rand(g, R, T, D), _rand(g, R, T, D), -_rand(g, D, N).abs(), _rand(g, R, T, N), _rand(g, R, T, N))
    d_out = _rand(g, R, T, D)
    want = plain.scan(*args, lengths=[40, 17], d_out=d_out)
    for name, (value, bound) in want.items():
        ops_plain.assert_within(value.float(), value, bound, torch.float32, name)
    later = plain.scan(*(t[:, 32:] if t.dim() == 3 else t for t in args), lengths=[8, 0])["out"][0]  # no carry at step 32
    bad = want["out"][0].clone()
    bad[:, 32:] = later
    with pytest.raises(AssertionError):
        ops_plain.assert_within(bad, want["out"][0], want["out"][1], torch.bfloat16, "carry")
    fewer = [t[..., 1:] if i < 2 else t[1:] if i == 2 else t for i, t in enumerate(args)]
    short = plain.scan(*fewer, lengths=[40, 17], d_out=d_out[..., 1:])
    for name in ("d_B", "d_C"):
        with pytest.raises(AssertionError):
            ops_plain.assert_within(short[name][0], *want[name], torch.bfloat16, name)
    full = plain.scan(*args, lengths=[40, 18], d_out=d_out)
    for name in ("h_n", "d_A", "d_dt", "out"):
        with pytest.raises(AssertionError):
            ops_plain.assert_within(full[name][0], *want[name], torch.bfloat16, name)


def test_public_names():
    for name in ("causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "clip_grad_norm"):
        assert name in P.__all__ and getattr(P, name) is getattr(ops, name)


@pytest.mark.parametrize("call", [
    lambda t: P.causal_conv(t(2, 3, 8), t(8, 4)),
    lambda t: P.causal_conv_step(t(2, 8), t(2, 3, 8), t(8, 4)),
    lambda t: P.selective_scan(t(2, 3, 8), t(2, 3, 8), t(8, 4), t(2, 3, 4), t(2, 3, 4)),
    lambda t: P.selective_scan_step(t(2, 8), t(2, 8), t(8, 4), t(2, 4), t(2, 4), t(2, 8, 4)),
    lambda t: P.clip_grad_norm([t(2, 8)], 1.0),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="HIP device"):
        call(torch.zeros)
    with pytest.raises(ValueError, match="must be a tensor"):
        call(lambda *shape: [0.0])


def test_clip_refuses_what_is_no_sequence_of_tensors():
    with pytest.raises(ValueError, match="sequence"):
        P.clip_grad_norm(torch.zeros(3), 1.0)
    with pytest.raises(ValueError, match="at least one"):
        P.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="at least one"):
        P.clip_grad_norm([None], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        P.clip_grad_norm([torch.zeros(3)], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        P.clip_grad_norm([torch.zeros(3)], float("nan"))
    with pytest.raises(ValueError, match="dense"):
        P.clip_grad_norm([torch.zeros(3).to_sparse()], 1.0)


# ---- the C ABI refuses before it touches a device ------------------------------------------------

ANY = ctypes.c_void_p(256)  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return require_extension().lib


def test_conv_refusals(lib):
    def fwd(dtype=0, wdtype=0, x=ANY, sb=32, st=8, B=2, T=4, C=8, W=4, w=ANY, y=ANY, state_n=ANY):
        return lib.plh_causal_conv_forward(dtype, wdtype, x, sb, st, B, T, C, W, w, None, None, None, 1, y, state_n, None)

    assert fwd(dtype=3) == PLH_ERR_INVALID and b"dtype" in lib.plh_last_error()
    assert fwd(wdtype=1) == PLH_ERR_INVALID and b"wdtype" in lib.plh_last_error()
    assert fwd(B=-1) == PLH_ERR_INVALID and fwd(T=-1) == PLH_ERR_INVALID
    assert fwd(W=0) == PLH_ERR_UNSUPPORTED and fwd(W=9) == PLH_ERR_UNSUPPORTED and b"width" in lib.plh_last_error()
    assert fwd(C=0) == PLH_ERR_UNSUPPORTED and fwd(C=(1 << 22) + 1) == PLH_ERR_UNSUPPORTED
    assert fwd(T=(1 << 30) + 1) == PLH_ERR_UNSUPPORTED
    assert fwd(B=1 << 26) == PLH_ERR_UNSUPPORTED and b"batch" in lib.plh_last_error()
    assert fwd(T=1 << 30, B=8) == PLH_ERR_UNSUPPORTED
    for name in ("x", "w", "y", "state_n"):
        assert fwd(**{name: None}) == PLH_ERR_INVALID
    assert fwd(sb=-1) == PLH_ERR_INVALID and fwd(B=0) == PLH_OK

    def step(state=ANY, y=ANY, state_n=ANY, B=2):
        return lib.plh_causal_conv_step(0, 0, ANY, 8, B, 8, 4, ANY, None, state, 1, y, state_n, None)

    assert step(state=None) == PLH_ERR_INVALID and step(y=None) == PLH_ERR_INVALID and step(state_n=None) == PLH_ERR_INVALID
    assert step(B=0) == PLH_OK

    need = lib.plh_causal_conv_workspace_bytes(2, 4, 8, 4)
    assert need > 0 and lib.plh_causal_conv_workspace_bytes(2, 4, 8, 9) == -1

    def back(d_y=ANY, T=4, d_w=ANY, d_state=None, ws=ANY, nws=need):
        return lib.plh_causal_conv_backward(0, 0, ANY, 32, 8, 2, T, 8, 4, ANY, None, None, None, 1, d_y, None, ANY, d_w,
                                            None, d_state, ws, nws, None)

    assert back(d_y=None) == PLH_ERR_INVALID
    assert back(ws=None) == PLH_ERR_INVALID and b"workspace" in lib.plh_last_error()
    assert back(nws=need - 1) == PLH_ERR_INVALID and back(ws=ctypes.c_void_p(260)) == PLH_ERR_INVALID
    assert back(T=0, d_state=ANY) == PLH_ERR_UNSUPPORTED


def _args(**changed):
    a = SelectiveScanArgs()
    a.batch, a.seq_len, a.channels, a.states, a.softplus = 2, 4, 8, 4, 1
    a.u = a.dt = a.B = a.C = a.A = 256
    for name, value in changed.items():
        if name.endswith("_stride"):
            getattr(a, name)[0] = value
        else:
            setattr(a, name, value)
    return a


def test_scan_refusals(lib):
    def fwd(out=ANY, ws=None, nws=0, **changed):
        a = _args(**changed)
        return lib.plh_selective_scan_forward(ctypes.byref(a), None, out, None, None, ws, nws, None)

    def step(h=ANY, out=ANY, h_n=ANY, **changed):
        a = _args(**{"seq_len": 1, **changed})
        return lib.plh_selective_scan_step(ctypes.byref(a), h, out, h_n, None)

    def back(states=ANY, d_out=ANY, ws=ANY, nws=1 << 40, grads=None, **changed):
        a = _args(**changed)
        g = SelectiveScanGrads()
        g.d_u = g.d_dt = g.d_z = 256
        for name in grads or ():
            setattr(g, name, None)
        return lib.plh_selective_scan_backward(ctypes.byref(a), states, d_out, None, ctypes.byref(g), ws, nws, None)

    for call in (fwd, step, back):
        assert call(dtype=3) == PLH_ERR_INVALID and b"dtype" in lib.plh_last_error()
        assert call(wdtype=1) == PLH_ERR_INVALID and b"wdtype" in lib.plh_last_error()
        assert call(batch=-1) == PLH_ERR_INVALID
        assert call(states=0) == PLH_ERR_UNSUPPORTED if call is not back else True
        assert call(channels=0) == PLH_ERR_UNSUPPORTED and call(channels=(1 << 20) + 1) == PLH_ERR_UNSUPPORTED
        if call is not step:
            assert call(batch=1 << 21, channels=9) == PLH_ERR_UNSUPPORTED and b"2^21" in lib.plh_last_error()
        for name in ("u", "dt", "B", "C", "A"):
            assert call(**{name: None}) == PLH_ERR_INVALID, name
        for name in ("u", "dt", "z", "B", "C"):
            assert call(**{name + "_stride": -1}) == PLH_ERR_INVALID and b"strides" in lib.plh_last_error()
    for a in (_args(states=0), _args(states=65)):
        assert lib.plh_selective_scan_forward(ctypes.byref(a), None, ANY, None, None, None, 0, None) == PLH_ERR_UNSUPPORTED
    assert fwd(seq_len=(1 << 30) + 1) == PLH_ERR_UNSUPPORTED and fwd(seq_len=1 << 30) == PLH_ERR_UNSUPPORTED
    assert fwd(out=None) == PLH_ERR_INVALID and fwd(batch=0) == PLH_OK
    assert lib.plh_selective_scan_forward(None, None, ANY, None, None, None, 0, None) == PLH_ERR_INVALID
    assert step(batch=1 << 24, channels=1 << 10) == PLH_ERR_UNSUPPORTED and b"2^32" in lib.plh_last_error()
    assert step(seq_len=2) == PLH_ERR_INVALID and step(lengths=256) == PLH_ERR_INVALID
    assert step(h=None) == PLH_ERR_INVALID and step(out=None) == PLH_ERR_INVALID and step(h_n=None) == PLH_ERR_INVALID
    assert back(states=None) == PLH_ERR_INVALID and back(d_out=None) == PLH_ERR_INVALID
    assert back(grads=["d_u"]) == PLH_ERR_INVALID and back(grads=["d_z"], z=256) == PLH_ERR_INVALID
    assert back(ws=None) == PLH_ERR_INVALID and b"workspace" in lib.plh_last_error()
    need = lib.plh_selective_scan_workspace_bytes(2, 4, 8, 4, 1)
    assert need > 0 and back(nws=need - 1) == PLH_ERR_INVALID and back(ws=ctypes.c_void_p(260)) == PLH_ERR_INVALID


def test_scan_sizes(lib):
    assert lib.plh_selective_scan_states(0) == 0 and lib.plh_selective_scan_states(1) == 1
    assert lib.plh_selective_scan_states(-1) == -1
    size = lib.plh_selective_scan_workspace_bytes
    assert size(-1, 1, 1, 1, 0) == -1 == size(1, 1, 0, 1, 0) == size(1, 1, 1, 65, 1)
    assert size(0, 5, 5, 5, 0) >= 0 and size(1000, 100, 512, 16, 0) == 0  # enough channels: the time axis is not split


def test_clip_refusals(lib):
    def call(n=8, dtype=0, src=256, dst=256, limit=1.0, norm=ANY, ws=ANY, nws=1 << 20, count=1):
        numel, dt = (ctypes.c_int64 * 1)(n), (ctypes.c_int * 1)(dtype)
        a, b = (ctypes.c_void_p * 1)(src), (ctypes.c_void_p * 1)(dst)
        return lib.plh_clip_grad_norm(count, dt, a, b, numel, limit, norm, ws, nws, None)

    assert call(count=-1) == PLH_ERR_INVALID and call(n=-1) == PLH_ERR_INVALID and call(dtype=5) == PLH_ERR_INVALID
    assert call(src=None) == PLH_ERR_INVALID and call(dst=None) == PLH_ERR_INVALID and call(norm=None) == PLH_ERR_INVALID
    assert call(limit=-1.0) == PLH_ERR_INVALID and call(limit=float("nan")) == PLH_ERR_INVALID
    assert call(ws=None) == PLH_ERR_INVALID and call(nws=7) == PLH_ERR_INVALID and b"workspace" in lib.plh_last_error()
    numel = (ctypes.c_int64 * 3)(1, 0, 1 << 30)
    assert 8 * 1 <= lib.plh_clip_grad_norm_workspace_bytes(3, numel) <= 8 * 4096
