"""What the block operators' autograd nodes do beside a first gradient on the GPU: second derivatives of every kind of
loss, where a gradient is a constant, and forward mode."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

import ops_plain as plain
import persistent_lstm_hip_amd as P

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _x(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


# ---- second derivatives ---------------------------------------------------------------------------

CURVED = {
    "layer_norm": lambda x, w: P.layer_norm(x, w),
    "gated_scan": lambda x, w: P.gated_scan(x.view(1, 3, 8) * w, output_gate=False)[0],
    "gated_scan c_n": lambda x, w: P.gated_scan(x.view(1, 3, 8) * w, output_gate=False)[1],
}


@pytest.mark.parametrize("name", CURVED)
@pytest.mark.parametrize("cotangent", ["sum", "constant"])
def test_a_second_derivative_of_a_linear_loss_raises(gpu, name, cotangent):
    """No incoming gradient is tracked here; the gradient still depends on x, and as a constant it would drop a
    penalty's term without an error."""
    _say(f"second derivative {name} {cotangent}")
    x, w = _x(3, 8).requires_grad_(True), torch.ones(8, device="cuda", requires_grad=True)
    y = CURVED[name](x, w)
    if cotangent == "sum":
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    else:
        g, = torch.autograd.grad(y, x, _x(*y.shape, seed=1), create_graph=True)
    assert g.requires_grad
    total = x.pow(3).sum() + g.square().sum()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(total, x, retain_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        total.backward()


def test_mixed_second_derivatives_raise(gpu):
    """A weight's gradient depends on x, an input's on the weight, a gate's on the state before it."""
    _say("mixed second derivatives")
    x, w = _x(3, 8).requires_grad_(True), torch.ones(8, device="cuda", requires_grad=True)
    c0 = _x(1, 4, seed=2).requires_grad_(True)
    for y, first, second in ((P.layer_norm(x, w), w, x), (P.layer_norm(x, w), x, w),
                             (P.gated_scan(x.view(1, 3, 8), c0, output_gate=False)[0], x, c0),
                             (P.gated_scan(x.view(1, 3, 8), c0, output_gate=False)[0], c0, x)):
        g, = torch.autograd.grad(y.sum(), first, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum(), second, allow_unused=True)


@pytest.mark.parametrize("layout", ["dense", "merged rows", "copied rows", "one row", "every second column"])
def test_a_norms_second_derivative_raises_in_every_layout(gpu, layout):
    _say(f"second derivative, norm of {layout}")
    leaf = _x(4, 6, 8).requires_grad_(True)
    x = {"dense": leaf, "merged rows": leaf[:, :, 2:6], "copied rows": leaf[:, :3], "one row": leaf[0, 0],
         "every second column": leaf[..., ::2]}[layout]
    g, = torch.autograd.grad(P.layer_norm(x).sum(), leaf, create_graph=True)
    assert g.shape == leaf.shape
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum(), leaf, allow_unused=True)
    dy = _x(*x.shape, seed=1)
    g, = torch.autograd.grad(P.layer_norm(x), leaf, dy)
    rows = x.detach().reshape(-1, x.shape[-1]).clone().requires_grad_(True)
    want, = torch.autograd.grad(P.layer_norm(rows), rows, dy.reshape(rows.shape))
    part = {"dense": g, "merged rows": g[:, :, 2:6], "copied rows": g[:, :3], "one row": g[0, 0],
            "every second column": g[..., ::2]}[layout]
    assert torch.equal(part.reshape(rows.shape), want) and torch.equal(g.count_nonzero(), want.count_nonzero())


def test_gradients_that_are_constants(gpu):
    """The operators are linear in these: without a tracked incoming gradient the second derivative is zero, and it does
    not take an error to say so."""
    _say("constant gradients")
    x, ones = _x(3, 8), torch.ones(8, device="cuda")
    w, c0 = ones.clone().requires_grad_(True), _x(1, 4).requires_grad_(True)
    for y, leaf in ((P.layer_norm(x, w), w), (P.gated_scan(x.view(1, 3, 8), c0, output_gate=False)[0], c0)):
        g, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        assert not g.requires_grad
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(P.dropout_add(leaf, p=0.25, seed=1).sum(), leaf, create_graph=True)
    assert not g.requires_grad
    keep = plain.keep(0, 24, 16384, 1, 0).view(3, 8)
    assert torch.equal(g.cpu(), torch.where(keep, torch.tensor(4.0 / 3.0), torch.tensor(0.0)))
    # a tracked incoming gradient: raises, as for the others
    g, = torch.autograd.grad(P.dropout_add(leaf, p=0.25, seed=1).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    # and a plain backward pass gives plain gradients
    P.layer_norm(leaf, w).sum().backward()
    assert not leaf.grad.requires_grad and not w.grad.requires_grad


def test_a_state_may_be_overwritten_before_the_backward_pass(gpu):
    """The states that a training pass saves hold c0's values: the buffer that carries it is free for the next chunk."""
    _say("c0 overwritten")
    z, c0 = _x(2, 70, 24).requires_grad_(True), _x(2, 8, seed=1)
    d = _x(2, 8, seed=2)
    want, = torch.autograd.grad(P.gated_scan(z, c0.clone())[1], z, d)
    _, c_n = P.gated_scan(z, c0)
    c0.copy_(c_n.detach())
    assert torch.equal(torch.autograd.grad(c_n, z, d)[0], want)


# ---- forward mode ---------------------------------------------------------------------------------


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(10))
def test_forward_mode_tangents_are_refused(gpu, which, grad):
    """A dual tensor has no requires_grad of its own; its tangent would be dropped."""
    _say(f"tangent {which} grad={grad}")
    x, w, c = _x(3, 8), _x(8, seed=1), _x(3, 4, seed=2)
    z = x.view(3, 1, 8)
    name, t, call = [
        ("x", x, lambda t: P.layer_norm(t, w, w)), ("weight", w, lambda t: P.layer_norm(x, t, w)),
        ("bias", w, lambda t: P.layer_norm(x, w, t)),
        ("x", x, lambda t: P.dropout_add(t, x, p=0.1, seed=1)), ("residual", x, lambda t: P.dropout_add(x, t, p=0.1, seed=1)),
        ("gates", z, lambda t: P.gated_scan(t, c, output_gate=False)),
        ("c0", c, lambda t: P.gated_scan(z, t, output_gate=False)),
        ("gates", x, lambda t: P.gated_scan_step(t, c, output_gate=False)),
        ("c", c, lambda t: P.gated_scan_step(x, t, output_gate=False)),
        ("c", c, lambda t: P.gated_scan_step(x, t, output_gate=False, inplace=True)),
    ][which]
    before = c.clone()
    with torch.set_grad_enabled(grad), fw.dual_level():
        with pytest.raises(ValueError, match=f"^{name} carries a forward-mode tangent"):
            call(fw.make_dual(t, torch.ones_like(t)))
        call(t)  # (as it is without one)
    if which < 9:
        assert torch.equal(c, before)


def test_a_tangent_of_an_incoming_gradient_is_refused(gpu):
    _say("tangent of a gradient")
    x = _x(3, 8).requires_grad_(True)
    for f in (P.layer_norm, lambda t: P.dropout_add(t, p=0.1, seed=1),
              lambda t: P.gated_scan(t.view(1, 3, 8), output_gate=False)[0],
              lambda t: P.gated_scan(t.view(1, 3, 8), output_gate=False)[1]):
        with fw.dual_level():
            y = f(x)
            with pytest.raises(ValueError, match="incoming gradient carries a forward-mode tangent"):
                torch.autograd.grad(y, x, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("transform", ["grad", "jvp", "vmap"])
def test_function_transforms_raise(gpu, transform):
    """torch.func's wrappers hold no storage: an error, never a value without its derivative."""
    _say(f"torch.func.{transform}")
    x = _x(3, 8)
    for f in (P.layer_norm, lambda t: P.dropout_add(t, p=0.1, seed=1),
              lambda t: P.gated_scan(t.view(1, 3, 8), output_gate=False)[0]):
        with pytest.raises((RuntimeError, ValueError)):
            if transform == "grad":
                torch.func.grad(lambda t: f(t).sum())(x)
            elif transform == "jvp":
                torch.func.jvp(f, (x,), (torch.ones_like(x),))
            else:
                torch.func.vmap(f)(x.expand(2, 3, 8))
