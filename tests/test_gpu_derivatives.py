"""Derivatives that the routed residual block's operators do not have are refused on the device, not lost: forward-mode tangents on an
input or on the gradient that a backward pass is given; the norm of gradients that are themselves recorded."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls():
    """(name, tensors by name, the call on them) of every operator with a backward pass"""
    from cpfn_amd import autograd_ops, ops
    g = torch.Generator().manual_seed(0)
    P, C, k, E = 6, 24, 2, 3
    rows = {n: torch.randn(P, C, generator=g).to(DEV) for n in ("x", "y", "gate")}
    rows.update({n: torch.randn(C, generator=g).to(DEV) for n in ("weight", "bias", "scale", "next_weight", "next_bias")})
    plan = ops.route_plan(torch.randint(0, E, (P, k), generator=g).to(DEV), E)
    return [("row_norm", {"x": rows["x"], "weight": rows["weight"], "bias": rows["bias"]}, lambda t: autograd_ops.row_norm(t["x"], t["weight"], t["bias"])),
            ("norm_residual", rows, lambda t: autograd_ops.norm_residual(**t)[1]),
            ("route_gather", {"rows": rows["x"]}, lambda t: autograd_ops.route_gather(t["rows"], plan)),
            ("route_combine", {"sorted_rows": torch.randn(P * k, C, generator=g).to(DEV), "weights": torch.randn(P, k, generator=g).to(DEV)},
             lambda t: autograd_ops.route_combine(t["sorted_rows"], t["weights"], plan))]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("trained", [True, False])
def test_forward_mode_tangents_are_refused(trained, grad_mode):
    for name, tensors, call in calls():
        want = call(tensors)
        for n in tensors:
            with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
                t = {m: v.clone().requires_grad_(trained) for m, v in tensors.items()}
                t[n] = fwd.make_dual(t[n], torch.ones_like(t[n]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(t)
                t[n] = fwd.unpack_dual(t[n]).primal            # (its value alone is an input like any other)
                assert torch.equal(call(t), want), (name, n)


def test_a_tangent_of_the_gradient_is_refused():
    """Forward over reverse: a backward pass whose incoming gradient carries a tangent."""
    for name, tensors, call in calls():
        t = {m: v.clone().requires_grad_() for m, v in tensors.items()}
        out = call(t)
        with fwd.dual_level():
            d = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, list(t.values()), d, retain_graph=True, allow_unused=True)
        got = torch.autograd.grad(out, list(t.values()), torch.ones_like(out), allow_unused=True)
        assert any(v is not None and bool(torch.isfinite(v).all()) for v in got), name


def test_the_norm_of_recorded_gradients_raises_where_it_is_differentiated():
    """A gradient penalty on optim.grad_norm would otherwise train as if the penalty were not there."""
    from cpfn_amd import optim
    torch.manual_seed(0)
    w = torch.nn.Parameter(torch.randn(7, 5, device=DEV))
    x = torch.randn(9, 7, device=DEV)
    loss = ((x @ w) ** 3).sum()
    (g,) = torch.autograd.grad(loss, [w], create_graph=True)
    for recorded in (g, w):
        plain = recorded.detach()
        for p in (1.0, 2.0, float("inf")):
            want = optim.grad_norm([plain], p)
            got = optim.grad_norm([recorded], p)
            assert not want.requires_grad and got.requires_grad and torch.equal(got.detach(), want)
            with pytest.raises(RuntimeError, match="grad_norm"):
                (loss + got ** 2).backward(retain_graph=True)
            with torch.no_grad():
                assert not optim.grad_norm([recorded], p).requires_grad
    w.grad = None
    loss.backward(create_graph=True)                       # clipping works on values, as torch.nn.utils.clip_grad_norm_ does
    before = w.grad.detach().clone()
    norm = optim.clip_grad_norm_([w], 1.0, error_if_nonfinite=True)
    assert not norm.requires_grad and torch.equal(norm, optim.grad_norm([before]))
    torch.testing.assert_close(w.grad.detach(), before / (norm + 1e-6), rtol=1e-6, atol=0.0)     # (three roundings)
    w.grad = None
    with fwd.dual_level():
        dual = fwd.make_dual(before.clone(), torch.ones_like(before))
        for call in (lambda: optim.grad_norm([dual]), lambda: optim.clip_grads_([dual], 1.0), lambda: optim.clip_grads_([before], 1.0, out=[dual])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
