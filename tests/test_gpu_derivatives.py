"""Derivatives that the routed residual block's operators do not have are refused on the device, not lost: forward-mode tangents on an
input or on the gradient that a backward pass is given."""
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
