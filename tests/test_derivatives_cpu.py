"""CPU: derivatives that the routed residual block's operators do not have are refused, not lost: a forward-mode tangent on any input, or on a
tensor of a gradient list.
(The refusal comes before the check of the device, so that it shows without a GPU.)"""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from cpfn_amd import autograd_ops, ops, optim


def _plan(rows, k, E):
    return ops.RoutePlan(torch.zeros(E + 1, dtype=torch.int32), torch.zeros(rows, k, dtype=torch.int32), E)


def calls():
    """(name, tensors by name, the call on them) of every operator with a backward pass"""
    C = 8
    rows = {n: torch.ones(4, C) for n in ("x", "y", "gate")}
    rows.update({n: torch.ones(C) for n in ("weight", "bias", "scale", "next_weight", "next_bias")})
    plan = _plan(4, 2, 3)
    return [("row_norm", {"x": rows["x"], "weight": rows["weight"], "bias": rows["bias"]}, lambda t: autograd_ops.row_norm(t["x"], t["weight"], t["bias"])),
            ("norm_residual", rows, lambda t: autograd_ops.norm_residual(**t)),
            ("route_gather", {"rows": rows["x"]}, lambda t: autograd_ops.route_gather(t["rows"], plan)),
            ("route_combine", {"sorted_rows": torch.ones(8, C), "weights": torch.ones(4, 2)},
             lambda t: autograd_ops.route_combine(t["sorted_rows"], t["weights"], plan))]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("trained", [True, False])
def test_forward_mode_tangents_are_refused(trained, grad_mode):
    for name, tensors, call in calls():
        for n in tensors:
            with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
                t = {m: v.clone().requires_grad_(trained) for m, v in tensors.items()}
                t[n] = fwd.make_dual(t[n], torch.ones_like(t[n]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(t)


def test_forward_mode_tangents_in_a_gradient_list_are_refused():
    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(torch.ones(5), torch.ones(5))
        for call in (lambda: optim.grad_norm([dual]), lambda: optim.clip_grads_([dual], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
