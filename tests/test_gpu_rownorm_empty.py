"""Norms of no rows: clouds without points keep their gate's rows, whose gradient is zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("groups", [0, 1, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clouds_without_points_and_a_gate_for_each(dtype, groups):
    from cpfn_amd import autograd_ops, ops
    C = 24
    x, y = (torch.zeros(0, C, dtype=dtype, device=DEV).requires_grad_() for _ in range(2))
    gate = torch.randn(groups, C, device=DEV).to(dtype).requires_grad_()
    w = torch.ones(C, device=DEV, requires_grad=True)
    out, normed = autograd_ops.norm_residual(x, y, w, gate=gate, gate_act="sigmoid", next_weight=w)
    assert out.shape == normed.shape == (0, C) and out.dtype == dtype
    g = torch.autograd.grad([out, normed], [x, y, gate, w], [torch.zeros_like(out)] * 2)
    for a, b in zip(g, (x, y, gate, w)):
        assert a.shape == b.shape and a.dtype == b.dtype and not bool(a.any())
    with torch.no_grad():
        assert ops.norm_residual_fwd(x, y, gate=gate)[0].shape == (0, C)
