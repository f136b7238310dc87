"""CPU: SPFNTrainer.grad_norm is the last step's: of a step that was skipped for its gradients too."""
import math

import pytest
import torch

import test_ddp_gloo as dp
from cpfn_amd import training


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_skipped_step_leaves_its_own_norm(value):
    torch.manual_seed(100)
    model = dp.TinyHeads()
    tr = training.SPFNTrainer(model, batch_size=2, multipliers=dp.LOCAL_MULT, fused_adam=False, max_grad_norm=0.05)
    assert tr.grad_norm is None
    tr.step(dp._batch(2, seed=0))
    assert math.isfinite(float(tr.grad_norm))
    weights = [p.detach().clone() for p in model.parameters()]
    first = next(p for p in model.parameters() if p.grad is not None)
    hook = first.register_hook(lambda g: torch.full_like(g, value))
    tr.step(dp._batch(2, seed=1))
    hook.remove()
    assert tr.skipped_steps == 1 and all(torch.equal(a, b) for a, b in zip(model.parameters(), weights))
    norm = float(tr.grad_norm)
    assert math.isnan(norm) if math.isnan(value) else norm == math.inf
    tr.step(dp._batch(2, seed=2))
    assert tr.skipped_steps == 1 and math.isfinite(float(tr.grad_norm))
