"""SPFNTrainer(max_grad_norm=): a step that is skipped for its gradients, and the norm that is reported."""
import contextlib
import io
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def trainer(**kw):
    from cpfn_amd import synthetic, training
    from cpfn_amd.PointNet2 import pn2_network
    from cpfn_amd.SPFN import fitter_factory
    with contextlib.redirect_stdout(io.StringIO()):
        fitter_factory.register_primitives(training.GLOBAL_SPFN_CLASSES)
    torch.manual_seed(0)
    model = pn2_network.PointNet2(dim_input=3, dim_pos=3, output_sizes=[3, 4, 28]).to(DEV)
    model.set_compute_dtype(torch.bfloat16)
    tr = training.SPFNTrainer(model, batch_size=2, max_grad_norm=0.05, **kw)
    batch = {k: v.to(DEV) for k, v in synthetic.training_batch(2, N=2048, n_prims=6, n_inst_points=128, seed=5).items()}
    bad = {k: v.clone() for k, v in batch.items()}
    bad["P"][1, 100, 2] = float("nan")
    return model, tr, batch, bad


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("fused", [True, False])
def test_training_goes_on_after_a_skipped_step(fused, graphs):
    """Parameters without a gradient (layers in front of a BatchNorm) keep a zero slice in the bucket, which a NaN factor must not reach:
    every later step would be skipped too."""
    model, tr, batch, bad = trainer(use_graphs=graphs, require_graphs=graphs, fused_adam=None if fused else False)
    skipped = 0
    for step, b in enumerate((batch, bad, batch, batch, bad, batch)):
        before = [p.detach().clone() for p in model.parameters()]
        tr.step(b)
        torch.cuda.synchronize()
        skipped += b is bad
        assert tr.skipped_steps == skipped, step
        same = all(torch.equal(p, q) for p, q in zip(model.parameters(), before))
        assert same == (b is bad), step
        assert all(p.grad is not None or not bool(v.any()) for p, v in zip(tr.bucket.params, tr.bucket.views)), step
    assert (tr._graph is not None) == graphs


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("fused", [True, False])
def test_the_norm_is_the_last_step_s(fused, graphs):
    """Nothing before the first step; of a skipped step its own, not the one before."""
    _, tr, batch, bad = trainer(use_graphs=graphs, require_graphs=graphs, fused_adam=None if fused else False)
    assert tr.grad_norm is None
    for step, b in enumerate((batch, bad, batch, batch, bad, batch)):
        tr.step(b)
        torch.cuda.synchronize()
        assert math.isfinite(float(tr.grad_norm)) == (b is batch), step
