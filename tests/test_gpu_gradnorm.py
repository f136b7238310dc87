"""optim.grad_norm / clip_grads_ / clip_grad_norm_, FlatAdam.step(max_grad_norm) and SPFNTrainer(max_grad_norm) against 64 bits.

Tolerances: sums are fp64 (far below one fp32 step), so the norm is off by its one rounding, u = 2^-24 relative, and the factor by
its own; a clipped value by the factor's rounding, the product's and the store's half step."""
import copy
import math

import pytest
import torch

from approx import Approx, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
INF = float("inf")


def lists(kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    sizes, types = {
        "one value": ([1], [torch.float32]),
        "mixed": ([5, 0, 1, 64, 4097, 130000, 16384, 16385, 7], [torch.float32, torch.bfloat16, torch.float16]),
        "many": ([(37 * i) % 601 for i in range(333)], [torch.bfloat16, torch.float32]),
        "large": ([40_000_003, 1_000_000, 9], [torch.float32]),
        "large16": ([40_000_003, 1_000_000, 9], [torch.bfloat16, torch.float16]),
    }[kind]
    return [(torch.randn(n, generator=g) * 10.0 ** -(i % 4)).to(types[i % len(types)]).to(DEV) for i, n in enumerate(sizes)]


def exact_norm(grads, p):
    wide = [t.double().reshape(-1) for t in grads if t.numel()]
    if not wide:
        return 0.0
    if p == INF:
        return max(float(t.abs().max()) for t in wide)
    return float(sum((t.abs() ** p).sum() for t in wide)) ** (1.0 / p)


def within(got, want64, factor):
    """A clipped tensor: (1 + u)^3 for factor, its conversion and the product, then half a step of its type."""
    fi = torch.finfo(got.dtype)
    tol = 3.01 * U * want64.abs() + 0.5 * fi.eps * want64.abs() + 0.5 * fi.smallest_normal * fi.eps
    return bool(((got.double() - want64).abs() <= tol * (1 + 1e-6)).all())


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("kind", ["one value", "mixed", "many", "large", "large16"])
def test_norm_and_clip_against_64_bits(kind, p):
    from cpfn_amd import optim
    grads = lists(kind)
    norm = exact_norm(grads, p)
    got = optim.grad_norm(grads, norm_type=p)
    assert got.shape == () and got.dtype == torch.float32 and got.device == grads[0].device
    assert abs(float(got) - norm) <= (1 + 1e-6) * U * norm
    before = [t.clone() for t in grads]
    for max_norm in (0.3 * norm, 0.0):
        coef = min(1.0, max_norm / (norm + 1e-6))
        want = [t.double() * coef for t in before]
        out = [torch.full(t.shape, float("nan"), dtype=torch.float32, device=DEV) for t in grads]
        assert float(optim.clip_grads_(grads, max_norm, norm_type=p, out=out)) == float(got)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        assert all(within(o, w, coef) for o, w in zip(out, want))
    same = [torch.empty_like(t) for t in grads]
    optim.clip_grads_(grads, 0.3 * norm, norm_type=p, out=same)
    assert float(optim.clip_grads_(grads, 0.3 * norm, norm_type=p)) == float(got)
    coef = min(1.0, 0.3 * norm / (norm + 1e-6))
    assert all(torch.equal(a, b) for a, b in zip(grads, same))
    assert all(within(t, b.double() * coef, coef) for t, b in zip(grads, before))


def test_within_the_bound_nothing_changes_and_out_is_a_copy():
    from cpfn_amd import optim
    grads = lists("mixed")
    before = [t.clone() for t in grads]
    out = [torch.zeros_like(t) for t in grads]
    for max_norm in (10 * exact_norm(grads, 2.0), INF):
        optim.clip_grads_(grads, max_norm)
        optim.clip_grads_(grads, max_norm, out=out)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        assert all(torch.equal(a, b) for a, b in zip(out, before))


def test_values_far_out_of_the_squares_range():
    """Squares of 1e30 and of 1e-40 are not fp32 numbers: the sums are fp64."""
    from cpfn_amd import optim
    for v in (1e30, 1e-40):
        t = torch.full((1000,), v, device=DEV)
        x = float(t[0].double())
        assert abs(float(optim.grad_norm([t])) - x * math.sqrt(1000)) <= U * x * math.sqrt(1000) * (1 + 1e-6) + 2.0 ** -150


def test_not_finite_gradients():
    from cpfn_amd import optim
    for p in (1.0, 2.0, INF):
        for where in (0, 4096, 29999):
            t = [torch.ones(30000, device=DEV), torch.ones(7, dtype=torch.bfloat16, device=DEV)]
            t[0][where] = -INF
            assert float(optim.grad_norm(t, p)) == INF
            optim.clip_grads_(t, 1.0, p)
            assert torch.isnan(t[0][where]) and float(t[0].nan_to_num().abs().sum()) == 0.0 and not bool(t[1].any())
            t = [torch.ones(30000, device=DEV), torch.ones(7, dtype=torch.bfloat16, device=DEV)]
            t[0][where] = float("nan")
            assert math.isnan(float(optim.grad_norm(t, p)))
            optim.clip_grads_(t, 1.0, p)
            assert all(bool(torch.isnan(x).all()) for x in t)


def test_any_alignment_and_order_of_dimensions():
    from cpfn_amd import optim
    g = torch.Generator().manual_seed(2)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for n in (1, 3, 8, 4099):
            for a in (0, 1, 3):
                for b in (0, 1, 5):
                    src = torch.randn(n + 16, generator=g).to(dt).to(DEV)[a:a + n]
                    buf = torch.full((n + 16,), 7.0, device=DEV)
                    norm = exact_norm([src], 2.0)
                    optim.clip_grads_([src], 0.5 * norm, out=[buf[b:b + n]])
                    assert within(buf[b:b + n], src.double() * (0.5 * norm / (norm + 1e-6)), 0.5)
                    assert bool((buf[:b] == 7.0).all()) and bool((buf[b + n:] == 7.0).all())
    t = torch.randn(6, 5, 4, generator=g).to(DEV)
    for v in (t.permute(2, 0, 1), t.t() if t.dim() == 2 else t.transpose(0, 2), torch.randn(2, 3, 4, 5, device=DEV).to(memory_format=torch.channels_last)):
        w = v.clone(memory_format=torch.preserve_format)
        norm = exact_norm([v], 2.0)
        optim.clip_grads_([w], 0.5 * norm)
        assert within(w, v.double() * (0.5 * norm / (norm + 1e-6)), 0.5)


def test_refusals_on_the_device():
    from cpfn_amd import optim
    a = torch.randn(100, device=DEV)
    b = torch.randn(50, device=DEV)
    keep = a.clone()
    for call in (lambda: optim.clip_grads_([a, b, a], 1e-3), lambda: optim.clip_grads_([a, a[50:]], 1e-3),
                 lambda: optim.clip_grads_([a[:60], b], 1e-3, out=[a[10:70], b]),
                 lambda: optim.clip_grads_([a[:50], b], 1e-3, out=[b, torch.empty(50, device=DEV)]),
                 lambda: optim.clip_grads_([a], 1e-3, out=[a.view(10, 10)]), lambda: optim.clip_grads_([a], 1e-3, out=[a.half()]),
                 lambda: optim.clip_grads_([a.view(10, 10)[:, :5]], 1e-3), lambda: optim.clip_grads_([a.double()], 1e-3),
                 lambda: optim.grad_norm([a[:1].expand(10)]), lambda: optim.clip_grads_([a], 1e-3, out=[]),
                 lambda: optim.grad_norm([a, torch.zeros(3)]), lambda: optim.clip_grads_([a], float("nan"))):
        with pytest.raises(RuntimeError):
            call()
    assert torch.equal(a, keep)
    assert abs(float(optim.grad_norm([a, a])) - exact_norm([a, a], 2.0)) < 1e-4      # (only reading it twice is fine)


def test_clip_grad_norm_of_parameters():
    from cpfn_amd import optim
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(33, 17), torch.nn.Linear(17, 5)).to(DEV)
    unused = torch.nn.Parameter(torch.zeros(3, device=DEV))
    (m(torch.randn(9, 33, device=DEV)) ** 2).sum().backward()
    mb = copy.deepcopy(m)
    for p, q in zip(m.parameters(), mb.parameters()):
        q.grad = p.grad.clone()
    got = optim.clip_grad_norm_(list(m.parameters()) + [unused], 0.5)
    want = torch.nn.utils.clip_grad_norm_(mb.parameters(), 0.5)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=0.0)              # (torch sums fp32 squares of <= 561 values: n u at most)
    for p, q in zip(m.parameters(), mb.parameters()):
        torch.testing.assert_close(p.grad, q.grad, rtol=2e-5, atol=0.0)
    assert unused.grad is None
    keep = [p.grad.clone() for p in m.parameters()]
    m[0].weight.grad[0, 0] = float("nan")
    keep[0][0, 0] = float("nan")
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm_(m.parameters(), 1e-4, error_if_nonfinite=True)
    for p, k in zip(m.parameters(), keep):
        assert torch.equal(p.grad.nan_to_num(), k.nan_to_num())


def test_streams_repeats_and_captured_graphs():
    from cpfn_amd import optim
    grads = lists("many") + [torch.zeros(3_000_001, device=DEV)]
    out = [torch.empty(t.shape, device=DEV) for t in grads]

    def both():
        return [optim.grad_norm(grads, INF), optim.clip_grads_(grads, 0.5, out=out)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        both()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                held = both()
            graphs.append((g, held))
    s.synchronize()
    for i in range(4):
        grads[-1].normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        want = [t.clone() for t in both() + out]
        for g, held in graphs:
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held + out, want))


def check_adam_step(opt, before, grad, t, max_norm, lr):
    """`opt` after step t (1, 2, ..) against Adam's formulas in 64 bits on its state `before` (parameters, moments) and the clipped
    gradient, the hyper-parameters being the fp32 numbers that they are.  Returns the clipping factor."""
    one = torch.ones(1, dtype=torch.float64, device=grad.device)
    b1, b2 = (float(torch.tensor(b, dtype=torch.float32)) for b in (0.9, 0.999))
    o1, o2 = (float(torch.tensor(1.0, dtype=torch.float32) - torch.tensor(b, dtype=torch.float32)) for b in (0.9, 0.999))
    lr, eps = (float(torch.tensor(v, dtype=torch.float32)) for v in (lr, 1e-8))
    p, m, v = (Approx(x.double()) for x in before)
    norm = exact_norm([grad], 2.0)
    assert abs(float(opt.grad_norm) - norm) <= (1 + 1e-6) * U * norm
    coef = min(1.0, max_norm / (norm + 1e-6))
    g = Approx(grad.double()) * Approx(coef * one, U * coef * one)
    m = m + (g - m) * o1
    v = v * b2 + g * g * o2
    step_size = Approx(one * lr) / Approx(one * (1 - b1 ** t), U * one)
    denom = v.sqrt() / Approx(one * (1 - b2 ** t), U * one * (1 - b2 ** t)).sqrt() + eps
    p = p - step_size * (m / denom)
    assert_within(opt.exp_avg, m, "exp_avg")
    assert_within(opt.exp_avg_sq, v, "exp_avg_sq")
    assert_within(opt.flat_p, p, "parameters")
    return coef


def _adam_pair(seed=3):
    from cpfn_amd import training
    from cpfn_amd.optim import FlatAdam
    torch.manual_seed(seed)
    ma = torch.nn.Sequential(torch.nn.Linear(70, 130), torch.nn.ReLU(), torch.nn.Linear(130, 51)).to(DEV)
    mb = copy.deepcopy(ma)
    bucket = training.FlatGradBucket(ma)
    return ma, mb, bucket, FlatAdam(bucket, lr=1e-2), torch.optim.Adam(mb.parameters(), lr=1e-2)


def test_adam_on_clipped_gradients():
    """FlatAdam.step(max_grad_norm) is Adam on the clipped gradients: the formulas in 64 bits on the gradients that every step read
    (with the hyper-parameters as the fp32 numbers they are), errors followed step by step (tests/approx.py).  The bucket keeps the
    gradients, the norm is left on the device."""
    ma, mb, bucket, oa, _ = _adam_pair()
    g = torch.Generator().manual_seed(0)
    for step in range(8):
        x = torch.randn(32, 70, generator=g).to(DEV)
        for q in ma.parameters():
            q.grad = None
        ((ma(x) * (10.0 if step % 2 else 0.01)) ** 2).mean().backward()
        bucket.collect()
        flat = bucket.flat.clone()
        state = [t.clone() for t in (oa.flat_p, oa.exp_avg, oa.exp_avg_sq)]
        oa.step(max_grad_norm=0.2)
        assert torch.equal(bucket.flat, flat)
        coef = check_adam_step(oa, state, flat, step + 1, 0.2, 1e-2)
        assert (coef < 1.0) == bool(step % 2)


def test_adam_within_the_bound_is_the_plain_step_bit_for_bit():
    from cpfn_amd.optim import FlatAdam
    ma, mb, bucket, oa, _ = _adam_pair()
    from cpfn_amd import training
    bb = training.FlatGradBucket(mb)
    ob = FlatAdam(bb, lr=1e-2)
    for i in range(3):
        bucket.flat.normal_()
        bb.flat.copy_(bucket.flat)
        oa.step(max_grad_norm=1e9)
        ob.step()
        assert torch.equal(oa.flat_p, ob.flat_p) and torch.equal(oa.exp_avg_sq, ob.exp_avg_sq)


def test_adam_skips_gradients_that_are_not_finite():
    ma, _, bucket, opt, _ = _adam_pair()
    skipped = torch.zeros((), device=DEV)
    for pos, val, skip in ((None, 0.0, False), (0, float("nan"), True), (bucket.flat.numel() - 1, INF, True), (777, 3.0e38, False)):
        bucket.flat.normal_()
        if pos is not None:
            bucket.flat[pos] = val
        before, steps = opt.flat_p.clone(), float(opt.step_count)
        opt.step(max_grad_norm=1.0, skipped=skipped)
        assert (float(opt.step_count) == steps) == skip and torch.equal(opt.flat_p, before) == skip
        assert bool(torch.isfinite(opt.flat_p).all())
    assert float(skipped) == 2.0
    with pytest.raises(RuntimeError):
        opt.step(max_grad_norm=-1.0)
    with pytest.raises(RuntimeError):
        opt.step(max_grad_norm=1.0, combine=(bucket.flat, bucket.flat, 1, bucket.flat))


@pytest.mark.parametrize("graphs", [False, True])
def test_trainer_clips_its_steps(graphs):
    """SPFNTrainer(max_grad_norm): every step of the network's training, eager and replayed, is Adam on the clipped bucket; a batch whose
    gradients are not finite is skipped."""
    import contextlib
    import io
    from cpfn_amd import synthetic, training
    from cpfn_amd.PointNet2 import pn2_network
    from cpfn_amd.SPFN import fitter_factory
    with contextlib.redirect_stdout(io.StringIO()):
        fitter_factory.register_primitives(training.GLOBAL_SPFN_CLASSES)
    torch.manual_seed(0)
    model = pn2_network.PointNet2(dim_input=3, dim_pos=3, output_sizes=[3, 4, 28]).to(DEV)
    model.set_compute_dtype(torch.bfloat16)
    tr = training.SPFNTrainer(model, batch_size=4, init_learning_rate=1e-3, use_graphs=graphs, require_graphs=graphs, max_grad_norm=0.05)
    batch = {k: v.to(DEV) for k, v in synthetic.training_batch(4, N=2048, n_prims=6, n_inst_points=128, seed=5).items()}
    opt = tr.optimizer
    for step in range(6):
        state = [t.clone() for t in (opt.flat_p, opt.exp_avg, opt.exp_avg_sq)]
        tr.step(batch, next_batch=batch)
        torch.cuda.synchronize()
        assert check_adam_step(opt, state, tr.bucket.flat.clone(), step + 1, 0.05, 1e-3) < 1.0
        assert tr.grad_norm is opt.grad_norm
    assert (tr._graph is not None) == graphs and tr.skipped_steps == 0
    bad = {k: v.clone() for k, v in batch.items()}
    bad["P"][1, 100, 2] = float("nan")
    state = [t.clone() for t in (opt.flat_p, opt.exp_avg, opt.exp_avg_sq)]
    tr.step(bad)
    torch.cuda.synchronize()
    assert tr.skipped_steps == 1
    assert all(torch.equal(a, b) for a, b in zip(state, (opt.flat_p, opt.exp_avg, opt.exp_avg_sq)))
    tr.step(batch)
    torch.cuda.synchronize()
    assert tr.skipped_steps == 1 and bool(torch.isfinite(opt.flat_p).all()) and not torch.equal(opt.flat_p, state[0])


def test_trainer_with_another_optimizer_clips_the_bucket():
    from cpfn_amd import training
    torch.manual_seed(1)
    m = torch.nn.Linear(40, 9).to(DEV)
    tr = training.SPFNTrainer(m, fused_adam=False, max_grad_norm=0.1)
    (m(torch.randn(8, 40, device=DEV)) ** 2).sum().backward()
    tr.bucket.collect()
    before = tr.bucket.flat.clone()
    tr._clipped_optimizer_step()
    norm = exact_norm([before], 2.0)
    assert norm > 0.1 and abs(float(tr.grad_norm) - norm) <= (1 + 1e-6) * U * norm
    assert within(tr.bucket.flat, before.double() * (0.1 / (norm + 1e-6)), 0.1)
    assert training.SPFNTrainer(m, fused_adam=False).grad_norm is None


def test_what_is_clipped_counts_as_changed():
    """Autograd notices that a tensor which it kept was scaled, in place and through `out`."""
    from cpfn_amd import optim
    for elsewhere in (False, True):
        leaf = torch.randn(100, device=DEV, requires_grad=True)
        a = leaf * 2.0
        b = (a * a).sum()                                           # (keeps a)
        d = a.detach()
        if elsewhere:
            optim.clip_grads_([torch.ones(100, device=DEV)], 0.5, out=[d])
        else:
            optim.clip_grads_([d], 0.5)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            b.backward()
    with torch.inference_mode():
        x = torch.randn(100, device=DEV)
        norm = optim.clip_grads_([x], 0.5)
    assert abs(float(x.double().norm()) - 0.5) < 1e-5 and abs(float(norm)) > 0.5


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
def test_the_smallest_and_the_largest_bound_and_out_in_place(p):
    from cpfn_amd import optim
    for kind in ("mixed", "many"):
        keep = lists(kind)
        for bound in (0.0, INF):
            g = [t.clone() for t in keep]
            norm = optim.clip_grads_(g, bound, norm_type=p)
            assert abs(float(norm) - exact_norm(keep, p)) <= 2 * U * exact_norm(keep, p)          # (its one rounding, and 1e-16s)
            for a, b in zip(g, keep):
                assert torch.equal(a, b if bound else torch.zeros_like(b))
        ours, theirs = [t.clone() for t in keep], [t.clone() for t in keep]
        optim.clip_grads_(ours, 0.1, norm_type=p, out=ours)
        optim.clip_grads_(theirs, 0.1, norm_type=p)
        assert all(torch.equal(a, b) for a, b in zip(ours, theirs))


def test_adam_on_the_clipped_gradients_of_a_long_bucket():
    """As many partial sums as a call leaves, and their sum by the one wave that prepares the step."""
    from cpfn_amd import lib, training
    from cpfn_amd.optim import FlatAdam
    torch.manual_seed(1)
    m = torch.nn.Linear(4001, 3001).to(DEV)
    bucket = training.FlatGradBucket(m)
    opt = FlatAdam(bucket, lr=1e-2)
    assert lib.lib().cpfn_grad_sumsq_blocks(bucket.flat.numel()) >= 1999
    bucket.flat.normal_()
    flat = bucket.flat.clone()
    state = [t.clone() for t in (opt.flat_p, opt.exp_avg, opt.exp_avg_sq)]
    opt.step(max_grad_norm=0.5)
    assert torch.equal(bucket.flat, flat)
    assert check_adam_step(opt, state, flat, 1, 0.5, 1e-2) < 1e-3
