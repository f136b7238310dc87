"""CPU: what the routed residual block's operators and the gradient lists refuse — at the Python entry points and at the C ABI (refused
before anything is launched, so no GPU is needed) —, and clipping in the trainer's host path, with one process and with two (gloo)."""
import ctypes
import os

import pytest
import torch
import torch.distributed as dist

import test_ddp_gloo as dp
from cpfn_amd import autograd_ops, lib, ops, optim, training


def test_python_entry_points_refuse_cpu_tensors_and_wrong_arguments():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for call in (lambda: autograd_ops.row_norm(x, w), lambda: autograd_ops.norm_residual(x, x), lambda: ops.norm_residual_fwd(x, x),
                 lambda: ops.norm_residual_bwd(x, x, w, None, None, "none", None, None, x, None),
                 lambda: ops.route_plan(torch.zeros(4, 2, dtype=torch.int32), 3),
                 lambda: autograd_ops.route_gather(x, ops.RoutePlan(torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), 3)),
                 lambda: autograd_ops.route_combine(x, None, ops.RoutePlan(torch.zeros(4, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32), 3)),
                 lambda: optim.grad_norm([x]), lambda: optim.clip_grads_([x], 1.0), lambda: optim.clip_grads_([], 1.0, out=[x])):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError, match="kind"):
        autograd_ops.row_norm(x, w, kind="batch")
    with pytest.raises(RuntimeError, match="gate_act"):
        autograd_ops.norm_residual(x, x, gate=x, gate_act="tanh")
    with pytest.raises(RuntimeError, match="norm_type"):
        optim.grad_norm([x], norm_type=3)
    with pytest.raises(RuntimeError, match="max_norm"):
        optim.clip_grads_([], -1.0)
    with pytest.raises(RuntimeError, match="RoutePlan"):
        autograd_ops.route_gather(x, (x, x))
    for bad in (3, None, "x"):
        with pytest.raises(RuntimeError):
            autograd_ops.row_norm(bad, w)
        with pytest.raises(RuntimeError):
            optim.grad_norm([bad])
    assert float(optim.grad_norm([])) == 0.0 and float(optim.clip_grads_([], 1.0)) == 0.0
    with pytest.raises(RuntimeError):
        training.SPFNTrainer(dp.TinyHeads(), fused_adam=False, max_grad_norm=-1.0)


EINVAL, EOVERLAP = -22, -16
A = 1 << 20                       # (an address that is never used: every call below is refused)


def test_c_abi_refuses_bad_norm_arguments():
    h = lib.lib()

    def fwd(x=A, y=A, gate=None, weight=A, bias=A, scale=A, nw=A, nb=A, P=8, C=16, gate_rows=0, dtype=1, eps=1e-5, out=A, normed=A):
        return h.cpfn_norm_residual_fwd(x, y, gate, weight, bias, scale, nw, nb, P, C, gate_rows, dtype, 0, 0, eps, out, normed, None)

    for kw in (dict(P=-1), dict(C=0), dict(C=4097), dict(dtype=3), dict(dtype=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None),
               dict(out=None), dict(nw=None), dict(weight=None), dict(gate=A, gate_rows=0), dict(gate=A, gate_rows=3), dict(y=None),
               dict(y=None, weight=None, bias=None, scale=None, gate=A, gate_rows=8)):
        assert fwd(**kw) == EINVAL, kw

    def bwd(x=A, y=A, gate=None, weight=A, bias=A, scale=A, nw=A, d_out=A, d_normed=A, P=8, C=16, gate_rows=0, dtype=1, eps=1e-5,
            d_gate=None, d_weight=A, d_bias=A, d_scale=A, d_nw=A, d_nb=A, ws=A):
        return h.cpfn_norm_residual_bwd(x, y, gate, weight, bias, scale, nw, d_out, d_normed, P, C, gate_rows, dtype, 0, 0, eps, A, A, d_gate, d_weight,
                                        d_bias, d_scale, d_nw, d_nb, ws, None)

    for kw in (dict(P=0), dict(C=0), dict(C=4097), dict(dtype=7), dict(ws=None), dict(d_out=None, d_normed=None, d_nw=None, d_nb=None),
               dict(weight=None), dict(scale=None), dict(d_gate=A), dict(d_normed=None), dict(nw=None), dict(x=None), dict(gate=A, gate_rows=5)):
        assert bwd(**kw) == EINVAL, kw
    assert h.cpfn_norm_residual_workspace(-1, 4, 0) == -1 and h.cpfn_norm_residual_workspace(6, 4, 4) == -1
    for P, C, G in ((1, 1, 0), (131072, 128, 0), (131072, 128, 16), (6, 4096, 6), (1 << 33, 4096, 0), (5000000, 8, 5000000 // 2)):
        assert 0 < h.cpfn_norm_residual_workspace(P, C, G) <= 5 * C * 4 * max(2 * 2048 + G, P * C >> 26), (P, C, G)


def test_c_abi_refuses_bad_routes():
    h = lib.lib()
    assert h.cpfn_route_plan(A, 0, 1 << 31, 4, A, A, A, None) == EINVAL
    assert h.cpfn_route_plan(A, 0, 8, 0, A, A, A, None) == EINVAL
    assert h.cpfn_route_plan(A, 0, 8, 2049, A, A, A, None) == EINVAL
    assert h.cpfn_route_plan(None, 0, 8, 4, A, A, A, None) == EINVAL
    assert h.cpfn_route_plan(A, 0, 8, 4, None, A, A, None) == EINVAL
    assert h.cpfn_route_plan(A, 0, 1 << 20, 4, A, A, None, None) == EINVAL
    assert h.cpfn_route_workspace(-1, 4) == -1 and h.cpfn_route_workspace(8, 4) == 0 and h.cpfn_route_workspace(1 << 20, 4) > 0
    assert h.cpfn_route_gather(A, A, A, 8, 0, 4, 16, 1, A, None) == EINVAL
    assert h.cpfn_route_gather(A, A, A, 8, 2, 4, 0, 1, A, None) == EINVAL
    assert h.cpfn_route_gather(A, A, A, 1 << 30, 2, 4, 16, 1, A, None) == EINVAL
    assert h.cpfn_route_gather(A, A, A, 8, 2, 4, 16, 9, A, None) == EINVAL
    assert h.cpfn_route_gather(A, None, A, 8, 2, 4, 16, 1, A, None) == EINVAL
    assert h.cpfn_route_combine(None, A, A, 8, 2, 16, 1, A, None) == EINVAL
    assert h.cpfn_route_combine_bwd(A, A, A, A, A, 8, 2, 4, 16, 1, None, None, None) == EINVAL
    assert h.cpfn_route_combine_bwd(A, None, A, A, A, 8, 2, 4, 16, 1, A, A, None) == EINVAL


def test_c_abi_refuses_rows_that_are_walked_out_of_32_bits():
    h = lib.lib()
    for R in (0, 1):
        assert h.cpfn_route_gather(A, A, A, R, 1, 4, (1 << 30) + 1, 1, A, None) == EINVAL
        assert h.cpfn_route_combine(A, A, A, R, 1, (1 << 30) + 1, 1, A, None) == EINVAL
        assert h.cpfn_route_combine_bwd(A, A, A, A, A, R, 1, 4, (1 << 30) + 1, 1, A, A, None) == EINVAL


def test_c_abi_refuses_bad_gradient_lists():
    h = lib.lib()

    def table(rows):
        k = len(rows)
        return ((ctypes.c_void_p * k)(*[r[0] for r in rows]), (ctypes.c_longlong * k)(*[r[1] for r in rows]), (ctypes.c_int * k)(*[r[2] for r in rows]))

    def clip(rows, out=None, max_norm=1.0, p=2, norm=A, ws=A):
        g, n, t = table(rows)
        o, _, ot = table(out) if out else (None, None, None)
        return h.cpfn_grad_clip(g, o, n, t, ot, len(rows), p, max_norm, norm, ws, None)

    one = (A, 100, 0)
    for status, rows, kw in ((EINVAL, [(A, -1, 0)], {}), (EINVAL, [(None, 4, 0)], {}), (EINVAL, [(A, 4, 3)], {}), (EINVAL, [one], dict(max_norm=-1.0)),
                             (EINVAL, [one], dict(max_norm=float("nan"))), (EINVAL, [one], dict(norm=None)), (EINVAL, [one], dict(ws=None)),
                             (EINVAL, [one], dict(ws=A + 4)), (EINVAL, [(A, 100, 1)], dict(out=[(4 * A, 100, 2)])), (EINVAL, [one], dict(out=[(None, 100, 0)])),
                             (EINVAL, [(A, 1 << 49, 0)], {}),
                             (EOVERLAP, [one, one], {}), (EOVERLAP, [one, (A + 396, 4, 1)], {}), (EOVERLAP, [one, (A - 4, 2, 0)], {}),
                             (EOVERLAP, [one], dict(out=[(A + 4, 100, 0)])), (EOVERLAP, [(A, 100, 1)], dict(out=[(A, 100, 0)])),
                             (EOVERLAP, [one, (2 * A, 5, 0)], dict(out=[(3 * A, 100, 0), (A + 8, 5, 0)])),
                             (EOVERLAP, [one, (2 * A, 5, 0)], dict(out=[(3 * A, 100, 0), (3 * A + 399, 5, 0)])), (EINVAL, [one], dict(p=3))):
        assert clip(rows, **kw) == status, (rows, kw)
    g, n, t = table([one])
    assert h.cpfn_grad_norm(g, n, t, 1, 5, A, A, None) == EINVAL and h.cpfn_grad_norm(g, n, t, -1, 2, A, A, None) == EINVAL
    assert h.cpfn_grad_norm(g, n, t, 1, 2, None, A, None) == EINVAL
    assert h.cpfn_grad_sumsq_blocks(-1) == -1 and h.cpfn_grad_sumsq(None, 5, A, None) == EINVAL
    assert h.cpfn_adam_flat_clip(A, A, A, A, 8, A, 0.9, 0.999, 1e-8, 0.0, A, A, None, A, None, 0, 0, None, -1.0, A, A, None) == EINVAL
    assert h.cpfn_adam_flat_clip(A, A, A, A, 8, A, 0.9, 0.999, 1e-8, 0.0, A, A, None, A, None, 0, 0, None, 1.0, None, A, None) == EINVAL


def _train(seeds_per_step, max_norm, world=1):
    torch.manual_seed(100)
    model = dp.TinyHeads()
    tr = training.SPFNTrainer(model, batch_size=4, multipliers=dp.LOCAL_MULT, fused_adam=False, max_grad_norm=max_norm)
    norms = []
    for seeds in seeds_per_step:
        tr.step(dp._cat([dp._batch(2, seed=s) for s in seeds]))
        norms.append(None if tr.grad_norm is None else float(tr.grad_norm))
    return model, tr, norms


def test_trainer_clips_on_the_host_path():
    """The same steps by hand: torch's own clip and Adam on the trainer's losses; without max_grad_norm nothing changes."""
    steps = [(0, 1), (10, 11), (20, 21)]
    model, tr, norms = _train(steps, 0.05)
    torch.manual_seed(100)
    hand = dp.TinyHeads()
    plain = training.SPFNTrainer(hand, batch_size=4, multipliers=dp.LOCAL_MULT, fused_adam=False)
    opt = torch.optim.Adam(hand.parameters(), lr=1e-3)
    for seeds, norm in zip(steps, norms):
        opt.zero_grad()
        plain.losses(dp._cat([dp._batch(2, seed=s) for s in seeds]))[0].backward()
        want = torch.nn.utils.clip_grad_norm_(hand.parameters(), 0.05)
        assert abs(norm - float(want)) <= 1e-5 * float(want) and norm > 0.05
        opt.step()
    for a, b in zip(model.parameters(), hand.parameters()):
        # (two trainings whose gradients agree to ~1e-6 relative; three steps of at most lr = 1e-3 each, so 1e-3 * 3 * 1e-4 leaves room
        #  for components whose gradient nearly cancels)
        torch.testing.assert_close(a, b, rtol=1e-5, atol=3e-7)
    assert _train(steps, None)[1].grad_norm is None


def _worker(rank, world, port, out_dir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.manual_seed(100 + rank)
    model = dp.TinyHeads()
    training.broadcast_parameters(model)
    tr = training.SPFNTrainer(model, batch_size=2 * world, multipliers=dp.LOCAL_MULT, fused_adam=False, max_grad_norm=0.05)
    norms = []
    for step in range(3):
        tr.step(dp._batch(2, seed=10 * step + rank))
        norms.append(float(tr.grad_norm))
    torch.save(({k: v.clone() for k, v in model.state_dict().items()}, norms), os.path.join(out_dir, "rank%d.pt" % rank))
    dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_two_ranks_clip_by_the_norm_of_the_mean_gradient(tmp_path):
    dp._spawn(_worker, 2, str(tmp_path))
    (a, na), (b, nb) = (torch.load(os.path.join(str(tmp_path), "rank%d.pt" % r)) for r in range(2))
    assert na == nb and all(torch.equal(a[k], b[k]) for k in a)
    model, _, norms = _train([(10 * s, 10 * s + 1) for s in range(3)], 0.05)
    assert all(abs(x - y) <= 1e-3 * y for x, y in zip(na, norms))
    for k, v in model.state_dict().items():
        torch.testing.assert_close(v, a[k], rtol=2e-4, atol=2e-6)          # (as test_ddp_gloo compares the two trainings without clipping)
