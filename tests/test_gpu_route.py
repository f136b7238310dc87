"""ops.route_plan and autograd_ops.route_gather / route_combine (csrc/route.hip): the order against a stable sort on the host, the moves
bit for bit, sums and gradients against 64 bits with tolerances from a running error analysis (tests/approx.py)."""
import pytest
import torch

from approx import Approx, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def order(choice, E):
    """offsets, place of a stable sort, on the host."""
    flat = choice.reshape(-1).cpu().long()
    ok = (flat >= 0) & (flat < E)
    entries = ok.nonzero().reshape(-1)
    entries = entries[torch.sort(flat[entries], stable=True)[1]]
    place = torch.full_like(flat, -1)
    place[entries] = torch.arange(entries.numel())
    offsets = torch.zeros(E + 1, dtype=torch.long)
    offsets[1:] = torch.bincount(flat[ok], minlength=E).cumsum(0)
    return offsets.int(), place.int().view(choice.shape)


def choices(R, k, E, seed=0, out_of=0.0, skew=False, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, E, (R, k), generator=g)
    if skew:
        c = torch.where(torch.rand(R, k, generator=g) < 0.7, torch.full_like(c, E // 2), c)
    if out_of:
        bad = torch.randint(0, 4, (R, k), generator=g)
        bad = torch.tensor([-1, E, E + 5, -2 ** 31])[bad]
        c = torch.where(torch.rand(R, k, generator=g) < out_of, bad, c)
    return c.to(dtype).to(DEV)


def check_plan(c, E):
    from cpfn_amd import ops
    plan = ops.route_plan(c, E)
    offsets, place = order(c, E)
    assert plan.offsets.dtype == plan.place.dtype == torch.int32 and plan.place.shape == c.shape
    assert torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(plan.place.cpu(), place)
    return plan


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("R,k,E", [(0, 2, 4), (1, 1, 1), (1, 2, 4), (63, 1, 3), (64, 1, 2), (65, 3, 28), (511, 8, 8), (512, 8, 2048),
                                   (4096, 1, 5), (4097, 1, 5), (2731, 3, 64), (32768, 8, 256), (32769, 8, 7), (100003, 2, 257),
                                   (32769, 8, 2047), (1000, 1, 1), (70000, 4, 1)])
def test_order_is_a_stable_sort(R, k, E, wide):
    """One tile, tiles that every workgroup sums by itself (up to 64, up to 256 experts) and the form with a scan in between; borders."""
    for out_of, skew in ((0.0, False), (0.3, True)):
        check_plan(choices(R, k, E, seed=R + E, out_of=out_of, skew=skew, dtype=torch.int64 if wide else torch.int32), E)


@pytest.mark.parametrize("R,k,E", [(300000, 2, 8), (300000, 2, 21), (300000, 2, 22), (524288, 1, 16), (524289, 1, 7), (600007, 1, 1), (64 * 2048, 1, 64),
                                   (64 * 2048 + 1, 1, 32), (64 * 2048 + 1, 1, 33), (2049, 1, 65)])
def test_order_at_the_borders_of_its_forms(R, k, E):
    """Longer lists, whose waves take more choices, and as many loads for the sums as a workgroup makes by itself, and one more."""
    check_plan(choices(R, k, E, seed=E, out_of=0.1), E)


def test_order_where_nothing_is_routed_and_where_all_go_to_one():
    for R, E in ((5000, 9), (5, 9), (300000, 300)):
        check_plan(torch.full((R, 2), -1, dtype=torch.int32, device=DEV), E)
        check_plan(torch.full((R, 2), E - 1, dtype=torch.int64, device=DEV), E)


def test_wide_indices_are_not_cut_to_32_bits():
    c = torch.tensor([[0, 2 ** 32], [2 ** 32 + 1, 1], [-2 ** 32, 2 ** 62]], device=DEV)
    plan = check_plan(c, 2)
    assert plan.place.tolist() == [[0, -1], [-1, 1], [-1, -1]]


def test_the_same_expert_twice_in_a_row():
    check_plan(torch.tensor([[1, 1, 0], [0, 1, 1]], dtype=torch.int32, device=DEV), 2)


def problem(R, k, E, C, dt, out_of=0.2, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(R, C, generator=g).to(dt).to(DEV).requires_grad_()
    mid = torch.randn(R * k, C, generator=g).to(dt).to(DEV).requires_grad_()
    w = torch.rand(R, k, generator=g).to(DEV).requires_grad_()
    d_sorted = torch.randn(R * k, C, generator=g).to(dt).to(DEV)
    d_out = torch.randn(R, C, generator=g).to(dt).to(DEV)
    return choices(R, k, E, seed, out_of), rows, mid, w, d_sorted, d_out


def check_moves(R, k, E, C, dt, out_of=0.2, seed=0, with_weights=True):
    from cpfn_amd import autograd_ops, ops
    c, rows, mid, w, d_sorted, d_out = problem(R, k, E, C, dt, out_of, seed)
    plan = ops.route_plan(c, E)
    place = plan.place.long()
    n = int(plan.offsets[-1])
    with torch.no_grad():                                          # what is behind the last expert's rows is not looked at
        mid[n:] = float("nan")
        d_sorted[n:] = float("nan")
    srt = autograd_ops.route_gather(rows, plan)
    there = place >= 0
    want = torch.zeros_like(mid)
    want[place[there]] = rows.detach().repeat_interleave(k, 0).view(R, k, C)[there]
    assert torch.equal(srt, want)
    out = autograd_ops.route_combine(mid, w if with_weights else None, plan)
    leaves = [rows, mid] + ([w] if with_weights else [])
    grads = torch.autograd.grad([srt, out], leaves, [d_sorted, d_out])
    wv = w.detach().double() if with_weights else torch.ones(R, k, dtype=torch.float64, device=DEV)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    picked = torch.where(there[:, :, None], mid.detach().double()[place.clamp(min=0)], zero)
    back = torch.where(there[:, :, None], d_sorted.double()[place.clamp(min=0)], zero)
    assert_within(out, (Approx(picked) * Approx(wv[:, :, None])).sum(1).view(R, C), "out")
    assert_within(grads[0], Approx(back).sum(1).view(R, C), "d_rows")
    d_mid = torch.zeros(R * k, C, dtype=torch.float64, device=DEV)
    d_mid[place[there]] = (wv[:, :, None] * d_out.double()[:, None, :])[there]
    assert_within(grads[1], Approx(d_mid, 2.0 ** -24 * d_mid.abs()), "d_sorted")
    assert not bool(grads[1][n:].any())
    if with_weights:
        assert_within(grads[2], (Approx(picked) * Approx(d_out.double()[:, None, :])).sum(2).view(R, k), "d_weights")
        assert not bool(grads[2][~there].any())
    return srt, out, grads


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,k,E,C", [(1, 1, 1, 1), (1, 2, 4, 1024), (7, 3, 5, 3), (33, 2, 4, 64), (50, 4, 8, 131), (200, 5, 28, 128),
                                     (19, 8, 16, 515), (12, 9, 3, 2048), (3, 2, 2, 5000), (4000, 2, 8, 24)])
def test_moves_against_64_bits(R, k, E, C, dtype):
    check_moves(R, k, E, C, T[dtype])


@pytest.mark.parametrize("out_of", [0.0, 1.0])
def test_moves_where_all_or_nothing_is_routed(out_of):
    srt, out, grads = check_moves(300, 2, 6, 72, torch.bfloat16, out_of=out_of)
    if out_of == 1.0:
        assert not bool(out.any()) and not bool(srt.any()) and not bool(grads[0].any())


def test_moves_without_weights():
    check_moves(100, 3, 6, 40, torch.float32, with_weights=False)


def test_no_rows():
    check_moves(0, 2, 4, 16, torch.bfloat16)


def test_a_sum_against_differences():
    """out is linear in the rows and in the weights: differences are exact up to rounding (u per product, summed over k and C)."""
    from cpfn_amd import autograd_ops, ops
    c, rows, mid, w, d_sorted, d_out = problem(64, 3, 5, 33, torch.float32)
    plan = ops.route_plan(c, 5)
    mid_g, w_g = torch.autograd.grad(autograd_ops.route_combine(mid, w, plan), [mid, w], [d_out])
    for leaf, grad in ((mid, mid_g), (w, w_g)):
        d = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(2)).to(DEV)
        with torch.no_grad():
            hi = autograd_ops.route_combine(mid + d if leaf is mid else mid, w + d if leaf is w else w, plan).double()
            lo = autograd_ops.route_combine(mid - d if leaf is mid else mid, w - d if leaf is w else w, plan).double()
        slope, want = float(((hi - lo) * d_out).sum() / 2), float((grad.double() * d).sum())
        scale = float(((hi.abs() + lo.abs()) * d_out.abs()).sum())
        assert abs(slope - want) <= 16 * 2.0 ** -24 * scale


def test_values_are_moved_bit_for_bit():
    """NaNs with their payloads, signed zeros, values below the smallest normal one."""
    from cpfn_amd import autograd_ops, ops
    for dt, it in ((torch.float32, torch.int32), (torch.bfloat16, torch.int16), (torch.float16, torch.int16)):
        g = torch.Generator().manual_seed(3)
        info = torch.iinfo(it)
        bits = torch.randint(info.min, info.max, (500, 35), generator=g).to(it).to(DEV)
        rows = bits.view(dt)
        plan = ops.route_plan(choices(500, 1, 7, seed=4), 7)
        srt = autograd_ops.route_gather(rows, plan)
        assert torch.equal(srt.view(it)[plan.place.long().view(-1)], bits)


def test_rows_that_start_anywhere_and_strides():
    from cpfn_amd import autograd_ops, ops
    c, rows, mid, w, d_sorted, d_out = problem(60, 2, 5, 48, torch.bfloat16)
    plan = ops.route_plan(c, 5)
    want = (autograd_ops.route_gather(rows, plan), autograd_ops.route_combine(mid, w, plan))

    def shifted(t, by):
        flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=DEV)
        return flat[by:by + t.numel()].view(t.shape).copy_(t.detach())
    for by in (1, 5):
        got = (autograd_ops.route_gather(shifted(rows, by), plan), autograd_ops.route_combine(shifted(mid, by), shifted(w, by), plan))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    t = rows.detach().t().contiguous().t()
    assert not t.is_contiguous() and torch.equal(autograd_ops.route_gather(t, plan), want[0])


def test_streams_repeats_and_captured_graphs():
    """The plan and the moves, forward and backward, as one graph: replayed on new choices with eager work in between, in two graphs."""
    from cpfn_amd import ops
    R, k, E, C = 6000, 2, 9, 64
    c, rows, mid, w, d_sorted, d_out = problem(R, k, E, C, torch.bfloat16)
    rows, mid, w = rows.detach(), mid.detach(), w.detach()

    def all_of_it():
        plan = ops.route_plan(c, E)
        back = ops.route_combine_bwd(d_out, mid, w, plan)
        return [plan.offsets, plan.place, ops.route_gather_fwd(rows, plan), ops.route_combine_fwd(mid, w, plan),
                ops.route_combine_fwd(d_sorted, None, plan), back[0], back[1]]
    want = all_of_it()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(s):
        got = all_of_it()
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                held = all_of_it()
            graphs.append((g, held))
    s.synchronize()
    for i in range(4):
        c.copy_(choices(R, k, E, seed=30 + i, out_of=0.1 * i))
        want = all_of_it()
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_offsets_that_pass_32_bits():
    from cpfn_amd import ops
    C, k = 4096, 2
    R = (1 << 31) // C // k + 5                                    # the sorted rows hold more than 2^31 values
    rows = torch.zeros(R, C, dtype=torch.bfloat16, device=DEV)
    rows[-1] = torch.arange(C, device=DEV).to(torch.bfloat16)
    c = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV).expand(R, k).contiguous()
    plan = ops.route_plan(c, 2)
    srt = ops.route_gather_fwd(rows, plan)
    assert torch.equal(srt[R - 1], rows[-1]) and torch.equal(srt[2 * R - 1], rows[-1])
    assert not bool(srt[:R - 1].any()) and not bool(srt[R:2 * R - 1].any())
    out = ops.route_combine_fwd(srt, None, plan)
    assert torch.equal(out[-1].float(), (2 * rows[-1].float()).to(torch.bfloat16).float()) and not bool(out[:-1].any())
    d_sorted, d_w = ops.route_combine_bwd(rows, srt, None, plan)
    assert torch.equal(d_sorted, srt) and not bool(d_w[:-1].any()) and bool((d_w[-1] > 0).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("C", [3, 40, 131])
def test_places_that_no_plan_left_are_choices_that_are_not_there(C, dtype):
    """A RoutePlan is two tensors that a caller can write to: places outside the sorted rows, and an end in front of them, are neither
    read from nor written to (results between guard rows, at the C ABI)."""
    from cpfn_amd import lib
    h, st = lib.lib(), torch.cuda.current_stream().cuda_stream
    R, k, E, guard = 50, 2, 4, 64
    dt, code = T[dtype], {"fp32": 0, "bf16": 1}[dtype]
    c, rows, mid, w, _, g = problem(R, k, E, C, dt, 0.0)
    n = R * k
    good = torch.randperm(n, generator=torch.Generator().manual_seed(1)).int().to(DEV).view(R, k)
    bad = torch.tensor([n, n + 1, -1, -2, -2 ** 31, 2 ** 31 - 1, 2 ** 30, n + 63], dtype=torch.int32, device=DEV)
    place = good.clone()
    place[::3, 0] = bad.repeat(R)[:place[::3].shape[0]]
    place[5, 1] = n
    there = (place >= 0) & (place < n)
    for end in (n, n + 1000, -1, -2 ** 31):
        offsets = torch.tensor([0] * E + [end], dtype=torch.int32, device=DEV)

        def held(count):
            return torch.full((count + 2 * guard, C), 7.0, dtype=dt, device=DEV)

        def inside(t):
            assert bool((t[:guard] == 7).all()) and bool((t[-guard:] == 7).all())
            return t[guard:-guard]
        srt, out, d_mid = held(n), held(R), held(n)
        d_w = torch.empty(R, k, device=DEV)
        size = C * srt.element_size() * guard
        assert h.cpfn_route_gather(rows.data_ptr(), place.data_ptr(), offsets.data_ptr(), R, k, E, C, code, srt.data_ptr() + size, st) == 0
        assert h.cpfn_route_combine(mid.data_ptr(), w.data_ptr(), place.data_ptr(), R, k, C, code, out.data_ptr() + size, st) == 0
        assert h.cpfn_route_combine_bwd(g.data_ptr(), mid.data_ptr(), w.data_ptr(), place.data_ptr(), offsets.data_ptr(), R, k, E, C, code,
                                        d_mid.data_ptr() + size, d_w.data_ptr(), st) == 0
        torch.cuda.synchronize()
        srt, out, d_mid = inside(srt), inside(out), inside(d_mid)
        if end >= n:                                              # (an earlier end's zeros and the rows are written in no order)
            want = torch.full((n, C), 7.0, dtype=dt, device=DEV)
            want[place[there].long()] = rows.detach().repeat_interleave(k, 0).view(R, k, C)[there]
            assert torch.equal(srt, want)
        picked = torch.where(there[:, :, None], mid.detach().double()[place.long().clamp(0, n - 1)], torch.zeros((), dtype=torch.float64, device=DEV))
        assert_within(out, (Approx(picked) * Approx(w.detach().double()[:, :, None])).sum(1).view(R, C), "out")
        assert_within(d_w, (Approx(picked) * Approx(g.double()[:, None, :])).sum(2).view(R, k), "d_weights")
        assert not bool(d_w[~there].any())


def test_only_one_of_rows_and_weights_is_differentiated_and_a_graph_is_walked_twice():
    from cpfn_amd import autograd_ops, ops
    c, rows, mid, w, d_sorted, d_out = problem(90, 3, 5, 44, torch.float32, 0.2)
    plan = ops.route_plan(c, 5)
    both = torch.autograd.grad(autograd_ops.route_combine(mid, w, plan), [mid, w], [d_out])
    only_w = torch.autograd.grad(autograd_ops.route_combine(mid.detach(), w, plan), [w], [d_out])
    only_mid = torch.autograd.grad(autograd_ops.route_combine(mid, w.detach(), plan), [mid], [d_out])
    assert torch.equal(only_w[0], both[1]) and torch.equal(only_mid[0], both[0])
    wt = w.detach().t().contiguous().t().requires_grad_()               # (weights in another order of memory)
    assert not wt.is_contiguous()
    turned = torch.autograd.grad(autograd_ops.route_combine(mid, wt, plan), [mid, wt], [d_out])
    assert all(torch.equal(a, b) for a, b in zip(turned, both))
    out = autograd_ops.route_combine(mid, w, plan)
    for _ in range(2):
        again = torch.autograd.grad(out, [mid, w], [d_out], retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(again, both))
    with torch.no_grad():
        assert torch.equal(autograd_ops.route_combine(mid, w, plan), out)
        assert torch.equal(autograd_ops.route_gather(rows, plan), autograd_ops.route_gather(rows.detach(), plan))
    plan.place[0, 0] = -1                                               # (a plan that changed under a recorded call)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, [mid], [d_out])
