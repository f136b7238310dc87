"""The operators of a routed residual block as they are used together: norm in front, router, rows to the experts and back, norm behind
with gate and residual scale, the next block's norm, loss, gradients, clipping — against the same block in float64 on the CPU, and a
training step of it as a captured graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class RoutedBlock(torch.nn.Module):
    """x, h = norm(x) -> out, next norm of out; each row of h goes to k of E experts (one layer each), weighted by the router."""

    def __init__(self, C, E, k, clouds):
        super().__init__()
        self.E, self.k, self.clouds = E, k, clouds
        self.router = torch.nn.Parameter(torch.randn(C, E) * 0.3)
        self.experts = torch.nn.Parameter(torch.randn(E, C, C) / C ** 0.5)
        self.norm_in = torch.nn.Parameter(1.0 + 0.1 * torch.randn(C))
        self.norm_out = torch.nn.Parameter(1.0 + 0.1 * torch.randn(C))
        self.bias_out = torch.nn.Parameter(0.1 * torch.randn(C))
        self.scale = torch.nn.Parameter(torch.full((C,), 0.5))
        self.norm_next = torch.nn.Parameter(1.0 + 0.1 * torch.randn(C))
        self.gate = torch.nn.Parameter(torch.randn(clouds, C))

    def forward(self, x, choice=None):
        from cpfn_amd import autograd_ops, ops
        h = autograd_ops.row_norm(x, self.norm_in, kind="layer")
        prob = torch.softmax(h.float() @ self.router, dim=1)
        if choice is None:
            choice = torch.topk(prob, self.k, dim=1)[1]
        weights = torch.gather(prob, 1, choice.clamp(min=0))
        plan = ops.route_plan(choice.contiguous(), self.E)
        rows = autograd_ops.route_gather(h, plan)
        ends = plan.offsets.tolist()
        parts = [rows[a:b] @ self.experts[e].to(rows.dtype) for e, (a, b) in enumerate(zip(ends[:-1], ends[1:]))]
        parts.append(rows[ends[-1]:])
        y = autograd_ops.route_combine(torch.cat(parts), weights, plan)
        out, nxt = autograd_ops.norm_residual(x, y, self.norm_out, self.bias_out, gate=self.gate.to(x.dtype), gate_act="sigmoid",
                                              scale=self.scale, next_weight=self.norm_next, kind="layer")
        return out, nxt, choice

    def plain(self, x, choice):
        """The same by torch operations, every row through all its experts in turn (float64 on the CPU)."""
        def norm(v, w, b=None):
            v = v - v.mean(1, keepdim=True)
            v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * w
            return v if b is None else v + b
        h = norm(x, self.norm_in)
        prob = torch.softmax(h @ self.router, dim=1)
        y = torch.zeros_like(x)
        for j in range(self.k):
            there = (choice[:, j] >= 0).to(x.dtype)[:, None]
            e = choice[:, j].clamp(min=0)
            per = torch.stack([h @ self.experts[i] for i in range(self.E)], 1)[torch.arange(x.shape[0]), e]
            y = y + there * prob.gather(1, e[:, None]) * per
        a = torch.sigmoid(self.gate).repeat_interleave(x.shape[0] // self.clouds, 0)
        out = x + self.scale * a * norm(y, self.norm_out, self.bias_out)
        return out, norm(out, self.norm_next)


@pytest.mark.parametrize("full", [False, True])
def test_block_against_float64(full):
    """fp32.  Every element is the end of about 12 operations on sums of 48 products: n u = 3e-6 relative each to the magnitudes that
    are added; 2e-4 of a tensor's norm leaves a factor of five for cancellation along the chain.  full: choices left out."""
    torch.manual_seed(3)
    P, C, E, k, clouds = 330, 48, 5, 2, 3
    block = RoutedBlock(C, E, k, clouds).to(DEV)
    x = torch.randn(P, C, device=DEV, requires_grad=True)
    g1, g2 = torch.randn(P, C, device=DEV), torch.randn(P, C, device=DEV)
    choice = None
    if full:
        choice = torch.randint(0, E, (P, k), device=DEV)
        choice[torch.rand(P, k, device=DEV) < 0.2] = -1
        choice[7] = -1
    out, nxt, choice = block(x, choice)
    ((out * g1).sum() + (nxt * g2).sum()).backward()
    twin = RoutedBlock(C, E, k, clouds).double()
    twin.load_state_dict({n: p.detach().cpu().double() for n, p in block.state_dict().items()})
    xd = x.detach().cpu().double().requires_grad_()
    o64, n64 = twin.plain(xd, choice.cpu())
    ((o64 * g1.cpu().double()).sum() + (n64 * g2.cpu().double()).sum()).backward()

    def near(a, b, name):
        off = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        assert off <= 2e-4, (name, off)
    near(out, o64, "out"); near(nxt, n64, "next"); near(x.grad, xd.grad, "x")
    for (n, p), q in zip(block.named_parameters(), twin.parameters()):
        near(p.grad, q.grad, n)


def test_block_trains_clipped_in_bf16():
    """A few optimizer steps with the clipped norm: everything runs, every parameter gets a finite gradient, the factor acts."""
    from cpfn_amd import optim
    torch.manual_seed(4)
    block = RoutedBlock(64, 4, 2, 2).to(DEV)
    opt = torch.optim.Adam(block.parameters(), lr=1e-3)
    x = torch.randn(512, 64, device=DEV).bfloat16()
    for _ in range(3):
        opt.zero_grad()
        out, nxt, _ = block(x)
        (nxt.float() ** 3).mean().backward()
        norm = optim.clip_grad_norm_(block.parameters(), 1e-3)
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in block.parameters())
        assert float(norm) > 1e-3
        after = float(torch.sqrt(sum((p.grad.double() ** 2).sum() for p in block.parameters())))
        assert abs(after - 1e-3 * float(norm) / (float(norm) + 1e-6)) <= 1e-6 * 1e-3
        opt.step()


def test_whole_step_as_one_graph():
    """Norm, plan, moves, one shared expert layer, norm behind, both backward passes and clipping as ONE graph (nothing in it needs the
    host), replayed on new rows and choices with eager work between the replays: the eager results, bit for bit."""
    from cpfn_amd import autograd_ops, ops, optim
    torch.manual_seed(5)
    P, C, E, k = 1200, 64, 6, 2
    x = torch.randn(P, C, device=DEV)
    choice = torch.randint(0, E, (P, k), device=DEV)
    weights = torch.rand(P, k, device=DEV)
    expert = torch.randn(C, C, device=DEV) / 8
    vec = torch.rand(3, C, device=DEV) + 0.5
    g = torch.randn(P, C, device=DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, weights, expert, vec[0], vec[1], vec[2])]
        lx, lw, le, n0, n1, n2 = leaves
        h = autograd_ops.row_norm(lx, n0)
        plan = ops.route_plan(choice, E)
        y = autograd_ops.route_combine(autograd_ops.route_gather(h, plan) @ le, lw, plan)
        out, nxt = autograd_ops.norm_residual(lx, y, n1, next_weight=n2)
        grads = torch.autograd.grad([out, nxt], leaves, [g, g])
        norm = optim.clip_grads_([t for t in grads], 0.5)
        return [out.detach(), nxt.detach(), norm] + [t.detach() for t in grads]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = step()
    s.synchronize()
    for i in range(4):
        gen = torch.Generator(device=DEV).manual_seed(i)
        x.normal_(generator=gen)
        choice.random_(-1, E, generator=gen)
        weights.uniform_(generator=gen)
        with torch.cuda.stream(s):
            want = step()
        s.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for j, (a, b) in enumerate(zip(held, want)):
            assert torch.equal(a, b), (i, j)


def test_two_threads_call_at_once():
    """The entry points from two host threads on their own streams: each gets its own results."""
    import threading
    from cpfn_amd import autograd_ops, ops, optim
    torch.manual_seed(6)
    data = [(torch.randn(900, 96, device=DEV), torch.randint(0, 7, (900, 2), device=DEV), torch.ones(96, device=DEV)) for _ in range(2)]

    def work(x, c, w):
        x = x.detach().requires_grad_()
        h = autograd_ops.row_norm(x, w)
        plan = ops.route_plan(c, 7)
        y = autograd_ops.route_combine(autograd_ops.route_gather(h, plan), None, plan)
        out, _ = autograd_ops.norm_residual(x, y, w)
        (gx,) = torch.autograd.grad(out.sum(), [x])
        return [out.detach(), gx, optim.grad_norm([gx, out.detach()])]
    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(30):
                    got[i] = work(*data[i])
            s.synchronize()
        except Exception as e:                       # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_bytes_are_counted_for_the_native_calls():
    from cpfn_amd import autograd_ops, lib
    x = torch.randn(64, 32, device=DEV, requires_grad=True)
    lib.byte_census(True)
    n = autograd_ops.row_norm(x, torch.ones(32, device=DEV))
    n.sum().backward()
    got = lib.byte_census(False)
    assert got["cpfn_norm_residual_fwd"] == (1, 2 * 64 * 32 * 4)
    assert got["cpfn_norm_residual_bwd"] == (1, 3 * 64 * 32 * 4)
    autograd_ops.row_norm(x, torch.ones(32, device=DEV))
    assert lib.byte_census(False) == {}


def test_a_captured_backward_pass_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """The leaf's accumulating node belongs to the default stream then, which cannot take part in a capture.  Without that graph the same
    pass is captured, and its replays leave the eager pass's gradients."""
    from cpfn_amd import autograd_ops, ops
    torch.manual_seed(3)
    P, C, k, E = 64, 32, 2, 4
    x = torch.randn(P, C, device=DEV, requires_grad=True)
    w = torch.rand(C, device=DEV, requires_grad=True)
    plan = ops.route_plan(torch.randint(0, E, (P, k), device=DEV), E)
    y = torch.randn(P * k, C, device=DEV, requires_grad=True)
    rw = torch.rand(P, k, device=DEV, requires_grad=True)
    g, gs = torch.randn(P, C, device=DEV), torch.randn(P * k, C, device=DEV)
    cases = ((lambda: autograd_ops.row_norm(x, w), g, [x, w]), (lambda: autograd_ops.route_gather(x, plan), gs, [x]),
             (lambda: autograd_ops.route_combine(y, rw, plan), g, [y, rw]))
    for call, d, leaves in cases:
        call().backward(d)
        want = [t.grad.clone() for t in leaves]
        for t in leaves:
            t.grad = None
        lives = call()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph, stream=s):
                call().backward(d)
        torch.cuda.synchronize()
        del lives
        assert all(t.grad is None for t in leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call().backward(d)
        for _ in range(3):
            for t in leaves:
                t.grad.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(t.grad, v) for t, v in zip(leaves, want))
        for t in leaves:
            t.grad = None
