"""autograd_ops.row_norm / norm_residual (csrc/rownorm_*.hip) against the formulas in 64 bits, with tolerances from a running error
analysis of fp32 arithmetic (tests/approx.py), and against differences; sizes from one row to many, odd channel counts, unaligned rows,
every gate; streams, captured graphs, repeated runs."""
import itertools

import pytest
import torch

from approx import Approx, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _normalise(v, kind):
    if kind == "layer":
        v = v - v.mean(1)
    r = ((v * v).mean(1) + EPS).rsqrt()
    return v * r, r


def reference(t, kind, act, d_out, d_normed):
    """All results and gradients of norm_residual (or, without "y", row_norm) as Approx, by the formulas."""
    f = {n: Approx(x.detach().double()) for n, x in t.items() if x is not None}
    P, C = t["x"].shape
    got, total = {}, f["x"]
    if "y" in f:
        hat = f["y"]
        u = hat
        if "weight" in f:
            hat, r = _normalise(f["y"], kind)
            u = hat * f["weight"]
            if "bias" in f:
                u = u + f["bias"]
        one = Approx(torch.ones(1, C, dtype=torch.float64, device=t["x"].device))
        a = one
        if "gate" in f:
            G = t["gate"].shape[0]
            a = Approx(f["gate"].v.repeat_interleave(P // G, 0))
            a = a.sigmoid(fast=t["x"].dtype != torch.float32) if act == "sigmoid" else a
        s = f.get("scale", one)
        total = total + s * (a * u)
        got["out"] = total
    if "next_weight" in f:
        hat1, r1 = _normalise(total, kind)
        got["normed"] = hat1 * f["next_weight"]
        if "next_bias" in f:
            got["normed"] = got["normed"] + f["next_bias"]
    D = None if d_out is None else Approx(d_out.double())
    if d_normed is not None:
        dn = Approx(d_normed.double())
        got["d_next_weight"] = (dn * hat1).sum(0).view(C)
        if "next_bias" in f:
            got["d_next_bias"] = dn.sum(0).view(C)
        dh = dn * f["next_weight"]
        inner = dh - hat1 * (dh * hat1).mean(1)
        if kind == "layer":
            inner = inner - dh.mean(1)
        D = r1 * inner if D is None else D + r1 * inner
    if D is None:
        return got
    got["d_x"] = D
    if "y" in f:
        du = D * s * a
        if "gate" in f:
            dg = D * s * u
            if act == "sigmoid":
                dg = dg * (a * (one - a))
            got["d_gate"] = dg.view(G, P // G, C).sum(1).view(G, C)
        # (the kernel's column sums: S1 = sum D a hat, S2 = sum D a)
        S1, S2 = (D * a * hat).sum(0), (D * a + Approx(torch.zeros_like(D.v))).sum(0)
        w, b = f.get("weight", one), f.get("bias")
        if "scale" in f:
            got["d_scale"] = (w * S1 + b * S2 if b is not None else w * S1).view(C)
        if "weight" in f:
            got["d_weight"] = (s * S1).view(C)
            if b is not None:
                got["d_bias"] = (s * S2).view(C)
            e = du * f["weight"]
            inner = e - hat * (e * hat).mean(1)
            if kind == "layer":
                inner = inner - e.mean(1)
            du = r * inner
        got["d_y"] = du
    return got


def inputs(P, C, dt, groups, post=True, nxt=True, bias=True, scale=True, y=True, seed=0, offset=0.0):
    g = torch.Generator().manual_seed(seed)

    def rows(n, sc=1.0):
        return (torch.randn(n, C, generator=g) * sc + offset).to(dt).to(DEV).requires_grad_()

    def vec(m):
        return (m + 0.3 * torch.randn(C, generator=g)).to(DEV).requires_grad_()
    t = {"x": rows(P), "y": rows(P, 2.0) if y else None, "weight": vec(1.0) if post and y else None,
         "bias": vec(0.0) if post and y and bias else None, "gate": rows(groups) if groups and y else None,
         "scale": vec(0.5) if scale and y else None, "next_weight": vec(1.0) if nxt else None,
         "next_bias": vec(0.0) if nxt and bias else None}
    d_out = torch.randn(P, C, generator=g).to(dt).to(DEV)
    d_normed = torch.randn(P, C, generator=g).to(dt).to(DEV)
    return t, d_out, d_normed


def call(t, kind, act):
    from cpfn_amd import autograd_ops
    if t["y"] is None:
        return None, autograd_ops.row_norm(t["x"], t["next_weight"], t["next_bias"], kind=kind, eps=EPS)
    return autograd_ops.norm_residual(t["x"], t["y"], t["weight"], t["bias"], gate=t["gate"], gate_act=act, scale=t["scale"],
                                      next_weight=t["next_weight"], next_bias=t["next_bias"], kind=kind, eps=EPS)


def run(t, kind, act, d_out, d_normed):
    out, normed = call(t, kind, act)
    got = {n: v.detach() for n, v in (("out", out), ("normed", normed)) if v is not None}
    pairs = [(o, g) for o, g in ((out, d_out), (normed, d_normed)) if o is not None and g is not None]
    names = [n for n, v in t.items() if v is not None and not (d_normed is None and n.startswith("next"))]
    grads = torch.autograd.grad([o for o, _ in pairs], [t[n] for n in names], [g for _, g in pairs])
    got.update({"d_" + n: g for n, g in zip(names, grads)})
    return got


def check(t, d_out, d_normed, kind, act):
    got = run(t, kind, act, d_out if t["y"] is not None else None, d_normed if t["next_weight"] is not None else None)
    want = reference(t, kind, act, d_out if t["y"] is not None else None, d_normed if t["next_weight"] is not None else None)
    assert set(got) == set(want), (sorted(got), sorted(want))
    for n in sorted(want):
        like = t["x"].dtype if n in ("out", "normed", "d_x", "d_y", "d_gate") else torch.float32
        assert got[n].dtype == like, n
        assert_within(got[n], want[n], n)
    return got


def _args(P, C, dtype, groups, **kw):
    return inputs(P, C, T[dtype], groups, **kw)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("P,C", [(1, 1), (1, 1024), (3, 8), (5, 7), (37, 64), (64, 65), (33, 128), (19, 131), (12, 259), (9, 513), (7, 1000),
                                 (4, 2047), (3, 4096)])
def test_every_size_against_64_bits(P, C, dtype):
    for kind in ("rms", "layer"):
        check(*_args(P, C, dtype, P), kind=kind, act="sigmoid")


@pytest.mark.parametrize("post,nxt,bias,scale", list(itertools.product([True, False], repeat=4)))
@pytest.mark.parametrize("gate", ["none", "full", "group"])
def test_every_part_on_and_off(post, nxt, bias, scale, gate):
    P, C = 24, 72
    groups = {"none": 0, "full": P, "group": 4}[gate]
    for dtype, kind, act in (("fp32", "layer", "sigmoid"), ("bf16", "rms", "none")):
        check(*_args(P, C, dtype, groups, post=post, nxt=nxt, bias=bias, scale=scale, seed=3), kind=kind, act=act)


@pytest.mark.parametrize("dtype,kind,bias", [("fp32", "rms", False), ("bf16", "layer", True), ("fp16", "rms", True)])
@pytest.mark.parametrize("P,C", [(1, 256), (100, 256), (1000, 40), (257, 1283)])
def test_the_norm_in_front_alone(P, C, dtype, kind, bias):
    check(*_args(P, C, dtype, 0, y=False, bias=bias), kind=kind, act="none")


@pytest.mark.parametrize("groups,each,C", [(1, 1, 64), (1, 3000, 64), (2, 1, 96), (3, 700, 128), (16, 1283, 24), (700, 2, 32), (1500, 3, 8),
                                           (5, 41, 1024), (40, 7, 2056)])
def test_a_gate_shared_by_groups_of_rows(groups, each, C):
    """One group, groups of one row, groups that several workgroups share and workgroups that take several groups."""
    for dtype, act in (("fp32", "none"), ("bf16", "sigmoid")):
        check(*_args(groups * each, C, dtype, groups, seed=groups), kind="rms", act=act)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("C", [40, 63, 104, 127, 240, 251, 472, 509, 520, 936, 1021, 1024, 1032, 1928, 2045, 3080, 4091])
def test_every_form_at_every_number_of_lanes(C, dtype):
    """Rows of one to eight waves, whole and ragged: the whole block with its own gate, a shared one and none, the norm in front, and what
    has no kernel of its own (no norm of y)."""
    for P, groups, kw in ((10, 10, {}), (10, 5, {}), (10, 0, {"bias": False}), (10, 0, {"y": False}), (10, 10, {"post": False}), (10, 0, {"nxt": False})):
        check(*_args(P, C, dtype, groups, seed=C, **kw), kind="layer", act="sigmoid")


@pytest.mark.parametrize("missing", ["out", "normed"])
@pytest.mark.parametrize("gate", [0, 30, 3])
def test_a_result_without_a_gradient(missing, gate):
    t, d_out, d_normed = inputs(30, 136, torch.bfloat16, gate, seed=5)
    d_out, d_normed = (None, d_normed) if missing == "out" else (d_out, None)
    got, want = run(t, "layer", "sigmoid", d_out, d_normed), reference(t, "layer", "sigmoid", d_out, d_normed)
    for n in got:
        assert_within(got[n], want[n], n)


def test_only_some_gradients_are_wanted():
    t, d_out, d_normed = inputs(48, 72, torch.float32, 4, seed=6)
    want = reference(t, "rms", "sigmoid", d_out, d_normed)
    for names in (["x"], ["y"], ["gate"], ["scale"], ["weight", "next_bias"], ["bias"], ["next_weight"], ["y", "next_weight"]):
        u = {n: (v if v is None else v.detach().requires_grad_(n in names)) for n, v in t.items()}
        out, normed = call(u, "rms", "sigmoid")
        grads = torch.autograd.grad([out, normed], [u[n] for n in names], [d_out, d_normed])
        for n, g in zip(names, grads):
            assert_within(g, want["d_" + n], n)


def test_gradients_against_differences():
    """The loss's change along a direction is the gradient's product with it: central differences of the kernel's own fp32 forward pass
    at a step h: the truncation is O(h^2) and the rounding of the loss ~ u |loss terms| / h; both are far under 1e-2 of the slope here."""
    t, d_out, d_normed = inputs(40, 50, torch.float32, 4, seed=7)
    got = run(t, "layer", "sigmoid", d_out, d_normed)
    h = 2.0 ** -7
    for n, v in t.items():
        d = torch.randn(v.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
        loss = []
        for sgn in (1.0, -1.0):
            u = dict(t)
            u[n] = v.detach() + sgn * h * d
            o, m = call(u, "layer", "sigmoid")
            loss.append(float(((o.double() * d_out).sum() + (m.double() * d_normed).sum()).detach()))
        slope = (loss[0] - loss[1]) / (2 * h)
        want = float((got["d_" + n].double() * d).sum())
        scale = float(got["d_" + n].double().norm() * d.double().norm())
        assert abs(slope - want) <= 1e-2 * scale / d.numel() ** 0.5 + 2e-3 * abs(want), (n, slope, want, scale)


def test_rows_that_start_anywhere():
    """Slices of a buffer (rows at any element), parameters inside a flat buffer: the same results as from fresh tensors."""
    for dtype, C in (("bf16", 128), ("fp32", 64), ("fp16", 77)):
        t, d_out, d_normed = inputs(33, C, T[dtype], 3, seed=8)
        want = run(t, "layer", "sigmoid", d_out, d_normed)
        for shift in (1, 3):
            u = {}
            for n, v in t.items():
                flat = torch.full((v.numel() + 16,), float("nan"), dtype=v.dtype, device=DEV)
                u[n] = flat[shift:shift + v.numel()].view(v.shape).copy_(v.detach()).detach().requires_grad_()
                assert u[n].data_ptr() % 16 != 0
            got = run(u, "layer", "sigmoid", d_out, d_normed)
            for n in want:
                assert torch.equal(got[n], want[n]), n


def test_not_contiguous_rows_and_expanded_gradients():
    t, d_out, d_normed = inputs(30, 64, torch.float32, 0, seed=9)
    want = run(t, "rms", "none", torch.ones_like(d_out), torch.ones_like(d_out))
    u = dict(t)
    u["x"] = t["x"].detach().t().contiguous().t().requires_grad_()
    u["y"] = torch.cat([t["y"].detach(), t["y"].detach()], 1)[:, :64].requires_grad_()
    out, normed = call(u, "rms", "none")
    gx, gy = torch.autograd.grad(out.sum() + normed.sum(), [u["x"], u["y"]])           # (the gradients of a sum: expanded ones)
    assert torch.equal(gx, want["d_x"]) and torch.equal(gy, want["d_y"])


def test_large_offsets_of_a_layer_norm():
    """Rows far from zero: the mean is taken off before the squares (x ~ 300 +- 1; squares in one pass would lose 2^-24 * 9e4)."""
    check(*_args(40, 200, "fp32", 0, seed=10, offset=300.0), kind="layer", act="none")


def test_zeros_infinities_and_nan_stay_in_their_rows():
    t, d_out, d_normed = inputs(16, 72, torch.bfloat16, 16, seed=11)
    clean = run(t, "layer", "none", d_out, d_normed)
    with torch.no_grad():
        t["x"][3] = 0.0
        t["y"][3] = 0.0
        t["y"][5, 7] = float("nan")
        t["y"][9, 0] = float("inf")
    got = run(t, "layer", "none", d_out, d_normed)
    rest = [i for i in range(16) if i not in (3, 5, 9)]
    for n in ("out", "normed", "d_x", "d_y", "d_gate"):
        assert torch.equal(got[n][rest], clean[n][rest]), n
        assert torch.isfinite(got[n][3].float()).all(), n
    assert torch.isnan(got["out"][5]).all() and torch.isnan(got["d_y"][9]).any()


def test_no_rows():
    t, _, _ = inputs(0, 64, torch.bfloat16, 0, seed=12)
    got = run(t, "layer", "none", torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV))
    assert got["out"].shape == (0, 64) and got["normed"].shape == (0, 64)
    for n in ("weight", "bias", "scale", "next_weight", "next_bias"):
        assert torch.equal(got["d_" + n], torch.zeros(64, device=DEV)), n


def test_repeated_runs_and_another_stream_are_bit_identical():
    t, d_out, d_normed = inputs(5000, 128, torch.bfloat16, 5, seed=13)
    want = run(t, "layer", "sigmoid", d_out, d_normed)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(t, "layer", "sigmoid", d_out, d_normed)
    s.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_captured_and_replayed_beside_eager_work():
    """Forward and backward in one graph, replayed on new contents of its inputs with eager work in between; two graphs that were
    captured one after the other hold their own workspaces."""
    from cpfn_amd import ops
    t, d_out, d_normed = inputs(700, 96, torch.bfloat16, 7, seed=14)
    v = {n: x.detach() for n, x in t.items()}

    def both():
        out, normed = ops.norm_residual_fwd(v["x"], v["y"], v["weight"], v["bias"], v["gate"], "sigmoid", v["scale"], v["next_weight"],
                                            v["next_bias"], "layer", EPS)
        back = ops.norm_residual_bwd(v["x"], v["y"], v["weight"], v["bias"], v["gate"], "sigmoid", v["scale"], v["next_weight"], d_out,
                                     d_normed, "layer", EPS)
        return [out, normed] + [back[n] for n in sorted(back)]
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
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        v["y"].copy_(torch.randn(v["y"].shape, generator=torch.Generator().manual_seed(20 + i)).to(v["y"].dtype))
        want = both()
        torch.cuda.synchronize()
        for g, held in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, held in graphs:
            for a, b in zip(held, want):
                assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    t, d_out, d_normed = inputs(4, 16, torch.float32, 0, seed=15)
    out, _ = call(t, "rms", "none")
    (gx,) = torch.autograd.grad(out.sum(), [t["y"]], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_a_long_tensor_whose_offsets_pass_32_bits():
    """2^31 + values: the last rows are where a 32-bit offset would miss them."""
    from cpfn_amd import ops
    C = 4096
    P = (1 << 31) // C + 3
    x = torch.zeros(P, C, dtype=torch.bfloat16, device=DEV)
    y = torch.zeros(P, C, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(1)
    tail = torch.randn(2, 4, C, generator=g).to(torch.bfloat16).to(DEV)
    x[-4:], y[-4:] = tail[0], tail[1]
    w = torch.ones(C, device=DEV)
    out, normed = ops.norm_residual_fwd(x, y, weight=w, next_weight=w)
    a, b = ops.norm_residual_fwd(tail[0].contiguous(), tail[1].contiguous(), weight=w, next_weight=w)
    assert torch.equal(out[-4:], a) and torch.equal(normed[-4:], b) and not bool(out[:-4].any())


def test_a_graph_is_walked_twice_and_nothing_is_recorded_without_gradients():
    from cpfn_amd import autograd_ops
    t, d_out, d_normed = inputs(50, 88, torch.bfloat16, 5, seed=9)
    out, normed = call(t, "rms", "sigmoid")
    leaves = [v for v in t.values() if v is not None]
    first = torch.autograd.grad([out, normed], leaves, [d_out, d_normed], retain_graph=True)
    again = torch.autograd.grad([out, normed], leaves, [d_out, d_normed])
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    detached = {n: None if v is None else v.detach() for n, v in t.items()}
    for grad_mode, u in ((False, t), (True, detached)):
        with torch.set_grad_enabled(grad_mode):
            o, n = call(u, "rms", "sigmoid")
        assert not o.requires_grad and not n.requires_grad and torch.equal(o, out) and torch.equal(n, normed)
    with torch.inference_mode():
        assert torch.equal(call(t, "rms", "sigmoid")[1], normed)
        turned = t["x"].detach().t().contiguous().t()
        assert not turned.is_contiguous()
        assert torch.equal(autograd_ops.row_norm(turned, t["next_weight"]), autograd_ops.row_norm(t["x"], t["next_weight"]))
