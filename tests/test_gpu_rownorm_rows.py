"""Norms of long tensors (csrc/rownorm_*.hip): every row counts, once.  A workgroup takes several row sets here, forward and backward, and
several gate groups; what it leaves is compared with 64 bits element by element, and column sums, whose tolerance as sums of n terms
would hide a whole row, are made of integers and have to be exact.

Sizes: the forward pass launches 2048 workgroups of 256 / L rows (L: lanes of a row; 4096, 2048 and 1024 workgroups of one row at 128, 256
and 512 lanes), so P is two to three times what they take at once."""
import numpy as np
import pytest
import torch

from test_gpu_rownorm import DEV, T, call, check, inputs, reference
from approx import assert_within

pytestmark = pytest.mark.gpu

LONG = [(140003, 24), (140003, 31), (70001, 63), (40011, 131), (20003, 259), (9001, 520), (9001, 640), (5003, 1283), (3001, 3001)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("P,C", LONG)
def test_several_row_sets_of_a_workgroup(P, C, dtype):
    """Each form of the kernels: a gate for each row, none, the norm in front, no norm of y."""
    for kind, act, groups, kw in (("layer", "sigmoid", P, {}), ("rms", "none", 0, {"bias": False}), ("layer", "none", 0, {"y": False}),
                                  ("rms", "none", P, {"post": False})):
        check(*inputs(P, C, T[dtype], groups, seed=C, **kw), kind=kind, act=act)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("groups,each,C", [(7, 20001, 31), (3, 13337, 131), (11, 819, 520), (5003, 2, 24), (5003, 3, 63), (2503, 9, 131), (4999, 2, 520),
                                           (3001, 2, 1283), (2053, 1, 3001)])
def test_several_row_sets_and_groups_behind_a_shared_gate(groups, each, C, dtype):
    check(*inputs(groups * each, C, T[dtype], groups, seed=groups), kind="layer", act="sigmoid")


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("C", [1, 2, 3, 5, 7, 9])
def test_short_rows_whose_last_chunk_is_shorter_than_a_piece(C, dtype):
    for P in (1, 2, 31, 32, 33, 65, 257, 8193):
        for groups in (0, P):
            t, d_out, d_normed = inputs(P, C, T[dtype], groups, seed=P)
            out, normed = call(t, "rms", "sigmoid")
            want = reference(t, "rms", "sigmoid", d_out, d_normed)
            assert_within(out.detach(), want["out"], "out")
            assert_within(normed.detach(), want["normed"], "normed")


def integers(P, C, groups, dt, seed, scale):
    """Rows of +-1: their rms norm with eps = 0 is themselves (C times the rounded 1 / C is 1 for these C, and the root of 1 is 1)."""
    assert float(np.float32(np.float64(C) * np.float64(np.float32(1) / np.float32(C)))) == 1.0
    g = torch.Generator(device=DEV).manual_seed(seed)

    def draw(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device=DEV).to(torch.float32 if len(shape) == 1 else dt)
    t = {"x": draw(0, 2, P, C) * 2 - 1, "y": draw(0, 2, P, C) * 2 - 1, "weight": draw(1, 3, C), "gate": draw(1, 3, groups, C) if groups else None,
         "scale": torch.full((C,), scale, device=DEV), "next_weight": torch.ones(C, device=DEV)}
    return t, draw(-1, 2, P, C)


# (the last row: more than 128 row sets for a workgroup, whose sums go to LDS in between, in one group, in parts of one and over several)
EXACT = [(0, 140003, 24), (0, 140003, 31), (0, 40011, 131), (0, 20003, 259), (0, 9001, 520), (0, 3001, 1283), (0, 2001, 3001), (0, 70000, 64),
         (0, 33, 5), (0, 257, 3), (140003, 1, 31), (20003, 1, 131), (7, 20001, 31), (3, 6007, 131), (11, 819, 520), (16, 1283, 259), (700, 2, 40),
         (5003, 3, 63), (2503, 9, 131), (3001, 2, 1283), (1200, 70, 24),
         (0, 2200003, 24), (0, 300007, 520), (0, 40009, 3001), (3, 1500001, 8), (600, 5003, 24), (100003, 33, 40), (1031, 63, 3001), (70, 9001, 131)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("groups,each,C", EXACT)
def test_column_sums_of_integers_are_exact(groups, each, C, dtype):
    """Every term is an integer of at most 8, every sum one below 2^24: in fp32 they are exact in any order, so one row more or less shows."""
    from cpfn_amd import ops
    P = each if groups == 0 else groups * each
    # behind y: out takes part with a gate and a scale of 2; no gradient comes through the next norm
    t, d = integers(P, C, groups, T[dtype], 1, 2.0)
    back = ops.norm_residual_bwd(t["x"], t["y"], t["weight"], None, t["gate"], "none", t["scale"], t["next_weight"], d, torch.zeros_like(d), "rms", 0.0)
    a = torch.ones(1, C, device=DEV) if groups == 0 else t["gate"].double().repeat_interleave(P // groups, 0)
    S1 = (d.double() * a * t["y"].double()).sum(0)
    assert torch.equal(back["weight"].double(), 2.0 * S1)
    assert torch.equal(back["scale"].double(), t["weight"].double() * S1)
    assert torch.equal(back["x"], d)
    if groups:
        u = (2.0 * d.double() * t["y"].double() * t["weight"].double()).view(groups, P // groups, C).sum(1)
        assert torch.equal(back["gate"], u.to(T[dtype]))
    bias = torch.zeros(C, device=DEV)
    back = ops.norm_residual_bwd(t["x"], t["y"], t["weight"], bias, t["gate"], "none", t["scale"], t["next_weight"], d, torch.zeros_like(d), "rms", 0.0)
    assert torch.equal(back["bias"].double(), 2.0 * (d.double() * a).sum(0))
    # behind the next norm: a scale of 0 leaves out = x
    t, d = integers(P, C, groups, T[dtype], 2, 0.0)
    back = ops.norm_residual_bwd(t["x"], t["y"], t["weight"], None, t["gate"], "none", t["scale"], t["next_weight"], torch.zeros_like(d), d, "rms", 0.0)
    assert torch.equal(back["next_weight"].double(), (d.double() * t["x"].double()).sum(0))
    assert torch.equal(back["next_bias"].double(), d.double().sum(0))
    back = ops.norm_residual_bwd(t["x"], None, None, None, None, "none", None, t["next_weight"], None, d, "rms", 0.0)
    assert torch.equal(back["next_weight"].double(), (d.double() * t["x"].double()).sum(0))
    assert torch.equal(back["next_bias"].double(), d.double().sum(0))


def test_column_sums_of_many_equal_terms():
    """Equal terms are rounded the same way at every step, so a long chain of fp32 additions drifts: n 2^-24 of the sum at most.  A lane adds
    up 128 row sets, then these sums (fewer than 20 here: a workgroup has up to 2344 row sets), then come the 32 row slots of a workgroup;
    then fp64, and one rounding."""
    from cpfn_amd import ops
    c = torch.full((), 0.1, device=DEV)
    tol = 1.01 * (128 + 20 + 31 + 1) * 2.0 ** -24

    def near(got, n, name):
        off = float((got.double() / (n * c.double()) - 1.0).abs().max())
        assert off <= tol, (name, off / 2.0 ** -24)
    P, C = 2048 * 512 * 32, 8
    ones, d, w = torch.ones(P, C, device=DEV), c.expand(P, C).contiguous(), torch.ones(C, device=DEV)
    back = ops.norm_residual_bwd(ones, None, None, None, None, "none", None, w, None, d, "rms", 0.0, needs=("next_weight", "next_bias"))
    near(back["next_weight"], P, "next_weight")
    near(back["next_bias"], P, "next_bias")
    for groups, each in ((600, 65536), (300000, 128)):
        P = groups * each
        ones, d, gate = torch.ones(P, C, device=DEV), c.expand(P, C).contiguous(), torch.ones(groups, C, device=DEV)
        back = ops.norm_residual_bwd(ones, ones, w, torch.zeros_like(w), gate, "none", w, None, d, None, "rms", 0.0, needs=("weight", "bias", "gate", "scale"))
        near(back["gate"], each, "gate")
        for n in ("weight", "bias", "scale"):
            near(back[n], P, n)
