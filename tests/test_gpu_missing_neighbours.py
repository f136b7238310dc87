"""Neighbours that are not there.  three_nn leaves the index M (one past the cloud's known points) where a query has fewer than three:
a query that is not finite, a cloud of one or two known points.  What reads rows by such an index takes the nearest row that there is, in
the last cloud too, whose row M is behind the tensor's end.  Small integers throughout: every sum is exact in any order."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_three_nn_names_no_row_for_a_query_that_is_not_finite():
    from cpfn_amd import ops
    g = torch.Generator().manual_seed(0)
    for M in (1, 2, 3, 40, 200):
        known, unknown = torch.rand(2, M, 3, generator=g), torch.rand(2, 70, 3, generator=g)
        unknown[1, 69, 1] = float("nan")
        _, idx, w = ops.three_nn_weights(unknown.to(DEV), known.to(DEV))
        assert int(idx.min()) >= 0 and bool((idx[1, 69] == M).all()) and bool(torch.isnan(w[1, 69]).all())
        assert bool((idx[:, :69].amax(2) == M).all()) if M < 3 else int(idx[:, :69].max()) < M
        feats = torch.randint(-8, 9, (2, M, 16), generator=g).float().to(DEV)
        out = ops.interp_rows_fwd(feats, idx, w)
        near = torch.gather(feats, 1, idx[..., 0].clamp(max=M - 1).long().unsqueeze(2).expand(-1, -1, 16))
        assert bool(torch.isnan(out[1, 69]).all()) and bool(torch.isfinite(out[0]).all())
        if M == 1:
            torch.testing.assert_close(out[0], near[0], rtol=1e-6, atol=0.0)       # (one neighbour: its weight is 1, the others' 0)


@pytest.mark.parametrize("B,M,N", [(1, 1, 5), (2, 2, 33), (3, 40, 130), (8, 128, 257)])
def test_rows_are_taken_from_the_own_cloud(B, M, N):
    from cpfn_amd import autograd_ops, ops
    C = 16
    g = torch.Generator().manual_seed(M)
    idx = torch.randint(-1, M + 2, (B, N, 3), generator=g).to(torch.int32)
    idx[-1, -1] = M                                          # (the last cloud's last query: all three)
    idx[-1, 0] = 2 ** 31 - 1
    w = torch.randint(0, 3, (B, N, 3), generator=g).float()
    feats, grad = torch.randint(-8, 9, (B, M, C), generator=g).float(), torch.randint(-3, 4, (B, N, C), generator=g).float()
    skip = torch.randint(-8, 9, (B, N, 8), generator=g).to(torch.bfloat16).to(DEV)
    inside = idx.clamp(0, M - 1).long()
    rows = torch.gather(feats.unsqueeze(1).expand(B, N, M, C), 2, inside.unsqueeze(3).expand(B, N, 3, C))
    want = (rows * w.unsqueeze(3)).sum(2)
    back = torch.zeros(B, M, C)
    for t in range(3):
        back.scatter_add_(1, inside[:, :, t:t + 1].expand(B, N, C), grad * w[:, :, t:t + 1])
    idx, w, want, back = idx.to(DEV), w.to(DEV), want.to(DEV), back.to(DEV)
    feats, grad = feats.to(DEV), grad.to(DEV)
    # channels first, fp32
    assert torch.equal(ops.three_interp_fwd(feats.transpose(1, 2).contiguous(), idx, w).transpose(1, 2), want)
    assert torch.equal(ops.three_interp_bwd(grad.transpose(1, 2).contiguous(), idx, w, M).transpose(1, 2), back)
    # rows, fp32
    f = feats.clone().requires_grad_()
    out = autograd_ops.interp_rows(f, idx, w)
    assert torch.equal(out, want)
    assert torch.equal(torch.autograd.grad(out, f, grad)[0], back)
    # rows, bf16: integers up to 256 are bf16 numbers; the adjoint is rounded once
    inv = ops.csr_build(idx.reshape(B, N * 3), M)
    for lists in (inv, None):
        f = feats.to(torch.bfloat16).requires_grad_()
        out = autograd_ops.interp_rows(f, idx, w, lists)
        assert torch.equal(out.float(), want)
        assert torch.equal(torch.autograd.grad(out, f, grad.to(torch.bfloat16))[0], back.to(torch.bfloat16))
        f = feats.to(torch.bfloat16).requires_grad_()
        out = autograd_ops.concat_interp(skip, f, idx, w, lists)
        assert torch.equal(out[..., 8:].float(), want) and torch.equal(out[..., :8], skip)
        d = torch.cat([torch.zeros_like(skip), grad.to(torch.bfloat16)], 2)
        assert torch.equal(torch.autograd.grad(out, f, d)[0], back.to(torch.bfloat16))


def test_rows_gathered_in_the_backward_pass_are_the_own_cloud_s():
    """The one-pass backward kernel that gathers its input rows, on indices behind the table (ball_query's N of an empty ball) and on the
    same indices brought inside: the same bits."""
    from cpfn_amd import lib as _l
    from cpfn_amd.ops import _ptr, _stream
    h = _l.lib()
    B, n_src, rpc, D = 5, 200, 8192, 128
    P = B * rpc
    g = torch.Generator().manual_seed(1)
    table, gy, y, W = (torch.randn(n, D, generator=g).to(torch.bfloat16).to(DEV) for n in (B * n_src, P, P, D))
    coef, scale, shift, xyz = (torch.randn(*n, generator=g).to(DEV) for n in ((3, D), (D,), (D,), (P, 3)))
    idx = torch.randint(0, n_src + 2, (P,), generator=g).to(torch.int32)
    idx[-64:] = n_src
    idx[:7] = 2 ** 31 - 1
    splits = h.cpfn_mlp_wgrad_splits(P, D, D)
    res = []
    for i in (idx.to(DEV), idx.clamp(max=n_src - 1).to(DEV)):
        ws, out, wx = torch.empty(splits * D * D, device=DEV), torch.empty(P, D, dtype=torch.bfloat16, device=DEV), torch.empty(splits * D * 3, device=DEV)
        _l.check(h.cpfn_mlp_bwd_fused_xt_gather(_ptr(gy), _ptr(table), _ptr(i), rpc, n_src, _ptr(W), P, D, D, _ptr(ws), _ptr(out), _ptr(y), _ptr(coef),
                                                _ptr(scale), _ptr(shift), _ptr(xyz), _ptr(wx), _stream()), "cpfn_mlp_bwd_fused_xt_gather")
        res.append((ws, out, wx))
    assert all(torch.equal(a, b) for a, b in zip(*res)) and bool(res[0][0].any())
