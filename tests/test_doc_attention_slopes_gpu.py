"""Slopes that the scale would take out of fp32 (doc_attention.hip)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
@pytest.mark.parametrize("scale,slope", [(1e-30, 1e10), (1e-30, 1e30),
                                         (1e-20, 1e25), (0.125, 3e38)])
def test_steep_slopes_leave_the_token_itself(scale, slope, heads, kv, dim):
    """slope |i - j| is past any score but at distance 0, so p is 1 there and 0
    elsewhere: o is v, nothing depends on q and k, and dv is do (of shared
    heads their sum, in fp32, rounded to 2^-8 of it)."""
    from deeplearning_cfn_amd.ops import functional as F_amd
    g = torch.Generator(device="cuda").manual_seed(dim)
    cu = torch.tensor([0, 100, 101, 300], dtype=torch.int32, device="cuda")
    q, k, v, do = (torch.randn(300, h, dim, generator=g, device="cuda")
                   .bfloat16() for h in (heads, kv, kv, heads))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu, scale=scale,
                                 slopes=torch.full((heads,), slope,
                                                   device="cuda"))
    assert torch.equal(o, v.repeat_interleave(heads // kv, 1))
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    want = do.double().unflatten(1, (kv, heads // kv)).sum(2)
    assert ((dv.double() - want).abs()
            <= want.abs() * 2.0 ** -8 + 2.0 ** -20 * heads).all()
    # D is do . o in fp32, and so is dP where p is 1: off by 2^-24 of dim
    # terms, next to a D of two parts (2^-16 of each term)
    room = scale * (2.0 ** -14 * (do.double().abs().amax() * v.double().abs()
                                  .amax()) * dim * 2 * heads)
    for d, t in ((dq, k), (dk, q)):
        assert (d.double().abs() <= room * t.double().abs().amax()).all()
