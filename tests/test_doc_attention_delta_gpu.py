"""D = do . o of document attention takes o in twice the type's bits
(doc_attention.hip)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [200, 1500, 3000])
def test_values_with_a_common_part(length, dim, heads, kv, dtype):
    """v = 16 + 0.1 x: the common part cancels in dS = P (dP - D), where dP - D is
    0.1 sqrt(dim).  With o's low part D keeps what rounding P leaves in o: 0.4 u
    of each of about length / e equal terms, 16 * 0.4 u * sqrt(e / length) in
    every dimension alike, times |sum do| = sqrt(dim).  That is the same for all
    keys of a query, so it meets sum_j p_ij k_j = q_i / sqrt(dim) in dq, and
    dP - D itself meets terms of random sign, sqrt(e / length) of them:
      16 * 0.4 u sqrt(dim) / sqrt(dim) / (0.1 sqrt(dim)) = 64 u / sqrt(dim),
    8 u of dq for 64, 5.7 u for 128; the rounding of dS is under u.  Two and a
    half times that leave room for short rows.  The oracle with a rounded o is
    past it."""
    from deeplearning_cfn_amd.ops import functional as F_amd
    u = torch.finfo(dtype).eps / 2
    bound = 2.5 * 64 * u / dim ** 0.5
    g = torch.Generator(device="cuda").manual_seed(length + dim)
    # in front of it a document that takes the call past 1024 tokens
    front = 1100
    q, k, v, do = (torch.randn(front + length, h, dim, generator=g,
                               device="cuda") for h in (heads, kv, kv, heads))
    q, k, v, do = (t.to(dtype) for t in (q, k, 16 + 0.1 * v, do))
    cu = torch.tensor([0, front, front + length], dtype=torch.int32,
                      device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu)
    got = torch.autograd.grad(o, leaves, do)[:2]

    at = torch.arange(heads, device="cuda") // (heads // kv)
    qd, kd, vd, gd = (t.detach()[front:].double() for t in (q, k, v, do))
    kh, vh = (t[:, at].transpose(0, 1).contiguous() for t in (kd, vd))
    qh, gh = (t.transpose(0, 1).contiguous() for t in (qd, gd))
    scale = dim ** -0.5
    p = torch.softmax(torch.bmm(qh, kh.mT.contiguous()) * scale, -1)
    dp = torch.bmm(gh, vh.mT.contiguous())

    def gradients(out):
        ds = p * (dp - (gh * out).sum(-1, keepdim=True)) * scale
        dk = torch.bmm(ds.mT.contiguous(), qh).unflatten(0, (kv, -1)).sum(1)
        return [torch.bmm(ds, kh).transpose(0, 1), dk.transpose(0, 1)]

    exact = torch.bmm(p, vh)
    want = gradients(exact)
    rounded = gradients(exact.to(dtype).double())
    for name, a, b, c in zip(("dq", "dk"), got, want, rounded):
        off = (a[front:].double() - b).norm() / b.norm()
        assert off <= bound, (name, (off / u).item())
        if name == "dq":
            assert (c - b).norm() / b.norm() > bound
