"""What a short document gets does not hang on what it is packed with
(doc_attention.hip): P and dS are taken in two parts by the document's own
length, or by that of a whole small call."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _exact(q, k, v, do):
    """o, dq, dk, dv of one document in 64 bits."""
    q, k, v = (t.double().requires_grad_(True) for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    at = torch.arange(q.shape[1], device="cuda") // group
    s = torch.bmm(q.transpose(0, 1).contiguous(),
                  k[:, at].permute(1, 2, 0).contiguous())
    p = torch.softmax(s * q.shape[-1] ** -0.5, -1)
    o = torch.bmm(p, v[:, at].transpose(0, 1).contiguous()).transpose(0, 1)
    return [o.detach(), *torch.autograd.grad(o, [q, k, v], do.double())]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
@pytest.mark.parametrize("lengths", [
    [3, 8000], [8000, 3], [64, 8000, 2, 3000], [40], [1024], [300, 724],
    [3, 8000, 0, 0]])
def test_short_documents_round_once(lengths, heads, kv, dim, dtype):
    """A term of a short document's products is off by u^2, the terms' sizes
    add up to at most 32 times the result's (sqrt(n) for n <= 1024 terms of
    random sign), which is 2^-11 for bf16; fp16's subnormals leave 2^-25 of a
    p or ds where typical ones are 2^-10 or more, 2^-15 of them, and its u^2
    is 2^-22: 2^-14.  What is left is the rounding of the result."""
    more = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -14
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    # the second call pads: eight waves by the call's mean, short by its own
    for padding in ((0, 6000) if ends[-1] < 64 else (0,)):
        tokens = ends[-1] + padding
        g = torch.Generator(device="cuda").manual_seed(tokens)
        q, k, v, do = (torch.randn(tokens, h, dim, generator=g, device="cuda")
                       .to(dtype) for h in (heads, kv, kv, heads))
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
        y = _f().document_attention(*leaves, cu)
        got = [y.detach(), *torch.autograd.grad(y, leaves, do)]
        small = 1024 if tokens <= 1024 else 64
        for a, b in zip(ends[:-1], ends[1:]):
            if not 1 < b - a <= small:
                continue
            want = _exact(*(t.detach()[a:b] for t in (q, k, v, do)))
            for name, x, w in zip(("o", "dq", "dk", "dv"), got, want):
                least = (w.to(dtype).double() - w).norm()
                off = (x[a:b].double() - w).norm()
                assert off <= least + more * w.norm(), (name, a, b)


@pytest.mark.parametrize("dim", [64, 128])
def test_short_document_in_any_company(dim):
    """The same bits of a document of up to 64 tokens, whatever is beside
    it."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    F_amd = _f()
    short = [torch.randn(50, 2, dim, generator=g, device="cuda").bfloat16()
             for _ in range(4)]
    got = []
    for beside in (0, 1500, 9000):
        big = [torch.cat([t, torch.randn(beside, 2, dim, generator=g,
                                         device="cuda").bfloat16()])
               for t in short]
        leaves = [t.requires_grad_(True) for t in big[:3]]
        cu = torch.tensor([0, 50, 50 + beside], dtype=torch.int32,
                          device="cuda")
        y = F_amd.document_attention(*leaves, cu)
        got.append([t[:50] for t in (y.detach(), *torch.autograd.grad(
            y, leaves, big[3]))])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
