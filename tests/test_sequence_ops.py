"""Embedding lookup, document attention and Newton-Schulz on the CPU: the
composed forms, the refusals, and the bindings' own checks."""

import pytest
import torch

from deeplearning_cfn_amd.ops import functional as F_amd


def test_embedding_sum_and_its_gradient():
    torch.manual_seed(0)
    tables = [torch.randn(v, 6, requires_grad=True) for v in (11, 5, 2)]
    ids = [torch.randint(0, v, (4, 7)) for v in (11, 5, 2)]
    ids[0][0] = 3
    scales = [2.0, 1.0, 0.5]
    y = F_amd.embedding_sum(ids, tables, scales)
    want = sum(w.detach().double()[i] * c
               for w, i, c in zip(tables, ids, scales))
    assert (y.double() - want).abs().max() <= 8 * 2.0 ** -24 * 8
    g = torch.randn_like(y)
    for d, w, i, c in zip(torch.autograd.grad(y, tables, g), tables, ids,
                          scales):
        ref = torch.zeros(w.shape, dtype=torch.float64).index_add_(
            0, i.reshape(-1), (g.double() * c).reshape(-1, 6))
        assert (d.double() - ref).abs().max() <= 30 * 2.0 ** -24 * 100


def test_embedding_is_one_table():
    w = torch.randn(5, 3)
    i = torch.tensor([4, 0, 4])
    assert torch.equal(F_amd.embedding(i, w, 2.0), 2.0 * w[i])


@pytest.mark.parametrize("ids,tables,scales", [
    ([], [], None),
    ([torch.zeros(2).long()] * 5, [torch.zeros(3, 4)] * 5, None),
    ([torch.zeros(2).long()], [torch.zeros(3, 4)] * 2, None),
    ([torch.zeros(2).long()], [torch.zeros(3, 4)], [1.0, 2.0]),
    ([torch.zeros(2)], [torch.zeros(3, 4)], None),
    ([torch.zeros(2).short()], [torch.zeros(3, 4)], None),
    ([torch.zeros(2).long(), torch.zeros(3).long()], [torch.zeros(3, 4)] * 2,
     None),
    ([torch.zeros(2).long()] * 2, [torch.zeros(3, 4), torch.zeros(3, 5)],
     None),
    ([torch.zeros(2).long()] * 2, [torch.zeros(3, 4), torch.zeros(3, 4).half()],
     None),
    ([torch.zeros(2).long()], [torch.zeros(3)], None),
])
def test_embedding_refusals(ids, tables, scales):
    with pytest.raises(ValueError, match="embedding_sum"):
        F_amd.embedding_sum(ids, tables, scales)


def _plain(q, k, v, ends, scale, slopes):
    """One masked softmax over all tokens, in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    T, H, D = q.shape
    doc = torch.full((T,), -1)
    for n, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        doc[a:b] = n
    see = (doc[:, None] == doc) & (doc >= 0)
    k, v = (t.repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    if slopes is not None:
        i = torch.arange(T).double()
        s = s - slopes.double()[:, None, None] * (i[:, None] - i).abs()
    p = torch.where(see, torch.exp(s - s.amax(-1, True)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.einsum("hij,jhd->ihd", p, v)


@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 2), (3, 1)])
@pytest.mark.parametrize("ends", [
    [0, 9], [0, 0, 1, 9, 9], [2, 5, 7], [9], [4, 4], [0, 3, 8]])
@pytest.mark.parametrize("bias", [False, True])
def test_document_attention_composed(heads, kv, ends, bias):
    torch.manual_seed(1)
    q, k, v = (torch.randn(9, h, 6, requires_grad=True)
               for h in (heads, kv, kv))
    slopes = torch.linspace(0.1, 1.0, heads) if bias else None
    o = F_amd.document_attention(q, k, v, torch.tensor(ends), slopes=slopes)
    want = _plain(q, k, v, ends, 6 ** -0.5, slopes)
    # 9 terms of size under 4, in fp32
    assert (o.double() - want).abs().max() <= 1e-5
    c = torch.randn_like(o)
    if o.grad_fn is not None:
        got = torch.autograd.grad(o, [q, k, v], c, allow_unused=True)
        ref = torch.autograd.grad(want, [q, k, v], c.double())
        for a, b in zip(got, ref):
            a = torch.zeros_like(b) if a is None else a
            assert (a.double() - b).abs().max() <= 1e-4


def test_document_attention_packed_entry():
    torch.manual_seed(2)
    qkv = torch.randn(7, 3, 2, 4, requires_grad=True)
    cu = torch.tensor([0, 3, 7], dtype=torch.int32)
    o = F_amd.document_attention_qkv(qkv, cu)
    assert torch.equal(o, F_amd.document_attention(*qkv.unbind(1), cu))
    o.sum().backward()
    assert qkv.grad.shape == qkv.shape


def _qkv(T=4, H=2, KV=2, D=8, dtype=torch.float32):
    return [torch.zeros(T, h, D, dtype=dtype) for h in (H, KV, KV)]


CU = torch.tensor([0, 4])


@pytest.mark.parametrize("args,kw", [
    ((*_qkv(H=3, KV=2), CU), {}),
    ((*_qkv()[:2], torch.zeros(4, 1, 8), CU), {}),
    ((_qkv()[0], *_qkv(D=16)[1:], CU), {}),
    ((_qkv()[0], *_qkv(T=5)[1:], CU), {}),
    ((*[t[0] for t in _qkv()], CU), {}),
    ((_qkv()[0], *_qkv(dtype=torch.float64)[1:], CU), {}),
    ((*_qkv(), CU.float()), {}),
    ((*_qkv(), CU[None]), {}),
    ((*_qkv(), CU[:0]), {}),
    ((*_qkv(), CU), {"scale": 0.0}),
    ((*_qkv(), CU), {"scale": -1.0}),
    ((*_qkv(), CU), {"scale": float("nan")}),
    ((*_qkv(), CU), {"scale": float("inf")}),
    ((*_qkv(), CU), {"scale": 1e-40}),
    ((*_qkv(H=0), CU), {"scale": 1e40}),
    ((*_qkv(), CU), {"slopes": torch.zeros(3)}),
    ((*_qkv(), CU), {"slopes": torch.zeros(2, 1)}),
    ((*_qkv(), CU), {"slopes": torch.zeros(2, requires_grad=True)}),
])
def test_document_attention_refusals(args, kw):
    with pytest.raises(ValueError, match="document_attention"):
        F_amd.document_attention(*args, **kw)


def test_document_attention_packed_refusals():
    with pytest.raises(ValueError, match="document_attention_qkv"):
        F_amd.document_attention_qkv(torch.zeros(4, 2, 2, 8), CU)
    with pytest.raises(ValueError, match="document_attention_qkv"):
        F_amd.document_attention_qkv(torch.zeros(4, 3, 8), CU)


def test_newton_schulz():
    torch.manual_seed(3)
    g = torch.randn(3, 20, 50)
    y = F_amd.newton_schulz(g)
    assert y.dtype == torch.bfloat16 and y.shape == g.shape
    s = torch.linalg.svdvals(y.float())
    # five steps of this polynomial bring singular values from 0.05 of the
    # largest up to between 0.66 and 1.22; bf16 moves them by under 0.02
    assert (s > 0.64).all() and (s < 1.24).all()
    assert torch.equal(F_amd.newton_schulz(g.mT).mT, y)
    assert torch.equal(F_amd.newton_schulz(g[1]), y[1])
    assert F_amd.newton_schulz(torch.zeros(4, 6)).eq(0).all()


@pytest.mark.parametrize("g,kw", [
    (torch.zeros(3), {}), (torch.zeros(3, 3).long(), {}),
    (torch.zeros(3, 3), {"steps": 0}), (torch.zeros(3, 3), {"steps": 101}),
    (torch.zeros(3, 3), {"eps": -1.0}),
    (torch.zeros(3, 3), {"eps": float("nan")})])
def test_newton_schulz_refusals(g, kw):
    with pytest.raises(ValueError, match="newton_schulz"):
        F_amd.newton_schulz(g, **kw)
