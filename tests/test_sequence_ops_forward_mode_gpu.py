"""Tangents of forward mode: the device's operators have no formula for them
and say so; the composed forms carry them."""

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _dual(t):
    return fw.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad", [False, True])
def test_embedding_refuses_a_tangent(grad):
    w = torch.randn(5, 8, device="cuda")
    other = torch.randn(5, 8, device="cuda", requires_grad=grad)
    i = torch.tensor([1, 2], device="cuda")
    with fw.dual_level():
        for tables in ([_dual(w), other], [other, _dual(w)], [_dual(w)]):
            with pytest.raises(RuntimeError, match="forward-mode"):
                _f().embedding_sum([i] * len(tables), tables)
            with torch.no_grad(), pytest.raises(RuntimeError,
                                                match="forward-mode"):
                _f().embedding_sum([i] * len(tables), tables)
        # inside a level, but without a tangent
        assert torch.equal(_f().embedding(i, w), w[i])


@pytest.mark.parametrize("grad", [False, True])
def test_attention_refuses_a_tangent(grad):
    q, k, v = (torch.randn(6, 2, 64, device="cuda").bfloat16()
               .requires_grad_(grad) for _ in range(3))
    cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    s = torch.ones(2, device="cuda")
    qkv = torch.randn(6, 3, 2, 64, device="cuda").half().requires_grad_(grad)
    f = _f()
    with fw.dual_level():
        for args in ((_dual(q), k, v), (q, _dual(k), v), (q, k, _dual(v))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f.document_attention(*args, cu)
        with pytest.raises(RuntimeError, match="forward-mode"):
            f.document_attention(q, k, v, cu, slopes=_dual(s))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f.document_attention_qkv(_dual(qkv), cu)
        assert f.document_attention(q, k, v, cu, slopes=s).shape == q.shape


def test_composed_forms_carry_it():
    """On the CPU the same calls give a tangent."""
    f = _f()
    w = torch.randn(5, 8)
    q = torch.randn(6, 2, 8)
    cu = torch.tensor([0, 6])
    with fw.dual_level():
        y = f.embedding(torch.tensor([1, 2]), _dual(w), 2.0)
        assert torch.equal(fw.unpack_dual(y).tangent, torch.full((2, 8), 2.0))
        # softmax weights add up to one: a tangent of ones in v stays one
        y = f.document_attention(q, q, _dual(q), cu)
        assert (fw.unpack_dual(y).tangent - 1).abs().max() <= 6 * 2.0 ** -23
