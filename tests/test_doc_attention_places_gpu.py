"""Document attention (doc_attention.hip) on tensors that begin anywhere in
their memory."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _at(t, off):
    """The same numbers, contiguous, `off` elements into a flat buffer."""
    flat = torch.zeros(t.numel() + 16, dtype=t.dtype, device=t.device)
    place = flat[off:off + t.numel()].view(t.shape)
    assert place.is_contiguous()
    return place.copy_(t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("lengths", [[1], [70, 3, 130]])
def test_inputs_cut_out_of_a_flat_buffer(lengths, dim, dtype):
    """q, k, v and the gradient that begin off a 16-byte border, all and one
    by one, give the bits of aligned copies."""
    F_amd = _f()
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(dim)
    base = [torch.randn(ends[-1], h, dim, generator=g, device="cuda").to(dtype)
            for h in (4, 2, 2, 4)]

    def run(offs):
        q, k, v, do = (_at(t, off) for t, off in zip(base, offs))
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = F_amd.document_attention(*leaves, cu)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want = run((0, 0, 0, 0))
    for offs in ((1, 1, 1, 1), (7, 0, 0, 0), (0, 2, 0, 0), (0, 0, 4, 0),
                 (0, 0, 0, 3)):
        for a, b in zip(run(offs), want):
            assert torch.equal(a, b), offs


@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("off", [1, 4])
def test_packed_projection_cut_out_of_a_flat_buffer(tokens, off):
    F_amd = _f()
    cu = torch.tensor([0, (tokens + 1) // 2, tokens], dtype=torch.int32,
                      device="cuda")
    base = torch.randn(tokens, 3, 2, 64, device="cuda").bfloat16()
    do = torch.randn(tokens, 2, 64, device="cuda").bfloat16()

    def run(qkv, grad):
        leaf = qkv.detach().requires_grad_(True)
        o = F_amd.document_attention_qkv(leaf, cu)
        return [o.detach(), *torch.autograd.grad(o, [leaf], grad)]

    want = run(base, do)
    for got in (run(_at(base, off), _at(do, off)), run(_at(base, off), do),
                run(base, _at(do, off))):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_one_token_of_any_stride():
    """A dimension of one element may have any stride."""
    F_amd = _f()
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    wide = torch.randn(3, 67, device="cuda").bfloat16()
    rows = [w[:64].view(1, 1, 64).as_strided((1, 1, 64), (67, 13, 1))
            for w in wide]
    o = F_amd.document_attention(*rows, cu)
    assert torch.equal(o, wide[2, :64].view(1, 1, 64))
