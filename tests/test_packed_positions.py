"""Positions of packed documents: where they end, and borders outside the
tokens."""

import pytest
import torch

from deeplearning_cfn_amd.models.bert import BertConfig, BertForPretraining


def _model(alibi=False, max_seq=16):
    torch.manual_seed(5)
    return BertForPretraining(BertConfig(
        vocab_size=211, hidden=64, layers=1, heads=2, intermediate=128,
        max_seq=max_seq, alibi=alibi))


def _ids(rows, seq):
    return torch.randint(0, 211, (rows, seq),
                         generator=torch.Generator().manual_seed(1))


def test_document_longer_than_the_table_raises():
    """It has no positions to take: neither do rows without borders."""
    model = _model()
    ids = _ids(2, 20)
    with pytest.raises(IndexError):
        model.encode(ids)
    with pytest.raises(IndexError):
        model.encode(ids, cu_seqlens=torch.tensor([0, 17, 40]))
    # 16 tokens fit, and documents of any length without such a table
    assert model.encode(ids, cu_seqlens=torch.tensor([0, 16, 32, 40])) \
        .isfinite().all()
    assert _model(True).encode(ids, cu_seqlens=torch.tensor([0, 17, 40])) \
        .isfinite().all()


@pytest.mark.gpu
def test_document_longer_than_the_table_is_nan():
    """On the GPU, where lengths are not known on the host, its own hidden
    states are NaN, and so is the loss; the others keep theirs."""
    model = _model().cuda().bfloat16().eval()
    ids = _ids(2, 20).cuda()
    cu = torch.tensor([0, 16, 33, 40], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        x = model.encode(ids, cu_seqlens=cu).reshape(40, -1)
        assert x[16:33].isnan().all()
        assert x[:16].isfinite().all() and x[33:].isfinite().all()
        fits = model.encode(ids, cu_seqlens=torch.tensor(
            [0, 16, 32, 40], dtype=torch.int32, device="cuda")).reshape(40, -1)
        assert fits.isfinite().all() and torch.equal(fits[:16], x[:16])
        assert model(ids, ids, cu_seqlens=cu).isnan()


def test_borders_outside_the_tokens():
    """They are cut off at the tokens: positions, and the whole model."""
    from deeplearning_cfn_amd.ops import functional as F_amd
    want = [0, 1, 2, 3, 0, 1, 2, 3, 4, 5]
    for ends in ([0, 4, 10], [-3, 4, 12], [-2 ** 40, 4, 2 ** 40],
                 [-1, 0, 4, 10, 10, 11]):
        assert F_amd.document_positions(torch.tensor(ends), 10).tolist() \
            == want
    for alibi in (False, True):
        model, ids = _model(alibi), _ids(1, 10)
        x = model.encode(ids, cu_seqlens=torch.tensor([0, 4, 10]))
        for ends in ([-3, 4, 12], [-2 ** 32 - 6, 4, 2 ** 32 + 5]):
            assert torch.equal(
                model.encode(ids, cu_seqlens=torch.tensor(ends)), x)
