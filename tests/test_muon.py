"""FlatMuon, and BERT on packed documents, on the CPU."""

import copy

import pytest
import torch

from tests.conftest import run_distributed

from deeplearning_cfn_amd.data import SyntheticBertBatches
from deeplearning_cfn_amd.engine.ddp import DataParallel
from deeplearning_cfn_amd.engine.optim import FlatMuon
from deeplearning_cfn_amd.models.bert import BertConfig, BertForPretraining
from deeplearning_cfn_amd.ops import functional as F_amd


def _tiny(alibi=False, **kw):
    torch.manual_seed(5)
    return BertForPretraining(BertConfig(
        vocab_size=211, hidden=64, layers=2, heads=4, intermediate=128,
        max_seq=32, alibi=alibi, **kw))


def _plain_step(named, state, t, lr, mu, wd, adam_lr, hidden):
    """One step of the rule, a parameter at a time."""
    for name, p in named:
        g = p.grad.double()
        if name in hidden:
            v = state.setdefault(name, torch.zeros_like(g))
            v.mul_(mu).add_(g)
            o = F_amd.newton_schulz((g + mu * v).float()).double()
            rows, cols = p.shape
            step = lr * max(1.0, rows / cols) ** 0.5
            p.data = ((1 - lr * wd) * p.double() - step * o).to(p.dtype)
        else:
            m, v = state.setdefault(name, [torch.zeros_like(g),
                                           torch.zeros_like(g)])
            m.mul_(0.9).add_(0.1 * g)
            v.mul_(0.999).add_(0.001 * g * g)
            w = p.double() * (1 - adam_lr * wd)
            p.data = (w - adam_lr * (m / (1 - 0.9 ** t))
                      / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)).to(p.dtype)


def test_flat_muon_is_the_rule():
    model = _tiny()
    plain = copy.deepcopy(model)
    engine = DataParallel(model, mode="local", bucket_bytes=64 << 10)
    opt = FlatMuon(engine, lr=0.02, weight_decay=0.1, adam_lr=1e-3)
    hidden = {n for n, p in plain.named_parameters()
              if p.dim() == 2 and n.split(".")[0] in ("blocks", "mlm_dense")}
    assert sum(len(s) for s in opt.groups.values()) == len(hidden)
    state = {}
    for t in range(1, 4):
        g = torch.Generator().manual_seed(t)
        engine.zero_grad()
        for (n, p), (_, q) in zip(model.named_parameters(),
                                  plain.named_parameters()):
            q.grad = torch.randn(q.shape, generator=g)
            p.grad.copy_(q.grad)
        opt.step()
        _plain_step(list(plain.named_parameters()), state, t, 0.02, 0.95, 0.1,
                    1e-3, hidden)
        for (n, p), (_, q) in zip(model.named_parameters(),
                                  plain.named_parameters()):
            # a step of 0.02 * 1.4 times an update of up to 1.3, whose bf16
            # rounding an input off in its last bit may turn (2^-8 of it);
            # elsewhere fp32 next to 64 bits
            room = 3 * 0.02 * 1.5 * 1.3 * 2.0 ** -8 * t if n in hidden \
                else 1e-5 * t
            assert (p - q).abs().max() <= room, n


def test_state_round_trip():
    model = _tiny()
    engine = DataParallel(model, mode="local")
    opt = FlatMuon(engine)
    for b in engine.plan.buckets:
        b.flat.normal_()
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    weights = [f.clone() for f in opt.flat_params]
    opt.step()
    want = [f.clone() for f in opt.flat_params]
    for f, w in zip(opt.flat_params, weights):
        f.copy_(w)
    opt.load_state_dict(saved)
    opt.step()
    for f, w in zip(opt.flat_params, want):
        assert torch.equal(f, w)


def test_positions():
    cu = torch.tensor([2, 5, 5, 6], dtype=torch.int32)
    assert F_amd.document_positions(cu, 9).tolist() \
        == [0, 0, 0, 1, 2, 0, 0, 0, 0]
    assert F_amd.document_positions(torch.tensor([0, 0, 3, 3, 3]), 3).tolist() \
        == [0, 1, 2]
    assert F_amd.document_positions(torch.tensor([4]), 3).tolist() == [0] * 3


def test_packed_batches():
    source = SyntheticBertBatches(3, seq_len=40, doc_len=12, seed=1)
    sizes = set()
    for _ in range(5):
        ids, mlm, nsp, cu = source.batch()
        assert ids.shape == mlm.shape == (3, 40) and cu.dtype == torch.int32
        n = cu[1:] - cu[:-1]
        assert cu[0] == 0 and cu[-1] == 120 and (n >= 0).all()
        assert {40, 80} <= set(cu.tolist())       # none across two rows
        assert ((nsp == -100) == (n == 0)).all()
        sizes.add(cu.numel())
    assert len(sizes) == 1


@pytest.mark.parametrize("alibi", [False, True])
def test_packed_is_document_by_document(alibi):
    """The loss of packed documents and its gradients are those of the
    documents one after the other."""
    model = _tiny(alibi)
    ids, mlm, nsp, cu = SyntheticBertBatches(
        2, seq_len=32, vocab_size=211, doc_len=9, mask_frac=0.4,
        seed=3).batch()
    loss = model(ids, mlm, nsp, cu)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    flat, labels = ids.reshape(-1), mlm.reshape(-1)
    total, marked, heads = 0.0, (labels != -100).sum(), (nsp != -100).sum()
    for d, (a, b) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
        if a == b:
            continue
        one = flat[None, a:b]
        x = model.encode(one)
        logits = model(one)[0]
        total = total + torch.nn.functional.cross_entropy(
            logits, labels[a:b], ignore_index=-100, reduction="sum") / marked
        total = total + torch.nn.functional.cross_entropy(
            model.nsp(x[:, 0]), nsp[d:d + 1], reduction="sum") / heads
    total.backward()
    assert (loss - total).abs() <= 2e-5
    for n, p in model.named_parameters():
        assert (got[n] - p.grad).abs().max() <= 2e-4 * (1 + p.grad.abs().max()), n


def test_default_path_is_unchanged():
    """Without cu_seqlens nothing of this runs."""
    model = _tiny()
    ids = torch.randint(0, 211, (2, 16))
    x = model.tok(ids) + model.pos(torch.arange(16)[None]) \
        + model.typ(torch.zeros_like(ids))
    x = model.ln(x)
    for blk in model.blocks:
        x = blk(x)
    assert torch.equal(model.encode(ids), x)


def _worker(rank, ws, path):
    torch.manual_seed(7)
    model = _tiny()
    engine = DataParallel(model, mode="dist_device_sync")
    opt = FlatMuon(engine, lr=0.02, adam_lr=1e-3)
    for step in range(2):
        batch = SyntheticBertBatches(2, seq_len=32, vocab_size=211, doc_len=9,
                                     seed=step, rank=rank).batch()
        engine.zero_grad()
        engine(*batch).backward()
        engine.finalize_backward()
        opt.step()
    torch.save([f.clone() for f in opt.flat_params], f"{path}/{rank}.pt")


def test_ranks_stay_in_step(tmp_path):
    run_distributed(_worker, 2, str(tmp_path))
    a, b = (torch.load(tmp_path / f"{r}.pt") for r in (0, 1))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_trainer_runs(tmp_path, monkeypatch):
    """The command with all three: packed documents, distance slopes, Muon."""
    from deeplearning_cfn_amd import train
    from deeplearning_cfn_amd.models import bert, registry
    monkeypatch.setenv("EFS_MOUNT", str(tmp_path))
    monkeypatch.setattr(
        registry, "build_bert",
        lambda size, seq_len, alibi: bert.BertForPretraining(bert.BertConfig(
            hidden=32, layers=1, heads=2, intermediate=64, max_seq=seq_len,
            alibi=alibi)))
    args = train.build_argparser().parse_args([
        "--network", "bert", "--batch-size", "2", "--seq-len", "24",
        "--steps-per-epoch", "2", "--disp-batches", "1", "--eval-steps", "1",
        "--optimizer", "muon", "--lr", "0.02", "--mom", "0.95",
        "--doc-len", "8", "--alibi", "--kv-store", "local"])
    out = train.train(args)
    assert out["steps"] == 2
    assert all(torch.isfinite(torch.tensor(x)) for x in out["losses"])
    with pytest.raises(ValueError, match="optimizer"):
        train.train(train.build_argparser().parse_args(
            ["--network", "bert", "--optimizer", "lion"]))
