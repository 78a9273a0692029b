"""Embedding, document attention and Muon together, as a training step of
BERT on packed documents runs them."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(alibi, dtype=torch.bfloat16, hidden=128, heads=2):
    from deeplearning_cfn_amd.models.bert import BertConfig, BertForPretraining
    from deeplearning_cfn_amd.utils import to_compute_dtype
    torch.manual_seed(11)
    model = BertForPretraining(BertConfig(
        vocab_size=997, hidden=hidden, layers=2, heads=heads,
        intermediate=256, max_seq=64, alibi=alibi)).cuda()
    return to_compute_dtype(model, dtype)


def _batch(seed=0):
    from deeplearning_cfn_amd.data import SyntheticBertBatches
    return [t.cuda() for t in SyntheticBertBatches(
        4, seq_len=64, vocab_size=997, doc_len=20, mask_frac=0.4,
        seed=seed).batch()]


@pytest.mark.parametrize("alibi", [False, True])
def test_step_against_fp32(alibi, monkeypatch):
    """Loss and gradients of the bf16 model are no further from the fp32
    model's than torch's composed form of the same bf16 model is."""
    model = _model(alibi)
    exact = copy.deepcopy(model).float()
    batch = _batch()

    def run(m):
        m.zero_grad()
        loss = m(*batch)
        loss.backward()
        return loss.item(), {n: p.grad.double()
                             for n, p in m.named_parameters()}

    loss, grads = run(model)
    from deeplearning_cfn_amd.ops import functional as F_amd
    monkeypatch.setattr(F_amd, "_doc_attention_native", lambda t: False)
    monkeypatch.setattr(F_amd, "embedding_sum", lambda ids, tables: sum(
        torch.nn.functional.embedding(i, w).float()
        for i, w in zip(ids, tables)).to(tables[0].dtype))
    plain_loss, plain = run(model)
    monkeypatch.undo()
    want_loss, want = run(exact)
    # logits are 128 products of numbers under 4 and weights of 0.02, each
    # rounded some ten times to 2^-9: off by 0.05 at most
    assert abs(loss - want_loss) <= 0.05 and abs(plain_loss - want_loss) <= 0.05
    ours = sum((grads[n] - want[n]).square().sum() for n in want).sqrt()
    theirs = sum((plain[n] - want[n]).square().sum() for n in want).sqrt()
    assert ours <= 1.5 * theirs, (ours, theirs)
    for n in want:
        assert grads[n].isfinite().all(), n


def test_documents_do_not_see_each_other():
    """A change in one document leaves the others' hidden states alone, bit
    for bit, in the whole model."""
    model = _model(True).eval()
    ids, _, _, cu = _batch()
    with torch.no_grad():
        a = model.encode(ids, cu_seqlens=cu).reshape(-1, 128)
        other = ids.clone().reshape(-1)
        s, e = cu[2].item(), cu[3].item()
        other[s:e] = (other[s:e] + 7) % 997
        b = model.encode(other.view_as(ids), cu_seqlens=cu).reshape(-1, 128)
    assert torch.equal(a[:s], b[:s]) and torch.equal(a[e:], b[e:])
    assert not torch.equal(a[s:e], b[s:e])


def _train(alibi, graphed, steps=4):
    from deeplearning_cfn_amd.engine import DataParallel
    from deeplearning_cfn_amd.engine.graph import GraphedStep
    from deeplearning_cfn_amd.engine.optim import FlatMuon
    engine = DataParallel(_model(alibi), mode="local", bucket_bytes=1 << 18)
    opt = FlatMuon(engine, lr=0.02, adam_lr=1e-3)

    def step(ins):
        engine.zero_grad()
        loss = engine(*ins)
        loss.backward()
        engine.finalize_backward()
        opt.step()
        return loss

    losses = []
    if graphed:
        runner = GraphedStep(step, _batch(0), warmup=1)
        # the warm-up pass and each replay are training steps of batch 0, 1, ..
        for k in range(1, steps):
            losses.append(runner.step(_batch(k)).item())
            torch.cuda.synchronize()
    else:
        for k in range(steps):
            losses.append(step(_batch(k)).item())
    return losses, [f.clone() for f in opt.flat_params], opt


def test_training_is_repeatable_and_moves_every_parameter():
    a, wa, opt = _train(False, False)
    b, wb, _ = _train(False, False)
    # the flat gradients of linear layers come from kernels with float
    # atomics, so runs agree to their rounding only
    for x, y in zip(a, b):
        assert abs(x - y) <= 0.05
    assert all(torch.isfinite(w).all() for w in wa)
    start = _model(False)
    for (n, p), q in zip(start.named_parameters(),
                         opt.engine.module.parameters()):
        assert not torch.equal(p, q), n


def test_captured_step():
    """A captured training step replays with new documents each time."""
    losses, weights, _ = _train(True, True)
    eager, want, _ = _train(True, False)
    assert all(torch.isfinite(w).all() for w in weights)
    for x, y in zip(losses, eager[1:]):
        assert abs(x - y) <= 0.1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("odd", [False, True])
def test_muon_kernels(dtype, odd):
    """Momentum and weights of 50 matrices (more than one launch holds) at odd
    places of a flat buffer, against 64 bits."""
    from deeplearning_cfn_amd.ops import native
    n, rows, cols = 50, 6, 34 if not odd else 35
    size = rows * cols
    off = 2 if not odd else 1
    flat = lambda t: torch.randn(n * size + off, device="cuda").to(t)  # noqa: E731
    g, p, v, w = flat(dtype), flat(dtype), flat(torch.float32), \
        flat(torch.float32)
    cut = lambda f: [f[off + i * size:off + (i + 1) * size]  # noqa: E731
                     for i in range(n)]
    u = torch.empty(n, rows, cols, device="cuda")
    v0 = v.clone()
    native().muon_momentum(cut(g), cut(v), u, 0.9, True)
    want = 0.9 * v0.double()[off:] + g.double()[off:]
    near = lambda a, b, s: ((a.double() - b).abs() <= s).all()  # noqa: E731
    f = 2.0 ** -22
    assert near(v[off:], want, f * (v0.abs().double() + g.abs().double())[off:])
    assert torch.equal(v[:off], v0[:off])
    assert near(u.reshape(-1), g.double()[off:] + 0.9 * want,
                4 * f * (v0.abs().double() + g.abs().double())[off:])
    o = torch.randn(n, rows, cols, device="cuda").bfloat16()
    for master in (cut(w), []):
        p0, w0 = p.clone(), w.clone()
        native().muon_apply(cut(p), master, o, 0.02, 0.99)
        src = w0 if master else p0
        ref = 0.99 * src.double()[off:] - 0.02 * o.double().reshape(-1)
        half = torch.finfo(dtype).eps / 2
        assert near(p[off:], ref, (half + 4 * f) * (ref.abs() + 0.1))
        if master:
            assert near(w[off:], ref, 4 * f * (ref.abs() + 0.1))
        assert torch.equal(p[:off], p0[:off])


def test_muon_refusals():
    from deeplearning_cfn_amd.ops import native
    g = torch.zeros(12, device="cuda")
    u = torch.zeros(1, 3, 4, device="cuda")
    with pytest.raises(RuntimeError, match="muon"):
        native().muon_momentum([g, g], [g, g], u, 0.9, True)
    with pytest.raises(RuntimeError, match="muon"):
        native().muon_momentum([g[:8]], [g], u, 0.9, True)
    with pytest.raises(RuntimeError, match="muon"):
        native().muon_momentum([g], [g.half()], u, 0.9, True)
    with pytest.raises(RuntimeError, match="muon"):
        native().muon_apply([g], [], u, 0.1, 1.0)
