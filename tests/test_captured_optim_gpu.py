"""Adam's step count in a captured step: replays go on where the eager steps
before them stopped."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _optimizer(kind, dtype):
    from deeplearning_cfn_amd.engine import DataParallel
    from deeplearning_cfn_amd.engine.optim import FlatAdam, FlatMuon
    torch.manual_seed(4)
    model = torch.nn.Sequential(
        torch.nn.Embedding(37, 48), torch.nn.Linear(48, 33),
        torch.nn.Linear(33, 48)).cuda().to(dtype)
    engine = DataParallel(model, mode="local")
    if kind == "muon":
        return FlatMuon(engine, lr=0.02, adam_lr=1e-2, betas=(0.8, 0.99))
    return FlatAdam(engine, lr=1e-2, betas=(0.8, 0.99))


def _gradients(opt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(b.flat.shape, generator=g, device="cuda")
            .to(b.flat.dtype) for b in opt.buckets]


def _step(opt):
    """The optimizer's part of a training step, from given gradients: no
    atomics of a backward pass, so the bits are the same each time."""
    def step(grads):
        for b, g in zip(opt.buckets, grads):
            b.flat.copy_(g)
        opt.step()
        return opt.flat_params[0].float().sum()
    return step


def _state(opt):
    return [t.clone() for t in (*opt.flat_params, *opt.m, *opt.v)] \
        + [t.clone() for t in opt.masters if t is not None]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_replays_count(kind, dtype):
    """Weights, moments and the count after 3 + 8 captured steps are, bit for
    bit, those of 11 eager ones; then an eager step, and a checkpoint."""
    from deeplearning_cfn_amd.engine.graph import GraphedStep
    eager, graphed = _optimizer(kind, dtype), _optimizer(kind, dtype)
    step = _step(eager)
    for seed in (0, 0, 0, 1, 2, 3, 4, 5, 6, 7, 8):
        step(_gradients(eager, seed))
    runner = GraphedStep(_step(graphed), _gradients(graphed, 0), warmup=3)
    for seed in range(1, 9):
        runner.step(_gradients(graphed, seed))
        torch.cuda.synchronize()
        _ = graphed.flat_params[0].double().sum().item()   # work in between
    assert eager.t == graphed.t == graphed.state_dict()["t"] == 11
    for a, b in zip(_state(eager), _state(graphed)):
        assert torch.equal(a, b)

    # eager again, after the replays
    saved = copy.deepcopy(graphed.state_dict())
    weights = [f.clone() for f in graphed.flat_params]
    for opt in (eager, graphed):
        _step(opt)(_gradients(opt, 20))
    assert eager.t == graphed.t == 12
    for a, b in zip(_state(eager), _state(graphed)):
        assert torch.equal(a, b)

    # a checkpoint of the replays, read while the graph lives
    for f, w in zip(graphed.flat_params, weights):
        f.copy_(w)
    graphed.load_state_dict(saved)
    assert graphed.t == 11
    runner.step(_gradients(graphed, 20))
    for a, b in zip(_state(eager), _state(graphed)):
        assert torch.equal(a, b)


def test_corrections_are_those_of_the_host():
    """1 / (1 - beta ** t) in fp32, the same bits as counted on the host."""
    from deeplearning_cfn_amd.ops import native
    for b1, b2 in ((0.9, 0.999), (0.8, 0.99), (0.0, 0.95)):
        steps = torch.zeros((), dtype=torch.int64, device="cuda")
        inverse = torch.empty(2, device="cuda")
        got = []
        for _ in range(400):
            native().adam_count(steps, inverse, b1, b2)
            got.append(inverse.clone())
        want = torch.tensor([[1 / (1 - b1 ** t), 1 / (1 - b2 ** t)]
                             for t in range(1, 401)], dtype=torch.float64)
        assert torch.equal(torch.stack(got).cpu(), want.float())
        assert steps.item() == 400


def test_counted_is_the_update_with_given_corrections():
    from deeplearning_cfn_amd.ops import native
    n = 1003
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in (torch.bfloat16, torch.float32):
        grad = torch.randn(n, generator=g, device="cuda").to(dtype)
        sets = []
        for _ in range(2):
            p = torch.linspace(-1, 1, n, device="cuda").to(dtype)
            sets.append([p, torch.zeros(n, device="cuda"),
                         torch.zeros(n, device="cuda"), p.float()])
        steps = torch.zeros((), dtype=torch.int64, device="cuda")
        inverse = torch.empty(2, device="cuda")
        for t in range(1, 4):
            p, m, v, w = sets[0]
            args = (1e-2, 0.9, 0.999, 1e-8, 0.1)
            bc = (1 - 0.9 ** t, 1 - 0.999 ** t)
            native().adam_count(steps, inverse, 0.9, 0.999)
            if dtype == torch.bfloat16:
                native().adamw_flat_master(p, grad, m, v, w, *args, *bc)
                native().adamw_flat_counted(sets[1][0], grad, *sets[1][1:],
                                            *args, inverse)
            else:
                native().adamw_flat(p, grad, m, v, *args, *bc)
                native().adamw_flat_counted(sets[1][0], grad, *sets[1][1:3],
                                            None, *args, inverse)
            for a, b in zip(*sets):
                assert torch.equal(a, b)


def test_refusals():
    from deeplearning_cfn_amd.ops import native
    steps = torch.zeros((), dtype=torch.int64, device="cuda")
    two = torch.empty(2, device="cuda")
    for args in ((steps.int(), two), (steps, two[:1]), (steps, two.double()),
                 (steps, torch.empty(4, device="cuda")[::2])):
        with pytest.raises(RuntimeError, match="adam_count"):
            native().adam_count(*args, 0.9, 0.999)
    z = torch.zeros(4, device="cuda")
    with pytest.raises(RuntimeError, match="adamw"):
        native().adamw_flat_counted(z, z, z, z, None, 1e-3, 0.9, 0.999, 1e-8,
                                    0.0, two[:1])
