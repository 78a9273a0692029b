"""Embedding lookup (embedding.hip) at the borders of what it takes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


@pytest.mark.parametrize("shape", [(), (0,), (3,), (2, 0), (2, 3)])
@pytest.mark.parametrize("width", [0, 5])
@pytest.mark.parametrize("rows", [0, 4])
def test_nothing_of_something(rows, width, shape):
    """No tokens, no width, no rows: outputs and gradients have their shapes,
    as on the CPU."""
    tokens = 1
    for n in shape:
        tokens *= n
    if rows == 0 and tokens and width:
        return                            # ids outside a table: NaN, not 0
    got = []
    for device in ("cuda", "cpu"):
        if device == "cpu" and rows == 0 and tokens:
            continue                      # raises there
        w = torch.ones(rows, width, device=device, requires_grad=True)
        v = torch.ones(7, width, device=device, requires_grad=True)
        i = torch.zeros(shape, dtype=torch.int64, device=device)
        y = _f().embedding_sum([i, i], [w, v], [1.0, 2.0])
        assert y.shape == (*shape, width)
        d = torch.autograd.grad(y, [w, v], torch.ones_like(y))
        assert d[0].shape == w.shape and d[1].shape == v.shape
        got.append([t.cpu() for t in (y, *d)])
    for a, b in zip(*got) if len(got) == 2 else ():
        assert torch.equal(a, b)


def test_large_tables_are_refused_before_the_lookup():
    """What has no gradient kernel raises in the forward pass, if a gradient
    is wanted of it; without one it is looked up."""
    rows = 2 ** 22
    big = torch.zeros(rows, 1, device="cuda", dtype=torch.bfloat16)
    big[-1] = 3
    small = torch.ones(5, 1, device="cuda", dtype=torch.bfloat16)
    i = torch.tensor([rows - 1, 0], device="cuda")
    j = torch.tensor([4, 4], device="cuda")
    f = _f().embedding_sum
    assert f([i], [big]).flatten().tolist() == [3, 0]
    y = f([i, j], [big, small.requires_grad_(True)])
    d, = torch.autograd.grad(y, [small], torch.ones_like(y))
    assert d.flatten().tolist() == [0, 0, 0, 0, 2]
    big.requires_grad_(True)
    for ids, tables in (([i], [big]), ([j, i], [small, big])):
        with pytest.raises(ValueError, match="embedding_sum.*2\\^22"):
            f(ids, tables)
        with torch.no_grad():
            assert f(ids, tables).isfinite().all()
    less = torch.zeros(rows - 1, 1, device="cuda", requires_grad=True)
    y = f([i - 1], [less])
    d, = torch.autograd.grad(y[:1], [less], torch.ones(1, 1, device="cuda"))
    assert d[rows - 2] == 1 and d.sum() == 1


@pytest.mark.parametrize("n", [900, 6000])
def test_any_order_of_the_tables(n):
    """A table's gradient has the same bits wherever it stands in the call."""
    rows, width = [3000, 2, 512, 2], 40
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = [torch.randint(0, r, (n,), generator=g, device="cuda") for r in rows]
    tables = [torch.randn(r, width, generator=g, device="cuda")
              .requires_grad_(True) for r in rows]
    scales = [1.0, 0.5, 2.0, -1.0]
    grad = torch.randn(n, width, generator=g, device="cuda")
    want = None
    for order in ((0, 1, 2, 3), (3, 2, 1, 0), (1, 3, 0, 2), (2, 0, 3, 1)):
        pick = lambda x: [x[k] for k in order]  # noqa: E731
        y = _f().embedding_sum(pick(ids), pick(tables), pick(scales))
        d = dict(zip(order, torch.autograd.grad(y, pick(tables), grad)))
        want = want or d
        for k in range(4):
            assert torch.equal(d[k], want[k])
