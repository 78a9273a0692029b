"""Embedding lookup and its gradient (embedding.hip) against 64 bits.

Bounds: the sums run in fp32, so n terms lose at most n * 2^-24 of the sum
of their sizes; the result is rounded once, eps / 2 of its value.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _close(got, want, size, terms):
    """got: rounded; want, size: 64 bits (the sum, and that of the sizes)."""
    half = torch.finfo(got.dtype).eps / 2
    # below the smallest normal number a step is absolute
    tiny = torch.finfo(got.dtype).smallest_normal * half
    bound = half * want.abs() * (1 + half) + terms * 2.0 ** -24 * size + tiny
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()


def _tables(sizes, width, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(v, width, generator=g, device="cuda").to(dtype)
            .requires_grad_(True) for v in sizes]


def _reference(ids, tables, scales, grad):
    y = sum(w.detach().double()[i.long()] * c
            for i, w, c in zip(ids, tables, scales))
    size = sum((w.detach().double()[i.long()] * c).abs()
               for i, w, c in zip(ids, tables, scales))
    grads = []
    for i, w, c in zip(ids, tables, scales):
        flat, g = i.reshape(-1).long(), grad.reshape(-1, w.shape[1]).double()
        d = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        a = torch.zeros_like(d)
        d.index_add_(0, flat, g * c)
        a.index_add_(0, flat, (g * c).abs())
        count = torch.bincount(flat, minlength=w.shape[0])[:, None]
        grads.append((d, a, count + 4.0))
    return y, size, grads


def _check(ids, tables, scales, seed=1):
    F_amd = _f()
    y = F_amd.embedding_sum(ids, tables, scales)
    width = tables[0].shape[1]
    assert y.shape == (*ids[0].shape, width) and y.dtype == tables[0].dtype
    g = torch.Generator(device="cuda").manual_seed(seed)
    grad = torch.randn(y.shape, generator=g, device="cuda").to(y.dtype)
    got = torch.autograd.grad(y, tables, grad)
    want, size, grads = _reference(ids, tables, scales, grad)
    _close(y.detach(), want, size, 2 * len(tables))
    for d, w, (ref, mag, count) in zip(got, tables, grads):
        assert d.shape == w.shape and d.dtype == w.dtype
        _close(d, ref, mag, count)
    return y, got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,width,rows", [
    (1, 8, 1), (1, 1, 5), (3, 13, 2), (64, 768, 100), (65, 104, 2048),
    (1000, 201, 7), (4097, 64, 30528), (2500, 1032, 300)])
def test_one_table(dtype, n, width, rows):
    g = torch.Generator(device="cuda").manual_seed(n)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    _check([ids], _tables([rows], width, dtype), [0.75])


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_three_tables_of_a_batch(ids_dtype):
    """Tokens by a power law with a hot one, positions, two segments."""
    n, h = (8, 512), 768
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    tok = (torch.exp(u * math.log(30529.0)).long() - 1).clamp(0, 30527)
    tok[torch.rand(n, generator=g, device="cuda") < 0.3] = 103
    pos = torch.arange(512, device="cuda").expand(n)
    seg = (pos > 300).long()
    ids = [t.to(ids_dtype) for t in (tok, pos, seg)]
    _check(ids, _tables([30528, 512, 2], h, torch.bfloat16),
           [math.sqrt(h), 1.0, 1.0])


@pytest.mark.parametrize("count", [63, 64, 65, 127, 128, 129, 256, 4096,
                                   40000])
def test_rows_of_many_tokens(count):
    """Around the sizes at which a row is cut into pieces."""
    ids = torch.full((count + 70,), 5, device="cuda")
    ids[::((count + 70) // 70)][:70] = torch.arange(70, device="cuda") + 20
    _check([ids], _tables([97], 72, torch.float32), [1.0])


def test_neighbouring_heavy_rows():
    ids = torch.arange(40, device="cuda").repeat_interleave(
        torch.arange(60, 100, device="cuda"))
    ids = ids[torch.randperm(len(ids), device="cuda")]
    _check([ids], _tables([40], 40, torch.float32), [1.0])


def test_large_vocabulary():
    """More rows than 256 blocks of the largest share."""
    rows = 600_000
    ids = torch.randint(0, rows, (5000,), device="cuda")
    ids[:300] = rows - 1
    _check([ids], _tables([rows], 8, torch.bfloat16), [1.0])


def test_same_bits_each_time():
    ids = torch.randint(0, 50, (20000,), device="cuda")
    w = _tables([50], 264, torch.float32)
    y = _f().embedding(ids, w[0])
    g = torch.randn_like(y)
    first, = torch.autograd.grad(y, w, g, retain_graph=True)
    for _ in range(4):
        again, = torch.autograd.grad(y, w, g, retain_graph=True)
        assert torch.equal(first, again)


def test_ids_outside_the_table():
    w = _tables([10], 16, torch.bfloat16)
    ids = torch.tensor([3, -1, 10, 3, 2 ** 40], device="cuda")
    y = _f().embedding(ids, w[0])
    assert y[[1, 2, 4]].isnan().all()
    assert torch.equal(y[0], w[0][3]) and torch.equal(y[3], w[0][3])
    d, = torch.autograd.grad(y, w, torch.ones_like(y))
    want = torch.zeros(10, 16, device="cuda", dtype=torch.bfloat16)
    want[3] = 2
    assert torch.equal(d, want)


def test_no_tokens_and_frozen_tables():
    F_amd = _f()
    w = _tables([10, 4], 16, torch.bfloat16)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    y = F_amd.embedding(none, w[0])
    assert y.shape == (0, 16)
    d, = torch.autograd.grad(y, w[:1], torch.empty_like(y))
    assert torch.equal(d, torch.zeros_like(w[0]))
    ids = torch.tensor([1, 2], device="cuda")
    frozen = w[0].detach()
    y = F_amd.embedding_sum([ids, ids], [frozen, w[1]])
    d, = torch.autograd.grad(y, [w[1]], torch.ones_like(y))
    assert d[1:3].eq(1).all() and d[0].eq(0).all() and d[3].eq(0).all()


def test_strided_inputs():
    """Ids, table and gradient that are views."""
    F_amd = _f()
    base = torch.randn(50, 48, device="cuda")
    w = base[:, 8:32].detach().requires_grad_(True)
    ids = torch.randint(0, 50, (30, 4), device="cuda").t()
    y = F_amd.embedding(ids, w, 2.0)
    assert torch.equal(y, 2.0 * w.detach()[ids])
    grad = torch.randn(24, 4, 30, device="cuda").permute(1, 2, 0)
    d, = torch.autograd.grad(y, [w], grad)
    want, size, grads = _reference([ids], [w], [2.0], grad)
    _close(d, *grads[0])


def test_captured_and_replayed():
    """The same graph over new inputs, with eager work in between."""
    F_amd = _f()
    w = [t.detach() for t in _tables([700, 2], 64, torch.bfloat16)]
    ids = [torch.randint(0, 700, (3000,), device="cuda"),
           torch.randint(0, 2, (3000,), device="cuda")]
    grad = torch.randn(3000, 64, device="cuda").bfloat16()
    from deeplearning_cfn_amd.ops import native

    def step():
        y = native().embed_sum_fwd(ids, w, [1.0, 1.0])
        return [y, *native().embed_sum_bwd(grad, ids, [700, 2], [1.0, 1.0])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        ids[0].copy_(torch.randint(0, 700 >> (3 * k), (3000,), device="cuda"))
        grad.copy_(torch.randn(3000, 64, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_on_another_stream():
    F_amd = _f()
    w = _tables([300], 128, torch.bfloat16)
    ids = torch.randint(0, 300, (4096,), device="cuda")
    want = F_amd.embedding(ids, w[0])
    g = torch.randn_like(want)
    dwant, = torch.autograd.grad(want, w, g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = F_amd.embedding(ids, w[0])
        d, = torch.autograd.grad(y, w, g)
    s.synchronize()
    assert torch.equal(y, want) and torch.equal(d, dwant)


def test_one_table_twice_and_expanded_ids():
    """The same table in two places of a sum; ids that are one row repeated."""
    F_amd = _f()
    w = _tables([40], 24, torch.float32)[0]
    a = torch.randint(0, 40, (1, 50), device="cuda").expand(30, 50)
    b = torch.randint(0, 40, (30, 50), device="cuda")
    y = F_amd.embedding_sum([a, b], [w, w], [1.0, -0.5])
    g = torch.randn_like(y)
    d, = torch.autograd.grad(y, [w], g)
    _, _, parts = _reference([a, b], [w, w], [1.0, -0.5], g)
    _close(d, parts[0][0] + parts[1][0], parts[0][1] + parts[1][1],
           parts[0][2] + parts[1][2])


def test_what_the_graph_refuses():
    F_amd = _f()
    w = _tables([10], 8, torch.float32)
    ids = torch.tensor([1, 2, 3], device="cuda")
    y = F_amd.embedding(ids, w[0])
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(y, w, torch.ones_like(y), create_graph=True)
    y = F_amd.embedding(ids, w[0])
    ids[0] = 5
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, w, torch.ones_like(y))


def test_many_short_rows():
    """More tokens than one block each, around the border at which the sort
    makes buckets first."""
    for n in (4095, 4096, 4097, 70000):
        ids = torch.randint(0, 3000, (n,), device="cuda")
        _check([ids], _tables([3000], 3, torch.float32), [1.0])


def test_backward_again():
    """With its graph kept a second pass gives the same; without it raises,
    and so does a graph whose ids were written to in between."""
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    ids = torch.randint(0, 20, (30,), device="cuda")
    y = _f().embedding_sum([ids], [w])
    first, = torch.autograd.grad(y.sum(), w, retain_graph=True)
    again, = torch.autograd.grad(y.sum(), w)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), w)
    y = _f().embedding_sum([ids], [w])
    ids.add_(0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), w)


def test_refusals_on_the_device():
    """The same errors as on the CPU."""
    f = _f().embedding_sum
    w, w2 = (torch.randn(4, n, device="cuda") for n in (8, 9))
    i = torch.zeros(3, dtype=torch.long, device="cuda")
    for ids, tables, scales in (
            ([i] * 5, [w] * 5, None), ([i], [w, w], None),
            ([i, i], [w, w], [1.0]), ([i.float()], [w], None),
            ([i, i[:2]], [w, w], None), ([i, i], [w, w2], None),
            ([i, i], [w, w.half()], None), ([i], [w[0]], None),
            ([i.cpu()], [w], None), ([i, i], [w, w.cpu()], None)):
        with pytest.raises(ValueError, match="embedding_sum"):
            f(ids, tables, scales)
