"""Document attention (doc_attention.hip) against 64 bits.

Bounds, element by element, u = eps / 2 of the inputs' type:
* a score is a sum of dim products and a bias in fp32, so it is off by at
  most e = 2^-24 (dim + 8) (scale sum |q||k| + |bias|) + 2^-22 (the exponential),
  and so is p, relatively; sums over L tokens add L 2^-24;
* p (and ds) is rounded to the inputs' type for the next product: u of each;
  fp16's subnormals make that at least 2^-25;
* the result is rounded: u.
* D = do . o takes the rounded o: u sum |do||o|.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _inputs(tokens, heads, kv, dim, dtype, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(tokens, h, dim, generator=g, device="cuda") * size)
            .to(dtype) for h in (heads, kv, kv, heads)]


def _slopes(heads):
    return torch.tensor([2.0 ** (-8 * (i + 1) / heads) for i in range(heads)],
                        device="cuda")


def _reference(q, k, v, do, ends, scale, slopes):
    """o, dq, dk, dv and what each may be off by, in 64 bits."""
    u = torch.finfo(q.dtype).eps / 2
    low = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    f = 2.0 ** -24
    T, H, D = q.shape
    group = H // k.shape[1]
    out = [torch.zeros(t.shape, dtype=torch.float64, device="cuda")
           for t in (q, q, k, v)]
    off = [torch.zeros_like(t) for t in out]
    for a, b in zip(ends[:-1], ends[1:]):
        L = b - a
        if L <= 0:
            continue
        for h in range(H):
            x = h // group
            qd, gd = q[a:b, h].double(), do[a:b, h].double()
            kd, vd = k[a:b, x].double(), v[a:b, x].double()
            s = scale * (qd @ kd.t())
            mag = scale * (qd.abs() @ kd.abs().t())
            if slopes is not None:
                i = torch.arange(L, device="cuda").double()
                bias = slopes[h].double() * (i[:, None] - i).abs()
                s, mag = s - bias, mag + bias
            p = torch.softmax(s, 1)
            # the exponent is held in base 2 next to the row's maximum
            e = f * (D + 8) * mag.amax() * 2 + 2.0 ** -21 + f * L
            o = p @ vd
            dp = gd @ vd.t()
            dl = (gd * o).sum(1, keepdim=True)
            ds = p * (dp - dl)
            o_off = (u + e) * (p @ vd.abs()) + low * vd.abs().sum(0) \
                + u * o.abs()
            dp_off = f * (D + 8) * (gd.abs() @ vd.abs().t()
                                    + (gd.abs() * o.abs()).sum(1, True)) \
                + (gd.abs() * o_off).sum(1, True)
            ds_off = (u + e) * ds.abs() + p * (1 + e) * dp_off + low
            p_off = (u + e) * p + low
            out[0][a:b, h] = o
            off[0][a:b, h] = o_off
            out[1][a:b, h] = scale * (ds @ kd)
            off[1][a:b, h] = scale * (ds_off @ kd.abs())
            out[2][a:b, x] += scale * (ds.t() @ qd)
            off[2][a:b, x] += scale * (ds_off.t() @ qd.abs())
            out[3][a:b, x] += p.t() @ gd
            off[3][a:b, x] += p_off.t() @ gd.abs()
            if h % group == group - 1:
                for n in (2, 3):
                    off[n][a:b, x] += (u + f * L * group) * out[n][a:b, x].abs()
            off[1][a:b, h] += (u + f * L) * out[1][a:b, h].abs()
    return out, [t * 1.01 + 1e-30 for t in off]


def _check(lengths, heads, kv, dim, dtype, front=0, back=0, bias=False,
           scale=None, size=1.0):
    F_amd = _f()
    ends = [front]
    for n in lengths:
        ends.append(ends[-1] + n)
    tokens = ends[-1] + back
    q, k, v, do = _inputs(tokens, heads, kv, dim, dtype, seed=tokens,
                          size=size)
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    slopes = _slopes(heads) if bias else None
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu, scale=scale, slopes=slopes)
    got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
    scale = dim ** -0.5 if scale is None else scale
    want, off = _reference(q.detach(), k.detach(), v.detach(), do, ends, scale,
                           slopes)
    for name, a, b, c in zip(("o", "dq", "dk", "dv"), got, want, off):
        bad = (a.double() - b).abs() / c
        bad = torch.where((a.double() == b), 0.0, bad)
        assert (bad <= 1).all(), (name, bad.max().item())
        # tokens in no document
        assert a[:front].eq(0).all() and a[tokens - back:].eq(0).all(), name
    return got


@pytest.mark.parametrize("lengths", [
    [1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [300],
    [1, 1, 1], [64, 64], [1, 63, 64, 65, 2], [0, 5, 0, 0, 70, 0],
    [200, 3, 129, 64, 1, 77]])
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths(lengths, dim):
    _check(lengths, 2, 2, dim, torch.bfloat16)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_widths_and_types(dim, dtype):
    _check([70, 130], 3, 3, dim, dtype, bias=True)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (6, 2), (12, 12),
                                      (16, 4)])
@pytest.mark.parametrize("dim", [64, 128])
def test_shared_heads(heads, kv, dim):
    _check([150, 20, 64], heads, kv, dim, torch.bfloat16, bias=True)


@pytest.mark.parametrize("front,back", [(1, 0), (0, 1), (70, 200), (129, 64)])
def test_tokens_in_no_document(front, back):
    _check([100, 28], 2, 1, 64, torch.bfloat16, front=front, back=back)


def test_no_document_at_all():
    _check([], 2, 2, 64, torch.bfloat16, front=90)
    _check([0, 0], 2, 2, 64, torch.bfloat16, back=10)


def test_many_documents():
    """More borders than one probe of a wave reaches (64, then 4096)."""
    g = torch.Generator().manual_seed(5)
    few = torch.randint(0, 12, (200,), generator=g).tolist()
    _check(few, 1, 1, 64, torch.bfloat16, front=3, back=5)
    many = torch.randint(0, 3, (5000,), generator=g)
    q, k, v, do = _inputs(int(many.sum()), 1, 1, 64, torch.bfloat16)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), many.cumsum(0)])
    cu = cu.int().cuda()
    o = _f().document_attention(q, k, v, cu)
    # one token: its own value; two: what the plain form says
    one = (many == 1).nonzero()[:, 0].cuda()
    at = cu.long()[one]
    assert torch.equal(o[at], v[at])
    two = cu.long()[(many == 2).nonzero()[:, 0].cuda()]
    s = [(q[two].double() * k[two + j].double()).sum(-1, True) / 8
         for j in (0, 1)]
    p = torch.softmax(torch.cat(s, -1), -1)
    want = p[..., :1] * v[two].double() + p[..., 1:] * v[two + 1].double()
    size = p[..., :1] * v[two].double().abs() \
        + p[..., 1:] * v[two + 1].double().abs()
    assert ((o[two].double() - want).abs() <= 2.0 ** -8 * 2.1 * size).all()


@pytest.mark.parametrize("bias", [False, True])
def test_long_documents(bias):
    _check([1500, 2100], 1, 1, 64, torch.bfloat16, bias=bias)
    _check([1300], 2, 1, 128, torch.float16, bias=bias)


def test_large_scores_and_scales():
    """Scores of thousands: a row is nearly one key."""
    _check([150], 2, 2, 64, torch.bfloat16, size=12.0)
    _check([150], 2, 2, 64, torch.bfloat16, scale=2.5)
    _check([150], 2, 2, 64, torch.bfloat16, scale=1e-4)


def test_nothing_passes_between_documents():
    """NaN and inf in one document leave the others' bits alone, and so does
    what padding holds."""
    F_amd = _f()
    q, k, v, do = _inputs(400, 2, 2, 64, torch.bfloat16)
    cu = torch.tensor([10, 75, 150, 339], dtype=torch.int32, device="cuda")

    def run():
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        o = F_amd.document_attention(*leaves, cu)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    clean = run()
    for t in (q, k, v, do):
        t[75:150] = float("nan")
        t[:10] = float("inf")
        t[339:] = float("nan")
    dirty = run()
    for a, b in zip(clean, dirty):
        assert torch.equal(a[10:75], b[10:75])
        assert torch.equal(a[150:339], b[150:339])
        assert b[:10].eq(0).all() and b[339:].eq(0).all()
        assert b[75:150].isnan().all()


def test_packed_projection_and_strides():
    """The packed entry, a slice of a wider buffer, rows of odd strides, and
    an expanded gradient all give the same bits."""
    F_amd = _f()
    T, H, D = 200, 3, 64
    cu = torch.tensor([0, 90, 200], device="cuda")
    wide = torch.randn(T, 3 * H * D + 64, device="cuda").bfloat16()
    qkv = wide[:, :3 * H * D].unflatten(1, (3, H, D)).requires_grad_(True)
    do = torch.randn(1, H, D, device="cuda").bfloat16().expand(T, H, D)
    o = F_amd.document_attention_qkv(qkv, cu)
    d, = torch.autograd.grad(o, [qkv], do)
    for make in (lambda t: t.contiguous(),
                 lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.cat([t, t[..., :3]], -1)[..., :D]):
        q, k, v = (make(t).detach().requires_grad_(True)
                   for t in qkv.detach().unbind(1))
        o2 = F_amd.document_attention(q, k, v, cu)
        d2 = torch.autograd.grad(o2, [q, k, v], do)
        assert torch.equal(o, o2)
        assert torch.equal(d, torch.stack(d2, 1))


def test_broadcast_keys():
    """Keys expanded over heads: the gradient is the sum over them."""
    F_amd = _f()
    q, _, v, do = _inputs(100, 4, 4, 64, torch.bfloat16)
    k1 = torch.randn(100, 1, 64, device="cuda").bfloat16().requires_grad_(True)
    cu = torch.tensor([0, 40, 100], device="cuda")
    o = F_amd.document_attention(q, k1.expand(100, 4, 64), v, cu)
    d, = torch.autograd.grad(o, [k1], do)
    k4 = k1.detach().expand(100, 4, 64).contiguous().requires_grad_(True)
    o4 = F_amd.document_attention(q, k4, v, cu)
    d4, = torch.autograd.grad(o4, [k4], do)
    want = d4.double().sum(1, True)
    # torch adds the four rounded gradients in fp32 or bf16 steps
    bound = 4 * 2.0 ** -8 * d4.double().abs().sum(1, True)
    assert ((d.double() - want).abs() <= bound).all()
    assert torch.equal(o, o4)


def test_same_bits_each_time():
    F_amd = _f()
    q, k, v, do = _inputs(3000, 4, 2, 64, torch.bfloat16)
    cu = torch.tensor([0, 700, 701, 3000], device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu)
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    for _ in range(3):
        assert torch.equal(o, F_amd.document_attention(*leaves, cu))
        for a, b in zip(first, torch.autograd.grad(o, leaves, do,
                                                   retain_graph=True)):
            assert torch.equal(a, b)


def test_borders_out_of_range_stay_inside():
    """Borders beyond the tokens are cut off at them."""
    F_amd = _f()
    q, k, v, _ = _inputs(100, 1, 1, 64, torch.bfloat16)
    cu = torch.tensor([-5, 50, 400], device="cuda", dtype=torch.int32)
    want = torch.tensor([0, 50, 100], device="cuda", dtype=torch.int32)
    assert torch.equal(F_amd.document_attention(q, k, v, cu),
                       F_amd.document_attention(q, k, v, want))


def test_gradient_against_differences():
    """A directional derivative of sum(o * c) from the fp64 formula's own
    differences agrees with the kernel's gradient."""
    F_amd = _f()
    T, D = 40, 64
    q, k, v, c = _inputs(T, 1, 1, D, torch.bfloat16, size=0.5)
    cu = torch.tensor([0, 17, 40], device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu, slopes=_slopes(1))
    got = torch.autograd.grad(o, leaves, c)

    def loss(qq, kk, vv):
        total = 0.0
        for a, b in ((0, 17), (17, 40)):
            i = torch.arange(b - a, device="cuda").double()
            s = qq[a:b, 0] @ kk[a:b, 0].t() / 8 \
                - _slopes(1).double() * (i[:, None] - i).abs()
            total = total + ((torch.softmax(s, 1) @ vv[a:b, 0])
                             * c[a:b, 0].double()).sum()
        return total

    base = [t.detach().double() for t in (q, k, v)]
    for n in range(3):
        d = torch.randn(base[n].shape, device="cuda", dtype=torch.float64)
        h = 1e-4
        up, down = list(base), list(base)
        up[n], down[n] = base[n] + h * d, base[n] - h * d
        diff = (loss(*up) - loss(*down)) / (2 * h)
        # each element of the gradient is off by a few roundings of 2^-8 of
        # the terms it sums; 2^-5 of the sum of sizes is over all of them
        room = 2.0 ** -5 * (got[n].double().abs() * d.abs()).sum() \
            / (T * D) ** 0.5 * 8
        assert (diff - (got[n].double() * d).sum()).abs() <= room


def test_captured_and_replayed():
    F_amd = _f()
    q, k, v, do = _inputs(700, 4, 2, 64, torch.bfloat16)
    cu = torch.tensor([0, 300, 650, 700], device="cuda", dtype=torch.int32)
    slopes = _slopes(4)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        o = F_amd.document_attention(*leaves, cu, slopes=slopes)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for ends in ([0, 1, 2, 700], [5, 600, 600, 610], [0, 300, 650, 700]):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_on_another_stream():
    F_amd = _f()
    q, k, v, do = _inputs(2000, 4, 4, 64, torch.bfloat16)
    cu = torch.tensor([0, 900, 2000], device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def run():
        o = F_amd.document_attention(*leaves, cu)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_extreme_scales():
    """Close to the borders of what scale may be, all stays finite and right:
    the mean of the values, and the value of the best key."""
    F_amd = _f()
    q, k, v, do = _inputs(60, 1, 1, 64, torch.bfloat16)
    cu = torch.tensor([0, 60], device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu, scale=1e-30)
    mean = v.double().mean(0, keepdim=True)
    size = v.double().abs().mean(0, keepdim=True)
    assert ((o.double() - mean).abs() <= 2.0 ** -7 * size).all()
    for g in torch.autograd.grad(o, leaves, do):
        assert g.isfinite().all()
    o = F_amd.document_attention(*leaves, cu, scale=1e5)
    best = (q[:, 0].double() @ k[:, 0].double().t()).argmax(1)
    # the best key's exponent is its score less the row's rounded one, up to
    # 2^22 * 2^-24 apart: its p is near 1, not 1, and is rounded (2^-8) before
    # it is divided by itself; the result is rounded again (2^-8)
    assert ((o.double() - v[best].double()).abs()
            <= 2.0 ** -7 * 1.01 * v[best].double().abs()).all()


def test_no_heads_and_no_tokens():
    F_amd = _f()
    cu = torch.tensor([0, 0], device="cuda", dtype=torch.int32)
    q = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16,
                    requires_grad=True)
    o = F_amd.document_attention(q, q, q, cu)
    assert o.shape == (0, 2, 64)
    d, = torch.autograd.grad(o, [q], torch.empty_like(o))
    assert d.shape == q.shape


def test_large_borders_in_int64():
    """Borders past 32 bits are cut off at the tokens like any other."""
    F_amd = _f()
    q, k, v, _ = _inputs(100, 1, 1, 64, torch.bfloat16)
    cu = torch.tensor([-2 ** 40, 50, 2 ** 32 + 7], device="cuda")
    want = torch.tensor([0, 50, 100], device="cuda", dtype=torch.int32)
    assert torch.equal(F_amd.document_attention(q, k, v, cu),
                       F_amd.document_attention(q, k, v, want))


def test_what_the_graph_refuses():
    """A graph of the gradients, and inputs changed before their use."""
    F_amd = _f()
    q, k, v, do = _inputs(50, 1, 1, 64, torch.bfloat16)
    cu = torch.tensor([0, 20, 50], device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = F_amd.document_attention(*leaves, cu)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(o, leaves, do, create_graph=True)
    o = F_amd.document_attention(*leaves, cu)
    cu[1] = 30
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o, leaves, do)


def test_only_some_gradients():
    F_amd = _f()
    q, k, v, do = _inputs(50, 2, 1, 64, torch.bfloat16)
    cu = torch.tensor([0, 20, 50], device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(F_amd.document_attention(*leaves, cu), leaves,
                               do)
    for n in range(3):
        some = [t.detach().requires_grad_(i == n)
                for i, t in enumerate(leaves)]
        got, = torch.autograd.grad(F_amd.document_attention(*some, cu),
                                   [some[n]], do)
        assert torch.equal(got, want[n])
    with torch.no_grad():
        o = F_amd.document_attention(*leaves, cu)
    assert not o.requires_grad
    with torch.inference_mode():
        assert torch.equal(F_amd.document_attention(*leaves, cu), o)


def test_two_calls_at_once():
    """Two streams, and two captured graphs replayed side by side."""
    F_amd = _f()
    sets = []
    for seed in (1, 2):
        q, k, v, do = _inputs(1500, 4, 1, 128, torch.bfloat16, seed)
        sets.append(([t.requires_grad_(True) for t in (q, k, v)], do))
    cu = torch.tensor([0, 700, 1500], device="cuda", dtype=torch.int32)

    def step(n):
        leaves, do = sets[n]
        o = F_amd.document_attention(*leaves, cu)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for n, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(step(n))
    torch.cuda.synchronize()
    graphs = []
    for n in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(n)
        graphs.append((g, out))
    for _ in range(3):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for n in range(2):
        for a, b, c in zip(want[n], got[n], graphs[n][1]):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2)])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("lengths", [
    [2], [1, 2, 2, 1], [3, 9, 1, 5], [17, 2, 30], [64, 63], [65, 200, 7],
    [33] * 40])
def test_short_documents_round_once(lengths, dim, heads, kv, dtype):
    """Few terms even nothing out, so P and dS keep twice the type's bits: a
    term is off by u^2, the terms' sizes add up to at most 16 times the
    result's (sqrt(n) for n terms of random sign, n <= 200), and fp16's
    subnormals leave 2^-25 of a p where typical ones are 2^-6 or more.  What
    is left is the rounding of the result."""
    more = 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -15
    for seed in range(4):
        q, k, v, do = _inputs(sum(lengths), heads, kv, dim, dtype, seed=seed)
        ends = [0]
        for n in lengths:
            ends.append(ends[-1] + n)
        cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
        for t in (q, k, v):
            t.requires_grad_(True)
        y = _f().document_attention(q, k, v, cu)
        got = [y, *torch.autograd.grad(y, [q, k, v], do)]
        with torch.no_grad():
            want = _reference(q, k, v, do, ends, dim ** -0.5, None)[0]
            for g, w in zip(got, want):
                size = w.norm()
                least = (w.to(dtype).double() - w).norm()
                assert (g.double() - w).norm() <= least + more * size


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_single_tokens_have_no_gradient_of_scores(heads, kv, dim):
    """Of one score the softmax is 1, whatever q and k are."""
    q, k, v, do = _inputs(100, heads, kv, dim, torch.bfloat16)
    cu = torch.arange(101, dtype=torch.int32, device="cuda")
    for t in (q, k, v):
        t.requires_grad_(True)
    y = _f().document_attention(q, k, v, cu)
    dq, dk, dv = torch.autograd.grad(y, [q, k, v], do)
    group = heads // kv
    assert (y == v.repeat_interleave(group, 1)).all()
    assert not dq.any() and not dk.any()
    want = do.double().unflatten(1, (kv, group)).sum(2)
    assert ((dv.double() - want).abs()
            <= want.abs() * 2.0 ** -8 + 2.0 ** -20 * group).all()


def test_refusals_on_the_device():
    """The same errors as on the CPU."""
    F_amd = _f()
    q, k, v, _ = _inputs(10, 4, 2, 64, torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    s = _slopes(4)
    for args, kw in (
            ((q, k[:5], v, cu), {}), ((q, k, v[..., :32], cu), {}),
            ((q, k.half(), v, cu), {}), ((q, k, v, cu.float()), {}),
            ((q, k, v, cu[None]), {}), ((q, k, v, cu[:0]), {}),
            ((q, k, v, cu.cpu()), {}), ((q[:, :3], k, v, cu), {}),
            ((q, k, v, cu), {"scale": 0.0}),
            ((q, k, v, cu), {"scale": float("nan")}),
            ((q, k, v, cu), {"slopes": s[:3]}),
            ((q, k, v, cu), {"slopes": s.cpu()}),
            ((q, k, v, cu), {"slopes": s.clone().requires_grad_(True)})):
        with pytest.raises(ValueError, match="document_attention"):
            F_amd.document_attention(*args, **kw)
    with pytest.raises(ValueError, match="document_attention_qkv"):
        F_amd.document_attention_qkv(torch.stack([q, q], 1), cu)


def test_borders_and_slopes_of_other_types():
    F_amd = _f()
    q, k, v, _ = _inputs(30, 4, 2, 64, torch.bfloat16)
    ends = [0, 7, 30]
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    s = _slopes(4)
    want = F_amd.document_attention(q, k, v, cu, slopes=s)
    wide = torch.tensor([[0, 1], [7, 1], [2 ** 40, 1]], device="cuda")[:, 0]
    got = F_amd.document_attention(q, k, v, wide, slopes=s.double())
    assert torch.equal(got, want)
