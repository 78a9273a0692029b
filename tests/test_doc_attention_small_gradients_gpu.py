"""fp16 gradients of document attention whose dS or P leave fp16's normal
numbers (doc_attention.hip).

dS and P are rounded to 2^-11 of each; the terms of a gradient have random
signs, so that leaves as much of it as rounding the result does: the error is
sqrt(2) times that of the rounded exact gradient (`least`, which counts the
result's own subnormals).  A bound of 1.6 leaves an eighth for fluctuation; up
to 64 tokens, and in calls of up to 1024, dS has twice the bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _gradients(q, k, v, do, cu, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = _f().document_attention(*leaves, cu, **kw)
    return torch.autograd.grad(o, leaves, do)


def _exact(q, k, v, do, ends):
    """dq, dk, dv in 64 bits."""
    q, k, v = (t.double().requires_grad_(True) for t in (q, k, v))
    at = torch.arange(q.shape[1], device="cuda") // (q.shape[1] // k.shape[1])
    total = 0.0
    for a, b in zip(ends[:-1], ends[1:]):
        s = torch.bmm(q[a:b].transpose(0, 1).contiguous(),
                      k[a:b][:, at].permute(1, 2, 0).contiguous())
        p = torch.softmax(s * q.shape[-1] ** -0.5, -1)
        o = torch.bmm(p, v[a:b][:, at].transpose(0, 1).contiguous())
        total = total + (o * do[a:b].double().transpose(0, 1)).sum()
    return torch.autograd.grad(total, (q, k, v))


def _inputs(tokens, heads, kv, dim, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(tokens, h, dim, generator=g, device="cuda").half()
            for h in (heads, kv, kv, heads)]


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (4, 1, 64), (2, 2, 128),
                                          (4, 1, 128)])
@pytest.mark.parametrize("ends", [[0, 60], [0, 1000], [0, 1100, 4000],
                                  [0, 50, 350, 1500]])
def test_small_gradients(ends, heads, kv, dim, size):
    q, k, v, do = _inputs(ends[-1], heads, kv, dim)
    do = (do.float() * size).half()
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    got = _gradients(q, k, v, do, cu)
    for name, a, w in zip(("dq", "dk", "dv"), got,
                          _exact(q, k, v, do, ends)):
        least = (w.half().double() - w).norm()
        off = (a.double() - w).norm()
        assert off <= 1.6 * least, (name, (off / least).item())


def test_gradients_of_many_sizes():
    """Rows and documents of sizes 1 to 1e-4 side by side, each by itself, and
    rows without any: a query's dS do not hang on another's."""
    ends = [0, 700, 1400, 3000]
    q, k, v, do = _inputs(3000, 2, 2, 64, seed=1)
    size = torch.logspace(0, -4, 5, device="cuda")[torch.arange(
        3000, device="cuda") % 5]
    size[700:1400] *= 0.03
    size[1400:1500] = 0
    do = (do.float() * size[:, None, None]).half()
    cu = torch.tensor(ends, dtype=torch.int32, device="cuda")
    got = _gradients(q, k, v, do, cu)
    want = _exact(q, k, v, do, ends)
    assert got[0][1400:1500].eq(0).all()
    for n in range(5):
        for a, b in zip(ends[:-1], ends[1:]):
            rows = torch.arange(a, b, device="cuda")
            rows = rows[(rows % 5 == n) & (size[rows] > 0)]
            w = want[0][rows]
            least = (w.half().double() - w).norm()
            assert (got[0][rows].double() - w).norm() <= 1.6 * least, (n, a)
    for x, w in zip(got[1:], want[1:]):
        for a, b in zip(ends[:-1], ends[1:]):
            least = (w[a:b].half().double() - w[a:b]).norm()
            assert (x[a:b].double() - w[a:b]).norm() <= 1.6 * least


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [50, 2000])
def test_gradients_that_do_not_fit(length, dim):
    """A dS past fp16's largest number, in gradients that are not.  Here q and
    k are so small that a row's p agree to four digits and round alike, so
    their rounding does not even out in dv: up to 2^-11 of it."""
    q, k, v, do = _inputs(length, 2, 2, dim, seed=2)
    q, k = q * 0.01, k * 0.01
    v, do = v * 200, do * 1500
    cu = torch.tensor([0, length], dtype=torch.int32, device="cuda")
    want = _exact(q, k, v, do, [0, length])
    assert max(w.abs().max() for w in want) < 60000
    for a, w, alike in zip(_gradients(q, k, v, do, cu), want,
                           (0, 0, 2.0 ** -11)):
        least = (w.half().double() - w).norm()
        assert (a.double() - w).norm() <= 1.6 * least + alike * w.norm()


def test_nan_stays_in_its_query():
    """NaN and infinity in a row of do reach that row's dq and the document's
    dk and dv, no other row's dq."""
    q, k, v, do = _inputs(2000, 2, 2, 64, seed=3)
    do[5], do[70] = float("nan"), float("inf")
    cu = torch.tensor([0, 1500, 2000], dtype=torch.int32, device="cuda")
    dq, dk, dv = _gradients(q, k, v, do, cu)
    bad = torch.zeros(2000, dtype=torch.bool, device="cuda")
    bad[5] = bad[70] = True
    assert dq[~bad].isfinite().all() and not dq[bad].isfinite().any()
    for d in (dk, dv):
        assert d[:1500].isnan().all() and d[1500:].isfinite().all()
    clean = do.clone()
    clean[bad] = 0
    assert torch.equal(_gradients(q, k, v, clean, cu)[0][~bad], dq[~bad])


def test_many_tokens_of_equal_weight():
    """p = 1 / 60000 is a subnormal number of fp16 that is off by 2^-9.5 of
    itself; dv is the mean of do.  P and the result are rounded, 2^-11 each,
    and 60000 fp32 sums of terms of one sign leave under 2^-12."""
    n = 60000
    g = torch.Generator(device="cuda").manual_seed(0)
    do = torch.rand(n, 1, 64, generator=g, device="cuda").half()
    z = torch.zeros(n, 1, 64, device="cuda", dtype=torch.half)
    v = torch.randn(n, 1, 64, generator=g, device="cuda").half()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    dv = _gradients(z, z, v, do, cu)[2]
    want = do.double().mean(0, keepdim=True)
    assert ((dv.double() - want).abs() <= (2 * 2.0 ** -11 + 2.0 ** -12)
            * want).all()
