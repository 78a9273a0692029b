"""Newton-Schulz orthogonalisation (newton_schulz.hip).

The result against 64 bits: a model of the kernel's roundings (fp16 operands,
fp32 sums, X in 15 bits) on the CPU, over four spectra and sizes from 64 to
1024, is off by 7e-4 to 2.9e-3; bf16's rounding of the result adds 1.7e-3
in the 2-norm.  Together at most 3.4e-3; a bound of 5.6e-3 leaves two
thirds of that for spectra that the model did not have.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BOUND = 5.6e-3


def _f():
    from deeplearning_cfn_amd.ops import functional
    return functional


def _exact(g, steps=5, eps=1e-7):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = (x.mT if tall else x).contiguous()
    x = x / (x.square().sum((-1, -2), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        a = x @ x.mT.contiguous()
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * a @ a) @ x
    return x.mT if tall else x


def _matrix(b, n, m, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    noise = torch.randn(b, n, m, generator=g, device="cuda")
    if kind == "flat":
        return noise
    r = min(n, m)
    k = torch.arange(1, r + 1, device="cuda").float()
    s = {"power": 1 / k, "steep": torch.exp(-8 * k / r),
         "low": torch.where(k < 9, 1.0, 1e-3)}[kind]
    u = torch.linalg.qr(torch.randn(b, n, r, generator=g, device="cuda"))[0]
    v = torch.linalg.qr(torch.randn(b, m, r, generator=g, device="cuda"))[0]
    return (u * s) @ v.mT.contiguous()


def _check(g, **kw):
    got = _f().newton_schulz(g, **kw)
    assert got.shape == g.shape and got.dtype == torch.bfloat16
    want = _exact(g, **kw)
    off = (got.double() - want).flatten(-2).norm(dim=-1)
    rel = off / want.flatten(-2).norm(dim=-1)
    assert (rel <= BOUND).all(), rel.max().item()


@pytest.mark.parametrize("n,m", [
    (1, 1), (1, 40), (40, 1), (2, 3), (17, 33), (64, 64), (64, 128),
    (127, 129), (128, 128), (129, 127), (200, 768), (768, 200), (333, 777),
    (768, 768), (100, 2500)])
def test_sizes(n, m):
    _check(_matrix(3, n, m, "flat"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,m", [
    (1, 5), (2, 2), (2, 9), (3, 3), (5, 6), (17, 9), (16, 16), (40, 64),
    (64, 200), (1, 300), (4, 400), (2100, 3), (40, 1000), (64, 257)])
def test_few_singular_values(n, m, dtype):
    """Up to 64 rows X, A and B have 22 bits.  Rounding the result costs at
    most 2^-8 of each element, so of the norm.  A step adds at most four
    roundings of 2^-22, and a step multiplies what is there already by at
    most |s p'(s) / p(s)| <= 5 for the s up to 1.21 that come up, so that
    five leave 4 * 2^-22 (1 + 5 + 25 + 125 + 625) = 7.5e-4."""
    g = _matrix(32, n, m, "flat", seed=3).to(dtype)
    want = _exact(g)
    off = (_f().newton_schulz(g).double() - want).flatten(-2).norm(dim=-1)
    rel = off / want.flatten(-2).norm(dim=-1)
    assert (rel <= 2 ** -8 + 7.5e-4).all(), rel.max().item()


@pytest.mark.parametrize("b,n,m", [
    (24, 512, 1100), (24, 1100, 512), (60, 500, 500), (23, 700, 768),
    (200, 130, 250)])
def test_many_matrices(b, n, m):
    """Enough of them for the larger tile, and next to that border."""
    _check(_matrix(b, n, m, "flat"))


@pytest.mark.parametrize("kind", ["flat", "power", "steep", "low"])
@pytest.mark.parametrize("n,m", [(64, 64), (256, 1024), (768, 512)])
def test_spectra(kind, n, m):
    _check(_matrix(2, n, m, kind))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("size", [1e-3, 1.0, 1e3])
def test_types_and_sizes_of_values(dtype, size):
    _check((_matrix(1, 96, 160, "power") * size).to(dtype))


def test_extreme_values():
    """Squares past fp32's range, and a matrix that eps dwarfs."""
    g = _matrix(1, 64, 96, "flat")
    want = _f().newton_schulz(g)
    # a power of two changes no rounding but that of eps
    for by in (2.0 ** 100, 2.0 ** 20):
        got = _f().newton_schulz(g * by)
        off = (got.double() - want.double()).norm() / want.double().norm()
        assert off <= 2 * BOUND
    small = _f().newton_schulz(g * 1e-12)
    assert small.isfinite().all()
    _check(g * 1e-9, eps=1e-7)


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 10])
def test_steps(steps):
    _check(_matrix(1, 150, 260, "power"), steps=steps)


def test_zero_matrix_and_no_matrix():
    F_amd = _f()
    g = _matrix(3, 50, 70, "flat")
    g[1] = 0
    y = F_amd.newton_schulz(g)
    assert y[1].eq(0).all()
    assert F_amd.newton_schulz(g[:0]).shape == (0, 50, 70)
    assert F_amd.newton_schulz(g[0]).shape == (50, 70)


def test_matrices_do_not_touch_each_other():
    """A batch gives the bits of its matrices alone, whatever its others."""
    F_amd = _f()
    g = _matrix(4, 200, 300, "power")
    alone = [F_amd.newton_schulz(g[i]) for i in range(4)]
    dirty = g.clone()
    dirty[2] = float("nan")
    y, z = F_amd.newton_schulz(g), F_amd.newton_schulz(dirty)
    for i in range(4):
        assert torch.equal(y[i], alone[i])
        if i != 2:
            assert torch.equal(z[i], alone[i])
    assert z[2].isnan().all()


def test_transpose():
    """A tall matrix gives the transposed bits of its transpose."""
    F_amd = _f()
    g = _matrix(2, 90, 210, "power")
    y = F_amd.newton_schulz(g)
    z = F_amd.newton_schulz(g.mT)          # a strided view
    assert torch.equal(y, z.mT)


def test_captured_and_replayed():
    F_amd = _f()
    g = _matrix(2, 130, 140, "power")
    F_amd.newton_schulz(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F_amd.newton_schulz(g)
    for seed in range(3):
        g.copy_(_matrix(2, 130, 140, "flat", seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, F_amd.newton_schulz(g))


def test_on_another_stream():
    F_amd = _f()
    g = _matrix(2, 256, 384, "flat")
    want = F_amd.newton_schulz(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F_amd.newton_schulz(g)
    s.synchronize()
    assert torch.equal(got, want)
