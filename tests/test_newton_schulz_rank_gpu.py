"""Newton-Schulz of matrices of few directions: a momentum of the first steps,
or of few tokens (newton_schulz.hip).

What is rounded in a direction without signal grows 3.4445 times a step, and
nothing else there does.  The rms of a relative rounding to p bits, over
mantissas as they come, is 0.2 * 2^(1 - p): 1.9e-4 for fp16 (p = 11), 0.025 of
that for e4m3's 4 bits of the rest, 1.5e-3 for the result's 8.  X_0 keeps 22
bits, X_1 to X_3 15, the last X 11, so the result holds 141 * 4.7e-6 = 6.7e-4
of X_1's loss, 1.9e-4 of X_2's, 6e-5 of X_3's and 3.44 * 1.9e-4 = 6.6e-4 of
the last one's; what A and B lose spreads over all rows and leaves 1 / sqrt(n)
of itself.  Together 9.7e-4; with as much again for mantissas that are not
spread so evenly (products of two short vectors), sqrt(1.5^2 + 1.94^2) / 1.5:
the result is off by 1.64 times what its own rounding costs."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _exact(g, steps=5):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = (x.mT if tall else x).contiguous()
    x = x / (x.square().sum((-1, -2), keepdim=True).sqrt() + 1e-7)
    for _ in range(steps):
        a = torch.bmm(x, x.mT.contiguous())
        x = 3.4445 * x + torch.bmm(-4.7750 * a + 2.0315 * torch.bmm(a, a), x)
    return x.mT if tall else x


def _check(g, steps=5):
    from deeplearning_cfn_amd.ops import functional as F_amd
    got = F_amd.newton_schulz(g, steps=steps)
    want = _exact(g, steps)
    least = (want.bfloat16().double() - want).flatten(-2).norm(dim=-1)
    off = (got.double() - want).flatten(-2).norm(dim=-1)
    assert (off <= 1.64 * least).all(), (off / least).max().item()


def _low(b, n, m, rank, noise=0.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return r(b, n, rank) @ r(b, rank, m) + noise * r(b, n, m)


@pytest.mark.parametrize("rank", [1, 4, 16, 64])
@pytest.mark.parametrize("b,n,m", [
    (2, 100, 400), (1, 768, 768), (2, 768, 2304), (2, 2304, 768),
    (2, 301, 701), (24, 512, 1100), (1, 1024, 4096)])
def test_few_directions(b, n, m, rank):
    """Tiles of 128 and 256, wide and tall."""
    _check(_low(b, n, m, rank))


@pytest.mark.parametrize("rank,noise", [(1, 1e-4), (1, 1e-2), (4, 1e-2)])
@pytest.mark.parametrize("n,m", [(768, 768), (300, 2500)])
def test_few_directions_and_noise(n, m, rank, noise):
    _check(_low(2, n, m, rank, noise))


@pytest.mark.parametrize("steps", [1, 2, 3, 4])
def test_fewer_steps(steps):
    """Each X's low part is read by the step it belongs to, from the first
    (alone the last one too, which has none) on."""
    _check(_low(2, 300, 500, 2), steps)


def test_transpose_and_batch():
    """The bits of a matrix do not hang on its side or its company."""
    from deeplearning_cfn_amd.ops import functional as F_amd
    g = _low(5, 300, 500, 3)
    y = F_amd.newton_schulz(g)
    assert torch.equal(F_amd.newton_schulz(g.mT), y.mT)
    assert torch.equal(F_amd.newton_schulz(g[3:4]), y[3:4])


@pytest.mark.parametrize("b,n,m", [
    (8, 768, 2304), (9, 768, 2304), (16, 1024, 1024), (17, 1024, 1024),
    (43, 768, 768), (56, 768, 768), (200, 256, 256), (43, 500, 500)])
def test_any_tile_gives_the_same_bits(b, n, m):
    """Batches on both sides of where the tiles change, of update and square:
    a matrix alone takes tiles of 128, and every tile adds in the order of k."""
    from deeplearning_cfn_amd.ops import functional as F_amd
    g = torch.randn(b, n, m, generator=torch.Generator(device="cuda")
                    .manual_seed(b), device="cuda")
    y = F_amd.newton_schulz(g)
    for k in (0, b // 2, b - 1):
        assert torch.equal(F_amd.newton_schulz(g[k]), y[k])
