"""Newton-Schulz of matrices whose norm is 0, or at fp32's ends."""

import pytest
import torch

from deeplearning_cfn_amd.ops import functional as F_amd

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# one launch, one launch of 128 rows, thin, tiles
SIZES = [(4, 6), (100, 200), (40, 300), (150, 260)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,m", SIZES)
@pytest.mark.parametrize("eps", [0.0, 1e-300, 1e-7])
def test_zero_stays_zero(n, m, eps, device):
    g = torch.randn(3, n, m, generator=torch.Generator().manual_seed(0))
    g[1] = 0
    g = g.to(device)
    y = F_amd.newton_schulz(g, eps=eps)
    assert y[1].eq(0).all()
    assert y[0].isfinite().all() and y[2].isfinite().all()
    assert F_amd.newton_schulz(g.mT, eps=eps)[1].eq(0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,m", SIZES)
@pytest.mark.parametrize("exp", [-136, -126, -110, 0, 100, 124])
def test_the_result_does_not_hang_on_the_size(n, m, exp, device):
    """Without eps a power of two changes no rounding: the same bits, as long
    as no entry of G loses its own (entries are whole multiples of 2^-12 up
    to 4, so that 2^-136 times them are still numbers of fp32)."""
    g = torch.randn(2, n, m, generator=torch.Generator().manual_seed(n))
    g = (g.clamp(-3.5, 3.5) * 2 ** 12).round() * 2.0 ** -12
    small = (g.double() * 2.0 ** exp).float()
    assert torch.equal(small.double(), g.double() * 2.0 ** exp)
    want = F_amd.newton_schulz(g.to(device), eps=0.0)
    assert want.isfinite().all() and want.ne(0).any()
    assert torch.equal(F_amd.newton_schulz(small.to(device), eps=0.0), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,m", SIZES)
def test_small_eps(n, m, device):
    """An eps under fp32's numbers still counts: with eps the norm itself X_0
    is half of what it is without."""
    g = torch.zeros(1, n, m)
    g[0, 0, 0] = 2.0 ** -149
    y = F_amd.newton_schulz(g.to(device), steps=1, eps=2.0 ** -149).cpu()
    # one step on a single singular value of 1/2; bf16 rounds the result, and
    # fp16 operands round A and B, each 2^-11 of numbers under 3.5: under 2e-3
    want = 3.4445 / 2 - 4.7750 / 8 + 2.0315 / 32
    assert (y[0, 0, 0].double() - want).abs() <= 2.0 ** -8 * want + 2e-3
    assert y.flatten()[1:].eq(0).all()
