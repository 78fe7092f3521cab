"""RMS norm to 8-bit codes with an eps that does not hold the mean of squares up: rows whose squares are below what fp32 holds."""

import math

import pytest
import torch

from conftest import announce
from oracle import w8a8 as ow

pytestmark = pytest.mark.gpu
U32 = 2.0**-24
# row lengths for every number of threads per row
LENGTHS = [16, 256, 272, 1024, 1040, 2048, 2064, 4096, 8192, 16384, 16400, 32768, 65536]


def rows(K, seed):
    """Rows of ordinary and of tiny numbers in turn (several share a wave where K is small), down to the smallest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(11, K, generator=g, dtype=torch.float64)
    size = [1.0, 1e-24, 1e-20, 1e-30, 1.0, 2.0**-50, 2.0**-51, 2.0**-64, 2.0**-75, 0.0, 1.0]
    x *= torch.tensor(size, dtype=torch.float64)[:, None]
    x[3, ::2] *= 1e5
    x = x.to(torch.bfloat16)
    x[8] = 2.0**-133  # the smallest number there is
    return x


@pytest.mark.parametrize("eps", [0.0, 2.0**-149, 2.0**-132, 2.0**-101, 2.0**-100, 1e-6])
@pytest.mark.parametrize("K", LENGTHS)
def test_rows_whose_squares_vanish(dev, K, eps):
    """Scales as the formula has them, within what a sum of squares and seven more operations round (52 U32: 64 + 22 additions at U32
    each, halved by the root); codes bit for bit.  A row of zeros with eps = 0 is 2^-100 / 0."""
    from nunchaku_amd.ops import rms_norm_quantize_w8a8

    x = rows(K, K)
    w = (1 + torch.randn(K, generator=torch.Generator().manual_seed(3)) / 4).to(torch.bfloat16)
    for r in (None, x.flip(0).contiguous()):
        announce(f"tiny rows {K} eps {eps} residual {r is not None}")
        codes, scales, h = rms_norm_quantize_w8a8(x.to(dev), w.to(dev), None if r is None else r.to(dev), eps=eps)
        want_codes, want, want_h = ow.rms_norm_quantize(x, w, r, eps)
        assert torch.equal(codes.cpu(), want_codes)
        assert r is None or torch.equal(h.cpu(), want_h)
        got = scales.cpu().double()
        fine = torch.isfinite(want)
        assert fine.sum() >= 10 and torch.equal(got[~fine], want[~fine])
        assert ((got - want).abs()[fine] <= 52 * U32 * want[fine]).all(), ((got - want).abs()[fine] / want[fine]).max()


def test_large_and_tiny_weights(dev):
    """A weight near the type's ends behind a row of tiny numbers: the scale is the formula's, or infinite where fp32 ends."""
    from nunchaku_amd.ops import rms_norm_quantize_w8a8

    K = 256
    g = torch.Generator().manual_seed(5)
    for size in (1e-24, 2.0**-60, 2.0**-51):
        for weight in (2.0**120, 2.0**64, 2.0**-45, 2.0**-90):
            announce(f"tiny rows {size} weight {weight}")
            x, w = (size * torch.randn(3, K, generator=g)).to(torch.bfloat16), (weight * (1 + torch.rand(K, generator=g) / 2)).to(torch.bfloat16)
            codes, scales, _ = rms_norm_quantize_w8a8(x.to(dev), w.to(dev), eps=0.0)
            want_codes, want, _ = ow.rms_norm_quantize(x, w, None, 0.0)
            assert torch.equal(codes.cpu(), want_codes)
            assert math.isfinite(want.max()) and want.max() < 2.0**127
            assert ((scales.cpu().double() - want).abs() <= 52 * U32 * want).all()
