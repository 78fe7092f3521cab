"""Layer norms of rows whose mean is far above their spread, on the GPU against the oracle in 64 bits.

Tolerance.  U = 2^-24 (fp32's rounding), u = half a step of the type.  h: exact where it is the input, U |b| more for a gate, U |h| for a residual: dh.
A sum of K numbers is right to 55 U of their magnitudes' sum; a mean, with the reciprocal's rounding and the product's, to 58 U of their mean: e0 = 58 U
mean |h| for the first, m.  What it is off by is the mean of the deviations h - m, right to 58 U (mean |d| + e0), and taken out of each of them: one rounding of
h - m and one of the difference, U (|d| + e0) each, and one of the product with 1 / std, U e0.
    dd = dh + mean(dh) + 2 U |d| + 58 U mean |d| + 61 U e0.
The deviations' squares, 58 U, less the square of their mean, which is at most half of them (else 64 bits take over): with w = e0 / std, 0.72 at most, relative
to the variance without eps (59 + 116 w + 3 w^2) U / (1 - w^2), half of that to the root, 5 U more for eps and the root, 8 U for the factors:
    |factor| (dd + |d| (rms(dd) / std + root + 8 U)) / std + U |y| + u |y|,
times 1.01 for the products of errors, and half the smallest step where the types end."""

import pytest
import torch

from conftest import announce
from oracle import blocks

pytestmark = pytest.mark.gpu
U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16]


def check(got, x, residual=None, eps=1e-6, **kw):
    y, h, parts = blocks.gated_norm(x, residual, "layer", eps=eps, **kw)
    u, end = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    b, d, std, factor = (parts[n] for n in ("b", "d", "std", "factor"))
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dh = U * (b.abs() * ("gate" in kw) + h.abs() * (residual is not None))
    e0 = 58 * U * mean(h.abs())
    dd = dh + mean(dh) + 2 * U * d.abs() + 58 * U * mean(d.abs()) + 61 * U * e0
    var = mean(d.square())
    w = (e0 / var.sqrt()).nan_to_num(0.72).clamp(max=0.72)  # (rows of zeros)
    root = 0.5 * U * (59 + 116 * w + 3 * w * w) / (1 - w * w) * var / (var + eps) + 5 * U
    bound = 1.01 * (factor.abs() * (dd + d.abs() * (mean(dd.square()).sqrt() / std + root + 8 * U)) / std + (U + u) * y.abs()) + end
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.cpu().double() - y).abs() - bound
    assert (off <= 0).all(), (off.max().item(), (off > 0).sum().item(), off.numel(), off.argmax().item() // x.shape[-1])


# one wave to a row and several, one, two and four pieces a thread; most are no powers of two and have reciprocals that are rounded
SIZES = [24, 328, 896, 1000, 1792, 3584, 4096, 7168, 9000, 21504, 32768]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", SIZES)
def test_constant_rows(dev, K, dtype):
    """All channels alike: nothing is left of them but the shift."""
    from nunchaku_amd.ops import gated_norm

    announce(f"gated_norm constant rows {K} {dtype}")
    x = torch.tensor([1000.0, 30000.0, -7.3, 0.001, -65000.0, 1.0, 0.0])[:, None].expand(-1, K).to(dtype).contiguous()
    g = torch.Generator().manual_seed(K)
    weight, scale, shift = ((0.5 * torch.randn(K, generator=g)).to(dtype) for _ in range(3))
    check(gated_norm(x.to(dev), norm="layer")[0], x)
    check(gated_norm(x.to(dev), norm="layer", weight=weight.to(dev), scale=scale.to(dev), shift=shift.to(dev))[0], x, weight=weight, scale=scale, shift=shift)
    # within a step of the shift
    step = torch.finfo(dtype).eps
    y = gated_norm(x.to(dev), norm="layer", shift=shift.to(dev))[0].cpu().float()
    assert ((y - shift.float()).abs() <= step * shift.float().abs() + 0.001).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", SIZES)
def test_small_spread_around_a_large_mean(dev, K, dtype):
    """Some channels a step or two above the others; a residual that is far from zero, with a small branch on it; one channel alone that differs."""
    from nunchaku_amd.ops import gated_norm

    announce(f"gated_norm small spread {K} {dtype}")
    g = torch.Generator().manual_seed(K + 1)
    base = torch.tensor([1000.0, 30000.0, -7.0, 100.0, -60000.0])[:, None].to(dtype).float()
    steps = torch.randint(0, 3, (5, K), generator=g).float()
    steps[3] = 0.0
    steps[3, K // 2] = 1.0
    x = (base * (1 + steps * torch.finfo(dtype).eps)).to(dtype)
    for n in (1000.0, 300.0, 17.0):
        check(gated_norm(x.to(dev), norm="layer")[0], x)
        small = (0.03 * torch.randn(5, K, generator=g)).to(dtype)
        gate = torch.randn(K, generator=g).to(dtype)
        far = torch.full((5, K), n).to(dtype)
        got = gated_norm(small.to(dev), far.to(dev), "layer", gate=gate.to(dev), residual_scale=0.75)
        check(got[0], small, far, gate=gate, residual_scale=0.75)
