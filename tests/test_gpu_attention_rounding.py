"""What attention rounds, by form: the sums of calls with few rows are those of the probabilities as they are, and fp16 keeps small
probabilities of many keys."""

import math

import pytest
import torch

from conftest import announce
from oracle import w8a8 as ow

pytestmark = pytest.mark.gpu
U32 = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16]


def tight_bound(q, k, v, valid, columns_of_ones):
    """The result in 64 bits and how far off it may be.  As in the tests of all shapes: probabilities rounded for the product (u), scores' and
    exponentials' errors e and fp32 sums in both sides of the division, the result rounded.  fp16: the largest probability in use is at
    least 2^7, so what a probability loses at the type's end, 2^-25, is n 2^-32 max |v| of the result; the result itself 2^-25.  With
    the sum made of the rounded probabilities, u |exact| and what they lose once more."""
    dtype, D, n = q.dtype, q.shape[-1], k.shape[1]
    u, s = torch.finfo(dtype).eps / 2, 1 / math.sqrt(D)
    want, A = ow.cross_attention(q, k, v, valid), ow.cross_attention(q, k, v.abs(), valid)
    e = (D + 8) * U32 * s * (q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()).item() + 16 * U32
    bound = 1.01 * (A * (u + 2 * e + 2 * n * U32) + (2 if columns_of_ones else 1) * u * want.abs())
    if dtype == torch.float16:
        bound = bound + 2.0**-25 + 1.01 * (2 if columns_of_ones else 1) * n * 2.0**-32 * v.double().abs().max()
    return want, bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 8), (2, 1, 63, 2, 1, 16), (3, 1, 65, 8, 2, 40), (1, 2, 513, 6, 3, 72), (2, 7, 257, 4, 4, 88), (1, 1, 3000, 4, 1, 120), (2, 5, 1000, 4, 2, 104),
                                   (2, 1, 4097, 4, 2, 128), (1, 16, 700, 4, 2, 64)])
def test_few_rows_sum_in_32_bits(dev, shape, dtype):
    """Up to 32 rows: the sum is that of the probabilities as they are, also where heads do not end on a multiple of 32."""
    from nunchaku_amd.ops import cross_attention

    announce(f"few rows {shape} {dtype}")
    B, Tq, Tk, H, Hkv, D = shape
    g = torch.Generator().manual_seed(sum(shape))
    q, k, v = ((f * torch.randn(B, T, n, D, generator=g)).to(dtype) for f, T, n in ((1.5, Tq, H), (1, Tk, Hkv), (1, Tk, Hkv)))
    valid = torch.arange(Tk) < torch.tensor([Tk, max(1, Tk // 2), 1][:B])[:, None]
    for kind in (None, valid):
        got = cross_attention(q.to(dev), k.to(dev), v.to(dev), key_lengths=None if kind is None else valid.sum(1).to(torch.int32).to(dev))
        want, bound = tight_bound(q, k, v, kind, False)
        off = (got.cpu().double() - want).abs() - bound
        assert (off <= 0).all(), (off.max().item(), (off > 0).sum().item())


@pytest.mark.parametrize("gap", [17.5, 19.0])
@pytest.mark.parametrize("D", [16, 64])
@pytest.mark.parametrize("form", ["few rows", "many rows"])
def test_many_small_probabilities_in_fp16(dev, form, D, gap):
    """One key ``gap`` above 65535 others, e^gap times as likely as each: together they are 1.6e-3 (3.7e-4) of the result.  V is zero at
    the one key and one at the others, so the result is their share.  Batch entries, or rows, are as many as keep the keys in one part."""
    from nunchaku_amd.ops import cross_attention

    announce(f"small probabilities {form} {D} {gap}")
    Tk = 65536
    B, Tq, H = (64, 1, 8) if form == "few rows" else (1, 65536, 1)
    q = torch.zeros(B, Tq, H, D, dtype=torch.float16, device=dev)
    q[..., 0] = 1.0
    k, v = torch.zeros(1, Tk, H, D, dtype=torch.float16, device=dev), torch.ones(1, Tk, H, D, dtype=torch.float16, device=dev)
    k[:, 0, :, 0] = gap
    v[:, 0] = 0.0
    got = cross_attention(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), scale=1.0).double()
    rest = (Tk - 1) * math.exp(-gap)
    want = rest / (1.0 + rest)
    u = 2.0**-11
    e = (D + 8) * U32 * gap + 16 * U32
    twice = 2 if form == "many rows" and D % 32 else 1
    bound = 1.01 * want * (u + 2 * e + 2 * Tk * U32 + twice * u) + 2.0**-25 + 1.01 * twice * Tk * 2.0**-32
    assert ((got - want).abs() <= bound).all(), (got.min().item(), got.max().item(), want, bound)
