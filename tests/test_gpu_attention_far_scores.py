"""Attention whose scores are so large that neighbouring fp32 numbers lie 8 or 16 apart in units of log2, where the exponentials' reference is a
rounded number.

q = (30000, 8, 0 ...), k = (30000, 8 j, 0 ...): 9e8 + 64 j, exact in fp32 (9e8 is a multiple of 256, the sum below 64 * 2^24).  Times the scale, j and
j + 1 lie 6.7 to 13 apart; the keys of step j hold it, so that the highest score rises from step to step.  V has a column for each j."""

import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu
U32 = 2.0**-24


@pytest.mark.parametrize("descending", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("Tq", [1, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_around_1e8(dev, dtype, Tq, sign, descending):
    """Scale and score are rounded to fp32 once (2 U32 of what lies between two scores, at most 15 * 13; the common part cancels), the
    exponential is within 16 U32, probability and result are rounded (u each), sums of 960 add 960 U32 each.  The rounded reference may be 8 above the
    highest score, which 64 keys have, so the sum is at least 64 * 2^-8 = 1 / 4; what a probability loses at its type's end (2^-25 in fp16, 2^-126
    in fp32's normal numbers, which bf16 shares) counts four times, and the result loses as much once."""
    from nunchaku_amd.ops import cross_attention

    B, H, D, each, steps = 2, 4, 64, 64, 15
    first = 30000.0 if dtype == torch.float16 else 29952.0  # (bf16: 117 * 256, 8 bits)
    step = torch.arange(steps).repeat_interleave(each)
    j = (step.flip(0) if descending else step).double()
    k = torch.zeros(B, steps * each, H, D, dtype=torch.float64)
    k[..., 0], k[..., 1] = sign * first, 8 * j[None, :, None]
    v = torch.zeros(B, steps * each, H, D, dtype=torch.float64)
    v[:, torch.arange(steps * each), :, j.long()] = 1.0
    q = torch.zeros(B, Tq, H, D, dtype=torch.float64)
    q[..., 0], q[..., 1] = first, 8.0
    raw = sign * first * first + 64 * j
    assert torch.equal(raw.float().double(), raw) and all(torch.equal(t.to(dtype).double(), t) for t in (q, k, v))
    on = [t.to(dtype).to(dev) for t in (q, k, v)]
    for scale in (0.1, 0.105, 0.111, 0.12, 0.131, 0.15, 0.17, 0.19, 0.2):
        announce(f"far scores {dtype} {Tq} {sign} {descending} {scale}")
        got = cross_attention(*on, scale=scale).cpu().double()
        p = torch.softmax(raw * scale, 0)
        want = torch.zeros(D, dtype=torch.float64).index_add_(0, j.long(), p)
        u = torch.finfo(dtype).eps / 2
        bound = 1.01 * want * (2 * u + 2 * (2 * U32 * 15 * 13 + 16 * U32 + 960 * U32)) + (2.0**-25 if dtype == torch.float16 else 2.0**-126) * (1 + 4 * 960)
        assert ((got - want).abs() <= bound).all(), (scale, (got - want).abs().max().item())


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("Tq", [1, 200])
def test_bf16_scores_around_1e9(dev, Tq, sign):
    """Up to 1.39e9 a reference is up to 64 off its score, which bf16's range holds: the 64 keys of the highest step share the result (the next
    step is e^-32 of it and less), so each column of V is its value there, rounded: probabilities, sums, division and result as above."""
    from nunchaku_amd.ops import cross_attention

    B, H, D, each, steps = 1, 2, 64, 64, 9
    first = 29952.0
    j = torch.arange(steps).repeat_interleave(each)
    k = torch.zeros(B, steps * each, H, D, dtype=torch.float64)
    k[..., 0], k[..., 1] = sign * first, 8.0 * j[None, :, None]
    q = torch.zeros(B, Tq, H, D, dtype=torch.float64)
    q[..., 0], q[..., 1] = first, 8.0
    v = (1.0 + j.double())[None, :, None, None].expand(B, -1, H, D)
    on = [t.to(torch.bfloat16).to(dev) for t in (q, k, v)]
    for scale in (0.51, 0.6, 0.77, 0.9, 1.1, 1.3, 1.49, 1.55):
        announce(f"scores around 1e9 {Tq} {sign} {scale}")
        got = cross_attention(*on, scale=scale).cpu().double()
        bound = steps * (2 * 2.0**-8 + 64 * U32 + 2 * 576 * U32) * 1.01 + steps * math.exp(-32)
        assert ((got - steps).abs() <= bound).all(), (scale, got.min().item(), got.max().item())
