"""Attention of few queries to many keys: every valid key counts once, whichever part, wave or step it falls to.

Among thousands of keys of random scores one key is worth less than a rounding of the result.  Here all scores are equal and V is zero but for
one key in each column, so a column's result is that key's value over the number of valid keys: zero if the key is lost, twice as much if
it is counted twice.  The columns of all heads together go over every key.

Tolerance there: probabilities are equal (each within 16 U32 of the exponential and u where it is rounded), the sum of n of them in fp32
adds n U32, the division and the result round once more: value / n * (2 u + 32 U32 + 2 n U32), times 1.01 for the products of errors."""

import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu
U32 = 2.0**-24
VALUE = 4096.0
DTYPES = [torch.bfloat16, torch.float16]
# single tokens and a few, in one part and in many; the last three are blocks of 128 rows whose keys are in parts
SHAPES = [
    (2, 1, 4097, 4, 2, 128), (1, 1, 1000, 5, 1, 64), (8, 1, 4096, 32, 8, 128), (3, 1, 5000, 6, 3, 72), (2, 3, 3001, 8, 2, 40), (1, 1, 20011, 2, 2, 128),
    (2, 1, 700, 4, 4, 80), (5, 2, 2111, 16, 16, 24), (1, 100, 5000, 2, 2, 120), (2, 45, 3001, 3, 1, 128), (2, 90, 1999, 4, 4, 96),
]


def validity(kind, B, Tk):
    """bool [B, Tk]: which keys count"""
    if kind == "all":
        return torch.ones(B, Tk, dtype=torch.bool)
    if kind == "mask":
        keep = torch.rand(B, Tk, generator=torch.Generator().manual_seed(B + Tk)) < 0.6
        keep[0, Tk - 1] = keep[B - 1, 0] = True
        keep[B - 1, 64:256] = False  # whole steps without a key
        return keep
    n = torch.tensor([Tk - 7, Tk // 3 + 1, 0, 129, 1, 64, Tk, 33][:B])
    return torch.arange(Tk) < n[:, None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["all", "lengths", "mask", "packed"])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_key_counts_once(dev, shape, kind, dtype):
    from nunchaku_amd.ops import cross_attention

    announce(f"every key {shape} {kind} {dtype}")
    B, Tq, Tk, H, Hkv, D = shape
    valid = validity(kind, B, Tk)
    keep = valid.to(dev)
    n = keep.sum(1).double().view(B, 1, 1)
    q = torch.randn(B, Tq, H, D, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    k = torch.zeros(B, Tk, Hkv, D, dtype=dtype, device=dev).masked_fill_(~keep[:, :, None, None], math.nan)
    args = {}
    if kind == "lengths":
        args["key_lengths"] = valid.sum(1).to(torch.int32).to(dev)
    elif kind == "mask":
        args["key_mask"] = keep
    elif kind == "packed":
        args["cu_seqlens_k"] = torch.cat((torch.zeros(1, dtype=torch.int64), valid.sum(1).cumsum(0))).to(torch.int32).to(dev)
        k = k[keep]
    tol = 1.01 * (torch.finfo(dtype).eps + 32 * U32 + 2 * n * U32)
    head, col = torch.arange(Hkv, device=dev)[:, None], torch.arange(D, device=dev)
    seen, wrong = torch.zeros(Tk, dtype=torch.int64, device=dev), torch.zeros((), dtype=torch.int64, device=dev)
    for base in range(0, Tk, Hkv * D):
        key = base + head * D + col  # the key that this column of this head shows
        inside = key < Tk
        at = key.clamp_max(Tk - 1)
        v = torch.zeros(B, Tk, Hkv, D, dtype=dtype, device=dev)
        v[:, at, head, col] = torch.where(inside, VALUE, 0.0).to(dtype)
        v.masked_fill_(~keep[:, :, None, None], math.nan)
        shown = inside & keep[:, at]
        want = torch.where(shown, VALUE / n.clamp_min(1), 0.0)  # [B, Hkv, D]
        got = cross_attention(q, k, v[keep] if kind == "packed" else v, **args).double().view(B, Tq, Hkv, H // Hkv, D)
        wrong += (~((got - want[:, None, :, None]).abs() <= (want * tol)[:, None, :, None])).sum()
        seen += torch.bincount(at[inside], minlength=Tk)
    assert wrong.item() == 0
    assert (seen == 1).all()
