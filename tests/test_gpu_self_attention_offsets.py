"""Attention within sequences whose offsets are out of range or order, where rows in no sequence become zeros: every row is written, once, by a sequence
that it lies in.

A sequence's keys all have its number, one more than its place, as their values: a row's result says whose it is (scores are equal, so are the rounded
probabilities, and a mean of equal numbers is off by less than one in a hundred)."""

import math
import random

import pytest
import torch

from conftest import announce
from test_gpu_self_attention import check, rand

pytestmark = pytest.mark.gpu


def owners(dev, cu, total, heads, keys, times=3):
    """Which sequence (from 1; 0: none) each row's result is of."""
    from nunchaku_amd.ops import self_attention

    S = len(cu) - 1
    H, Hkv, D = heads
    number = torch.arange(1, S + 1).repeat_interleave(keys)
    v = torch.zeros(S * keys, Hkv, D)
    v[..., 0::2], v[..., 1::2] = (number % 128).float()[:, None, None], (number // 128).float()[:, None, None]
    q = rand(total, H, D, dtype=torch.bfloat16, seed=1).to(dev)
    v = v.to(torch.bfloat16).to(dev)
    offs, cu_k = torch.tensor(cu, dtype=torch.int32, device=dev), torch.arange(0, S * keys + 1, keys, dtype=torch.int32, device=dev)
    results = []
    for _ in range(times):
        del_me = torch.full_like(q, math.nan)  # (where the result is likely to be)
        del del_me
        results.append(self_attention(q, torch.zeros_like(v), v, offs, cu_k))
    torch.cuda.synchronize()
    for r in results:
        assert r.isfinite().all() and torch.equal(r, results[0])
    r = results[0].float().cpu()
    assert (r - r.round()).abs().max() < 0.5 and (r[..., 0::2] == r[:, :1, :1]).all() and (r[..., 1::2] == r[:, :1, 1:2]).all()
    return (r[:, 0, 0].round() + 128 * r[:, 0, 1].round()).int().tolist()


def look_over(got, cu, total):
    S, starts = len(cu) - 1, [min(max(c, 0), total) for c in cu]
    for t, s in enumerate(got):
        if s:
            assert starts[s - 1] <= t < starts[s], (t, s)
        else:
            assert t < starts[0] or t >= starts[S], t
    # a sequence whose offsets are in order with all others has all its rows
    for s in range(S):
        if all(c <= starts[s] for c in starts[:s]) and all(c >= starts[s + 1] for c in starts[s + 2:]) and starts[s] <= starts[s + 1]:
            assert all(got[t] == s + 1 for t in range(starts[s], starts[s + 1])), s


def disorder(S, total, many, seed):
    g = random.Random(seed)
    cu = sorted(g.randint(0, total) for _ in range(S + 1))
    for _ in range(many):
        cu[g.randrange(S + 1)] = g.choice([g.randint(-5, total + 5), -(2**31), 2**31 - 1, 0, total])
    return cu


# (offsets, rows): a few sequences
FEW = [([0, 20, 5], 50), ([900, 0, 900, 0, 900, 1000], 1000), ([30, 10, -5], 50), ([2**31 - 1, -(2**31), 4], 50), ([-7, 20, 2**31 - 1], 50), ([0, 20, 1000], 50), ([40, 40, 3, 3, 60], 50)]


@pytest.mark.parametrize("keys", [1, 300])
@pytest.mark.parametrize("heads", [(2, 1, 64), (8, 8, 72), (3, 1, 128)])
@pytest.mark.parametrize("case", FEW)
def test_a_few_sequences(dev, case, heads, keys):
    announce(f"offsets {case} {heads} {keys}")
    cu, total = case
    look_over(owners(dev, cu, total, heads, keys), cu, total)


# up to 64 regions of rows, up to 256, more; keys in parts for long ones of few heads; an offset out of order, some, all
@pytest.mark.parametrize("many", [0, 1, 7, 10000])
@pytest.mark.parametrize("shape", [(62, 500, 2, 1, 64, 40), (63, 500, 2, 1, 64, 40), (70, 70, 4, 1, 128, 3000), (128, 128, 2, 1, 64, 5000), (200, 3000, 1, 1, 32, 7), (254, 600, 4, 4, 128, 200),
                                   (255, 255, 8, 2, 128, 600), (1000, 5000, 2, 2, 64, 3), (5000, 9000, 1, 1, 64, 1), (9000, 2000, 3, 1, 40, 1)])
def test_many_sequences(dev, shape, many):
    announce(f"offsets {shape} {many}")
    S, total, H, Hkv, D, keys = shape
    cu = disorder(S, total, many, S + many) if many < 10000 else [random.Random(S).randint(-20, total + 20) for _ in range(1)] + [random.Random(i).randint(-20, total + 20) for i in range(S)]
    look_over(owners(dev, cu, total, (H, Hkv, D), keys), cu, total)


@pytest.mark.parametrize("causal", [True, False])
def test_the_first_sequence_of_descending_offsets(dev, causal):
    from nunchaku_amd.ops import self_attention

    q = rand(50, 2, 64, dtype=torch.float16, seed=1)
    g = q.to(dev)
    for offs in ([0, 20, 1000], [0, 20, 5], [0, 20, -3], [0, 20, 20, 4]):
        got = self_attention(g, g, g, torch.tensor(offs, dtype=torch.int32, device=dev), causal=causal)
        check(got[:20], q[:20], q[:20], q[:20], causal)
        assert got.isfinite().all()
        if offs[-1] <= 20:
            assert not got[20:].any()
