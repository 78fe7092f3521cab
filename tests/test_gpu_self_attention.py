"""Attention within sequences on the GPU against the oracle in 64 bits.

Tolerance: that of attention to an encoder's states.  u = half a step of the type.  A probability's relative error: its score's absolute one, (D + 8) U32 times the
sum of the products' magnitudes times the scale, the exponential's own (16 U32), and u where it is rounded for the second product; sums over n keys
n U32.  With A = sum p |v| and e the probability's error without u, in numerator and denominator:
    |out - exact| <= A (u + 2 e + 2 n U32) + u |exact|, times 1.01 for the products of errors,
another u |exact| where the sum is that of the rounded probabilities, and half the smallest step where fp16 ends: 2^-25 for the result and, twice, n 2^-25
max |v| for the probabilities (whose sum is at least 1 / 2), twice again where their sum is that of the rounded ones."""

import math

import pytest
import torch

from conftest import announce
from gpu_util import Guarded
from oracle import blocks

pytestmark = pytest.mark.gpu
U32 = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16]


def bound(want, q, k, v, causal, scale=None):
    dtype, D, n = q.dtype, q.shape[-1], k.shape[0]
    u = torch.finfo(dtype).eps / 2
    A = blocks.self_attention(q, k, v.abs(), causal, scale)
    s = scale or 1 / math.sqrt(D)
    most = q.double().norm(dim=-1).max() * k.double().nan_to_num(0).norm(dim=-1).max() if n and q.shape[0] else torch.tensor(0.0)
    e = (D + 8) * U32 * s * most.item() + 16 * U32
    b = 1.01 * (A * (u + 2 * e + 2 * n * U32) + 2 * u * want.abs())
    if dtype == torch.float16 and n:
        b = b + 2.0**-25 + 4 * n * 2.0**-25 * v.double().nan_to_num(0, 0, 0).abs().max()
    return b


def check(got, q, k, v, causal, scale=None, rows=None):
    """One sequence; rows: those to look at"""
    want = blocks.self_attention(q, k, v, causal, scale)
    off = (got.cpu().double() - want).abs() - bound(want, q, k, v, causal, scale)
    if rows is not None:
        off = off[rows]
    assert got.shape == q.shape and got.dtype == q.dtype
    assert (off <= 0).all(), (off.max().item(), (~(off <= 0)).sum().item(), off.numel())


def rand(*shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def offsets(lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


# (lengths, heads, heads of keys, head size): one token, none, blocks and steps that end everywhere, every head size's kernel, odd groups
PACKED = [
    ([1], 1, 1, 8), ([5, 0, 1, 64], 2, 1, 16), ([63, 65, 2, 128], 4, 4, 32), ([0, 0, 33], 6, 2, 40), ([130, 1, 257], 8, 2, 64), ([31, 32, 33, 1, 1, 1], 5, 1, 72),
    ([300, 129], 3, 3, 80), ([77, 400], 12, 4, 96), ([200, 56, 511], 2, 2, 104), ([1000], 4, 1, 128), ([1025, 1, 255, 640], 6, 3, 128), ([513, 700], 7, 1, 112), ([256, 512], 16, 2, 120),
    ([3] * 70 + [90], 2, 2, 64), ([2049], 1, 1, 128), ([900, 300, 20], 16, 8, 88), ([1500, 700], 8, 8, 24),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", PACKED)
def test_packed(dev, case, causal, dtype):
    from nunchaku_amd.ops import self_attention

    lens, H, Hkv, D = case
    announce(f"self_attention packed {case} {causal} {dtype}")
    total = sum(lens)
    qkv = rand(total, (H + 2 * Hkv) * D, dtype=dtype, seed=total, scale=1.2)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([H * D, Hkv * D, Hkv * D], -1))
    gq, gk, gv = (t.unflatten(-1, (-1, D)) for t in qkv.to(dev).split([H * D, Hkv * D, Hkv * D], -1))
    cu = offsets(lens).to(dev)
    out = Guarded((total, H, D), dtype, dev)
    got = self_attention(gq, gk, gv, cu_seqlens_q=cu, causal=causal, out=out.t)
    assert got is out.t
    for a, n in zip(offsets(lens).tolist(), lens):
        check(got[a:a + n], q[a:a + n], k[a:a + n], v[a:a + n], causal)
    out.check("out")
    assert torch.equal(self_attention(gq, gk, gv, cu, cu, causal=causal), got)


# (queries, keys) of each sequence: fewer and more queries than keys, none of either
CHUNKS = [
    [(1, 1)], [(1, 700), (1, 0), (0, 9), (3, 64)], [(5, 300), (33, 33), (40, 7), (1, 129)], [(16, 2000), (17, 1999), (1, 5)], [(200, 650), (64, 4000), (300, 100)],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(8, 2, 128), (3, 3, 72), (16, 4, 64), (4, 1, 96)])
@pytest.mark.parametrize("chunks", CHUNKS)
def test_new_tokens_over_a_cache_and_packed_keys(dev, chunks, heads, dtype):
    from nunchaku_amd.ops import self_attention

    H, Hkv, D = heads
    announce(f"self_attention chunks {chunks} {heads} {dtype}")
    new, lens = [m for m, _ in chunks], [n for _, n in chunks]
    S, T = len(lens), max(lens) + 3
    q = rand(sum(new), H, D, dtype=dtype, seed=1, scale=1.5)
    k, v = (rand(S, T, Hkv, D, dtype=dtype, seed=s) for s in (2, 3))
    behind = torch.arange(T) >= torch.tensor(lens)[:, None]
    for t in (k, v):
        t.masked_fill_(behind[:, :, None, None], math.nan)
    n = torch.tensor(lens, dtype=torch.int32).to(dev)
    cu = offsets(new)
    for causal in (True, False):
        got = self_attention(q.to(dev), k.to(dev), v.to(dev), cu_seqlens_q=cu.to(dev), key_lengths=n, causal=causal)
        for s, (a, m) in enumerate(zip(cu.tolist(), new)):
            check(got[a:a + m], q[a:a + m], k[s, :lens[s]], v[s, :lens[s]], causal)
        if sum(lens):
            packed = [torch.cat([t[s, :lens[s]] for s in range(S)]).to(dev) for t in (k, v)]
            again = self_attention(q.to(dev), *packed, cu_seqlens_q=cu.to(dev), cu_seqlens_k=offsets(lens).to(dev), causal=causal)
            for s, (a, m) in enumerate(zip(cu.tolist(), new)):
                check(again[a:a + m], q[a:a + m], k[s, :lens[s]], v[s, :lens[s]], causal)


BATCHES = [(1, 1, 1, 2, 1, 64), (4, 77, 77, 12, 12, 64), (2, 300, 300, 6, 2, 72), (3, 40, 1000, 8, 8, 128), (1, 1100, 1100, 4, 2, 128), (2, 700, 260, 4, 4, 32), (2, 513, 2050, 3, 1, 80)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", BATCHES)
def test_batches(dev, shape, dtype):
    """[B, T, heads, D] with and without lengths, heads first in memory, another scale; lengths beyond both ends."""
    from nunchaku_amd.ops import self_attention

    B, Tq, Tk, H, Hkv, D = shape
    announce(f"self_attention batch {shape} {dtype}")
    q = rand(B, H, Tq, D, dtype=dtype, seed=1).transpose(1, 2)
    k, v = (rand(B, Hkv, Tk, D, dtype=dtype, seed=s).transpose(1, 2) for s in (2, 3))
    g = [t.transpose(1, 2).to(dev).transpose(1, 2) for t in (q, k, v)]
    for causal in (True, False):
        got = self_attention(*g, causal=causal, scale=0.17)
        for b in range(B):
            check(got[b], q[b], k[b], v[b], causal, 0.17)
        lens = [max(0, Tk - 7 * b) for b in range(B)]
        n = torch.tensor(lens, dtype=torch.int32)
        n[0] = 2**31 - 1
        if B > 2:
            n[1], lens[1] = -3, 0
        got = self_attention(*g, key_lengths=n.to(dev), causal=causal)
        for b in range(B):
            check(got[b], q[b], k[b, :lens[b]], v[b, :lens[b]], causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("total_keys", [60, 3000])
def test_rows_in_no_sequence(dev, causal, total_keys):
    """In front of the first sequence and behind the last: zeros, or left as they are in `out`; the keys there have no effect."""
    from nunchaku_amd.ops import self_attention

    lens, keys, front, behind = [5, 0, 40], [total_keys, 3, 50], 3, 100
    total = front + sum(lens) + behind
    q = rand(total, 4, 64, dtype=torch.bfloat16, seed=1).to(dev)
    k, v = (rand(4 + sum(keys) + 9, 2, 64, dtype=torch.bfloat16, seed=s).to(dev) for s in (2, 3))
    for t in (k, v):
        t[:4] = math.nan
        t[-9:] = math.inf
    cq, ck = offsets(lens, front).to(dev), offsets(keys, 4).to(dev)
    got = self_attention(q, k, v, cq, ck, causal=causal)
    inside = slice(front, total - behind)
    assert got[inside].isfinite().all() and not got[:front].any() and not got[total - behind:].any()
    out = torch.full_like(q, 3.0)
    self_attention(q, k, v, cq, ck, causal=causal, out=out)
    assert torch.equal(out[inside], got[inside]) and (out[:front] == 3).all() and (out[total - behind:] == 3).all()
    for a, n, b, m in zip(cq.tolist(), lens, ck.tolist(), keys):
        check(got[a:a + n], *(t.cpu() for t in (q[a:a + n], k[b:b + m], v[b:b + m])), causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(200, 4, 2, 128), (700, 8, 8, 64), (90, 3, 1, 72), (1030, 2, 1, 96)])
def test_what_a_query_does_not_see_has_no_effect(dev, shape, dtype):
    """NaN and infinities in the last keys and values of a causal sequence: the queries in front of them are as they were."""
    from nunchaku_amd.ops import self_attention

    T, H, Hkv, D = shape
    announce(f"self_attention unseen {shape} {dtype}")
    q, k, v = rand(T, H, D, dtype=dtype, seed=1), rand(T, Hkv, D, dtype=dtype, seed=2), rand(T, Hkv, D, dtype=dtype, seed=3)
    cu = offsets([T]).to(dev)
    for at, what in ((T - 1, math.nan), (T - 9, math.inf), (T // 2, math.nan), (0, math.inf)):
        bad = v.clone()
        bad[at, :, 1::2] = what
        got = self_attention(q.to(dev), k.to(dev), bad.to(dev), cu, causal=True)
        check(got, q, k, v, True, rows=slice(0, at))
        assert not got[at:, :, 1::2].isfinite().any()
        # (the columns without any are right in all rows)
        off = (got.cpu().double() - (want := blocks.self_attention(q, k, v, True))).abs() - bound(want, q, k, v, True)
        assert (off[..., 0::2] <= 0).all()
    bad = k.clone()
    bad[T - 1] = math.nan
    got = self_attention(q.to(dev), bad.to(dev), v.to(dev), cu, causal=True)
    # (not the same bits: the maximum that a row's exponentials refer to moves with its neighbours', the sums' order with a second pass)
    check(got, q, k, v, True, rows=slice(0, T - 1))
    assert got[T - 1].isnan().all()


def test_offsets_out_of_order(dev):
    """Offsets beyond the rows or descending: nothing outside is read or written, and what is well-formed is right."""
    from nunchaku_amd.ops import self_attention

    q = rand(50, 2, 64, dtype=torch.float16, seed=1)
    out = Guarded((50, 2, 64), torch.float16, dev)
    for offs in ([0, 20, 1000], [-7, 20, 2**31 - 1], [0, 20, 5], [30, 10, -5], [2**31 - 1, -(2**31), 4]):
        cu = torch.tensor(offs, dtype=torch.int32, device=dev)
        self_attention(q.to(dev), q.to(dev), q.to(dev), cu, causal=True, out=out.t)
        torch.cuda.synchronize()
        out.check("out")
        if offs[:2] == [0, 20]:
            check(out.t[:20], q[:20], q[:20], q[:20], True)


def test_no_keys(dev):
    from nunchaku_amd.ops import self_attention

    q = rand(2, 3, 4, 64, dtype=torch.bfloat16, seed=1).to(dev)
    k = q.new_empty(2, 0, 2, 64)
    assert not self_attention(q, k, k).any()
    assert not self_attention(q, k, k, key_lengths=torch.tensor([3, 0], dtype=torch.int32, device=dev), causal=True).any()
    assert self_attention(q[:, :0], k, k).shape == (2, 0, 4, 64)
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device=dev)
    assert not self_attention(q[0], k[0], k[0], cu, torch.zeros_like(cu)).any()


@pytest.mark.parametrize("scale", [30.0, 1e4])
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_scores(dev, dtype, scale):
    """Scores that leave one key of each row (the others have e^-60 of it at most): its value, off by the roundings of its probability and of the result."""
    from nunchaku_amd.ops import self_attention

    g = torch.Generator().manual_seed(2)
    T, D = 300, 64
    k = torch.sign(torch.randn(T, 1, D, generator=g)).to(dtype)  # (a row's own key is ahead by 2 for each channel that differs)
    v = rand(T, 1, D, dtype=dtype, seed=3)
    got = self_attention(k.to(dev)[None], k.to(dev)[None], v.to(dev)[None], causal=True, scale=scale)
    u = torch.finfo(dtype).eps / 2
    assert ((got[0].cpu().double() - v.double()).abs() <= 1.01 * (2 * u + 4 * U32) * v.double().abs() + 2.0**-24).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [(40, 2, 2, 64), (300, 4, 1, 128), (700, 8, 8, 64), (90, 3, 1, 72), (1030, 2, 1, 96), (2100, 16, 16, 128), (2100, 16, 16, 32)])
def test_a_nan_of_one_query_stays_with_it(dev, shape, causal):
    """Infinities and NaN in some queries and one head: all other rows are right."""
    from nunchaku_amd.ops import self_attention

    T, H, Hkv, D = shape
    announce(f"self_attention query nan {shape} {causal}")
    q, k, v = rand(T, H, D, dtype=torch.bfloat16, seed=1), rand(T, Hkv, D, dtype=torch.bfloat16, seed=2), rand(T, Hkv, D, dtype=torch.bfloat16, seed=3)
    bad = q.clone()
    rows = sorted({0, 7, T // 2, T - 1})
    for i, t in enumerate(rows):
        bad[t, i % H, 3] = (math.nan, math.inf)[i % 2]
    got = self_attention(bad[None].to(dev), k[None].to(dev), v[None].to(dev), causal=causal)[0].cpu()
    for i, t in enumerate(rows):
        if t or not causal:  # (a query that sees itself alone has no other score to compare with: NaN or its value)
            assert got[t, i % H].isnan().all()
        got[t, i % H] = 0
        q[t, i % H] = 0
    heads = sorted({0, H - 1} | {i % H for i in range(len(rows))})
    want, b = (f(q[:, heads], k, v, causal) if Hkv == 1 else f(q[:, heads], k[:, [h * Hkv // H for h in heads]], v[:, [h * Hkv // H for h in heads]], causal)
               for f in (blocks.self_attention, lambda q, k, v, c: bound(blocks.self_attention(q, k, v, c), q, k, v, c)))
    off = (got[:, heads].double() - want).abs() - b
    for i, t in enumerate(rows):
        off[t, heads.index(i % H)] = -1
    assert (off <= 0).all(), (off.max().item(), (~(off <= 0)).sum().item())


# (queries, keys) of each entry or sequence, heads, heads of keys, head size: causal, so few heads that the keys are divided, blocks whose keys end in the first part, and rows in
# front of all keys
@pytest.mark.parametrize("case", [([(2300, 2300)], 1, 1, 128), ([(1500, 1500)], 2, 1, 64), ([(1100, 1900)] * 2, 1, 1, 96), ([(1300, 700)], 2, 2, 72), ([(129, 4200), (1, 64), (900, 900)], 3, 1, 128),
                                  ([(1024, 1024)] * 2, 2, 2, 32)])
def test_parts_of_keys_under_a_causal_mask(dev, case):
    from nunchaku_amd.ops import self_attention

    lens, H, Hkv, D = case
    announce(f"self_attention parts {case}")
    new, keys = ([n[i] for n in lens] for i in (0, 1))
    q = rand(sum(new), H, D, dtype=torch.bfloat16, seed=5, scale=1.5)
    k, v = (rand(sum(keys), Hkv, D, dtype=torch.bfloat16, seed=s) for s in (6, 7))
    out = Guarded((sum(new), H, D), torch.bfloat16, dev)
    self_attention(q.to(dev), k.to(dev), v.to(dev), offsets(new).to(dev), offsets(keys).to(dev), causal=True, out=out.t)
    out.check("out")
    results = [out.t]
    if len(set(lens)) == 1:
        S = len(lens)
        results.append(self_attention(*(t.to(dev).unflatten(0, (S, -1)) for t in (q, k, v)), causal=True).flatten(0, 1))
    for got in results:
        for a, m, b, n in zip(offsets(new).tolist(), new, offsets(keys).tolist(), keys):
            check(got[a:a + m], q[a:a + m], k[b:b + n], v[b:b + n], True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [(3, 5, 2, 1, 64), (2, 300, 4, 4, 72), (4, 1, 8, 2, 128)])
def test_a_batch_of_queries_over_packed_keys(dev, shape, causal):
    from nunchaku_amd.ops import self_attention

    S, T, H, Hkv, D = shape
    lens = [0, 700, 33, 129][:S]
    q = rand(S, T, H, D, dtype=torch.float16, seed=1)
    k, v = (rand(sum(lens), Hkv, D, dtype=torch.float16, seed=s) for s in (2, 3))
    cu = offsets(lens)
    got = self_attention(q.to(dev), k.to(dev), v.to(dev), cu_seqlens_k=cu.to(dev), causal=causal)
    for s, (a, n) in enumerate(zip(cu.tolist(), lens)):
        check(got[s], q[s], k[a:a + n], v[a:a + n], causal)


# heads of every kernel of blocks of 128 and of 256 rows, with and without a column of ones
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", [(900, 2, 2, 64), (900, 1, 1, 72), (700, 2, 1, 128), (600, 4, 4, 24), (700, 64, 64, 128), (700, 64, 64, 72), (700, 48, 48, 96)])
def test_scores_that_rise_along_the_keys(dev, shape, causal):
    """By 30, 80, 100 and 3000 over all keys, or by 90 at one key between two others: within fp32's range of an old maximum's exponentials, at its end and beyond."""
    from nunchaku_amd.ops import self_attention

    T, H, Hkv, D = shape
    dtype = torch.bfloat16
    announce(f"self_attention rising {shape} {causal}")
    way = torch.sign(rand(1, 1, D, dtype=torch.float32, seed=1))
    q = (way * (1 + 0.05 * rand(T, H, 1, dtype=torch.float32, seed=2))).to(dtype)
    v = rand(T, Hkv, D, dtype=dtype, seed=3)
    at = torch.arange(T, dtype=torch.float32)[:, None, None] / T
    for rise in (30.0, 80.0, 100.0, 3000.0, None):
        size = rise * at if rise else 90.0 * (at == 333 / T) - 3.0 * at
        k = (way * size / math.sqrt(D) + 0.02 * rand(T, Hkv, D, dtype=torch.float32, seed=4)).to(dtype)
        check(self_attention(*(t.to(dev)[None] for t in (q, k, v)), causal=causal)[0], q, k, v, causal)


@pytest.mark.parametrize("shape", [(500, 2, 2, 64), (700, 64, 64, 128), (700, 64, 64, 72)])
def test_first_keys_of_no_weight(dev, shape):
    """Scores of minus infinity for more than a block's first keys: as if those keys were not there."""
    from nunchaku_amd.ops import self_attention

    T, H, Hkv, D = shape
    for dtype in DTYPES:
        q, v = rand(T, H, D, dtype=dtype, seed=1).abs() + 0.125, rand(T, Hkv, D, dtype=dtype, seed=3)
        k = rand(T, Hkv, D, dtype=dtype, seed=2)
        for first in (40, 130):
            k[:first] = -math.inf
            check(self_attention(*(t.to(dev)[None] for t in (q, k, v)))[0], q, k[first:], v[first:], False)
