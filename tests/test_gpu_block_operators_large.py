"""Sizes at which the operators between a block's linear layers take another way: attention's keys in parts among 65 to 256 regions of rows, rows and tokens of more
than one launch.  Tolerances are those of the operators' own tests."""

import ctypes

import pytest
import torch

import test_gpu_gated_norm as norm_test
import test_gpu_rotary_axes as rotary_test
import test_gpu_self_attention as attention_test
from conftest import announce
from nunchaku_amd import _native as nv

pytestmark = pytest.mark.gpu


def workspace(S, H, Hkv, D, q_len, k_len, packed, causal):
    """Bytes that a call needs: not zero where it divides the keys."""
    i64x3 = ctypes.c_int64 * 3
    some, none = 1 << 20, (0, 0, 0)  # (an address is not followed)
    args = nv.SelfAttentionArgs(some, some, some, some, some if packed else None, None, None, None, 0, S, H, Hkv, D, q_len, k_len, *(i64x3(*none) for _ in range(4)), 1.0, causal, 0, 0)
    n = ctypes.c_int64()
    assert nv.lib().svdq_self_attention_workspace(ctypes.byref(args), ctypes.byref(n)) == 0
    return n.value


# sequences, new tokens of each (packed, then about so many, under a causal mask; a batch, without), heads, heads of keys, head size, keys of the cache
PARTS = [(62, 1, 8, 2, 128, 1500), (63, 1, 8, 2, 128, 1500), (64, 1, 8, 2, 64, 2000), (70, 1, 2, 1, 128, 3000), (100, 3, 4, 1, 72, 2500), (128, 1, 1, 1, 32, 4000), (127, 1, 2, 1, 96, 2000),
         (254, 2, 3, 1, 64, 3000), (80, 32, 3, 1, 128, 2000), (66, 100, 1, 1, 64, 4000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("case", PARTS)
def test_keys_in_parts_among_many_sequences(dev, case, packed, dtype):
    """New tokens over a cache of very different lengths, none among them; NaN behind each."""
    from nunchaku_amd.ops import self_attention

    S, new, H, Hkv, D, T = case
    announce(f"parts among many {case} {packed} {dtype}")
    g = torch.Generator().manual_seed(S)
    lens = torch.randint(0, T + 1, (S,), generator=g)
    lens[S // 3], lens[S // 2], lens[-1] = 0, T, T - 1
    each = [new] * S
    if packed and new > 1:
        each = torch.randint(0, 2 * new, (S,), generator=g).tolist()
    total = sum(each)
    assert workspace(S, H, Hkv, D, total if packed else new, T, packed, packed) > 0
    q = attention_test.rand(total, H, D, dtype=dtype, seed=1, scale=1.5)
    k, v = (attention_test.rand(S, T, Hkv, D, dtype=dtype, seed=s) for s in (2, 3))
    behind = torch.arange(T) >= lens[:, None]
    gk, gv = (t.masked_fill(behind[:, :, None, None], float("nan")).to(dev) for t in (k, v))
    cu, n = attention_test.offsets(each), lens.to(torch.int32).to(dev)
    if packed:
        call = lambda: self_attention(q.to(dev), gk, gv, cu.to(dev), key_lengths=n, causal=True)  # noqa: E731
    else:
        call = lambda: self_attention(q.to(dev).view(S, new, H, D), gk, gv, key_lengths=n).flatten(0, 1)  # noqa: E731
    got = call()
    assert torch.equal(call(), got)
    for s, (a, m, length) in enumerate(zip(cu.tolist(), each, lens.tolist())):
        attention_test.check(got[a:a + m], q[a:a + m], k[s, :length], v[s, :length], packed)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_norms_of_more_rows_than_a_launch(dev, norm):
    """2^21 rows and some, of a batch and packed: the rows of the second launch as in a call of their own, gates of the right entries."""
    from nunchaku_amd.ops import gated_norm

    announce(f"norm in two launches {norm}")
    B, T, K, dtype = 3, 2**21 // 3 + 50, 16, torch.bfloat16
    M, seam = B * T, 2**21
    x, res = (norm_test.rand(M, K, dtype=dtype, seed=i, scale=2.0) for i in (1, 2))
    gate, scale, shift = (norm_test.rand(B, K, dtype=dtype, seed=3 + i) for i in range(3))
    gx, gr = x.to(dev), res.to(dev)
    v = {n: t.to(dev) for n, t in (("gate", gate), ("scale", scale), ("shift", shift))}
    y, h = gated_norm(gx.view(B, T, K), gr.view(B, T, K), norm, **v)
    cu = torch.tensor([0, T, 2 * T, M - 7], dtype=torch.int32, device=dev)
    py, ph = gated_norm(gx, gr, norm, cu_seqlens=cu, **v)
    for part, packed in ((y, py), (h, ph)):
        assert torch.equal(part.view(M, K)[:M - 7], packed[:M - 7]) and not packed[M - 7:].any()
    entry = torch.arange(M) // T
    for rows in (slice(0, 40), slice(T - 20, T + 20), slice(seam - 20, seam + 20), slice(M - 20, M)):
        e = entry[rows]
        norm_test.check((y.view(M, K)[rows], h.view(M, K)[rows]), x[rows], res[rows], norm, gate=gate[e], scale=scale[e], shift=shift[e])
    e = entry.to(dev)[seam:]
    alone = gated_norm(gx[seam:], gr[seam:], norm, **{n: t[e] for n, t in v.items()})
    assert torch.equal(alone[0], y.view(M, K)[seam:]) and torch.equal(alone[1], h.view(M, K)[seam:])


def test_rotation_of_more_tokens_than_a_launch(dev):
    """2^25 tokens and some, a wave each: those of the second launch as in a call of their own."""
    from nunchaku_amd.ops import rotary_axes

    announce("rotation in two launches")
    seam, more, D, dtype = 2**25, 77, 8, torch.bfloat16
    q = torch.randn(seam + more, 1, D, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(dtype)
    pos = torch.arange(seam + more, dtype=torch.int32, device=dev).remainder_(100003)[:, None]
    got = rotary_axes(q, None, pos, (D,))[0]
    for rows in (slice(0, 5000), slice(seam - 50, seam + more)):
        assert torch.equal(rotary_axes(q[rows], None, pos[rows], (D,))[0], got[rows])
        rotary_test.check(got[rows], q[rows].cpu(), pos[rows].cpu(), (D,))
    assert got.isfinite().all()
