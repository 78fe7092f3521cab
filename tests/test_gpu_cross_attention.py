"""Attention to an encoder's states on the GPU against the oracle in 64 bits.

Tolerance.  u = half a step of the type.  A probability's relative error: its score's absolute one, (D + 8) U32 times the sum of the
products' magnitudes times the scale (fp32 sums in any order, the factor, the subtraction of the maximum), the exponential's own
(16 U32), and u where it is rounded for the second product.  Sums over n keys in fp32: n U32.  So with A = sum p |v| and e the
probability's error without u, in numerator and denominator:
    |out - exact| <= A (u + 2 e + 2 n U32) + u |exact|, times 1.01 for the products of errors,
and half the smallest step where fp16 ends: 2^-25 for the result, and n 2^-25 max |v| for probabilities (whose sum is at least 1 / 2:
twice that).
Where the sum is that of the rounded probabilities (heads that do not end on a multiple of 32, many rows), p (1 + d) with |d| <= u stands
in both: out - exact = sum p d (v - exact) / sum p (1 + d), and |v - exact| <= |v| + |exact|: another u |exact|, and for what
fp16 loses of the probabilities n 2^-25 |exact| <= n 2^-25 max |v|, twice."""

import math

import pytest
import torch

from conftest import announce
from gpu_util import Guarded
from oracle import w8a8 as ow

pytestmark = pytest.mark.gpu
U32 = 2.0**-24


def inputs(B, Tq, Tk, H, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn(B, Tq, H, D, generator=g)).to(dtype)
    k, v = (torch.randn(B, Tk, Hkv, D, generator=g).to(dtype) for _ in range(2))
    return q, k, v


def check(got, q, k, v, valid=None, scale=None):
    dtype, D, n = q.dtype, q.shape[-1], k.shape[1]
    u = torch.finfo(dtype).eps / 2
    want = ow.cross_attention(q, k, v, valid, scale)
    keep = torch.ones(k.shape[:2], dtype=torch.bool) if valid is None else valid
    k0, v0 = k.double().masked_fill(~keep[:, :, None, None], 0), v.double().masked_fill(~keep[:, :, None, None], 0)
    A = ow.cross_attention(q, k, v.abs(), valid, scale)
    s = scale or 1 / math.sqrt(D)
    G = q.shape[2] // k.shape[2]
    most = (q.double().abs().amax((1, 3)) * k0.abs().amax((1, 3)).repeat_interleave(G, 1)).max().item()  # |q_i k_i|
    e = (D + 8) * U32 * s * min(D * most, (q.double().norm(dim=-1).max() * k0.norm(dim=-1).max()).item()) + 16 * U32
    bound = 1.01 * (A * (u + 2 * e + 2 * n * U32) + (2 if D % 32 else 1) * u * want.abs())
    if dtype == torch.float16:
        bound = bound + 2.0**-25 + (4 if D % 32 else 2) * n * 2.0**-25 * v0.abs().max()
    off = (got.cpu().double() - want).abs() - bound
    assert got.shape == q.shape and got.dtype == dtype
    assert (off <= 0).all(), (off.max().item(), (off > 0).sum().item(), off.numel())
    return want


DTYPES = [torch.bfloat16, torch.float16]
# every head size's kernel, both forms, lengths on both sides of a step of 64 keys, of 32 and of 128 rows
SHAPES = [
    (1, 1, 1, 1, 1, 8), (2, 1, 63, 2, 1, 16), (1, 1, 64, 4, 4, 32), (3, 1, 65, 8, 2, 40), (1, 1, 1000, 5, 1, 64), (2, 1, 4097, 4, 2, 128), (1, 2, 513, 6, 3, 72),
    (1, 33, 130, 2, 2, 80), (2, 7, 257, 10, 2, 96), (1, 128, 128, 1, 1, 112), (1, 129, 77, 3, 3, 120), (2, 31, 1024, 2, 1, 24), (1, 300, 300, 2, 2, 104),
    (4, 1100, 77, 8, 8, 64), (2, 1024, 333, 20, 20, 72), (3, 260, 190, 16, 8, 128), (8, 500, 100, 8, 8, 32), (9, 130, 129, 30, 15, 96), (4, 1030, 64, 8, 8, 16),
    (16, 128, 65, 16, 16, 88), (4, 4090, 150, 4, 4, 32), (2, 2040, 65, 16, 4, 128), (1, 7937, 193, 8, 8, 72), (1, 4096, 128, 16, 16, 64), (2, 4000, 1, 8, 8, 96),
    (1, 2550, 257, 96, 4, 112),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_all_keys(dev, shape, dtype):
    from nunchaku_amd.ops import cross_attention

    announce(f"attention {shape} {dtype}")
    q, k, v = inputs(*shape, dtype, sum(shape))
    out = Guarded(q.shape, dtype, dev)
    kg, vg = Guarded(k.shape, dtype, dev), Guarded(v.shape, dtype, dev)
    kg.raw.view(dtype).fill_(math.nan)  # in front of the keys and behind them
    vg.raw.view(dtype).fill_(math.nan)
    kg.t.copy_(k)
    vg.t.copy_(v)
    got = cross_attention(q.to(dev), kg.t, vg.t, out=out.t)
    assert got is out.t
    check(got, q, k, v)
    out.check("out")


VALID_SHAPES = [(4, 1, 200, 4, 2, 128), (5, 3, 700, 2, 2, 72), (4, 260, 150, 16, 16, 64), (6, 257, 333, 12, 12, 80), (3, 40, 129, 4, 1, 32), (8, 1030, 70, 4, 4, 128),
                (8, 2030, 260, 4, 4, 128), (4, 4090, 150, 4, 4, 72), (3, 8000, 193, 3, 3, 24),
                # blocks of 128 rows with the keys in parts
                (3, 70, 1100, 4, 2, 72), (4, 45, 2000, 3, 1, 80), (4, 100, 1100, 6, 6, 128), (4, 33, 5000, 2, 2, 120), (3, 120, 2500, 5, 5, 56)]


def spoil(t, keep):
    """NaN, infinities and the largest numbers where no key counts."""
    t = t.clone()
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(t.dtype).max], dtype=t.dtype)
    return torch.where(keep[:, :, None, None], t, bad[torch.arange(t.numel()).view(t.shape) % 4])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", VALID_SHAPES)
def test_lengths(dev, shape, dtype):
    from nunchaku_amd.ops import cross_attention

    B, Tk = shape[0], shape[2]
    announce(f"lengths {shape} {dtype}")
    q, k, v = inputs(*shape, dtype, sum(shape))
    n = torch.tensor([Tk, 0, 1, 65, Tk - 1, 63, 64, 128][:B], dtype=torch.int32)
    keep = torch.arange(Tk) < n[:, None]
    got = cross_attention(q.to(dev), spoil(k, keep).to(dev), spoil(v, keep).to(dev), key_lengths=n.to(dev))
    check(got, q, k, v, keep)
    assert not got[1].any()
    # out of range: all keys, none
    n2 = n.clone()
    n2[0], n2[1] = 2**31 - 1, -5
    assert torch.equal(cross_attention(q.to(dev), spoil(k, keep).to(dev), spoil(v, keep).to(dev), key_lengths=n2.to(dev)), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", VALID_SHAPES)
def test_mask(dev, shape, dtype):
    from nunchaku_amd.ops import cross_attention

    B, Tk = shape[0], shape[2]
    announce(f"mask {shape} {dtype}")
    q, k, v = inputs(*shape, dtype, sum(shape))
    keep = torch.rand(B, Tk, generator=torch.Generator().manual_seed(1)) < 0.7
    keep[0] = False
    keep[0, Tk - 1] = True  # the last key alone
    keep[1] = False         # none
    keep[2, :min(Tk - 1, 128)] = False  # whole steps without any
    wide = torch.ones(B, Tk + 5, dtype=torch.bool)
    wide[:, 3:Tk + 3] = keep  # rows at odd addresses
    got = cross_attention(q.to(dev), spoil(k, keep).to(dev), spoil(v, keep).to(dev), key_mask=wide.to(dev)[:, 3:Tk + 3])
    check(got, q, k, v, keep)
    assert not got[1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", VALID_SHAPES)
def test_packed(dev, shape, dtype):
    from nunchaku_amd.ops import cross_attention

    B, Tk = shape[0], shape[2]
    announce(f"packed {shape} {dtype}")
    q, k, v = inputs(*shape, dtype, sum(shape))
    n = torch.tensor([65, 0, 1, Tk, 63, 64, 2, 3][:B])
    keep = torch.arange(Tk) < n[:, None]
    cu = torch.cat((torch.zeros(1, dtype=torch.int64), n.cumsum(0))).to(torch.int32)
    pk, pv = k[keep], v[keep]
    behind = torch.full((9, *pk.shape[1:]), math.nan, dtype=dtype)  # rows of no sequence
    got = cross_attention(q.to(dev), torch.cat((pk, behind)).to(dev), torch.cat((pv, behind)).to(dev), cu_seqlens_k=cu.to(dev))
    check(got, q, k, v, keep)
    assert not got[1].any()
    # offsets out of order or range read nothing outside the tensors: each entry has the keys between its two offsets, as far as they exist
    bad = cu.clone()
    bad[-1] = 2**31 - 1
    bad[0] = -7
    check(cross_attention(q.to(dev), pk.to(dev), pv.to(dev), cu_seqlens_k=bad.to(dev)), q, k, v, keep)
    assert not cross_attention(q.to(dev), pk.to(dev), pv.to(dev), cu_seqlens_k=cu.flip(0).contiguous().to(dev)).any()


@pytest.mark.parametrize("Tq", [1, 200])
def test_strides(dev, Tq):
    """Heads first, parts of wider tensors, keys and values side by side, a broadcast batch; what lies beside the output stays."""
    from nunchaku_amd.ops import cross_attention

    announce(f"strides {Tq}")
    B, Tk, H, D = 3, 150, 4, 64
    q, k, v = inputs(B, Tq, Tk, H, H, D, torch.float16, 3)
    want = cross_attention(q.to(dev), k.to(dev), v.to(dev))
    check(want, q, k, v)
    heads_first = [t.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(cross_attention(*heads_first), want)
    kv = torch.cat((k.flatten(2), v.flatten(2)), -1).to(dev)
    out = torch.full((B, Tq, H + 2, D), 7.0, dtype=torch.float16, device=dev)
    cross_attention(q.to(dev), kv[..., :H * D].view(B, Tk, H, D), kv[..., H * D:].view(B, Tk, H, D), out=out[:, :, 1:-1])
    assert torch.equal(out[:, :, 1:-1], want) and (out[:, :, 0] == 7).all() and (out[:, :, -1] == 7).all()
    one = cross_attention(q.to(dev), k[:1].to(dev).expand(B, -1, -1, -1), v[:1].to(dev).expand(B, -1, -1, -1))
    check(one, q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Tq", [1, 300])
def test_scores_of_any_size(dev, Tq, dtype):
    """Scores that grow along the keys (the maximum moves at every step), that are far apart, all equal, and far below zero."""
    from nunchaku_amd.ops import cross_attention

    announce(f"scores {Tq} {dtype}")
    q, k, v = inputs(2, Tq, 400, 8, 8, 64, dtype, 5)
    up = torch.linspace(-1, 1, 400).view(1, 400, 1, 1)
    for name, qq, kk in (("growing", q.abs(), (k.abs() * 0.1 + up).to(dtype)), ("falling", q.abs(), (k.abs() * 0.1 - up).to(dtype)), ("equal", q, torch.zeros_like(k)),
                         ("far", q * 4, k * 4), ("low", q.abs() + 1, (-k.abs() * 8 - 8).to(dtype))):
        announce(name)
        check(cross_attention(qq.to(dev), kk.to(dev), v.to(dev)), qq, kk, v)
    check(cross_attention(q.to(dev), k.to(dev), v.to(dev), scale=0.01), q, k, v, scale=0.01)
    check(cross_attention(q.to(dev), k.to(dev), v.to(dev), scale=0.7), q, k, v, scale=0.7)


def test_nan_and_infinity_in_valid_places_reach_their_rows_only(dev):
    from nunchaku_amd.ops import cross_attention

    for Tq in (2, 300):
        announce(f"nan in valid places {Tq}")
        q, k, v = (t.to(dev) for t in inputs(2, Tq, 100, 4, 4, 64, torch.bfloat16, 6))
        want = cross_attention(q, k, v)
        q[0, 1, 2, 5] = math.nan
        k[1, 70, 1, 3] = math.nan
        v[1, 3, 0, 9] = math.inf
        got = cross_attention(q, k, v)
        assert torch.isnan(got[0, 1, 2]).all() and torch.isnan(got[1, :, 1]).all()
        assert not torch.isfinite(got[1, :, 0, 9]).any()
        got[0, 1, 2] = want[0, 1, 2]
        got[1, :, :2] = want[1, :, :2]
        assert torch.equal(got, want)


@pytest.mark.parametrize("Tq", [3, 8200])
def test_key_offset_beyond_32_bits(dev, Tq):
    """Keys and values of a batch entry that stand more than 2^32 bytes into their tensors, and tokens as far apart as is allowed."""
    from nunchaku_amd.ops import cross_attention

    announce(f"offset beyond 32 bits {Tq}")
    q, k, v = inputs(2, Tq, 200, 2, 2, 64, torch.bfloat16, 7)
    big = torch.empty(2 * (2**31 + 2**20), dtype=torch.bfloat16, device=dev)  # 8 GiB
    kd, vd = (big.as_strided((2, 200, 2, 64), (2**31 + 2**20, 2**20, 64, 1), o) for o in (0, 128))
    kd.copy_(k)
    vd.copy_(v)
    check(cross_attention(q.to(dev), kd, vd), q, k, v)
    far, vfar = (big.as_strided((2, 200, 2, 64), (64 * 2, 2**24 - 8, 64, 1), o) for o in (0, 512))
    far.copy_(k)
    vfar.copy_(v)
    check(cross_attention(q.to(dev), far, vfar), q, k, v)


def test_streams_and_graphs(dev):
    """A call whose keys are divided among workgroups, on a user's stream and in two captured graphs replayed in turn: workspaces are
    the calls' own."""
    from nunchaku_amd.ops import cross_attention

    announce("streams and graphs")
    sets = [[t.to(dev) for t in inputs(2, 1, 3000 + 500 * i, 4, 2, 128, torch.bfloat16, i)] for i in range(2)]
    want = [cross_attention(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [cross_attention(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cross_attention(*s))
        graphs.append(g)
    for turn in range(4):
        for s in sets:
            s[0].mul_(-0.9)
        eager = [cross_attention(*s) for s in sets]
        for o in outs:
            o.zero_()
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_rows_in_parts_on_streams_and_in_graphs(dev):
    """As above, with blocks of 128 rows; lengths change between the replays."""
    from nunchaku_amd.ops import cross_attention

    announce("rows in parts, graphs")
    sets = [[t.to(dev) for t in inputs(2, 100 + i, 2000 + 700 * i, 4, 2, 128, torch.float16, i)] for i in range(2)]
    lengths = [torch.tensor([n, 77], dtype=torch.int32, device=dev) for n in (2000, 1500)]
    graphs, outs = [], []
    for s, n in zip(sets, lengths):
        cross_attention(*s, key_lengths=n)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cross_attention(*s, key_lengths=n))
        graphs.append(g)
    side = torch.cuda.Stream()
    for turn in range(4):
        for n in lengths:
            n[1] += 311 * turn
            n[0] //= 2
        eager = [cross_attention(*s, key_lengths=n) for s, n in zip(sets, lengths)]
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = [cross_attention(*s, key_lengths=n) for s, n in zip(sets, lengths)]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(outs, eager, beside))
    for i, (s, n) in enumerate(zip(sets, lengths)):
        check(outs[i], *[t.cpu() for t in s], torch.arange(s[1].shape[1]) < n.cpu()[:, None])


def test_same_from_run_to_run(dev):
    from nunchaku_amd.ops import cross_attention

    for shape in ((2, 1, 5000, 8, 2, 128), (2, 513, 300, 16, 16, 64)):
        q, k, v = (t.to(dev) for t in inputs(*shape, torch.bfloat16, 8))
        want = cross_attention(q, k, v)
        for _ in range(5):
            assert torch.equal(cross_attention(q, k, v), want)


def test_empty_calls(dev):
    from nunchaku_amd.ops import cross_attention

    q, k, v = (t.to(dev) for t in inputs(2, 3, 5, 4, 2, 16, torch.bfloat16, 9))
    assert not cross_attention(q, k[:, :0], v[:, :0]).any()
    assert cross_attention(q[:, :0], k, v).shape == (2, 0, 4, 16)
    assert cross_attention(q[:0], k[:0], v[:0]).shape == (0, 3, 4, 16)


def test_refusals(dev):
    from nunchaku_amd.ops import cross_attention

    q, k, v = (t.to(dev) for t in inputs(2, 3, 8, 4, 2, 64, torch.bfloat16, 9))
    n = torch.tensor([1, 2], dtype=torch.int32, device=dev)
    with pytest.raises(NotImplementedError):
        cross_attention(q.float(), k.float(), v.float())
    with pytest.raises(ValueError, match="one type"):
        cross_attention(q, k.half(), v)
    with pytest.raises(ValueError, match="divides"):
        cross_attention(q[:, :, :3], k, v)
    with pytest.raises(ValueError, match="at most one"):
        cross_attention(q, k, v, key_lengths=n, key_mask=torch.ones(2, 8, dtype=torch.bool, device=dev))
    with pytest.raises(NotImplementedError, match="added"):
        cross_attention(q, k, v, key_mask=torch.zeros(2, 8, dtype=torch.bfloat16, device=dev))
    with pytest.raises(ValueError, match="key_mask"):
        cross_attention(q, k, v, key_mask=torch.ones(2, 7, dtype=torch.bool, device=dev))
    with pytest.raises(ValueError, match="key_lengths"):
        cross_attention(q, k, v, key_lengths=n.long())
    with pytest.raises(ValueError, match="key_lengths"):
        cross_attention(q, k, v, key_lengths=n.cpu())
    with pytest.raises(ValueError, match="cu_seqlens_k"):
        cross_attention(q, k[0], v[0], cu_seqlens_k=n)
    with pytest.raises(ValueError):
        cross_attention(q, k, v, cu_seqlens_k=torch.zeros(3, dtype=torch.int32, device=dev))
    for s in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            cross_attention(q, k, v, scale=s)
    with pytest.raises(ValueError, match="head_dim"):
        cross_attention(q[..., :60].contiguous(), k[..., :60].contiguous(), v[..., :60].contiguous())
    with pytest.raises(ValueError, match="aligned"):
        cross_attention(q[..., 4:60], k[..., 4:60], v[..., 4:60])
    with pytest.raises(ValueError, match="next to each other"):
        cross_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v)
    with pytest.raises(ValueError, match="out must"):
        cross_attention(q, k, v, out=q[:, :2])
    with pytest.raises(ValueError, match="expanded"):
        cross_attention(q, k, v, out=q[:1].expand(2, 3, 4, 64))
    with pytest.raises(ValueError, match="multiples of 8"):
        wide = torch.zeros(2, 8, 2, 68, dtype=torch.bfloat16, device=dev)[..., :64]
        cross_attention(q, wide, wide)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_attention_block(dev, dtype):
    """The operators together, as a decoder block uses them: residual and norm to codes, 8-bit projections of the tokens and of the
    encoder's states, attention over states of several lengths, 8-bit output projection; for a prompt and for single tokens.  Each step
    is checked by itself elsewhere: here against the same block of the oracle on the same codes, in 64 bits from step to step, where a
    code on the border of two may go either way: half a percent of the result's norm, what such codes are worth at most (one step of
    127 on every fourth code)."""
    from nunchaku_amd.models import W8A8Linear
    from nunchaku_amd.ops import cross_attention, rms_norm_quantize_w8a8

    torch.manual_seed(3)
    C, H, D, Tk = 256, 4, 64, 90
    q_proj, kv_proj, o_proj = (W8A8Linear.from_linear(torch.nn.Linear(C, n, dtype=dtype), device=dev) for n in (C, 2 * C, C))
    weight = (1 + 0.1 * torch.randn(C)).to(dtype)
    states, lengths = torch.randn(3, Tk, C).to(dtype), torch.tensor([Tk, 17, 0], dtype=torch.int32)
    keep = torch.arange(Tk) < lengths[:, None]

    def layer(m, codes, scales):
        return ow.gemm(codes, m.qweight.cpu(), scales, m.wscales.cpu(), m.bias.cpu()).to(dtype)

    for T in (1, 200):
        announce(f"block of {T} tokens {dtype}")
        x, r = torch.randn(3, T, C).to(dtype), torch.randn(3, T, C).to(dtype)
        codes, scales, h = rms_norm_quantize_w8a8(x.to(dev), weight.to(dev), r.to(dev))
        q = q_proj.forward_quant(codes, scales, out_dtype=dtype).view(3, T, H, D)
        kv = kv_proj(states.to(dev)).view(3, Tk, 2, H, D)
        a = cross_attention(q, kv[:, :, 0], kv[:, :, 1], key_lengths=lengths.to(dev))
        y = o_proj(a.flatten(2)) + h
        c1, s1, h1 = ow.rms_norm_quantize(x.view(-1, C), weight, r.view(-1, C))
        q1 = layer(q_proj, c1, s1).view(3, T, H, D)
        kv1 = layer(kv_proj, *ow.quantize_rows(states.view(-1, C))).view(3, Tk, 2, H, D)
        a1 = ow.cross_attention(q1, kv1[:, :, 0], kv1[:, :, 1], keep).to(dtype)
        y1 = layer(o_proj, *ow.quantize_rows(a1.flatten(2).view(-1, C))).double().view(3, T, C) + h1.double().view(3, T, C)
        assert ((y.cpu().double() - y1).norm() / y1.norm()).item() < 5e-3
        assert not a[2].any()


def test_attention_on_the_outputs_of_the_fused_projection(dev):
    """q, k and v as ``fused_qkv_norm_rottary`` writes them apart, NaN keys behind the last token included."""
    from gpu_util import make_module
    from nunchaku_amd.ops import cross_attention, fused_qkv_norm_rottary
    from oracle import layouts, synth

    heads, K, T, pad = 2, 256, 300, 512
    m = make_module(synth.make_layer(3 * heads * 128, K, 16, seed=11), dev)

    class Norm:
        weight = torch.ones(128, dtype=torch.bfloat16, device=dev)

    angles = torch.rand(pad, 64) * 6.28
    rot = torch.from_numpy(layouts.pack_rotemb(torch.stack((angles.sin(), angles.cos()), -1).view(pad, 128).numpy())).view(1, pad, 128).to(dev)
    outs = tuple(torch.empty(1, heads, pad, 128, dtype=torch.float16, device=dev) for _ in range(3))
    announce("attention on the fused projection's outputs")
    fused_qkv_norm_rottary(synth.make_activations(T, K, seed=12).to(dev).view(1, T, K), m, Norm, Norm, rot, output=outs, attn_tokens=T)
    q, k, v = (t.transpose(1, 2) for t in outs)
    assert torch.isnan(k[:, T:]).all()
    got = cross_attention(q[:, :T], k, v, key_lengths=torch.tensor([T], dtype=torch.int32, device=dev))
    check(got, q[:, :T].cpu(), k[:, :T].cpu(), v[:, :T].cpu())
    # (not the same bits: into how many parts the keys are divided goes by the tensors' length)
    check(cross_attention(q[:, :T], k[:, :T], v[:, :T]), q[:, :T].cpu(), k[:, :T].cpu(), v[:, :T].cpu())


def test_calls_from_several_threads(dev):
    """Every thread on a stream of its own, products and keys in parts among them: the results of one thread alone."""
    import threading

    from nunchaku_amd.ops import cross_attention, gemm_w8a8, quantize_w8a8_act

    announce("threads")

    def work(i):
        q, k, v = (t.to(dev) for t in inputs(2, 1 + 60 * (i % 2), 1500 + i, 4, 2, 64 + 8 * i, torch.bfloat16, i))
        o = cross_attention(q, k, v)
        codes, scales = quantize_w8a8_act(k[0].reshape(k.shape[1], -1))
        return [o, codes, scales, gemm_w8a8(codes[:5 + 40 * (i % 2)], codes[:300], scales[:5 + 40 * (i % 2)], scales[:300])]

    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = work(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 (reported below, in the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
