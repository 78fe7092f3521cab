"""Rotary positions with several axes on the GPU against the oracle in 64 bits.

Tolerance.  U = 2^-24, u = half a step of the type.  The norm's factor: eight squares of a thread and 5 exchanges 14 U of the sum, half of it and 4 for the root, the
mean and the division, two products: 13 U.  Cosine and sine: 4 U of the function, the angle's rounding to fp32 (at most a whole number times pi, 2^-25 of it): 2 U
more, and positions up to 2^21 nothing beside.  Two products and a sum: 2 U.  Together 21 U of |x| + |y| of the pair; then u of the result."""

import pytest
import torch

from conftest import announce
from gpu_util import Guarded
from oracle import blocks

pytestmark = pytest.mark.gpu
U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16]


def check(got, x, positions, axes, **kw):
    want, size = blocks.rotary(x, positions, axes, **kw)
    u, end = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    bound = 1.01 * (21 * U * size + u * want.abs()) + end
    off = (got.cpu().double() - want).abs() - bound
    assert got.shape == x.shape and got.dtype == x.dtype
    assert (off <= 0).all(), (off.max().item(), (off > 0).sum().item(), off.numel())


def inputs(B, T, H, Hkv, D, A, dtype, seed, most=5000):
    g = torch.Generator().manual_seed(seed)
    q, k = ((1.5 * torch.randn(B, T, n, D, generator=g)).to(dtype) for n in (H, Hkv))
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]
    return q, k, w, torch.randint(-most, most, (B, T, A), generator=g, dtype=torch.int32)


# heads of every number of lanes, axes that end inside a piece of eight channels, channels that pass
CASES = [
    ((1, 1, 1, 1, 8), (8,), True), ((2, 3, 5, 1, 16), (4, 6), True), ((1, 7, 3, 3, 32), (10, 12, 10), True), ((3, 65, 4, 2, 40), (14, 14, 12), True), ((2, 33, 8, 8, 64), (16, 24, 24), False),
    ((1, 1157, 2, 1, 72), (24, 24, 24), True), ((1, 129, 6, 2, 80), (16, 24, 24), False), ((2, 50, 12, 4, 96), (32, 64), False), ((1, 20, 7, 7, 128), (44, 42, 42), True),
    ((8, 1, 32, 8, 128), (128,), False), ((1, 4099, 3, 1, 128), (16, 56, 56), True), ((2, 5, 3, 2, 256), (64, 64, 64, 64), True), ((1, 9, 2, 2, 200), (2, 96, 94), False), ((2, 4, 5, 5, 120), (2, 2), True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_queries_and_keys(dev, case, dtype):
    from nunchaku_amd.ops import rotary_axes

    shape, axes, interleaved = case
    announce(f"rotary {case} {dtype}")
    q, k, w, pos = inputs(*shape, len(axes), dtype, sum(shape))
    for spectrum in ("axis", "head"):
        for norm in (False, True):
            oq, ok = Guarded(q.shape, dtype, dev), Guarded(k.shape, dtype, dev)
            kw = dict(interleaved=interleaved, spectrum=spectrum)
            got = rotary_axes(q.to(dev), k.to(dev), pos.to(dev), axes, norm_q=w[0].to(dev) if norm else None, norm_k=w[1].to(dev) if norm else None, out_q=oq.t, out_k=ok.t, **kw)
            assert got[0] is oq.t and got[1] is ok.t
            check(oq.t, q, pos, axes, weight=w[0] if norm else None, **kw)
            check(ok.t, k, pos, axes, weight=w[1] if norm else None, **kw)
            oq.check("q")
            ok.check("k")
            again = rotary_axes(q.to(dev), k.to(dev), pos.to(dev), list(axes), norm_q=w[0].to(dev) if norm else None, norm_k=w[1].to(dev) if norm else None, **kw)
            assert torch.equal(again[0], oq.t) and torch.equal(again[1], ok.t)


@pytest.mark.parametrize("interleaved", [True, False])
def test_positions(dev, interleaved):
    """Far positions (2^21), 64-bit and fp32 ones, between whole numbers, by strides, shared by the batch; several thetas."""
    from nunchaku_amd.ops import rotary_axes

    q, k, _, pos = inputs(2, 37, 4, 2, 64, 2, torch.float16, 3, most=1 << 21)
    axes, theta = (32, 32), (10000.0, 500.0)
    kw = dict(theta=theta, interleaved=interleaved)
    for p in (pos, pos.long(), (pos.float() / 7.0), pos[:1].expand(2, -1, -1), pos[0], pos.transpose(1, 2).contiguous().transpose(1, 2)):
        g = p.to(dev)
        if p.stride() != g.stride() and p.dim() == 3 and p.stride(0):
            g = p.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        got = rotary_axes(q.to(dev), k.to(dev), g, axes, **kw)
        check(got[0], q, p, axes, **kw)
        check(got[1], k, p, axes, **kw)
    # whole numbers in each type: the same bits; position zero: nothing turns
    a = rotary_axes(q.to(dev), None, pos.to(dev) // 512, axes, **kw)[0]
    assert torch.equal(a, rotary_axes(q.to(dev), None, (pos // 512).float().to(dev), axes, **kw)[0])
    assert torch.equal(rotary_axes(q.to(dev), None, torch.zeros_like(pos).to(dev), axes, **kw)[0], q.to(dev))


def test_strides_in_place_and_packed(dev):
    """q and k as parts of a fused projection's rows, turned in place; the same tokens packed."""
    from nunchaku_amd.ops import rotary_axes

    B, T, H, Hkv, D, axes = 2, 19, 6, 2, 72, (24, 24, 24)
    q, k, w, pos = inputs(B, T, H, Hkv, D, 3, torch.bfloat16, 5)
    qkv = torch.cat((q.flatten(2), k.flatten(2), k.flatten(2)), -1).to(dev)
    gq, gk, gv = (t.unflatten(-1, (-1, D)) for t in qkv.split([H * D, Hkv * D, Hkv * D], -1))
    want = rotary_axes(gq, gk, pos.to(dev), axes, norm_q=w[0].to(dev))
    check(want[0], q, pos, axes, weight=w[0])
    check(want[1], k, pos, axes)
    packed = rotary_axes(gq.flatten(0, 1), gk.flatten(0, 1), pos.flatten(0, 1).to(dev), axes, norm_q=w[0].to(dev))
    assert torch.equal(packed[0], want[0].flatten(0, 1)) and torch.equal(packed[1], want[1].flatten(0, 1))
    heads_first = gq.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rotary_axes(heads_first, None, pos.to(dev), axes, norm_q=w[0].to(dev))[0], want[0])
    rotary_axes(gq, gk, pos.to(dev), axes, norm_q=w[0].to(dev), out_q=gq, out_k=gk)
    assert torch.equal(gq, want[0]) and torch.equal(gk, want[1]) and torch.equal(gv.cpu(), k)


def test_norms_beyond_fp32(dev):
    """bf16 heads whose squares overflow fp32, or vanish in it."""
    from nunchaku_amd.ops import rotary_axes

    q, _, w, pos = inputs(1, 3, 4, 1, 128, 1, torch.bfloat16, 8)
    q[0, :, 1] *= 2.0**100
    q[0, :, 2] *= 2.0**-90
    for eps in (0.0, 1e-6):
        check(rotary_axes(q.to(dev), None, pos.to(dev), (128,), norm_q=w[0].to(dev), eps=eps)[0], q, pos, (128,), weight=w[0], eps=eps)
    assert torch.equal(rotary_axes(q[:, :0].to(dev), None, pos[:, :0].to(dev), (128,))[0], q[:, :0].to(dev))
