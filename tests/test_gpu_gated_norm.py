"""Norms with gate, residual and modulation on the GPU against the oracle in 64 bits.

Tolerance.  U = 2^-24 (fp32's rounding), u = half a step of the type.  A thread adds at most 32 numbers, then come 6 exchanges and 16 waves: a sum of K
numbers of one sign is right to 55 U of it, one of squares to 56 U.  The root of the mean plus eps: half of that and 4 more, 32 U; all factors of b: 36 U |b|.  With
dh = 36 U |b| + 2 U (|b| + |h|) for h, 60 U mean |h| for the mean, d = h - m and its error dd = dh + mean(dh) + 60 U mean |h| + U |d|:
    1 / std is off by rms(dd) / std + 32 U, relative;  y by |factor| (dd + |d| (rms(dd) / std + 38 U)) / std + U |y| + u |y|,
times 1.01 for the products of errors, and half the smallest step where the types end."""

import math

import pytest
import torch

from conftest import announce
from gpu_util import Guarded
from oracle import blocks

pytestmark = pytest.mark.gpu
U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16]


def bounds(y, h, parts, dtype, layer):
    u, end = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    b, d, std, factor = (parts[n] for n in ("b", "d", "std", "factor"))
    dh = 36 * U * b.abs() + 2 * U * (b.abs() + h.abs())
    dd = dh + U * d.abs()
    if layer:
        dd = dd + dh.mean(-1, keepdim=True) + 60 * U * h.abs().mean(-1, keepdim=True)
    r = dd.square().mean(-1, keepdim=True).sqrt() / std
    by = factor.abs() * (dd + d.abs() * (r + 38 * U)) / std + U * y.abs() + u * y.abs()
    return 1.01 * by + end, 1.01 * (dh + u * h.abs()) + end


def check(got, x, residual=None, norm="rms", **kw):
    """got (y, h) of rows [M, K]; vectors in kw [K] or [M, K]"""
    y, h, parts = blocks.gated_norm(x, residual, norm, **kw)
    by, bh = bounds(y, h, parts, x.dtype, norm == "layer")
    for name, g, want, bound in (("y", got[0], y, by), ("h", got[1], h, bh)):
        if g is None:
            assert name == "h" and residual is None
            continue
        assert g.dtype == x.dtype
        off = (g.cpu().double().view(want.shape) - want).abs() - bound
        assert (off <= 0).all(), (name, off.max().item(), (off > 0).sum().item(), off.numel())


def rand(*shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


# every number of threads and pieces: one row, odd numbers of rows, channels on both sides of each
SHAPES = [(1, 8), (3, 24), (5, 256), (2, 264), (7, 512), (9, 520), (3, 1024), (4, 1032), (2, 2048), (5, 2056), (1157, 2304), (3, 4096), (2, 4104), (3, 8192), (2, 8200), (2, 16384), (1, 16392), (2, 32768)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("shape", SHAPES)
def test_everything_at_once(dev, shape, norm, dtype):
    from nunchaku_amd.ops import gated_norm

    announce(f"gated_norm {shape} {norm} {dtype}")
    M, K = shape
    x, res = (rand(M, K, dtype=dtype, seed=i, scale=3.0) for i in (1, 2))
    v = {n: rand(K, dtype=dtype, seed=10 + i, scale=0.5) for i, n in enumerate(("weight", "gate", "scale", "shift", "branch_weight"))}
    y, h = Guarded((M, K), dtype, dev), Guarded((M, K), dtype, dev)
    got = gated_norm(x.to(dev), res.to(dev), norm=norm, residual_scale=0.75, out=y.t, residual_out=h.t, **{n: t.to(dev) for n, t in v.items()})
    assert got[0] is y.t and got[1] is h.t
    check(got, x, res, norm, residual_scale=0.75, **v)
    y.check("y")
    h.check("h")
    again = gated_norm(x.to(dev), res.to(dev), norm=norm, residual_scale=0.75, **{n: t.to(dev) for n, t in v.items()})
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_what_is_not_given_is_left_out(dev, norm):
    from nunchaku_amd.ops import gated_norm

    names = ("residual", "weight", "gate", "scale", "shift", "branch_weight")
    x = rand(6, 328, dtype=torch.bfloat16, seed=0, scale=2.0)
    for mask in range(1 << len(names)):
        given = {n: rand(6, 328, dtype=x.dtype, seed=5) if n == "residual" else rand(328, dtype=x.dtype, seed=i + 6) for i, n in enumerate(names) if mask >> i & 1}
        got = gated_norm(x.to(dev), norm=norm, **{n: t.to(dev) for n, t in given.items()})
        assert (got[1] is None) == ("residual" not in given)
        check(got, x, given.pop("residual", None), norm, **given)


def test_vectors_of_entries_and_tokens(dev):
    """[B, K] as parts of a modulation layer's row, [B, 1, K], [B, T, K]; x a part of longer rows."""
    from nunchaku_amd.ops import gated_norm

    B, T, K, dtype = 3, 5, 712, torch.float16
    x, res, tok = (rand(B, T, K, dtype=dtype, seed=i) for i in range(3))
    mod = rand(B, 3 * K, dtype=dtype, seed=4)
    gate, scale, shift = mod.to(dev).chunk(3, 1)
    rows = [t.repeat_interleave(T, 0) for t in mod.chunk(3, 1)]
    check(gated_norm(x.to(dev), res.to(dev), "layer", gate=gate, scale=scale[:, None], shift=shift), x.view(-1, K), res.view(-1, K), "layer", gate=rows[0], scale=rows[1], shift=rows[2])
    check(gated_norm(x.to(dev), res.to(dev), gate=tok.to(dev), scale=scale), x.view(-1, K), res.view(-1, K), gate=tok.view(-1, K), scale=rows[1])
    wide = rand(B * T, 2 * K + 8, dtype=dtype, seed=7)
    part, per_row = wide.to(dev)[:, 8:K + 8], wide.to(dev)[:, K + 8:]
    check(gated_norm(part, shift=per_row), wide[:, 8:K + 8], shift=wide[:, K + 8:])
    one = rand(B, K, dtype=dtype, seed=9)  # a token of each entry
    check(gated_norm(one.to(dev), gate=gate), one, gate=mod[:, :K])


@pytest.mark.parametrize("K", [64, 512, 4096])
@pytest.mark.parametrize("lens", [[7], [0, 3, 0, 0, 5, 1, 0], [1] * 130, [5, 200]])
def test_packed_sequences(dev, lens, K):
    """Each sequence its gate, scale and shift; rows in front of the first and behind the last are zeros, or left as they are."""
    from nunchaku_amd.ops import gated_norm

    announce(f"gated_norm packed {len(lens)} {K}")
    dtype, S, front, behind = torch.bfloat16, len(lens), 2, 3
    total = front + sum(lens) + behind
    cu = torch.tensor([front + sum(lens[:i]) for i in range(S + 1)], dtype=torch.int32)
    x, res = (rand(total, K, dtype=dtype, seed=i) for i in range(2))
    mod = [rand(S, K, dtype=dtype, seed=3 + i) for i in range(3)]
    entry = torch.repeat_interleave(torch.arange(S), torch.tensor(lens))
    inside = slice(front, total - behind)
    call = lambda **kw: gated_norm(x.to(dev), res.to(dev), gate=mod[0].to(dev), scale=mod[1].to(dev), shift=mod[2].to(dev), cu_seqlens=cu.to(dev), **kw)  # noqa: E731
    y, h = call()
    check((y[inside], h[inside]), x[inside], res[inside], gate=mod[0][entry], scale=mod[1][entry], shift=mod[2][entry])
    outside = torch.ones(total, dtype=torch.bool, device=dev)
    outside[inside] = False
    assert not y[outside].any() and not h[outside].any()
    o, ho = (torch.full((total, K), 7.0, dtype=dtype, device=dev) for _ in range(2))
    call(out=o, residual_out=ho)
    assert torch.equal(o[inside], y[inside]) and torch.equal(ho[inside], h[inside])
    assert (o[outside] == 7).all() and (ho[outside] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place(dev, dtype):
    from nunchaku_amd.ops import gated_norm

    x, res, g = rand(33, 1000, dtype=dtype, seed=1).to(dev), rand(33, 1000, dtype=dtype, seed=2).to(dev), rand(1000, dtype=dtype, seed=3).to(dev)
    want = gated_norm(x, res, "layer", gate=g)
    a, b = x.clone(), res.clone()
    got = gated_norm(a, b, "layer", gate=g, out=a, residual_out=b)
    assert got[0] is a and got[1] is b and torch.equal(a, want[0]) and torch.equal(b, want[1])


@pytest.mark.parametrize("K", [40, 1000, 8192])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_squares_beyond_fp32(dev, norm, K):
    """bf16 rows of numbers around 2^100, 2^-80 and of one large mean: finite and right; a row with an infinity or a NaN is NaN, its neighbours are not."""
    from nunchaku_amd.ops import gated_norm

    x = rand(6, K, dtype=torch.float32, seed=K)
    x[1] *= 2.0**100
    x[2] *= 2.0**-80
    x[3] = 1000.0 + x[3]
    x = x.to(torch.bfloat16)
    for after in (None, torch.ones(K, dtype=torch.bfloat16)):
        for eps in (0.0, 1e-6):
            got = gated_norm(x.to(dev), norm=norm, eps=eps, branch_weight=None if after is None else after.to(dev))
            check((got[0][:4], None), x[:4], None, norm, eps=eps, branch_weight=after)
    x[4, 3], x[5, 7] = math.inf, math.nan
    y = gated_norm(x.to(dev), norm=norm)[0].cpu()
    assert y[4:].isnan().any(1).all() and y[:4].isfinite().all()


def test_zero_rows(dev):
    from nunchaku_amd.ops import gated_norm

    x = torch.zeros(3, 256, dtype=torch.float16, device=dev)
    s = torch.full((256,), 2.0, dtype=torch.float16, device=dev)
    for norm in ("rms", "layer"):
        assert torch.equal(gated_norm(x, norm=norm, shift=s)[0], s.expand(3, 256))
    y, h = gated_norm(x[:0], x[:0])
    assert y.shape == h.shape == (0, 256)


def test_no_rows(dev):
    """Empty batches and entries: empty results, vectors of their shape taken all the same."""
    from nunchaku_amd.ops import gated_norm

    for shape in ((0, 16), (0, 5, 16), (3, 0, 16), (2, 0, 4, 16)):
        x = torch.empty(shape, dtype=torch.float16, device=dev)
        y, h = gated_norm(x, x.clone(), gate=x.clone(), scale=torch.ones(16, dtype=x.dtype, device=dev))
        assert y.shape == h.shape == x.shape
        out = torch.empty_like(x)
        assert gated_norm(x, out=out)[0] is out
    with pytest.raises(ValueError):
        gated_norm(torch.empty(2, 3, 0, dtype=torch.float16, device=dev), gate=torch.empty(2, 3, 0, dtype=torch.float16, device=dev))


@pytest.mark.parametrize("tokens", [5, 2**32, 2**40 + 1])
def test_entries_longer_than_the_rows(dev, tokens):
    """The C entry: all rows belong to the first entry, however many rows one would have."""
    import ctypes

    from nunchaku_amd import _native as nv

    x, gate, y = rand(5, 64, dtype=torch.float16, seed=1), rand(5, 64, dtype=torch.float16, seed=2), torch.empty(5, 64, dtype=torch.float16, device=dev)
    gx, gg, two = x.to(dev), gate.to(dev), ctypes.c_int64 * 2
    args = nv.GatedNormArgs(gx.data_ptr(), None, y.data_ptr(), None, None, None, gg.data_ptr(), None, None, None, 5, 64, tokens, 0, 64, 0, 64, 0, two(1 << 40, 64), two(0, 0), two(0, 0),
                            1.0, 1e-6, 0, 0, 1)
    assert nv.lib().svdq_gated_norm(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    check((y, None), x, gate=gate)
