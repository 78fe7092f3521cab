"""The 8-bit linear operators on the GPU against the oracle: codes bit for bit, products against exact integer sums."""

import math

import pytest
import torch

from conftest import announce
from gpu_util import Guarded
from oracle import w8a8 as ow

pytestmark = pytest.mark.gpu
U32 = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16]


def rand(shape, seed, dtype, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if outliers:
        x[..., :: max(1, shape[-1] // 3)] *= 20
    return x.to(dtype)


def check_codes(codes, scales, want_codes, want_scales, rel):
    assert torch.equal(codes.cpu().view(want_codes.shape), want_codes), (codes.cpu().view(want_codes.shape) != want_codes).sum()
    got, want = scales.cpu().double().view(-1), want_scales.double().view(-1)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert ((got - want).abs()[fine] <= rel * want[fine]).all(), ((got - want).abs()[fine] / want[fine]).max()


# row lengths on both sides of every number of threads per row
SIZES = [(1, 16), (3, 64), (5, 240), (9, 256), (7, 272), (9, 512), (5, 528), (6, 1024), (3, 1040), (2100, 1040), (2050, 2048), (5, 2032), (2, 2048), (4, 2064), (3, 4096), (2, 4112), (2, 8192), (1, 8208), (3, 16384), (2, 16400), (3, 32768), (2, 32784), (1, 65536), (1157, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", SIZES)
def test_quantize(dev, M, K, dtype):
    from nunchaku_amd.ops import quantize_w8a8_act

    announce(f"quantize {M} x {K} {dtype}")
    x = rand((M, K), M + K, dtype)
    codes, scales = Guarded((M, K), torch.int8, dev), Guarded((M,), torch.float32, dev)
    got = quantize_w8a8_act(x.to(dev), codes.t, scales.t)
    assert got[0] is codes.t and got[1] is scales.t
    check_codes(*got, *ow.quantize_rows(x), 0.0)
    codes.check("codes")
    scales.check("scales")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", SIZES)
def test_norm(dev, M, K, residual, dtype):
    """Scales: the sum of squares adds positive terms along at most 64 + 22 additions (relative error U32 each, halved by the root),
    and seven more operations round once: 52 U32."""
    from nunchaku_amd.ops import rms_norm_quantize_w8a8

    announce(f"norm {M} x {K} residual {residual} {dtype}")
    x, w = rand((M, K), M + K, dtype), (1 + rand((K,), K, dtype, False).float() / 4).to(dtype)
    r = rand((M, K), K, dtype) if residual else None
    codes, scales, h = rms_norm_quantize_w8a8(x.to(dev), w.to(dev), None if r is None else r.to(dev))
    want = ow.rms_norm_quantize(x, w, r)
    check_codes(codes, scales, want[0], want[1], 52 * U32)
    assert (h is None) if r is None else torch.equal(h.cpu(), want[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_special_values(dev, dtype):
    """Zeros, the smallest and largest numbers, infinities and NaN: each in a row of its own, which alone shows it."""
    from nunchaku_amd.ops import quantize_w8a8_act, rms_norm_quantize_w8a8

    f = torch.finfo(dtype)
    x = rand((10, 4096), 1, dtype)
    x[1] = 0
    x[2] = f.tiny
    x[3] = 0
    x[3, 77] = f.smallest_normal / 4  # below the smallest normal number
    x[4, 5] = f.max
    x[5, 4095] = math.inf
    x[6, 0] = -math.inf
    x[7, 2048] = math.nan
    x[8] = math.nan
    announce(f"special values {dtype}")
    check_codes(*quantize_w8a8_act(x.to(dev)), *ow.quantize_rows(x), 0.0)
    x[4] = 0  # (its square would overflow fp32 in bf16; the test below)
    codes, scales, h = rms_norm_quantize_w8a8(x.to(dev), torch.ones(4096, dtype=dtype, device=dev), torch.zeros_like(x).to(dev), eps=1e-5)
    want = ow.rms_norm_quantize(x, torch.ones(4096, dtype=dtype), None, eps=1e-5)
    check_codes(codes, scales, want[0], want[1], 52 * U32)
    assert torch.equal(torch.isnan(h.cpu()), torch.isnan(x)) and torch.equal(h.cpu().nan_to_num(), x.nan_to_num())


def test_sum_of_squares_that_overflows_is_nan(dev):
    from nunchaku_amd.ops import rms_norm_quantize_w8a8

    x = rand((2, 64), 3, torch.bfloat16)
    x[1, 3] = 3e38
    codes, scales, _ = rms_norm_quantize_w8a8(x.to(dev), torch.ones(64, dtype=torch.bfloat16, device=dev))
    assert torch.isfinite(scales[0]) and torch.isnan(scales[1]) and not codes[1].any()


def test_fp16_sum_that_overflows_is_nan(dev):
    from nunchaku_amd.ops import rms_norm_quantize_w8a8

    x = rand((2, 64), 3, torch.float16)
    x[1, 3] = 60000.0
    codes, scales, h = rms_norm_quantize_w8a8(x.to(dev), torch.ones(64, dtype=torch.float16, device=dev), x.to(dev))
    assert torch.isinf(h[1, 3]) and torch.isnan(scales[1]) and torch.isfinite(scales[0])


def test_rows_of_longer_rows_and_in_place(dev):
    """Inputs that are columns of wider tensors, more dimensions, the residual updated in place; what lies beside the columns stays."""
    from nunchaku_amd.ops import quantize_w8a8_act, rms_norm_quantize_w8a8

    announce("strided rows")
    wide = rand((2, 7, 1024), 4, torch.bfloat16).to(dev)
    x, r = wide[..., 128:640], wide.flip(0).contiguous()[..., 512:]
    codes, scales = quantize_w8a8_act(x)
    assert codes.shape == (2, 7, 512) and scales.shape == (2, 7)
    check_codes(codes, scales, *ow.quantize_rows(x.cpu()), 0.0)
    w = torch.ones(512, dtype=torch.bfloat16, device=dev)
    want = ow.rms_norm_quantize(x.cpu(), w.cpu(), r.cpu())
    keep = r._base.clone() if r._base is not None else r.clone()
    codes, scales, h = rms_norm_quantize_w8a8(x, w, r, residual_out=r)
    assert h is r and torch.equal(r.cpu(), want[2])
    check_codes(codes, scales, want[0], want[1], 52 * U32)
    if r._base is not None:
        assert torch.equal(r._base.view(2, 7, 1024)[..., :512], keep.view(2, 7, 1024)[..., :512])
    # the stream in x's place
    x2, r2 = x.contiguous(), rand((2, 7, 512), 5, torch.bfloat16).to(dev)
    want = ow.rms_norm_quantize(x2.cpu(), w.cpu(), r2.cpu())
    assert rms_norm_quantize_w8a8(x2, w, r2, residual_out=x2)[2] is x2 and torch.equal(x2.cpu(), want[2])


def codes_of(rows, K, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8), torch.rand(rows, generator=g) * 0.02 + 1e-3


def check_gemm(got, act, wgt, sa, sw, bias, dtype):
    """Rounded: the sum to fp32, the factor, their product, the bias's addition (U32 relative to the main term, twice to the result at
    most), and the result to the type (half a step; below its smallest normal number half its smallest step)."""
    main = ow.gemm(act, wgt, sa, sw)
    want = main if bias is None else main + bias.double()
    bound = 4 * U32 * (main.abs() + want.abs()) + torch.finfo(dtype).eps / 2 * want.abs() * 1.0001 + (2.0**-25 if dtype == torch.float16 else 0)
    off = (got.cpu().double().view(want.shape) - want).abs() - bound
    assert (off <= 0).all(), (off.max(), (off > 0).sum())


GEMM_SIZES = [
    (1, 1, 16), (1, 7, 32), (1, 256, 4096), (2, 33, 80), (16, 48, 64), (17, 130, 1008), (32, 64, 528), (33, 64, 128), (33, 65, 144), (64, 7, 2064),
    (65, 200, 256), (127, 129, 112), (128, 384, 400), (200, 1000, 1040), (257, 513, 272), (505, 1152, 2304), (1000, 1, 640), (3, 5000, 2064),
    (4096, 1536, 144), (2049, 6145, 96), (4100, 4104, 208),
]


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, True), (torch.float16, False)])
@pytest.mark.parametrize("M,N,K", GEMM_SIZES)
def test_gemm(dev, M, N, K, dtype, bias):
    from nunchaku_amd.ops import gemm_w8a8

    announce(f"gemm {M} x {N} x {K} {dtype}")
    (act, sa), (wgt, sw) = codes_of(M, K, M), codes_of(N, K, N + 1)
    b = rand((N,), N, dtype) if bias else None
    out = Guarded((M, N), dtype, dev)
    got = gemm_w8a8(act.to(dev), wgt.to(dev), sa.to(dev), sw.to(dev), bias=None if b is None else b.to(dev), out=out.t)
    assert got is out.t
    check_gemm(got, act, wgt, sa, sw, b, dtype)
    out.check("out")


# every form of the kernel, whole and with K in parts (of which a small kernel adds the sums)
GEMM_FORMS = [
    (8, 8810, 144), (5, 30, 8208), (13, 100, 4112), (19, 44, 1488), (64, 7, 2064), (17, 700, 13728), (3052, 5, 1936), (8311, 4, 16), (6594, 4, 14496),
    (8483, 198, 48), (9971, 273, 48), (10, 8764, 10688), (8531, 643, 16), (67, 8993, 8928), (6615, 1807, 32), (414, 5461, 11840),
]


@pytest.mark.parametrize("M,N,K", GEMM_FORMS)
def test_gemm_forms(dev, M, N, K):
    """... and the same bits from run to run, and through a call that names its output."""
    from nunchaku_amd.ops import gemm_w8a8

    announce(f"gemm forms {M} x {N} x {K}")
    (act, sa), (wgt, sw) = codes_of(M, K, M), codes_of(N, K, N + 1)
    on = [t.to(dev) for t in (act, wgt, sa, sw)]
    b = rand((N,), N, torch.bfloat16).to(dev)
    got = gemm_w8a8(*on, bias=b)
    check_gemm(got, act, wgt, sa, sw, b.cpu(), torch.bfloat16)
    out = Guarded((M, N), torch.bfloat16, dev)
    for _ in range(3):
        assert torch.equal(gemm_w8a8(*on, bias=b, out=out.t), got)
    out.check("out")


def test_gemm_streams_and_graphs(dev):
    """Products with K in parts on a user's stream and in two captured graphs replayed in turn: workspaces are the calls' own."""
    from nunchaku_amd.ops import gemm_w8a8

    announce("gemm streams and graphs")
    sets = []
    for i, (M, N, K) in enumerate([(5, 500, 16384), (64, 700, 8208)]):
        (act, sa), (wgt, sw) = codes_of(M, K, i), codes_of(N, K, i + 7)
        sets.append([t.to(dev) for t in (act, wgt, sa, sw)])
    want = [gemm_w8a8(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [gemm_w8a8(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(gemm_w8a8(*s))
        graphs.append(g)
    for turn in range(4):
        for s in sets:
            s[0].bitwise_xor_(turn)
            s[2].mul_(1.25)
        eager = [gemm_w8a8(*s) for s in sets]
        for o in outs:
            o.zero_()
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_more_rows_than_a_launch_takes(dev):
    """2^25 rows a launch: the rows around that one, and the last."""
    from nunchaku_amd.ops import quantize_w8a8_act, rms_norm_quantize_w8a8

    announce("2^25 + 77 rows")
    M, K = (1 << 25) + 77, 16
    x = torch.randn(M, K, device=dev, dtype=torch.bfloat16)
    w = rand((K,), 1, torch.bfloat16, False)
    picks = [slice(0, 9), slice((1 << 25) - 5, (1 << 25) + 6), slice(M - 3, M)]
    codes, scales = quantize_w8a8_act(x)
    for p in picks:
        check_codes(codes[p], scales[p], *ow.quantize_rows(x[p].cpu()), 0.0)
    codes, scales, h = rms_norm_quantize_w8a8(x, w.to(dev), x)
    for p in picks:
        want = ow.rms_norm_quantize(x[p].cpu(), w, x[p].cpu())
        check_codes(codes[p], scales[p], want[0], want[1], 52 * U32)
        assert torch.equal(h[p].cpu(), want[2])


def test_gemm_largest_sums(dev):
    """K just below the limit with codes of the largest magnitude: the integer sums reach 2^31 - 127^2 and are still exact."""
    from nunchaku_amd.ops import gemm_w8a8

    K = 131056
    for M in (3, 40):
        announce(f"largest sums, {M} rows")
        act, wgt = torch.full((M, K), 127, dtype=torch.int8), torch.full((24, K), 127, dtype=torch.int8)
        wgt[1::2] = -128
        act[1::2] = -128
        one = torch.ones(1)
        got = gemm_w8a8(act.to(dev), wgt.to(dev), one.expand(M).contiguous().to(dev), one.expand(24).contiguous().to(dev))
        check_gemm(got, act, wgt, one.expand(M), one.expand(24), None, torch.bfloat16)


@pytest.mark.parametrize("M", [2, 24, 100, 700])
def test_gemm_rows_of_longer_rows(dev, M):
    from nunchaku_amd.ops import gemm_w8a8

    announce(f"gemm strided {M}")
    (act, sa), (wgt, sw) = codes_of(M, 512, 1), codes_of(96, 768, 2)
    wide = torch.full((M, 300), 7.0, dtype=torch.bfloat16, device=dev)
    for first in (0, 3):  # aligned for wide stores, and not
        out = wide[:, first:first + 96]
        gemm_w8a8(act.to(dev)[:, 96:400], wgt.to(dev)[:, 416:720], sa.to(dev), sw.to(dev), out=out)
        check_gemm(out.contiguous(), act[:, 96:400], wgt[:, 416:720], sa, sw, None, torch.bfloat16)
        assert (wide[:, 96 + first:] == 7).all() and (wide[:, :first] == 7).all()
        wide.fill_(7.0)


def test_gemm_nan_scale_stays_in_its_row(dev):
    from nunchaku_amd.ops import gemm_w8a8

    for M in (4, 80):
        (act, sa), (wgt, sw) = codes_of(M, 256, 1), codes_of(40, 256, 2)
        sa[1] = math.nan
        got = gemm_w8a8(act.to(dev), wgt.to(dev), sa.to(dev), sw.to(dev))
        assert torch.isnan(got[1]).all() and torch.isfinite(got[0]).all() and torch.isfinite(got[2:]).all()


def test_empty_calls(dev):
    from nunchaku_amd.ops import gemm_w8a8, quantize_w8a8_act, rms_norm_quantize_w8a8

    x = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    codes, scales = quantize_w8a8_act(x)
    assert codes.shape == (0, 64) and scales.shape == (0,)
    assert rms_norm_quantize_w8a8(x, torch.ones(64, dtype=torch.bfloat16, device=dev), x)[2].shape == (0, 64)
    w, ws = torch.zeros(8, 64, dtype=torch.int8, device=dev), torch.ones(8, device=dev)
    assert gemm_w8a8(codes, w, scales, ws).shape == (0, 8)
    assert gemm_w8a8(w, w[:0], ws, ws[:0]).shape == (8, 0)


def test_refusals(dev):
    from nunchaku_amd.ops import gemm_w8a8, quantize_w8a8_act, rms_norm_quantize_w8a8

    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=dev)
    w = x[0].clone()
    with pytest.raises(NotImplementedError):
        quantize_w8a8_act(x.float())
    with pytest.raises(ValueError, match="K"):
        quantize_w8a8_act(x[:, :24].contiguous())
    with pytest.raises(ValueError, match="aligned"):
        quantize_w8a8_act(x[:, 4:52])
    with pytest.raises(ValueError, match="next to each other"):
        quantize_w8a8_act(x.t())
    with pytest.raises(ValueError, match="multiple of 8"):
        quantize_w8a8_act(torch.zeros(4, 68, dtype=torch.bfloat16, device=dev)[:, :64])
    with pytest.raises(ValueError, match="output"):
        quantize_w8a8_act(x, torch.empty(4, 32, dtype=torch.int8, device=dev))
    with pytest.raises(ValueError, match="weight"):
        rms_norm_quantize_w8a8(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        rms_norm_quantize_w8a8(x, w, x[:2])
    with pytest.raises(ValueError, match="residual_out"):
        rms_norm_quantize_w8a8(x, w, residual_out=x)
    with pytest.raises(ValueError, match="overlap"):
        rms_norm_quantize_w8a8(x, w, x.clone(), residual_out=x[:1].expand(4, 64))
    c, s = quantize_w8a8_act(x)
    with pytest.raises(ValueError, match="wgt"):
        gemm_w8a8(c, c[:, :32].contiguous(), s, s)
    with pytest.raises(ValueError, match="ascales"):
        gemm_w8a8(c, c, s[:2], s)
    with pytest.raises(ValueError, match="bias"):
        gemm_w8a8(c, c, s, s, bias=w[:4].half(), out_dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        gemm_w8a8(c, c, s, s, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="out must"):
        gemm_w8a8(c, c, s, s, out=torch.empty(4, 5, dtype=torch.bfloat16, device=dev))
    with pytest.raises(ValueError, match="overlap"):
        gemm_w8a8(c, c, s, s, out=torch.empty(4, dtype=torch.bfloat16, device=dev).expand(4, 4))
    with pytest.raises(ValueError, match="int8"):
        gemm_w8a8(c.view(torch.uint8), c, s, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer(dev, dtype):
    """The module's forward is its two operators, on a user's stream and replayed from a graph, and near the layer in 64 bits: every
    code is off by half a step at most, on both sides."""
    from nunchaku_amd.models import W8A8Linear

    torch.manual_seed(1)
    lin = torch.nn.Linear(320, 200, dtype=dtype)
    m = W8A8Linear.from_linear(lin, device=dev)
    for M in (1, 50, 300):
        announce(f"layer {M} {dtype}")
        x = rand((2, M, 320), M, dtype)
        y = m(x.to(dev))
        assert y.shape == (2, M, 200) and y.dtype == dtype
        codes, sa = ow.quantize_rows(x.view(-1, 320))
        check_gemm(y, codes, m.qweight.cpu(), sa, m.wscales.cpu(), lin.bias.detach(), dtype)
        xd, wd, sw = x.double().view(-1, 320), lin.weight.detach().double(), m.wscales.cpu().double()
        full = xd @ wd.t() + lin.bias.detach().double()
        # |x'w' - xw| <= |x'| |w' - w| + |w| |x' - x|, a code within 0.5005 steps
        most = (codes.double().abs().sum(1) * sa.double())[:, None] * sw * 0.5005 + sa.double()[:, None] * 0.5005 * wd.abs().sum(1)
        assert ((y.cpu().double().view(-1, 200) - full).abs() <= most + torch.finfo(dtype).eps * full.abs() + 1e-4).all()
    x = rand((1, 77, 320), 9, dtype).to(dev)
    want = m(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(m(x), want)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = m(x)
    for seed in (9, 10, 11):
        x.copy_(rand((1, 77, 320), seed, dtype))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m(x))


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_with_and_without_given_outputs(dev, dtype):
    """Calls that name their outputs, or come with an integer eps, take another way to the kernels: the same bits."""
    from nunchaku_amd.ops import gemm_w8a8, quantize_w8a8_act, rms_norm_quantize_w8a8

    x, r, w = (rand(s, i, dtype).to(dev) for i, s in enumerate([(2, 11, 528), (2, 11, 528), (528,)]))
    codes, scales = quantize_w8a8_act(x)
    out = torch.empty_like(codes), torch.empty_like(scales)
    quantize_w8a8_act(x, *out)
    assert torch.equal(codes, out[0]) and torch.equal(scales, out[1])
    wide = torch.zeros(22, 1056, dtype=dtype, device=dev)
    wide[:, 528:] = x.view(22, 528)
    again = quantize_w8a8_act(wide[:, 528:])
    assert torch.equal(codes.view(22, 528), again[0]) and torch.equal(scales.view(22), again[1])
    a = rms_norm_quantize_w8a8(x, w, r, 0.0)
    b = rms_norm_quantize_w8a8(x, w, r, 0)
    c = rms_norm_quantize_w8a8(x, w, r, 0.0, *out, residual_out=torch.empty_like(x))
    assert all(torch.equal(p, q) and torch.equal(p, s) for p, q, s in zip(a, b, c))
    wc, ws = quantize_w8a8_act(r[0])
    y = gemm_w8a8(codes, wc, scales, ws, out_dtype=dtype)
    z = torch.empty(2, 11, 11, dtype=dtype, device=dev)
    assert gemm_w8a8(codes, wc, scales, ws, out=z) is z and torch.equal(y, z)


def test_a_token_without_a_batch(dev):
    """[K] -> [N], as a linear layer takes it; and a layer cast with its model."""
    from nunchaku_amd.models import W8A8Linear

    torch.manual_seed(2)
    m = W8A8Linear.from_linear(torch.nn.Linear(528, 72)).to(dev).half()
    x = rand((3, 528), 1, torch.float16).to(dev)
    y = m(x)
    assert y.dtype == torch.float16 and y.shape == (3, 72)
    one = m(x[1])
    assert one.shape == (72,) and torch.equal(one, y[1])


def test_results_in_inference_mode_are_as_torch_makes_them(dev):
    from nunchaku_amd.ops import cross_attention, gemm_w8a8, rms_norm_quantize_w8a8

    def run():
        x = rand((4, 1, 64), 3, torch.bfloat16).to(dev)
        codes, scales, h = rms_norm_quantize_w8a8(x, x[0, 0], x)
        y = gemm_w8a8(codes, codes.view(4, 64), scales, scales.view(4))
        return codes, scales, h, y, cross_attention(x.view(1, 4, 1, 64), x.view(1, 4, 1, 64), x.view(1, 4, 1, 64))

    with torch.inference_mode():
        inside = run()
    outside = run()
    assert all(t.is_inference() and t.is_contiguous() for t in inside) and not any(t.is_inference() or t.requires_grad for t in outside)
    assert all(torch.equal(a, b) for a, b in zip(inside, outside))
    outside[3].add_(1)  # an ordinary tensor: changed in place, and counted
    assert outside[3]._version == 1
