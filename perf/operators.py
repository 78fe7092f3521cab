"""What the speed of the 8-bit linear layer and of attention to an encoder's states is measured on: the operators of a
cross-attention block, from one token to whole images, through ``nunchaku_amd.ops``.

Kinds of case:

``quantize``  ``quantize_w8a8_act``: rows of M x K activations (or channels of a weight) to 8-bit codes with a scale each
``norm``      ``rms_norm_quantize_w8a8``: the residual's addition, RMS norm and 8-bit codes with a scale for each token
``gemm``      ``gemm_w8a8``: codes [M, K] times codes [N, K], scales for each token and channel, bias
``attention`` ``cross_attention``: Tq queries of each batch entry over Tk keys of an encoder, of which ``lengths`` / a mask /
              packed sequences leave some valid; H query heads share Hkv heads of keys and values

Codes are returned as the values they stand for (code times scale) in the type of the activations.  ``own`` false: the
plain form of each operator in elementary torch operations; true: the framework's operators.
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

#: rows whose largest magnitude is below this are quantized with the scale of this
FLOOR = 2.0**-100


def listed():
    return [
        # A handful of tokens being decoded, on their way into an output projection: pure latency.
        dict(name="quantize_bf16_8x4096", kind="quantize", M=8, K=4096, dtype="bf16"),
        # The hidden states of an MLP for a batch of images: bandwidth.
        dict(name="quantize_fp16_16384x8192", kind="quantize", M=16384, K=8192, dtype="fp16"),
        # One token of a decoder in front of its projection.
        dict(name="norm_fp16_1x4096", kind="norm", M=1, K=4096, dtype="fp16", residual=True),
        # The encoder's states of a few prompts, odd count, no residual.
        dict(name="norm_bf16_1157x2304", kind="norm", M=1157, K=2304, dtype="bf16", residual=False),
        # The tokens of a batch of images, residual stream updated on the way.
        dict(name="norm_bf16_9216x5120", kind="norm", M=9216, K=5120, dtype="bf16", residual=True),
        # One token times a layer: weight traffic.
        dict(name="gemm_bf16_1x4096x12288", kind="gemm", M=1, K=4096, N=12288, dtype="bf16", bias=True),
        # Key and value projection of a prompt's states, odd count of tokens.
        dict(name="gemm_fp16_505x2304x4608", kind="gemm", M=505, K=2304, N=4608, dtype="fp16", bias=True),
        # The first layer of an MLP on a full-size image's tokens, the largest.
        dict(name="gemm_bf16_4608x4096x16384", kind="gemm", M=4608, K=4096, N=16384, dtype="bf16", bias=False),
        # Single tokens of eight sequences over long encoder states of their own lengths, four query heads to a key head.
        dict(name="attention_bf16_decode_4096", kind="attention", B=8, Tq=1, Tk=4096, H=32, Hkv=8, D=128, dtype="bf16", valid="lengths", heads_first=False),
        # Image tokens over a prompt with holes in its mask, odd sizes, one prompt empty.
        dict(name="attention_bf16_1157x333_mask", kind="attention", B=4, Tq=1157, Tk=333, H=16, Hkv=16, D=72, dtype="bf16", valid="mask", heads_first=False),
        # Image tokens over prompts stored one behind the other.
        dict(name="attention_fp16_1024x300_packed", kind="attention", B=8, Tq=1024, Tk=300, H=32, Hkv=32, D=64, dtype="fp16", valid="packed", heads_first=False),
        # A full-size image over text and image keys, heads apart as the fused QKV projection writes them, rows behind the last token NaN.
        dict(name="attention_fp16_4096x4573", kind="attention", B=1, Tq=4096, Tk=4608, H=24, Hkv=24, D=128, dtype="fp16", valid="lengths", heads_first=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: 1 .. 16384 tokens, rows of 256 .. 16384 (any multiple of 16), any number of output
    channels, 1 .. 8192 keys, heads of 16 .. 128 (any multiple of 8); no more work than the largest listed one."""
    kind = rng.choice(["quantize", "norm", "norm", "gemm", "gemm", "gemm", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if kind in ("quantize", "norm"):
            c = dict(kind=kind, M=_log_int(rng, 1, 16384), K=16 * _log_int(rng, 16, 1024), dtype=dtype)
            if kind == "norm":
                c["residual"] = rng.random() < 0.6
        elif kind == "gemm":
            c = dict(kind=kind, M=_log_int(rng, 1, 9216), K=16 * _log_int(rng, 16, 1024), N=_log_int(rng, 64, 16384), dtype=dtype, bias=rng.random() < 0.5)
        else:
            Hkv = rng.choice([1, 2, 4, 8, 16, 20, 24])
            Tq = 1 if rng.random() < 0.3 else _log_int(rng, 1, 4608)
            c = dict(kind=kind, B=rng.choice([1, 1, 2, 4, 8]), Tq=Tq, Tk=_log_int(rng, 1, 8192), H=Hkv * rng.choice([1, 1, 1, 2, 4, 5]), Hkv=Hkv,
                     D=rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 112, 120, 128, 128]), dtype=dtype,
                     valid=rng.choice(["all", "lengths", "lengths", "mask", "packed"]), heads_first=rng.random() < 0.3)
            c["heads_first"] = c["heads_first"] and c["valid"] != "packed"
            if c["B"] * c["H"] * c["Tq"] * c["Tk"] > 24 * 4096 * 4608:  # (the plain form holds all scores)
                continue
        w = work(c)
        if w["bytes"] <= 6e8 and w["flops"] <= 2.0 * 4608 * 4096 * 16384:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _activations(M, K, dtype, g, dev):
    """Normal values, one channel in a hundred 20 times as large."""
    x = torch.randn(M, K, generator=g, device=dev)
    x[:, torch.randperm(K, generator=g, device=dev)[: math.ceil(K / 100)]] *= 20.0
    return x.to(dtype)


def _codes(x):
    """Codes and scales as a loader makes them from a layer's weights (and a user's earlier call from its activations)."""
    a = x.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
    return (x * (127.0 / a)).round_().to(torch.int8), (a / 127.0).view(-1)


def _valid_lengths(case, g, dev):
    """How many keys each batch entry has: the first all of them, one none where there are several."""
    B, Tk = case["B"], case["Tk"]
    n = torch.randint(max(1, Tk // 2), Tk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    n[0] = Tk
    if B == 1:
        n[0] = max(1, Tk - Tk // 130)
    elif case["valid"] != "packed":
        n[B - 1] = 0
    return n


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype}
    if case["kind"] in ("quantize", "norm"):
        M, K = case["M"], case["K"]
        state["x"] = _activations(M, K, dtype, g, dev)
        state["values"] = torch.empty(M, K, dtype=dtype, device=dev)
        if case["kind"] == "norm":
            state["weight"] = (1.0 + 0.2 * torch.randn(K, generator=g, device=dev)).to(dtype)
            state["residual"] = _activations(M, K, dtype, g, dev) if case["residual"] else None
        return state
    if case["kind"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        state["act"], state["ascales"] = _codes(_activations(M, K, dtype, g, dev).float())
        state["wgt"], state["wscales"] = _codes(0.02 * torch.randn(N, K, generator=g, device=dev))
        state["bias"] = (0.02 * torch.randn(N, generator=g, device=dev)).to(dtype) if case["bias"] else None
        return state
    B, Tq, Tk, H, Hkv, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hkv", "D"))

    def heads(T, n):
        t = torch.randn(B, n, T, D, generator=g, device=dev).to(dtype)
        return t.transpose(1, 2) if case["heads_first"] else t.transpose(1, 2).contiguous()

    state["q"], state["k"], state["v"] = 1.5 * heads(Tq, H), heads(Tk, Hkv), heads(Tk, Hkv)
    state.update(key_lengths=None, key_mask=None, cu_seqlens_k=None)
    at = torch.arange(Tk, device=dev)
    if case["valid"] == "lengths":
        state["key_lengths"] = _valid_lengths(case, g, dev)
        state["valid"] = at < state["key_lengths"][:, None]
    elif case["valid"] == "mask":
        state["key_mask"] = (at < _valid_lengths(case, g, dev)[:, None]) & (torch.rand(B, Tk, generator=g, device=dev) < 0.9)
        state["valid"] = state["key_mask"]
    elif case["valid"] == "packed":
        n = _valid_lengths(case, g, dev)
        state["valid"] = at < n[:, None]
        state["cu_seqlens_k"] = torch.cat((torch.zeros(1, dtype=torch.int32, device=dev), n.cumsum(0).to(torch.int32)))
        state["k"], state["v"] = state["k"][state["valid"]], state["v"][state["valid"]]
    else:
        state["valid"] = torch.ones(B, Tk, dtype=torch.bool, device=dev)
    if case["valid"] in ("lengths", "mask"):  # what lies behind the last token, as the fused QKV projection leaves it
        state["k"].masked_fill_(~state["valid"][:, :, None, None], math.nan)
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------


def _quantized(g, factor=1.0):
    """(codes as fp32, scales [M, 1]) of rows g whose values are factor * g."""
    a = g.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
    return torch.round(g * (127.0 / a)), a * factor / 127.0


def _plain_quantize(s):
    codes, scales = _quantized(s["x"].float())
    return (codes * scales).to(s["dtype"]), scales.view(-1)


def _plain_norm(s):
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["dtype"])
    x = h.float()
    codes, scales = _quantized(x * s["weight"].float(), torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6))
    out = ((codes * scales).to(s["dtype"]), scales.view(-1))
    return out if s["residual"] is None else (*out, h)


def _plain_gemm(s):
    y = (s["act"].float() @ s["wgt"].float().t()) * (s["ascales"][:, None] * s["wscales"])
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["dtype"])


def _padded(s, x):
    """Packed keys or values as a user's plain program unpacks them, zeros behind each sequence's last."""
    out = torch.zeros(*s["valid"].shape, *x.shape[1:], dtype=F32, device=x.device)
    out[s["valid"]] = x.float()
    return out


def _plain_attention(s):
    case = s["case"]
    G, D = case["H"] // case["Hkv"], case["D"]
    packed = case["valid"] == "packed"
    k, v = (_padded(s, s[n]) if packed else s[n].float() for n in "kv")
    keep = s["valid"][:, None, None, :]
    k = torch.where(s["valid"][:, :, None, None], k, 0.0).repeat_interleave(G, 2).permute(0, 2, 3, 1).contiguous()
    v = torch.where(s["valid"][:, :, None, None], v, 0.0).repeat_interleave(G, 2).transpose(1, 2).contiguous()
    scores = (s["q"].float().transpose(1, 2) @ k) * (1.0 / math.sqrt(D))
    scores = torch.where(keep, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3.0e38)  # (a row without keys has none)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    return out.transpose(1, 2).contiguous().to(s["dtype"])


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"quantize": _plain_quantize, "norm": _plain_norm, "gemm": _plain_gemm, "attention": _plain_attention}[kind](state)
    from nunchaku_amd import ops

    if kind == "quantize":
        codes, scales = ops.quantize_w8a8_act(state["x"])
        return torch.mul(codes, scales[:, None], out=state["values"]), scales
    if kind == "norm":
        codes, scales, h = ops.rms_norm_quantize_w8a8(state["x"], state["weight"], residual=state["residual"], eps=1e-6)
        out = (torch.mul(codes, scales[:, None], out=state["values"]), scales)
        return out if h is None else (*out, h)
    if kind == "gemm":
        return ops.gemm_w8a8(state["act"], state["wgt"], state["ascales"], state["wscales"], bias=state["bias"], out_dtype=state["dtype"])
    return ops.cross_attention(state["q"], state["k"], state["v"], key_lengths=state["key_lengths"], key_mask=state["key_mask"],
                               cu_seqlens_k=state["cu_seqlens_k"])


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gemm":
        y = torch.matmul(s["act"].to(F64), s["wgt"].to(F64).t()).mul_(s["ascales"].to(F64)[:, None]).mul_(s["wscales"].to(F64))
        return y if s["bias"] is None else y.add_(s["bias"].to(F64))
    if case["kind"] in ("quantize", "norm"):
        y, tail = s["x"].to(F64), ()
        if case["kind"] == "norm":
            if case["residual"]:
                h = (y + s["residual"].to(F64)).to(s["dtype"])  # (a sum of two such values is exact in 64 bits)
                y, tail = h.to(F64), (h.to(F64),)
            y = y / torch.sqrt((y * y).mean(1, keepdim=True) + 1e-6) * s["weight"].to(F64)
        step = torch.linalg.vector_norm(y, math.inf, dim=1, keepdim=True).clamp_min(FLOOR) / 127
        return (torch.round(y / step) * step, step[:, 0], *tail)
    # a batch entry and a head at a time: its valid keys alone
    B, H, G = case["B"], case["H"], case["H"] // case["Hkv"]
    out = torch.zeros(B, case["Tq"], H, case["D"], dtype=F64, device=s["q"].device)
    for b in range(B):
        if case["valid"] == "packed":
            span = s["cu_seqlens_k"].tolist()
            k, v = s["k"][span[b]:span[b + 1]], s["v"][span[b]:span[b + 1]]
        else:
            k, v = s["k"][b][s["valid"][b]], s["v"][b][s["valid"][b]]
        if k.shape[0] == 0:
            continue
        for h in range(H):
            e = torch.matmul(s["q"][b, :, h].to(F64), k[:, h // G].to(F64).t().contiguous()) / math.sqrt(case["D"])
            out[b, :, h] = torch.matmul(torch.softmax(e, 1), v[:, h // G].to(F64).contiguous())
    return out


def work(case):
    """Each input read once, each output written once (codes as the bytes they are)."""
    if case["kind"] in ("quantize", "norm"):
        M, K = case["M"], case["K"]
        more = (2.0 * K + (4.0 * M * K if case["residual"] else 0)) if case["kind"] == "norm" else 0
        return {"bytes": 3.0 * M * K + 4.0 * M + more, "flops": 4.0 * M * K}
    if case["kind"] == "gemm":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": 1.0 * K * (M + N) + 4.0 * (M + N) + (2.0 * N if case["bias"] else 0) + 2.0 * M * N, "flops": 2.0 * M * N * K}
    B, Tq, Tk, H, Hkv, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hkv", "D"))
    # (the share of the keys that is valid, on average over the seeds)
    share = 1.0
    if case["valid"] != "all":
        share = 1.0 if B == 1 else (1.0 + 0.75 * (B - (1 if case["valid"] == "packed" else 2))) / B
    if case["valid"] == "mask":
        share *= 0.9
    return {"bytes": 4.0 * B * Tq * H * D + 4.0 * B * Tk * share * Hkv * D, "flops": 4.0 * B * Tq * Tk * share * H * D}
