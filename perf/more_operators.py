"""What the speed of the operators between a transformer block's linear layers is measured on, from one decoded token to
whole videos, through ``nunchaku_amd.ops``.

Kinds of case:

``norm``       ``gated_norm``: a block's output, normed or not, joins the residual stream through a gate; the stream is normed for the
               next block and modulated.  ``entries`` says who shares a gate, scale and shift: every token of a batch entry, or of a
               packed sequence
``rotary``     ``rotary_axes``: norms and rotation of q and k by positions of one to three axes (time, height, width)
``attention``  ``self_attention``: queries of packed sequences or of a batch to the keys of the same sequence, causal or not, ``new``
               queries at the end of ``lens`` keys each; H query heads share Hkv heads of keys and values

Lengths stand in a case as text, "5,130" for two sequences of 5 and of 130 tokens.  ``own`` false: the plain form of each operator in
elementary torch operations; true: the framework's operators.
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # One token of a decoder between two blocks with norms before and behind each: pure latency.
        dict(name="norm_fp16_1x4096_after", kind="norm", entries="batch", B=1, lens="1", K=4096, norm="rms", dtype="fp16", residual=True, after=True, gate=False, modulate=False),
        # Image tokens on their way into the first block, odd count, an entry's timestep modulates them.
        dict(name="norm_bf16_2x1157x2304", kind="norm", entries="batch", B=2, lens="1157", K=2304, norm="layer", dtype="bf16", residual=False, after=False, gate=False, modulate=True),
        # Images of different sizes and their prompts one behind the other, each with a timestep of its own, norms before and behind the block.
        dict(name="norm_fp16_packed_7943x2560_after", kind="norm", entries="packed", B=6, lens="4096,77,2305,1,1024,440", K=2560, norm="rms", dtype="fp16", residual=True, after=True,
             gate=True, modulate=True),
        # The tokens of two full-size images: gate, residual, layer norm and modulation in one pass.
        dict(name="norm_bf16_2x4608x5120", kind="norm", entries="batch", B=2, lens="4608", K=5120, norm="layer", dtype="bf16", residual=True, after=False, gate=True, modulate=True),
        # One token of eight sequences being decoded, far positions, halves of a head paired.
        dict(name="rotary_bf16_8x1_far", kind="rotary", B=8, T=1, H=32, Hkv=8, D=128, axes="128", interleaved=False, spectrum="axis", positions="far", norm=False, dtype="bf16"),
        # Text and image tokens of a vision model: part of a head is rotated, positions between whole numbers.
        dict(name="rotary_fp16_2x1157_part", kind="rotary", B=2, T=1157, H=16, Hkv=16, D=80, axes="16,24,24", interleaved=False, spectrum="head", positions="resized", norm=True, dtype="fp16"),
        # A video's tokens, norms of q and k fused, three axes.
        dict(name="rotary_bf16_32760_video", kind="rotary", B=1, T=32760, H=24, Hkv=24, D=128, axes="44,42,42", interleaved=True, spectrum="axis", positions="grid", norm=True, dtype="bf16"),
        # A few short prompts in a text encoder with a causal mask.
        dict(name="attention_fp16_77_causal", kind="attention", form="batch", lens="77,77,77,77", new="77,77,77,77", H=12, Hkv=12, D=64, causal=True, dtype="fp16"),
        # Chunks of new tokens, one of them single, behind what their sequences have in the cache already, four query heads to a key head.
        dict(name="attention_bf16_chunks_8192", kind="attention", form="cache", lens="8192,4000,1023,130,6001,8000,64,2500", new="1,32,17,1,64,5,64,8", H=32, Hkv=8, D=128, causal=True,
             dtype="bf16"),
        # Images of different sizes one behind the other, every token sees its whole image.
        dict(name="attention_fp16_packed_images", kind="attention", form="packed", lens="4096,1024,2305,555", new="4096,1024,2305,555", H=16, Hkv=16, D=72, causal=False, dtype="fp16"),
        # Prompts of different lengths one behind the other, grouped heads.
        dict(name="attention_bf16_packed_prompts", kind="attention", form="packed", lens="4096,1,300,2047,129,1600", new="4096,1,300,2047,129,1600", H=32, Hkv=8, D=128, causal=True, dtype="bf16"),
        # One long prompt, the largest.
        dict(name="attention_bf16_16384_causal", kind="attention", form="batch", lens="16384", new="16384", H=24, Hkv=8, D=128, causal=True, dtype="bf16"),
    ]


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_norm(rng, dtype):
    packed = rng.random() < 0.3
    B = rng.choice([2, 3, 5, 8]) if packed else rng.choice([1, 1, 2, 4])
    lens = [_log_int(rng, 1, 8192) for _ in range(B)] if packed else [_log_int(rng, 1, 16384 // B)]
    residual = rng.random() < 0.7
    return dict(kind="norm", entries="packed" if packed else "batch", B=B, lens=_text(lens), K=8 * _log_int(rng, 32, 2048), norm=rng.choice(["rms", "layer"]), dtype=dtype,
                residual=residual, after=residual and rng.random() < 0.4, gate=residual and rng.random() < 0.6, modulate=packed or rng.random() < 0.6)


def _draw_rotary(rng, dtype):
    D = rng.choice([32, 40, 64, 64, 72, 80, 96, 112, 128, 128, 128])
    interleaved = rng.random() < 0.6
    # (halves are whole groups of eight channels)
    rotated = D if interleaved or D % 16 == 0 else D - 8
    if rng.random() < 0.25 and rotated > 32:
        rotated -= 16
    count = rng.choice([1, 2, 3, 3])
    rest, axes = rotated, []
    for i in range(count - 1):
        axes.append(max(2, rest // (count - i) // 4 * 4 + rng.choice([-2, 0, 2])))
        rest -= axes[-1]
    Hkv = rng.choice([1, 2, 4, 8, 12, 16, 24])
    return dict(kind="rotary", B=rng.choice([1, 1, 2, 4, 8]), T=1 if rng.random() < 0.2 else _log_int(rng, 1, 32768), H=Hkv * rng.choice([1, 1, 1, 2, 4]), Hkv=Hkv, D=D, axes=_text([*axes, rest]),
                interleaved=interleaved, spectrum=rng.choice(["axis", "axis", "head"]), positions=rng.choice(["grid", "far", "resized"]), norm=rng.random() < 0.6, dtype=dtype)


def _draw_attention(rng, dtype):
    form = rng.choice(["batch", "packed", "packed", "packed", "cache", "cache"])
    Hkv = rng.choice([1, 2, 4, 8, 8, 12, 16, 24])
    S = rng.choice([1, 2, 4, 8]) if form == "batch" else rng.choice([1, 2, 3, 5, 8, 13])
    lens = [_log_int(rng, 1, 16384)] * S if form == "batch" else [_log_int(rng, 1, 8192) for _ in range(S)]
    new = [min(n, 1 if rng.random() < 0.4 else _log_int(rng, 1, 256)) for n in lens] if form == "cache" else lens
    return dict(kind="attention", form=form, lens=_text(lens), new=_text(new), H=Hkv * rng.choice([1, 1, 1, 2, 3, 4, 8]), Hkv=Hkv,
                D=rng.choice([32, 40, 64, 64, 72, 80, 96, 112, 128, 128, 128]), causal=form == "cache" or rng.random() < 0.7, dtype=dtype)


def draw(rng):
    """Another case of the same ranges: 1 .. 16384 tokens of 256 .. 16384 channels (any multiple of 8) for the norms, heads of 32 .. 128
    (multiples of 8), 1 .. 32768 tokens to rotate, up to 13 sequences of 1 .. 16384 tokens; no more work than the largest listed one."""
    most = {c["kind"]: work(c) for c in listed()}  # (the last of a kind is its largest)
    while True:
        make = rng.choice([_draw_norm, _draw_rotary, _draw_attention, _draw_attention])
        c = make(rng, rng.choice(["bf16", "bf16", "fp16"]))
        w = work(c)
        # (the plain form of attention works out all scores of a sequence, masked or not)
        scores = sum(m * n for m, n in zip(_numbers(c["new"]), _numbers(c["lens"]))) * c["H"] if c["kind"] == "attention" else 0
        if w["bytes"] <= most[c["kind"]]["bytes"] and w["flops"] <= most[c["kind"]]["flops"] and scores <= 24 * 16384**2:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _activations(rows, K, dtype, g, dev):
    """Normal values, one channel in a hundred 20 times as large."""
    x = torch.randn(rows, K, generator=g, device=dev)
    x[:, torch.randperm(K, generator=g, device=dev)[: math.ceil(K / 100)]] *= 20.0
    return x.to(dtype)


def _weight(n, dtype, g, dev):
    return (1.0 + 0.2 * torch.randn(n, generator=g, device=dev)).to(dtype)


def _offsets(lens, dev):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


def _prepare_norm(case, g, dev, dtype):
    lens, B, K = _numbers(case["lens"]), case["B"], case["K"]
    packed = case["entries"] == "packed"
    rows = sum(lens) if packed else B * lens[0]
    shape = (rows, K) if packed else (B, lens[0], K)
    # gate, scale and shift side by side, as a modulation layer writes them
    modulation = (0.5 * torch.randn(B, 3 * K, generator=g, device=dev)).to(dtype)
    gate, scale, shift = modulation.chunk(3, 1)
    return dict(
        x=_activations(rows, K, dtype, g, dev).view(shape),
        residual=_activations(rows, K, dtype, g, dev).view(shape) if case["residual"] else None,
        after=_weight(K, dtype, g, dev) if case["after"] else None,
        weight=_weight(K, dtype, g, dev) if case["norm"] == "rms" else None,
        gate=gate if case["gate"] else None,
        scale=scale if case["modulate"] else None,
        shift=shift if case["modulate"] else None,
        cu_seqlens=_offsets(lens, dev) if packed else None,
        entry=torch.repeat_interleave(torch.arange(B, device=dev), torch.tensor(lens if packed else lens * B, device=dev), output_size=rows),
    )


def _positions(case, g, dev):
    """[B, T, axes]: the places of a grid of tokens behind some of text, far ones, or a grid's of another resolution."""
    B, T, A = case["B"], case["T"], len(_numbers(case["axes"]))
    at = torch.arange(T, device=dev)
    width = max(1, int(math.sqrt(T / 4.0)))
    columns = [at // (width * width), at // width % width, at % width] if A == 3 else [at // width, at % width] if A == 2 else [at]
    p = torch.stack(columns, -1).to(torch.int32).expand(B, T, A)
    if case["positions"] == "far":
        return p + torch.randint(1 << 10, 1 << 20, (B, 1, 1), generator=g, device=dev, dtype=torch.int32)
    if case["positions"] == "resized":
        return p.float() * (0.25 + torch.rand(B, 1, 1, generator=g, device=dev))
    return (p * (at >= T // 10)[:, None]).contiguous()


def _prepare_rotary(case, g, dev, dtype):
    B, T, H, Hkv, D = (case[n] for n in ("B", "T", "H", "Hkv", "D"))
    # q, k and v side by side, as a fused projection writes them
    qkv = torch.empty(B, T, (H + 2 * Hkv) * D, dtype=dtype, device=dev)
    for b in range(B):
        qkv[b] = 1.5 * torch.randn(T, (H + 2 * Hkv) * D, generator=g, device=dev)
    q, k, _ = qkv.split([H * D, Hkv * D, Hkv * D], -1)
    norms = [_weight(D, dtype, g, dev) if case["norm"] else None for _ in "qk"]
    return dict(q=q.unflatten(-1, (H, D)), k=k.unflatten(-1, (Hkv, D)), positions=_positions(case, g, dev), norm_q=norms[0], norm_k=norms[1], axes=_numbers(case["axes"]))


def _prepare_attention(case, g, dev, dtype):
    lens, new, H, Hkv, D = _numbers(case["lens"]), _numbers(case["new"]), case["H"], case["Hkv"], case["D"]
    S = len(lens)
    state = dict(cu_seqlens_q=None, cu_seqlens_k=None, key_lengths=None)
    if case["form"] == "cache":
        # a cache of one size for all sequences: NaN behind what they have written
        T = max(lens)
        state["q"] = (1.5 * torch.randn(sum(new), H, D, generator=g, device=dev)).to(dtype)
        state["k"], state["v"] = (torch.randn(S, T, Hkv, D, generator=g, device=dev).to(dtype) for _ in "kv")
        state["key_lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        state["cu_seqlens_q"] = _offsets(new, dev)
        behind = torch.arange(T, device=dev) >= state["key_lengths"][:, None]
        for n in "kv":
            state[n].masked_fill_(behind[:, :, None, None], math.nan)
        return state
    qkv = torch.randn(sum(lens), (H + 2 * Hkv) * D, generator=g, device=dev).to(dtype)
    qkv[:, : H * D] *= 1.5
    q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], -1)
    state["q"], state["k"], state["v"] = (t.unflatten(-1, (-1, D)) for t in (q, k, v))
    if case["form"] == "batch":
        for n in "qkv":
            state[n] = state[n].unflatten(0, (S, lens[0]))
    else:
        state["cu_seqlens_q"] = _offsets(lens, dev)
    return state


_PREPARE = {"norm": _prepare_norm, "rotary": _prepare_rotary, "attention": _prepare_attention}


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    return {"case": case, "dtype": dtype, **_PREPARE[case["kind"]](case, g, dev, dtype)}


# ---- the plain forms --------------------------------------------------------------------------------------------------


def _plain_norm(s):
    K = s["x"].shape[-1]
    h = s["x"].float().view(-1, K)
    if s["after"] is not None:
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["after"].float()
    if s["gate"] is not None:
        h = h * s["gate"].float()[s["entry"]]
    if s["residual"] is not None:
        h = s["residual"].float().view(-1, K) + h
    y = h if s["case"]["norm"] == "rms" else h - h.mean(-1, keepdim=True)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    if s["weight"] is not None:
        y = y * s["weight"].float()
    if s["scale"] is not None:
        y = y * (1.0 + s["scale"].float()[s["entry"]]) + s["shift"].float()[s["entry"]]
    y = y.to(s["dtype"]).view(s["x"].shape)
    return y if s["residual"] is None else (y, h.to(s["dtype"]).view(s["x"].shape))


def _angles(s):
    """[B, T, pairs] in 64 bits: each pair's frequency times its axis' position."""
    case, axes = s["case"], s["axes"]
    freqs, columns, before = [], [], 0
    for a, n in enumerate(axes):
        i = torch.arange(n // 2, dtype=F64, device=s["q"].device)
        freqs.append(10000.0 ** (-(2.0 * i / n if case["spectrum"] == "axis" else 2.0 * (i + before) / sum(axes))))
        columns += [a] * (n // 2)
        before += n // 2
    return s["positions"].double()[..., torch.tensor(columns, device=s["q"].device)] * torch.cat(freqs)


def _plain_rotary(s):
    angles = _angles(s)
    cos, sin = torch.cos(angles).float()[:, :, None], torch.sin(angles).float()[:, :, None]
    R = 2 * cos.shape[-1]
    out = []
    for x, w in ((s["q"], s["norm_q"]), (s["k"], s["norm_k"])):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        y = x.clone()
        at = (slice(0, R, 2), slice(1, R, 2)) if s["case"]["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        y[..., at[0]] = x[..., at[0]] * cos - x[..., at[1]] * sin
        y[..., at[1]] = x[..., at[0]] * sin + x[..., at[1]] * cos
        out.append(y.to(s["dtype"]))
    return tuple(out)


def _sequences(s):
    """(queries [m, H, D], keys and values [n, Hkv, D]) of every sequence."""
    case = s["case"]
    lens, new = _numbers(case["lens"]), _numbers(case["new"])
    at = 0
    for b, (m, n) in enumerate(zip(new, lens)):
        if case["form"] == "batch":
            yield s["q"][b], s["k"][b], s["v"][b]
        elif case["form"] == "packed":
            yield tuple(s[x][at:at + n] for x in "qkv")
        else:
            yield s["q"][at:at + m], s["k"][b, :n], s["v"][b, :n]
        at += m


def _plain_attention(s):
    case = s["case"]
    H, G, D = case["H"], case["H"] // case["Hkv"], case["D"]
    outs = []
    for q, k, v in _sequences(s):
        m, n = q.shape[0], k.shape[0]
        q = q.float().transpose(0, 1).contiguous()
        k = k.float().repeat_interleave(G, 1).permute(1, 2, 0).contiguous()
        v = v.float().repeat_interleave(G, 1).transpose(0, 1).contiguous()
        out = torch.empty(m, H, D, dtype=s["dtype"], device=q.device)
        at_once = max(1, (1 << 28) // (m * n))  # heads whose scores are held together
        for h in range(0, H, at_once):
            scores = (q[h:h + at_once] @ k[h:h + at_once]) * (1.0 / math.sqrt(D))
            if case["causal"]:
                behind = torch.arange(n, device=q.device) > torch.arange(n - m, n, device=q.device)[:, None]
                scores.masked_fill_(behind, -math.inf)
            p = torch.exp(scores.sub_(scores.amax(-1, keepdim=True)))
            out[:, h:h + at_once] = ((p @ v[h:h + at_once]) / p.sum(-1, keepdim=True)).transpose(0, 1).to(s["dtype"])
        outs.append(out)
    return torch.stack(outs) if case["form"] == "batch" else torch.cat(outs)


_PLAIN = {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention}


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return _PLAIN[kind](state)
    from nunchaku_amd import ops

    s, case = state, state["case"]
    if kind == "norm":
        y, h = ops.gated_norm(s["x"], s["residual"], norm=case["norm"], weight=s["weight"], gate=s["gate"], scale=s["scale"], shift=s["shift"], branch_weight=s["after"],
                              cu_seqlens=s["cu_seqlens"], eps=EPS)
        return y if h is None else (y, h)
    if kind == "rotary":
        return ops.rotary_axes(s["q"], s["k"], s["positions"], s["axes"], norm_q=s["norm_q"], norm_k=s["norm_k"], interleaved=case["interleaved"], spectrum=case["spectrum"], eps=EPS)
    return ops.self_attention(s["q"], s["k"], s["v"], cu_seqlens_q=s["cu_seqlens_q"], cu_seqlens_k=s["cu_seqlens_k"], key_lengths=s["key_lengths"], causal=case["causal"])


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------


def _exact_norm(s):
    def per_row(v):
        return 0.0 if v is None else v.to(F64).index_select(0, s["entry"])

    K = s["x"].shape[-1]
    branch = s["x"].to(F64).reshape(-1, K)
    if s["after"] is not None:
        branch = branch / torch.sqrt((branch * branch).sum(1, keepdim=True) / K + EPS) * s["after"].to(F64)
    if s["gate"] is not None:
        branch = branch * per_row(s["gate"])
    h = branch if s["residual"] is None else s["residual"].to(F64).reshape(-1, K) + branch
    mean = h.sum(1, keepdim=True) / K if s["case"]["norm"] == "layer" else 0.0
    y = (h - mean) / torch.sqrt(((h - mean) ** 2).sum(1, keepdim=True) / K + EPS)
    if s["weight"] is not None:
        y = y * s["weight"].to(F64)
    y = (y + y * per_row(s["scale"]) + per_row(s["shift"])).reshape(s["x"].shape)
    return y if s["residual"] is None else (y, h.reshape(s["x"].shape))


def _exact_rotary(s):
    case, axes = s["case"], s["axes"]
    R, dev = sum(axes), s["q"].device
    turn = []  # a unit complex number for each token and pair
    for a, n in enumerate(axes):
        for i in range(n // 2):
            power = 2.0 * i / n if case["spectrum"] == "axis" else (sum(axes[:a]) + 2.0 * i) / R
            angle = s["positions"][..., a].to(F64) * math.exp(-power * math.log(10000.0))
            turn.append(torch.polar(torch.ones_like(angle), angle))
    turn = torch.stack(turn, -1)
    out = []
    for x, w in ((s["q"], s["norm_q"]), (s["k"], s["norm_k"])):
        y = torch.empty(x.shape, dtype=F64, device=dev)
        for h in range(x.shape[2]):
            z = x[:, :, h].to(F64)
            if w is not None:
                z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS) * w.to(F64)
            y[:, :, h] = z
            pairs = z[..., :R].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1)).movedim(-1 if case["interleaved"] else -2, 0)
            moved = torch.complex(pairs[0], pairs[1]) * turn
            y[:, :, h, :R] = torch.stack((moved.real, moved.imag), -1 if case["interleaved"] else -2).flatten(-2)
        out.append(y)
    return tuple(out)


def _exact_attention(s):
    # a sequence and a head at a time, some thousand queries of it: softmax over the keys up to a query's own
    case = s["case"]
    G, outs = case["H"] // case["Hkv"], []
    for q, k, v in _sequences(s):
        m, n = q.shape[0], k.shape[0]
        out = torch.empty(q.shape, dtype=F64, device=q.device)
        for h in range(case["H"]):
            keys, values = k[:, h // G].to(F64).t().contiguous(), v[:, h // G].to(F64).contiguous()
            for first in range(0, m, 4096):
                rows = q[first:first + 4096, h].to(F64)
                seen = n - m + first + rows.shape[0] if case["causal"] else n  # of the last of these queries
                e = torch.matmul(rows, keys[:, :seen].contiguous()) / math.sqrt(case["D"])
                if case["causal"]:
                    e = torch.where(torch.ones_like(e, dtype=torch.bool).tril_(seen - rows.shape[0]), e, -math.inf)
                out[first:first + 4096, h] = torch.matmul(torch.softmax(e, 1), values[:seen])
        outs.append(out)
    return torch.stack(outs) if case["form"] == "batch" else torch.cat(outs)


def exact(case, seed):
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention}[case["kind"]](prepare(case, seed))


def work(case):
    """Each input read once, each output written once; the products of the keys that a query sees."""
    if case["kind"] == "norm":
        lens, B, K = _numbers(case["lens"]), case["B"], case["K"]
        rows = sum(lens) if case["entries"] == "packed" else B * lens[0]
        vectors = case["after"] + (case["norm"] == "rms") + B * (case["gate"] + 2 * case["modulate"])
        return {"bytes": 2.0 * K * (rows * (4 if case["residual"] else 2) + vectors), "flops": 10.0 * rows * K}
    if case["kind"] == "rotary":
        tokens, heads, A = case["B"] * case["T"], case["H"] + case["Hkv"], len(_numbers(case["axes"]))
        return {"bytes": 4.0 * tokens * heads * case["D"] + 4.0 * tokens * A + (4.0 * case["D"] if case["norm"] else 0), "flops": (7.0 if case["norm"] else 3.0) * tokens * heads * case["D"]}
    lens, new, H, Hkv, D = _numbers(case["lens"]), _numbers(case["new"]), case["H"], case["Hkv"], case["D"]
    seen = sum(m * n - (m * (m - 1) // 2 if case["causal"] else 0) for m, n in zip(new, lens))
    return {"bytes": 4.0 * sum(new) * H * D + 4.0 * sum(lens) * Hkv * D, "flops": 4.0 * seen * H * D}
