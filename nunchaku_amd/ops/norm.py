"""The norms before and behind a block with its gate, residual and modulation (``gated_norm``)."""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _native as nv
from .w8a8 import DTYPES, _row_stride
from .w8a8 import _rows as _filled_rows

NORMS = {"rms": 0, "layer": 1}


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    return _filled_rows(x if x.numel() or x.dim() < 3 else x.flatten(0, -2), name)


def _vector(v: torch.Tensor | None, name: str, x: torch.Tensor, entries: int | None) -> tuple[int, int]:
    """(entry, token) strides of a gate, scale or shift for rows ``x``; ``entries``: of packed sequences."""
    if v is None:
        return 0, 0
    K = x.shape[-1]
    if v.device != x.device or v.dtype != x.dtype:
        raise ValueError(f"{name} must be {x.dtype} on {x.device}")
    if v.dim() == 0 or v.shape[-1] != K or (K > 1 and v.stride(-1) != 1):
        raise ValueError(f"the last dimension of {name} must be {K} elements next to each other, got {tuple(v.shape)} with strides {v.stride()}")
    if v.dim() == 1:
        return 0, 0
    if entries is not None:
        if v.shape != (entries, K):
            raise ValueError(f"{name} must be [{K}] or, one for each sequence, [{entries}, {K}], got {tuple(v.shape)}")
        return (v.stride(0) if entries > 1 else 0), 0
    if v.shape == x.shape:  # one for each token
        rows = _rows(v, name)
        ld = rows.stride(0) if rows.shape[0] > 1 else 0
        return ld * math.prod(x.shape[1:-1]), ld
    if x.dim() > 2 and v.numel() == x.shape[0] * K and v.shape[0] == x.shape[0]:  # one for each batch entry
        return (v.stride(0) if v.shape[0] > 1 else 0), 0
    raise ValueError(f"{name} must be [{K}], [{x.shape[0]}, {K}] or {tuple(x.shape)}, got {tuple(v.shape)}")


def gated_norm(
    x: torch.Tensor,
    residual: torch.Tensor | None = None,
    norm: str = "rms",
    weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    branch_weight: torch.Tensor | None = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
    cu_seqlens: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The end of one block and the beginning of the next for ``x`` bf16 / fp16 [..., K], a block's output:

        b = x, or x / sqrt(mean(x^2) + eps) * branch_weight
        h = residual_scale * residual + gate * b                      (gate * b without a residual)
        y = N(h) * weight * (1 + scale) + shift

    with N(h) = h / sqrt(mean(h^2) + eps) (``norm`` "rms") or (h - mean(h)) / sqrt(var(h) + eps) ("layer"); what is not given is left out.
    Returns (y, h), h None without a residual.  Everything between is fp32, y and h are rounded once: y is made of h as it was before.
    Rows of finite numbers whose squares leave fp32's range are normed in 64 bits.

    ``weight`` and ``branch_weight`` are [K].  ``gate``, ``scale`` and ``shift`` are [K], one for each batch entry (x [B, ..., K]: [B, K], parts of
    longer rows too) or for each token (the shape of x).  With ``cu_seqlens`` int32 [S + 1], x is [total, K], sequences one behind the other, and
    they are [K] or [S, K]; rows in no sequence become zeros, or are left as they are in ``out`` and ``residual_out`` when given.

    K is a multiple of 8 up to 32768.  The rows of x and residual may be parts of longer ones.  ``out`` may be ``x``, ``residual_out`` may be
    ``residual`` or ``x`` (the stream is then updated in place).  Forward only: results carry no gradient."""
    if out is None and residual_out is None:
        y = nv.host().gated_norm(x, residual, norm, weight, gate, scale, shift, branch_weight, residual_scale, eps, cu_seqlens)
        if y is not None:
            return y
    # not the plain case: say what is wrong, or take the call with the caller's outputs or on another device than the current one
    rows = _rows(x, "x")
    M, K = rows.shape
    if norm not in NORMS:
        raise ValueError(f'norm must be "rms" or "layer", got {norm!r}')
    for name, w in (("weight", weight), ("branch_weight", branch_weight)):
        if w is not None and (w.device != x.device or w.dtype != x.dtype or w.shape != (K,) or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {x.dtype} vector of {K} elements on {x.device}")
    entries = None
    if cu_seqlens is not None:
        if cu_seqlens.device != x.device or cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2 or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must be a contiguous int32 vector of at least 2 elements on {x.device}")
        if x.dim() != 2:
            raise ValueError(f"with cu_seqlens x is [total, K], got {tuple(x.shape)}")
        entries = cu_seqlens.shape[0] - 1
    strides = [_vector(v, name, x, entries) for name, v in (("gate", gate), ("scale", scale), ("shift", shift))]
    if residual is None and residual_out is not None:
        raise ValueError("residual_out is the sum with a residual: none is given")
    res = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)} on {x.device}")
        res = _rows(residual, "residual")
    if not (0.0 <= eps < math.inf):
        raise ValueError(f"eps must be a finite number not below zero, got {eps}")
    zero_rest = 0
    outs = []
    for bit, name, t, wanted in ((1, "out", out, True), (2, "residual_out", residual_out, residual is not None)):
        if t is None:
            zero_rest |= bit
            t = torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None
        elif t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f"{name} must be {x.dtype} {tuple(x.shape)} on {x.device}")
        outs.append(t)
    out, residual_out = outs
    o, ro = _rows(out, "out"), None if residual_out is None else _rows(residual_out, "residual_out")
    for name, t in (("out", o), ("residual_out", ro)):
        if t is not None and M > 1 and t.stride(0) < K:
            raise ValueError(f"the rows of {name} must not overlap")
    if ro is not None and ro.data_ptr() == o.data_ptr() and M:
        raise ValueError("out and residual_out must not be the same tensor")
    if M == 0:
        return out, residual_out
    i64x2 = ctypes.c_int64 * 2
    args = nv.GatedNormArgs(
        rows.data_ptr(), nv.ptr(res), o.data_ptr(), nv.ptr(ro), nv.ptr(weight), nv.ptr(branch_weight), nv.ptr(gate), nv.ptr(scale), nv.ptr(shift), nv.ptr(cu_seqlens),
        M, K, M // x.shape[0] if x.dim() > 2 else 1, entries or 0, _row_stride(rows), 0 if res is None else _row_stride(res), _row_stride(o), 0 if ro is None else _row_stride(ro),
        *(i64x2(*s) for s in strides), residual_scale, eps, NORMS[norm], zero_rest, DTYPES[x.dtype],
    )
    nv.launch(nv.lib().svdq_gated_norm, ctypes.byref(args), x.device)
    return out, residual_out
