"""Softmax attention: to an encoder's states (``cross_attention``), and within sequences (``self_attention``)."""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _native as nv
from .w8a8 import DTYPES


def _strides(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(batch, token, head) strides; of a dimension of one element, none."""
    s, n = t.stride(), t.shape
    if n[-1] > 1 and s[-1] != 1:
        raise ValueError(f"the elements of a head of {name} must be next to each other (strides {s})")
    s = tuple(a if b > 1 else 0 for a, b in zip(s[:-1], n[:-1]))
    return s if len(s) == 3 else (0, *s)


def _vector(t: torch.Tensor, name: str, n: int, device: torch.device) -> None:
    if t.device != device or t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of {n} elements on {device}")


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    key_lengths: torch.Tensor | None = None,
    key_mask: torch.Tensor | None = None,
    cu_seqlens_k: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(scale * q k^T) v of the queries [B, Tq, H, D] over an encoder's keys and values [B, Tk, Hkv, D], bf16 or fp16;
    H / Hkv query heads share a head of keys.  Returns [B, Tq, H, D].

    Which keys count, at most one of: ``key_lengths`` int32 [B] (the first so many; values beyond 0..Tk count as the nearer of the
    two), ``key_mask`` bool [B, Tk] (True: counts), ``cu_seqlens_k`` int32 [B + 1] with k and v [total, Hkv, D], the sequences one
    behind the other.  A query without any key gets zeros; what k and v hold in places that do not count (NaN included) has no effect.

    D is a multiple of 8 up to 128.  Tensors go by their strides (multiples of 8, elements of a head next to each other): the fp16
    [B, heads, tokens, 128] outputs of ``fused_qkv_norm_rottary`` are taken as ``t.transpose(1, 2)``.  ``out`` takes the result when
    given and must not overlap the inputs.  ``scale``: 1 / sqrt(D) by default, positive.  Forward only: the result carries no gradient.

    Scores, maxima, exponentials and sums are fp32; the probabilities are rounded to the inputs' type for their product with v, which with
    the result's own rounding is up to one and a half steps of the type, relative to sum(p |v|) (typically a relative error of 0.0023 in bf16
    and 0.0003 in fp16, where the rounding of the result alone is 0.0017 and 0.0002).  Scores (scale * q k^T) up to 1.8e8 in fp16 and 1.4e9 in
    bf16 are in range; larger ones may give infinities or NaN."""
    if out is None:
        y = nv.host().attention(q, k, v, key_lengths, key_mask, cu_seqlens_k, scale)
        if y is not None:
            return y
    # not the plain case: say what is wrong, or take the call with the caller's output or on another device than the current one
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must live on a GPU (got {t.device}); this path has no CPU implementation")
        if t.dtype not in DTYPES:
            raise NotImplementedError(f"{name} must be bf16 or fp16, got {t.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must have one type and be on one device")
    if q.dim() != 4 or k.dim() != (4 if cu_seqlens_k is None else 3) or k.shape != v.shape:
        raise ValueError(f"q is [B, Tq, H, D], k and v [B, Tk, Hkv, D] (with cu_seqlens_k [total, Hkv, D]); got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Tq, H, D = q.shape
    Tk, Hkv = k.shape[-3], k.shape[-2]
    if k.shape[-1] != D or (cu_seqlens_k is None and k.shape[0] != B) or Hkv == 0 or H % Hkv:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)}: same batch and head sizes, Hkv divides H")
    if (key_lengths is not None) + (key_mask is not None) + (cu_seqlens_k is not None) > 1:
        raise ValueError("at most one of key_lengths, key_mask and cu_seqlens_k can be given")
    mask_stride = 0
    if key_lengths is not None:
        _vector(key_lengths, "key_lengths", B, q.device)
    elif cu_seqlens_k is not None:
        _vector(cu_seqlens_k, "cu_seqlens_k", B + 1, q.device)
    elif key_mask is not None:
        if key_mask.dtype != torch.bool:
            raise NotImplementedError(f"key_mask must be bool (True: the key counts), got {key_mask.dtype}: masks that are added to scores are not supported")
        if key_mask.shape != (B, Tk) or key_mask.device != q.device or (Tk > 1 and key_mask.stride(1) != 1):
            raise ValueError(f"key_mask must be [{B}, {Tk}] on {q.device}, a row's elements next to each other")
        mask_stride = key_mask.stride(0) if B > 1 else 0
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be a positive number, got {scale}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out must be {q.dtype} {tuple(q.shape)} on {q.device}")
        if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise ValueError("out must not be an expanded tensor")
    if out.numel() == 0:
        return out
    if Tk == 0:
        return out.zero_()
    i64x3 = ctypes.c_int64 * 3
    args = nv.CrossAttentionArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), nv.ptr(key_lengths), nv.ptr(key_mask), nv.ptr(cu_seqlens_k), None, 0,
        B, H, Hkv, D, Tq, Tk, i64x3(*_strides(q, "q")), i64x3(*_strides(k, "k")), i64x3(*_strides(v, "v")), i64x3(*_strides(out, "out")),
        mask_stride, scale, DTYPES[q.dtype],
    )
    nv.launch_with_workspace(nv.lib().svdq_cross_attention_workspace, nv.lib().svdq_cross_attention, args, q.device)
    return out


def self_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor | None = None,
    cu_seqlens_k: torch.Tensor | None = None,
    key_lengths: torch.Tensor | None = None,
    causal: bool = False,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(scale * q k^T) v of the queries of several sequences over the keys of the same sequence, causal or not; bf16 or fp16, H / Hkv query heads
    share a head of keys.  Returns the shape of q.

    Queries: q [B, Tq, H, D], or packed, [total, H, D] with ``cu_seqlens_q`` int32 [S + 1], the sequences one behind the other.
    Keys: k and v [B, Tk, Hkv, D] (packed queries: [S, Tk, Hkv, D], a cache), of which ``key_lengths`` int32 [B] says how many each sequence has (all by
    default; values beyond 0..Tk count as the nearer of the two), or packed, [total, Hkv, D] with ``cu_seqlens_k`` int32 [S + 1]: those of the queries
    by default.  Lengths stay on the GPU: nothing waits for them, and a captured graph takes others.

    ``causal``: query i of a sequence of n_q queries and n_k keys sees the keys j <= i + n_k - n_q; the last one sees all, so that new tokens see those
    before them.  A query without any key gets zeros.  What k and v hold for keys that a query does not see (NaN included) has no effect on it.  Rows of q in
    no sequence get zeros, or are left as they are in ``out`` when given.

    D is a multiple of 8 up to 128.  Tensors go by their strides (multiples of 8, elements of a head next to each other).  ``out`` takes the result
    when given and must not overlap the inputs.  ``scale``: 1 / sqrt(D) by default, positive.  Forward only: the result carries no gradient.  Precision
    and range of scores are those of ``cross_attention``; finite bf16 scores of a row that rise by more than 44 within 448 keys take 2.4 times as long.

    Batches without a causal mask can go to either operator: from about a thousand queries and keys on this one is faster (4608 tokens, 24 heads of 128 244 us,
    ``cross_attention`` 293), with some hundred keys or single tokens the other (300 tokens 9.4 us, this 11.1)."""
    if out is None:
        y = nv.host().self_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, key_lengths, causal, scale)
        if y is not None:
            return y
    # not the plain case: say what is wrong, or take the call with the caller's output or on another device than the current one
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must live on a GPU (got {t.device}); this path has no CPU implementation")
        if t.dtype not in DTYPES:
            raise NotImplementedError(f"{name} must be bf16 or fp16, got {t.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must have one type and be on one device")
    if q.dim() != (4 if cu_seqlens_q is None else 3) or k.dim() not in (3, 4) or k.shape != v.shape:
        raise ValueError(f"q is [B, Tq, H, D] (with cu_seqlens_q [total, H, D]), k and v [B, Tk, Hkv, D] or packed [total, Hkv, D]; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dim() == 3 and cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    if (k.dim() == 3) != (cu_seqlens_k is not None):
        raise ValueError("packed keys [total, Hkv, D] come with cu_seqlens_k, and only they")
    if key_lengths is not None and cu_seqlens_k is not None:
        raise ValueError("key_lengths are for keys [B, Tk, Hkv, D]: packed ones have cu_seqlens_k")
    offsets = cu_seqlens_q if cu_seqlens_q is not None else cu_seqlens_k
    S = q.shape[0] if cu_seqlens_q is None else offsets.shape[0] - 1 if offsets.dim() == 1 else -1
    H, D = q.shape[-2:]
    Tk, Hkv = k.shape[-3], k.shape[-2]
    for name, t in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        if t is not None:
            _vector(t, name, max(S, 0) + 1, q.device)
    if S < 1 and (cu_seqlens_q is not None or q.numel()):
        raise ValueError("cu_seqlens_q must hold the offsets of one sequence at least")
    if k.shape[-1] != D or (k.dim() == 4 and k.shape[0] != S) or Hkv == 0 or H % Hkv:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)} of {S} sequences: as many entries, the same head size, Hkv divides H")
    if key_lengths is not None:
        _vector(key_lengths, "key_lengths", S, q.device)
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be a positive number, got {scale}")
    zero_rest = out is None
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out must be {q.dtype} {tuple(q.shape)} on {q.device}")
        if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise ValueError("out must not be an expanded tensor")
    if out.numel() == 0:
        return out
    keys, values = (k, v) if Tk else (torch.zeros(*k.shape[:-3], 1, Hkv, D, dtype=k.dtype, device=k.device) for _ in "kv")
    if Tk == 0 and key_lengths is None and cu_seqlens_k is None:
        key_lengths = torch.zeros(S, dtype=torch.int32, device=q.device)
    elif Tk == 0:
        # (no rows of keys at all: whatever the lengths say, no sequence has any)
        key_lengths, cu_seqlens_k = (key_lengths.new_zeros(S), None) if key_lengths is not None else (None, torch.zeros_like(cu_seqlens_k))
    i64x3 = ctypes.c_int64 * 3
    args = nv.SelfAttentionArgs(
        q.data_ptr(), keys.data_ptr(), values.data_ptr(), out.data_ptr(), nv.ptr(cu_seqlens_q), nv.ptr(cu_seqlens_k), nv.ptr(key_lengths), None, 0,
        S, H, Hkv, D, q.shape[-3], keys.shape[-3], i64x3(*_strides(q, "q")), i64x3(*_strides(keys, "k")), i64x3(*_strides(values, "v")), i64x3(*_strides(out, "out")),
        scale, causal, zero_rest, DTYPES[q.dtype],
    )
    nv.launch_with_workspace(nv.lib().svdq_self_attention_workspace, nv.lib().svdq_self_attention, args, q.device)
    return out
