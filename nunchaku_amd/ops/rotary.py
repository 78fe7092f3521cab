"""Rotary positions with several axes for queries and keys (``rotary_axes``)."""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _native as nv
from .w8a8 import DTYPES

POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
SPECTRA = {"axis": 0, "head": 1}


def _heads(t: torch.Tensor, name: str, packed: bool) -> tuple[int, int, int]:
    """(batch, token, head) strides; of a dimension of one element, none."""
    s, n = t.stride(), t.shape
    if n[-1] > 1 and s[-1] != 1:
        raise ValueError(f"the elements of a head of {name} must be next to each other (strides {s})")
    s = tuple(a if b > 1 else 0 for a, b in zip(s[:-1], n[:-1]))
    return (0, *s) if packed else s


def rotary_axes(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    axes: tuple[int, ...] | list[int],
    theta: float | tuple[float, ...] | list[float] = 10000.0,
    norm_q: torch.Tensor | None = None,
    norm_k: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = True,
    spectrum: str = "axis",
    out_q: torch.Tensor | None = None,
    out_k: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotates ``q`` [B, T, H, D] and ``k`` [B, T, Hkv, D] (or packed: [T, H, D]; ``k`` may be None), bf16 or fp16, by ``positions`` of one to four axes
    (time, height, width), behind an RMS norm of every head where ``norm_q`` / ``norm_k`` [D] are given.  Returns (q, k).

    ``axes``: the channels of each axis, even numbers; the R = sum(axes) first channels of a head are rotated, the others pass (normed).  Pair i of
    them is (2 i, 2 i + 1), or (i, i + R / 2) with ``interleaved`` false (R is then a multiple of 16).  Axis a has the next axes[a] / 2 pairs.  Pair j of an
    axis of n channels turns by position * theta^(-2 j / n) (``spectrum`` "axis"); with "head" pair i of the head turns by its axis' position *
    theta^(-2 i / R), as where the axes share one spectrum.  ``theta``: one number, or one for each axis.
    ``positions`` int32, int64 or fp32 (between whole numbers, too) [B, T, len(axes)] or [T, len(axes)], by any strides.  An angle is right to 2^-55 of
    itself before its whole revolutions are dropped: positions up to 2^31 lose nothing that fp32 could hold, one of 2^40 up to 3e-5 radians.  The rest is fp32, rounded once.

    D is a multiple of 8 up to 256.  q and k go by their strides (multiples of 8, elements of a head next to each other), as parts of a fused
    projection do.  ``out_q`` and ``out_k`` take the results when given; they may be ``q`` and ``k`` themselves.  Forward only."""
    if out_q is None and out_k is None:
        y = nv.host().rotary_axes(q, k, positions, axes, theta, norm_q, norm_k, eps, interleaved, spectrum)
        if y is not None:
            return y
    # not the plain case: say what is wrong, or take the call with the caller's outputs or on another device than the current one
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must live on a GPU (got {t.device}); this path has no CPU implementation")
        if t.dtype not in DTYPES:
            raise NotImplementedError(f"{name} must be bf16 or fp16, got {t.dtype}")
        if t.dim() not in (3, 4):
            raise ValueError(f"{name} must be [B, T, heads, D] or [T, heads, D], got {tuple(t.shape)}")
    packed = q.dim() == 3
    if k is not None and (k.dtype != q.dtype or k.device != q.device or k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)}: the same type, device, tokens and head size")
    B, T = (1, q.shape[0]) if packed else q.shape[:2]
    H, D = q.shape[-2:]
    Hkv = 0 if k is None else k.shape[-2]
    axes = [int(n) for n in axes]
    A = len(axes)
    if not 1 <= A <= 4 or any(n <= 0 or n % 2 for n in axes) or sum(axes) > D:
        raise ValueError(f"axes must be one to four even positive numbers of at most {D} channels together, got {axes}")
    thetas = [float(theta)] * A if isinstance(theta, (int, float)) else [float(x) for x in theta]
    if len(thetas) != A or not all(0.0 < x < math.inf for x in thetas):
        raise ValueError(f"theta must be a positive number, or one for each axis, got {theta}")
    if spectrum not in SPECTRA:
        raise ValueError(f'spectrum must be "axis" or "head", got {spectrum!r}')
    if positions.device != q.device or positions.dtype not in POSITION_TYPES:
        raise ValueError(f"positions must be int32, int64 or fp32 on {q.device}, got {positions.dtype} on {positions.device}")
    if positions.shape not in ((T, A), (B, T, A)) or (packed and positions.dim() != 2):
        raise ValueError(f"positions must be [{T}, {A}]{'' if packed else f' or [{B}, {T}, {A}]'}, got {tuple(positions.shape)}")
    for name, w in (("norm_q", norm_q), ("norm_k", norm_k)):
        if w is not None and (w.device != q.device or w.dtype != q.dtype or w.shape != (D,) or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {q.dtype} vector of {D} elements on {q.device}")
    if k is None and (norm_k is not None or out_k is not None):
        raise ValueError("norm_k and out_k belong to k: none is given")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be a finite number not below zero, got {eps}")
    outs = []
    for name, t, o in (("out_q", q, out_q), ("out_k", k, out_k)):
        if t is not None and o is None:
            o = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        elif t is not None:
            if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device:
                raise ValueError(f"{name} must be {t.dtype} {tuple(t.shape)} on {t.device}")
            if any(n > 1 and s == 0 for n, s in zip(o.shape, o.stride())):
                raise ValueError(f"{name} must not be an expanded tensor")
        outs.append(o)
    out_q, out_k = outs
    if B * T == 0 or H + Hkv == 0:
        return out_q, out_k
    if H == 0 or (k is not None and Hkv == 0):
        raise ValueError(f"q and k must have heads, got {H} and {Hkv}")
    i64x3, none = ctypes.c_int64 * 3, (0, 0, 0)
    ps = tuple(a if n > 1 else 0 for a, n in zip(positions.stride(), positions.shape))
    args = nv.RotaryAxesArgs(
        q.data_ptr(), nv.ptr(k), out_q.data_ptr(), nv.ptr(out_k), nv.ptr(norm_q), nv.ptr(norm_k), positions.data_ptr(), B, T, H, Hkv, D, A,
        (ctypes.c_int64 * 4)(*axes), (ctypes.c_double * 4)(*thetas), i64x3(*_heads(q, "q", packed)), i64x3(*(none if k is None else _heads(k, "k", packed))),
        i64x3(*_heads(out_q, "out_q", packed)), i64x3(*(none if k is None else _heads(out_k, "out_k", packed))), i64x3(*(ps if len(ps) == 3 else (0, *ps))),
        eps, POSITION_TYPES[positions.dtype], not interleaved, SPECTRA[spectrum], DTYPES[q.dtype],
    )
    nv.launch(nv.lib().svdq_rotary_axes, ctypes.byref(args), q.device)
    return out_q, out_k
