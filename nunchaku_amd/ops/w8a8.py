"""8-bit linear layers: activations and weights as int8 codes with one fp32 scale per token and per output channel.

The layers a model keeps at 8 bits beside its 4-bit ones take three operators: ``quantize_w8a8_act`` or
``rms_norm_quantize_w8a8`` makes codes of activations (the former also of a weight's rows), ``gemm_w8a8`` multiplies them.
bf16 and fp16; forward only, like every operator here: results carry no gradient."""

from __future__ import annotations

import ctypes

import torch

from .. import _native as nv

DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """``x`` [..., K] as rows [M, K] without a copy; the elements of a row are next to each other, rows a multiple of 8 apart."""
    if not x.is_cuda:
        raise RuntimeError(f"{name} must live on a GPU (got {x.device}); this path has no CPU implementation")
    if x.dtype not in DTYPES:
        raise NotImplementedError(f"{name} must be bf16 or fp16, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError(f"{name} must have a last dimension of channels")
    if x.dim() != 2:
        try:
            x = x.view(-1, x.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name} {tuple(x.shape)} with strides {x.stride()} is not rows at one distance") from None
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError(f"the elements of a row of {name} must be next to each other (strides {x.stride()})")
    return x


def _row_stride(x: torch.Tensor) -> int:
    """Elements between rows; a single row has none to speak of."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _outputs(x: torch.Tensor, shape, output, oscales):
    M, K = x.shape
    if output is None:
        output = torch.empty(shape, dtype=torch.int8, device=x.device)
    elif output.device != x.device or output.dtype != torch.int8 or output.numel() != M * K or output.shape[-1] != K or not output.is_contiguous():
        raise ValueError(f"output must be a contiguous int8 tensor of {M} x {K} elements on {x.device}")
    if oscales is None:
        oscales = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    elif oscales.device != x.device or oscales.dtype != torch.float32 or oscales.numel() != M or not oscales.is_contiguous():
        raise ValueError(f"oscales must be a contiguous fp32 tensor of {M} elements on {x.device}")
    return output, oscales


def quantize_w8a8_act(x: torch.Tensor, output: torch.Tensor | None = None, oscales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``x`` bf16 / fp16 [..., K] to int8 codes [..., K] and fp32 scales [...]: with a = max(max |x|, 2^-100) of the row,
    code = round(x * (127 / a)) (ties to even), scale = a / 127.  A row that holds an infinity or a NaN gets the scale NaN and codes 0.

    K is a multiple of 16 up to 65536.  The rows of ``x`` may be parts of longer ones.  ``output`` and ``oscales`` take the results
    when given.  A weight [N, K] goes to its codes and channel scales the same way."""
    if output is None and oscales is None:
        y = nv.host().w8a8_quantize(x)
        if y is not None:
            return y
    # not the plain case: say what is wrong, or take the call with the caller's outputs or on another device than the current one
    rows = _rows(x, "x")
    codes, scales = _outputs(rows, x.shape, output, oscales)
    M, K = rows.shape
    if M == 0:
        return codes, scales
    args = nv.QuantizeW8A8Args(rows.data_ptr(), None, None, None, codes.data_ptr(), scales.data_ptr(), M, K, _row_stride(rows), 0, 0, 0.0, DTYPES[x.dtype])
    nv.launch(nv.lib().svdq_quantize_w8a8_act, ctypes.byref(args), x.device)
    return codes, scales


def rms_norm_quantize_w8a8(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    output: torch.Tensor | None = None,
    oscales: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """RMS norm of ``x`` bf16 / fp16 [..., K], behind the residual's addition, to int8 codes with a scale for each token.

    h = ``x`` + ``residual``, rounded to the type (``x`` itself without a residual); y = h / sqrt(mean(h^2) + eps) * ``weight``, not
    rounded; codes and scales of y as in ``quantize_w8a8_act``, but for the smallest rows: with a = max(max |h * weight|, 2^-100) a code is
    round(h * weight * (127 / a)) and the scale a / 127 / sqrt(mean(h^2) + eps).  A row whose sum of squares overflows fp32 gets the
    scale NaN and codes 0, too.  Returns (codes int8 [..., K], scales fp32 [...], h), h None without
    a residual.  ``residual_out`` takes h when given; it may be ``residual`` or ``x`` itself (the stream is then updated in place)."""
    if output is None and oscales is None and residual_out is None:
        y = nv.host().w8a8_norm(x, weight, residual, eps)
        if y is not None:
            return y
    rows = _rows(x, "x")
    M, K = rows.shape
    if weight.device != x.device or weight.dtype != x.dtype or weight.numel() != K or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous {x.dtype} vector of {K} elements on {x.device}")
    res = out = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)} on {x.device}")
        res = _rows(residual, "residual")
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        elif residual_out.shape != x.shape or residual_out.dtype != x.dtype or residual_out.device != x.device:
            raise ValueError(f"residual_out must be {x.dtype} {tuple(x.shape)} on {x.device}")
        out = _rows(residual_out, "residual_out")
        if M > 1 and out.stride(0) < K:
            raise ValueError("the rows of residual_out must not overlap")
    elif residual_out is not None:
        raise ValueError("residual_out is the sum with a residual: none is given")
    codes, scales = _outputs(rows, x.shape, output, oscales)
    if M == 0:
        return codes, scales, residual_out
    args = nv.QuantizeW8A8Args(
        rows.data_ptr(), nv.ptr(res), weight.data_ptr(), nv.ptr(out), codes.data_ptr(), scales.data_ptr(), M, K, _row_stride(rows),
        0 if res is None else _row_stride(res), 0 if out is None else _row_stride(out), eps, DTYPES[x.dtype],
    )
    nv.launch(nv.lib().svdq_rms_norm_quantize_w8a8, ctypes.byref(args), x.device)
    return codes, scales, residual_out


def _code_rows(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on a GPU (got {t.device}); this path has no CPU implementation")
    if t.dtype != torch.int8 or t.dim() == 0:
        raise ValueError(f"{name} must be int8 rows of codes, got {t.dtype} {tuple(t.shape)}")
    if t.dim() != 2:
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name} {tuple(t.shape)} with strides {t.stride()} is not rows at one distance") from None
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"the codes of a row of {name} must be next to each other (strides {t.stride()})")
    return t


def gemm_w8a8(
    act: torch.Tensor,
    wgt: torch.Tensor,
    ascales: torch.Tensor,
    wscales: torch.Tensor,
    bias: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """out[..., n] = sum_k act[..., k] * wgt[n, k] * (ascales[...] * wscales[n]) + bias[n], rounded once to bf16 or fp16.

    act int8 [..., K] and ascales fp32 [...] as ``quantize_w8a8_act`` writes them, wgt int8 [N, K], wscales fp32 [N], bias [N] of the
    output's type.  The integer sums are exact.  ``out_dtype``: bf16 by default, or the type of ``out`` or ``bias`` when given.
    K is a multiple of 16 below 131072; any numbers of rows and columns, from a single token on.  The rows of act, wgt and out may be
    parts of longer ones."""
    if out is None:
        y = nv.host().w8a8_gemm(act, wgt, ascales, wscales, bias, out_dtype)
        if y is not None:
            return y
    a, w = _code_rows(act, "act"), _code_rows(wgt, "wgt")
    M, K = a.shape
    N = w.shape[0]
    if wgt.dim() != 2 or w.shape[1] != K or w.device != a.device:
        raise ValueError(f"wgt must be [N, {K}] on {a.device}, got {tuple(wgt.shape)} on {wgt.device}")
    for name, t, n in (("ascales", ascales, M), ("wscales", wscales, N)):
        if t.device != a.device or t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp32 tensor of {n} elements on {a.device}")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else bias.dtype if bias is not None else torch.bfloat16
    if out_dtype not in DTYPES:
        raise NotImplementedError(f"the output must be bf16 or fp16, got {out_dtype}")
    if bias is not None and (bias.device != a.device or bias.dtype != out_dtype or bias.numel() != N or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous {out_dtype} vector of {N} elements on {a.device}")
    shape = (*act.shape[:-1], N)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=a.device)
        ld = N
    else:
        if out.shape != shape or out.dtype != out_dtype or out.device != a.device:
            raise ValueError(f"out must be {out_dtype} {shape} on {a.device}")
        o = _rows(out, "out")
        ld = _row_stride(o)
        if M > 1 and ld < N:
            raise ValueError("the rows of out must not overlap")
    if M == 0 or N == 0:
        return out
    args = nv.GemmW8A8Args(
        a.data_ptr(), w.data_ptr(), ascales.data_ptr(), wscales.data_ptr(), nv.ptr(bias), out.data_ptr(), M, N, K,
        _row_stride(a), _row_stride(w), ld, None, 0, DTYPES[out_dtype],
    )
    nv.launch_with_workspace(nv.lib().svdq_gemm_w8a8_workspace, nv.lib().svdq_gemm_w8a8, args, a.device)
    return out
