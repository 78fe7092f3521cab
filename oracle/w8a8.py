"""CPU restatement, in 64 bits, of the 8-bit linear operators and of attention to an encoder's states."""

from __future__ import annotations

import math

import torch

MIN_AMAX = 2.0**-100


def quantize_rows(g: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (int8) and scales (fp32) of rows ``g`` (fp32, exact), in the operator's own fp32 steps: these are bit-exact."""
    g = g.float()
    bad = ~torch.isfinite(g).all(-1)
    a = torch.where(bad, 1.0, g.abs().nan_to_num(0.0, 0.0, 0.0).amax(-1)).clamp_min(MIN_AMAX)
    codes = torch.round(torch.where(bad[..., None], 0.0, g) * (torch.tensor(127.0) / a)[..., None]).to(torch.int8)
    return codes, torch.where(bad, math.nan, a / 127.0)


def rms_norm_quantize(x, weight, residual=None, eps=1e-6):
    """(codes, scales in 64 bits, h): the codes in the operator's fp32 steps (bit-exact), the scales as the formula has them."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    g = h.float() * weight.float()
    codes, scales = quantize_rows(g)
    a = g.double().abs().amax(-1).clamp_min(MIN_AMAX)
    exact = a / torch.sqrt(h.double().square().mean(-1) + eps) / 127.0
    return codes, torch.where(torch.isnan(scales), math.nan, exact), h


def gemm(act, wgt, ascales, wscales, bias=None):
    y = (act.double() @ wgt.double().t()) * ascales.double().view(-1, 1) * wscales.double()
    return y if bias is None else y + bias.double()


def cross_attention(q, k, v, valid=None, scale=None):
    """q [B, Tq, H, D], k and v [B, Tk, Hkv, D], valid bool [B, Tk]: out [B, Tq, H, D] in 64 bits; rows without keys are zero."""
    B, Tq, H, D = q.shape
    G = H // k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Tq, H, D, dtype=torch.float64)
    for b in range(B):
        keep = torch.ones(k.shape[1], dtype=torch.bool) if valid is None else valid[b]
        kb, vb = k[b][keep].double(), v[b][keep].double()
        if not kb.shape[0]:
            continue
        for h in range(H):
            p = torch.softmax(q[b, :, h].double() @ kb[:, h // G].t() * scale, -1)
            out[b, :, h] = p @ vb[:, h // G]
    return out
