"""CPU restatement, in 64 bits, of the operators between a block's linear layers: norms with gate, residual and modulation, rotary positions with
several axes, attention within sequences."""

from __future__ import annotations

import math

import torch


def gated_norm(x, residual=None, norm="rms", weight=None, gate=None, scale=None, shift=None, branch_weight=None, residual_scale=1.0, eps=1e-6):
    """(y, h, parts) of rows x [M, K]; vectors [K] or [M, K].  parts: what the bound of the fp32 steps is made of."""
    def wide(v):
        return None if v is None else v.double()

    b = x.double()
    if branch_weight is not None:
        b = b / torch.sqrt(b.square().mean(-1, keepdim=True) + eps) * wide(branch_weight)
    if gate is not None:
        b = b * wide(gate)
    h = b if residual is None else residual_scale * wide(residual) + b
    d = h - h.mean(-1, keepdim=True) if norm == "layer" else h
    std = torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    factor = torch.ones_like(h)
    if weight is not None:
        factor = factor * wide(weight)
    if scale is not None:
        factor = factor * (1 + wide(scale))
    y = d / std * factor
    if shift is not None:
        y = y + wide(shift)
    return y, h, {"b": b, "d": d, "std": std, "factor": factor}


def angles(positions, axes, theta=10000.0, spectrum="axis"):
    """positions [..., axes] -> angles [..., pairs]"""
    thetas = theta if isinstance(theta, (tuple, list)) else [theta] * len(axes)
    out, before = [], 0
    for a, n in enumerate(axes):
        for j in range(n // 2):
            e = 2 * j / n if spectrum == "axis" else 2 * (before + j) / sum(axes)
            out.append(positions[..., a].double() * math.pow(thetas[a], -e))
        before += n // 2
    return torch.stack(out, -1)


def pairs(R, interleaved):
    i = torch.arange(R // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)


def rotary(x, positions, axes, theta=10000.0, weight=None, eps=1e-6, interleaved=True, spectrum="axis"):
    """(y, size) of x [..., T, heads, D], positions [..., T, axes]; size: the magnitudes that each channel's sum has."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    phi = angles(positions, axes, theta, spectrum).unsqueeze(-2)
    i, j = pairs(sum(axes), interleaved)
    y, size = x.clone(), x.abs().clone()
    y[..., i] = x[..., i] * torch.cos(phi) - x[..., j] * torch.sin(phi)
    y[..., j] = x[..., i] * torch.sin(phi) + x[..., j] * torch.cos(phi)
    size[..., i] = size[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, size


def self_attention(q, k, v, causal=False, scale=None):
    """One sequence: q [m, H, D], k and v [n, Hkv, D] -> out [m, H, D]; a query without keys gets zeros, a key that it does not see has no part in it,
    whatever it holds."""
    (m, H, D), n = q.shape, k.shape[0]
    G = H // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    seen = torch.arange(n) <= torch.arange(m)[:, None] + (n - m) if causal else torch.ones(m, n, dtype=torch.bool)
    out = torch.zeros(m, H, D, dtype=torch.float64)
    if n == 0:
        return out
    some = seen.any(1)
    for h in range(H):
        values = v[:, h // G].double()
        e = (q[:, h].double() @ k[:, h // G].double().t() * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(e[some], -1).masked_fill(~seen[some], 0.0)
        bad = ~torch.isfinite(values)
        y = p @ values.masked_fill(bad, 0.0)
        y[(seen[some].double() @ bad.double()) > 0] = math.nan
        out[some, h] = y
    return out
