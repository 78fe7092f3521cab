"""Rotary positions far from zero on the GPU against angles of 60 digits.

Heads hold (a, 0) in every pair, so that the result is (a cos phi, a sin phi), a power of two.  Tolerance, U = 2^-24, u = half a step of the type: 4 U of each function,
U |phi| for the angle as fp32 has it, less its whole revolutions, and the frequency's error, (3 j + 3 e log(theta) + 4) 2^-64 of the whole angle for pair
j, whose frequency is theta^-e; u of the result, half the smallest step where fp16 ends."""

import decimal
import math
import random

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu
U = 2.0**-24
PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def angles(positions, n, theta):
    """(phi less whole revolutions, its error) of positions (whole numbers or floats) and the pairs of an axis of n channels"""
    with decimal.localcontext() as c:
        c.prec = 75
        log = decimal.Decimal(theta).ln()
        freqs = [(-log * 2 * j / n).exp() for j in range(n // 2)]
        phi, off = [], []
        for x in positions:
            whole = [decimal.Decimal(x) * f for f in freqs]
            phi.append([float(w - (w / (2 * PI)).to_integral_value() * 2 * PI) for w in whole])
            off.append([abs(float(w)) * (3 * j + 3 * abs(float(log)) * 2 * j / n + 4) * 2.0**-64 for j, w in enumerate(whole)])
    return torch.tensor(phi, dtype=torch.float64), torch.tensor(off, dtype=torch.float64)


def positions(kind, count, seed):
    g = random.Random(seed)
    if kind == "int32":
        return torch.tensor([2**31 - 1, -(2**31), 2**31 - 2, *(g.choice([-1, 1]) * g.randint(2**30, 2**31 - 1) for _ in range(count - 3))], dtype=torch.int32)
    if kind == "fp32":
        return torch.tensor([g.choice([-1, 1]) * 10.0 ** g.uniform(5, 15) for _ in range(count)], dtype=torch.float32)
    bits = int(kind[6:])
    ends = [2**63 - 1, -(2**63), -(2**63) + 5] if bits == 63 else [2**bits + 1, -(2**bits) - 1, 2**bits - 1]
    return torch.tensor([*ends, *(g.choice([-1, 1]) * g.randint(2 ** (bits - 1), 2**bits - 1) for _ in range(count - 3))], dtype=torch.int64)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("theta", [10000.0, 500.0, 1e6])
@pytest.mark.parametrize("kind", ["int32", "fp32", "int64_31", "int64_40", "int64_53", "int64_54", "int64_63"])
def test_far_positions(dev, kind, theta, interleaved):
    from nunchaku_amd.ops import rotary_axes

    announce(f"rotary far {kind} {theta} {interleaved}")
    T, D, a = 1500, 128, 512.0
    pos = positions(kind, T, len(kind))
    q = torch.zeros(T, 1, D, dtype=torch.float16)
    first, second = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, D // 2), slice(D // 2, None))
    q[..., first] = a
    got = rotary_axes(q.to(dev), None, pos[:, None].to(dev), (D,), theta=theta, interleaved=interleaved)[0][:, 0].cpu().double()
    phi, off = angles(pos.tolist(), D, theta)
    for y, f, other in ((got[:, first], phi.cos(), phi.sin()), (got[:, second], phi.sin(), phi.cos())):
        want = a * f
        bound = 1.01 * (a * (4 * U * f.abs() + U * phi.abs() * other.abs() + off) + 2.0**-11 * want.abs()) + 2.0**-25
        over = (y - want).abs() - bound
        assert (over <= 0).all(), (over.max().item(), (over > 0).sum().item(), over.numel())
    if kind == "int64_31":  # whole numbers of another type: the same bits
        again = rotary_axes(q[3:].to(dev), None, pos[3:, None].int().to(dev), (D,), theta=theta, interleaved=interleaved)[0]
        assert torch.equal(again[:, 0].cpu().double(), got[3:])


@pytest.mark.parametrize("theta", [1e-30, 1e-60, 1e-200])
def test_theta_near_zero(dev, theta):
    """Frequencies beyond fp32: position zero turns nothing, others stay finite."""
    from nunchaku_amd.ops import rotary_axes

    q = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    pos = torch.tensor([0, 1, 5, -7], dtype=torch.int32, device=dev)[:, None]
    got = rotary_axes(q, None, pos, (64,), theta=theta)[0]
    assert torch.equal(got[0], q[0]) and got.isfinite().all()
