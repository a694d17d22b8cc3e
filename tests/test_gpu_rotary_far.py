"""Rotary positions far out, against turn counts in whole-number arithmetic.

The angle is the exact product of the whole-number position and the float64
frequency.  Its fraction of a turn is taken with 1 / (2 pi) to 60 digits in
fractions, so that the reference's own error is below 1e-30 turns.  Bound: as
in test_gpu_rotary without a term for the angle: 6 u (|a| + |b|), and half a
step of fp32 of the result.
"""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# 1 / (2 pi), to 60 digits
PER_TURN = Fraction("0.159154943091895335768883763372514362034459645740456448747667")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("bits", [20, 31, 40, 53, 63])
def test_rotary_of_far_positions(cuda, layout, bits):
    from pyramidkv.rope import rotary_apply
    T, P = 40, 16
    g = torch.Generator().manual_seed(bits)
    top = 2 ** bits - 1
    pos = torch.randint(-top, top, (T,), generator=g)
    pos[0], pos[1] = top, -top
    if bits == 63:
        pos[2] = -2 ** 63
    inv = 10000.0 ** (-torch.arange(P, dtype=torch.float64) / P)
    x = torch.randn(T, 2, 2 * P, generator=g)
    out = rotary_apply(x.to(cuda), pos.to(cuda), inv.to(cuda), layout=layout).double().cpu()
    turns = [[float(f - round(f)) for f in (int(p) * Fraction(float(w)) * PER_TURN for w in inv)]
             for p in pos]
    ang = 2 * math.pi * torch.tensor(turns, dtype=torch.float64)[:, None]
    xd = x.double()
    a, b = (xd[..., :P], xd[..., P:]) if layout == "half" else (xd[..., ::2], xd[..., 1::2])
    want = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    got = (out[..., :P], out[..., P:]) if layout == "half" else (out[..., ::2], out[..., 1::2])
    for y, ref in zip(got, want):
        assert ((y - ref).abs() <= 6 * U * (a.abs() + b.abs()) + U * ref.abs()).all()
