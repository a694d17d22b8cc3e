"""Rotary positions (pyramidkv.rope.rotary_apply) against 64-bit rotations.

Bound of each result, with u = 2^-24: the cosine and sine come from sinpi /
cospi (documented error 1 ulp = 2 u), are corrected and scaled (2 u); the two
products and their sum add 2 u: at most 6 u scale (|a| + |b|), plus the
angle's float64 error 2^-50 |position| inv_freq (the longest a step of its
product), plus half a step of the result's type.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _exact(x, pos, inv, axis, layout, scale, sign=1.0):
    """(value, bound) for x [T, H, D], pos [T, A]."""
    P, xd = inv.numel(), x.double()
    axis = torch.zeros(P, dtype=torch.long, device=x.device) if axis is None else axis.long()
    ang = pos.double()[:, axis] * inv
    c, s = scale * ang.cos()[:, None], sign * scale * ang.sin()[:, None]
    slack = 6 * U + 2.0 ** -50 * ang.abs()[:, None]
    if layout == "half":
        a, b = xd[..., :P], xd[..., P:2 * P]
    else:
        a, b = xd[..., 0:2 * P:2], xd[..., 1:2 * P:2]
    re, im = a * c - b * s, a * s + b * c
    bound = abs(scale) * (a.abs() + b.abs()) * slack
    val, err = xd.clone(), torch.zeros_like(xd)
    if layout == "half":
        val[..., :P], val[..., P:2 * P] = re, im
        err[..., :P] = err[..., P:2 * P] = bound
    else:
        val[..., 0:2 * P:2], val[..., 1:2 * P:2] = re, im
        err[..., 0:2 * P:2] = err[..., 1:2 * P:2] = bound
    return val, err + torch.finfo(x.dtype).eps / 2 * val.abs()


def _within(got, want, name):
    value, bound = want
    tiny = 6e-8 if got.dtype == HF else 1e-37
    assert torch.isfinite(got.float()).all(), name
    off = ((got.double() - value).abs() - bound - tiny).max().item()
    assert off <= 0, f"{name}: over its bound by {off:.3e}"


def _data(cuda, T, H, HK, D, P, A, dt, span, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, H, D, generator=g).to(cuda, dt)
    k = torch.randn(T, HK, D, generator=g).to(cuda, dt)
    pos = torch.randint(-span, span + 1, (T, A), generator=g).to(cuda)
    inv = (10000.0 ** (-torch.arange(P, dtype=torch.float64) / max(P, 1))).to(cuda)
    axis = (torch.arange(P, dtype=torch.int32) * A // max(P, 1)).int().to(cuda)
    return q, k, pos, inv, axis


CASES = [
    # tokens, heads, key heads, D, pairs, axes, layout, type, largest position
    (1, 12, 4, 128, 64, 1, "half", BF, 1_000_000),
    (333, 12, 12, 128, 64, 3, "interleaved", BF, 200),
    (77, 3, 1, 128, 32, 1, "half", HF, 70_000),
    (50, 2, 2, 64, 32, 2, "interleaved", FP, 5000),
    (20, 5, 3, 66, 33, 1, "half", BF, 100),          # odd pairs: single elements
    (20, 5, 3, 90, 31, 4, "interleaved", HF, 100),
    (9, 1, 7, 12, 6, 3, "half", FP, 10),             # accesses of 2 elements
    (1200, 24, 8, 256, 128, 1, "interleaved", BF, 1 << 40),
    (2, 1, 1, 4096, 2048, 1, "half", FP, 4096),      # a table for one token
    (5, 2, 2, 7, 3, 1, "interleaved", FP, 50),       # an odd head
    (5, 2, 2, 8, 0, 1, "half", BF, 50),              # nothing turns
    (700, 7, 5, 90, 31, 1, "half", BF, 1000),
    (700, 7, 5, 90, 45, 2, "interleaved", BF, 1000),
    (40, 3, 2, 74, 34, 1, "interleaved", FP, 100),
]


@pytest.mark.parametrize("T,H,HK,D,P,A,layout,dt,span", CASES)
def test_rotary_and_gradients(cuda, T, H, HK, D, P, A, layout, dt, span):
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv, axis = _data(cuda, T, H, HK, D, P, A, dt, span, seed=T + D)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    scale = 1.25
    q.requires_grad_(True)
    k.requires_grad_(True)
    qo, ko = rotary_apply((q, k), pos, inv, axis, layout=layout, scale=scale)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for got, x, sign in ((qo, q, 1.0), (ko, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        _within(got, _exact(x.detach(), pos, inv, axis, layout, scale, sign), f"{sign}")
        assert torch.equal(got[..., 2 * P:], x[..., 2 * P:])
    with torch.no_grad():
        one = rotary_apply(q, pos, inv, axis, layout=layout, scale=scale)
    assert torch.equal(one, qo)
    assert torch.equal(torch.autograd.grad(
        rotary_apply((q, k), pos, inv, axis, layout=layout, scale=scale)[1], k, dk)[0], gk)


def test_rotary_gradient_against_differences(cuda):
    """The rotation is linear in x: f(x + v) - f(x - v) over 2 is exact in the
    64-bit definition, and must be what the gradient says along v."""
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv, axis = _data(cuda, 30, 4, 4, 64, 32, 1, FP, 1000)
    dq = torch.randn_like(q)
    v = torch.randn_like(q)
    q.requires_grad_(True)
    g, = torch.autograd.grad(rotary_apply(q, pos, inv, layout="half", scale=0.5), q, dq)
    up = _exact(q.detach().double() + v.double(), pos, inv, None, "half", 0.5)[0]
    down = _exact(q.detach().double() - v.double(), pos, inv, None, "half", 0.5)[0]
    diff = ((up - down) * dq.double()).sum() / 2
    bound = (_exact(dq, pos, inv, None, "half", 0.5, -1.0)[1] * v.abs()).sum()
    assert ((g.double() * v).sum() - diff).abs() <= bound + 1e-9


def test_rotary_strided_shaped_and_expanded(cuda):
    """Slices of a fused QKV projection, [B, L] leading shapes, gradients that
    are expanded, and heads that lie transposed."""
    from pyramidkv.rope import rotary_apply
    g = torch.Generator().manual_seed(2)
    B, L, H, D = 2, 9, 3, 64
    qkv = torch.randn(B, L, 3 * H * D, generator=g).to(cuda, BF)
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:2 * H * D].unflatten(-1, (H, D))
    pos = torch.arange(L).expand(B, L).to(cuda)
    inv, axis = _data(cuda, 1, 1, 1, D, 32, 1, BF, 1)[3:]
    qo, ko = rotary_apply((q, k), pos, inv)
    flat = pos.reshape(-1, 1)
    _within(qo.view(-1, H, D), _exact(q.reshape(-1, H, D), flat, inv, None, "interleaved", 1.0), "q")
    _within(ko.view(-1, H, D), _exact(k.reshape(-1, H, D), flat, inv, None, "interleaved", 1.0), "k")
    t = torch.randn(H, L, D, generator=g).to(cuda, FP).transpose(0, 1).requires_grad_(True)
    to = rotary_apply(t, pos[0].int(), inv, layout="half")
    _within(to, _exact(t.detach(), pos[0, :, None], inv, None, "half", 1.0), "transposed")
    dy = torch.randn(D, generator=g).to(cuda).expand(L, H, D)
    gt, = torch.autograd.grad(to, t, dy)
    _within(gt, _exact(dy, pos[0, :, None], inv, None, "half", 1.0, -1.0), "expanded")


def test_rotary_offsets_past_32_bits(cuda):
    from pyramidkv.rope import rotary_apply
    T, H, D = 1_100_003, 16, 128
    q, _, _, inv, _ = _data(cuda, 5, H, 1, D, 64, 1, BF, 1)
    x = torch.zeros(T, H, D, dtype=BF, device=cuda)
    x[-5:] = q
    pos = torch.arange(T, device=cuda)
    out = rotary_apply(x, pos, inv, layout="half")
    _within(out[-5:], _exact(q, pos[-5:, None], inv, None, "half", 1.0), "tail")
    assert (out[:5] == 0).all()


def test_rotary_matches_the_block_rotation(cuda):
    """With a video's (t, y, x) axes it is the rotation causal_rope_apply
    makes from the model's tables, to fp32 arithmetic and one bf16 step."""
    from causal_dit.model import rope_table
    from pyramidkv.rope import axial_frequencies, causal_rope_apply, rotary_apply
    F_, Hh, Ww, H, D, t0 = 3, 5, 7, 4, 128, 11
    T = F_ * Hh * Ww
    x = torch.randn(1, T, H, D, device=cuda).to(BF)
    inv, axis = axial_frequencies((44, 42, 42), device=cuda)
    i = torch.arange(T, device=cuda)
    pos = torch.stack([t0 + i // (Hh * Ww), i // Ww % Hh, i % Ww], dim=1)
    got = rotary_apply(x, pos[None], inv, axis)
    want = causal_rope_apply(x, None, rope_table(D).to(cuda), start_frame=t0,
                             grid_int=((F_, Hh, Ww),))
    step = torch.finfo(BF).eps * want.double().abs() + 6 * U * 2 * x.double().abs().amax()
    assert ((got.double() - want.double()).abs() <= step).all()


def test_rotary_streams_graph_and_no_tokens(cuda):
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv, axis = _data(cuda, 2000, 6, 2, 128, 64, 3, BF, 500)
    want = rotary_apply((q, k), pos, inv, axis)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = rotary_apply((q, k), pos, inv, axis)
    with torch.cuda.stream(s2):
        b = rotary_apply((q, k), pos, inv, axis)
    torch.cuda.synchronize()
    for got in (a, b):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    ps = pos.clone()
    with torch.cuda.graph(graph):
        out = rotary_apply((q, k), ps, inv, axis)
    ps.copy_(pos + 3)
    graph.replay()
    later = rotary_apply((q, k), pos + 3, inv, axis)
    torch.cuda.synchronize()
    assert torch.equal(out[0], later[0]) and torch.equal(out[1], later[1])
    none = rotary_apply(q[:0], pos[:0], inv, axis)
    assert none.shape == (0, 6, 128)


def test_rotary_refusals(cuda):
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv, axis = _data(cuda, 4, 2, 2, 64, 32, 2, BF, 10)
    with pytest.raises(ValueError, match="layout"):
        rotary_apply(q, pos, inv, axis, layout="other")
    with pytest.raises(ValueError, match="leading shape"):
        rotary_apply(q, pos[:3], inv, axis)
    with pytest.raises(ValueError, match="whole numbers"):
        rotary_apply(q, pos.float(), inv, axis)
    with pytest.raises(ValueError, match="agree"):
        rotary_apply((q, k[:3]), pos, inv, axis)
    for p, f, a in ((pos, inv, None),                                 # two axes, no names
                    (pos, inv.float(), axis), (pos, inv, axis.long()),
                    (pos, inv.cpu(), axis), (pos[:, :1], torch.cat([inv, inv]), None)):
        with pytest.raises(RuntimeError, match="pkv_rotary"):
            rotary_apply(q, p, f, a)
    with pytest.raises(RuntimeError, match="inv_freq"):
        rotary_apply(q, pos, inv.clone().requires_grad_(True), axis)
    x = torch.randn(4, 2, 64, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(rotary_apply(x, pos, inv, axis).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="bf16, fp16 or fp32"):
        rotary_apply(q.double(), pos, inv, axis)
    assert math.isfinite(float(q.float().sum()))
