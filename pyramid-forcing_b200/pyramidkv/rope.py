"""3D RoPE of the query block, one fused kernel per sample.

``causal_rope_apply`` has the signature and results of the reference's
wan/modules/causal_model.py:30-63 (the model rotates Q with it before
``MegaCache.attend``; K is stored raw and rotated by the pack): pairs of
head_dim are complex numbers multiplied in float64 by the time / row / column
frequencies of each token's (frame, h, w) position and cast back to bf16 as
torch casts float64 (through float32).
The reference builds a float64 copy of the block and a broadcast frequency
tensor per call; here ``adahead.pkv_rope_q`` reads bf16 and writes bf16.

``rotary_apply`` is the general form beside it: 1 to 4 position axes given per
token, interleaved or half pairing, part of the head, scaled frequencies
(``rotary_frequencies``, ``axial_frequencies``), q and k in one launch of
``adahead.pkv_rotary``, with its gradient.
"""
from __future__ import annotations

import math

import torch

from . import _ops

_TABLES: dict = {}


def _tables(freqs: torch.Tensor, c: int, device) -> tuple:
    """float64 (re, im) tables of the t / y / x parts of a complex128 [rows, c]
    frequency tensor, cached per tensor."""
    key = (freqs.data_ptr(), tuple(freqs.shape), str(device))
    t = _TABLES.get(key)
    if t is None:
        parts = freqs.split([c - 2 * (c // 3), c // 3, c // 3], dim=1)
        t = tuple(torch.view_as_real(p.to(device=device, dtype=torch.complex128))
                  .reshape(p.shape[0], -1).contiguous() for p in parts)
        _TABLES.clear()
        _TABLES[key] = t
    return t


def causal_rope_apply(x: torch.Tensor, grid_sizes, freqs: torch.Tensor, start_frame: int = 0,
                      grid_int=None) -> torch.Tensor:
    """x [B, L, n, 2c] bf16 on CUDA, grid_sizes [B, 3] (f, h, w), freqs
    complex128 [rows, c]; returns x rotated, same dtype (the reference's)."""
    if not x.is_cuda or x.dtype != torch.bfloat16:
        raise ValueError("causal_rope_apply: x must be a bf16 CUDA tensor")
    c = x.size(3) // 2
    ft, fy, fx = _tables(freqs, c, x.device)
    grid = grid_int if grid_int is not None else grid_sizes.tolist()
    ops = _ops.ops()
    out = [ops.pkv_rope_q(x[i], ft, fy, fx, int(start_frame), int(f), int(h), int(w))
           for i, (f, h, w) in enumerate(grid)]
    return torch.stack(out)


# ---- rotary positions of any axes, layout and frequencies ----------------------------


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: str = "none",
                       factor: float = 1.0, original_length: int = 8192, beta_fast: float = 32.0,
                       beta_slow: float = 1.0, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq float64 [dim / 2], scale) for ``rotary_apply``.

    ``scaling`` stretches a table trained on ``original_length`` positions to
    ``factor`` times as many: "linear" divides every frequency by the factor;
    "ntk" raises the base so that only the slowest reaches that; "yarn" leaves
    pairs that turn more than beta_fast times over the original length alone,
    divides those below beta_slow turns, blends in between, and returns the
    scale 0.1 ln(factor) + 1 of the rotated part (1 for the others).
    """
    if dim <= 0 or dim % 2:
        raise ValueError("rotary_frequencies: dim must be even and positive")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    if factor < 1.0:
        raise ValueError("rotary_frequencies: factor must be at least 1")
    n = dim // 2
    if scaling == "ntk":
        base = base * factor ** (n / max(1, n - 1))
    inv = base ** (-torch.arange(n, dtype=torch.float64) / n)
    scale = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        turns = original_length * inv / (2.0 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    return inv.to(device), scale


def axial_frequencies(dims, base: float = 10000.0, device=None):
    """(inv_freq float64 [P], axis int32 [P]) of a head whose leading dims[a]
    elements (even) belong to position axis a, each with its own table: a
    video's (t, y, x) is dims (44, 42, 42) of a head of 128."""
    parts = [rotary_frequencies(d, base)[0] for d in dims]
    axis = torch.cat([torch.full((p.numel(),), a, dtype=torch.int32)
                      for a, p in enumerate(parts)])
    return torch.cat(parts).to(device), axis.to(device)


def rotary_apply(x, positions: torch.Tensor, inv_freq: torch.Tensor,
                 axis: torch.Tensor | None = None, *, layout: str = "interleaved",
                 scale: float = 1.0):
    """Rotary positions of x, or of a pair (q, k) in one launch.

    x: CUDA bf16, fp16 or fp32 [..., heads, D]; q and k may differ in heads.
    positions: int64 of x's leading shape [...] (one axis) or [..., A] with
    ``axis`` naming the axis of each pair (1 <= A <= 4).  Pair p turns by
    ``positions[..., axis[p]] * inv_freq[p]`` and is multiplied by ``scale``;
    pairs are elements (2p, 2p + 1) ("interleaved") or (p, p + P) ("half"),
    P = len(inv_freq); elements from 2P on are copied.  Differentiable (once) in x.
    """
    if layout not in ("interleaved", "half"):
        raise ValueError(f"rotary_apply: unknown layout {layout!r}")
    q, k = x if isinstance(x, (tuple, list)) else (x, None)
    for t in (q, k):
        if t is not None and (not t.is_cuda or t.dim() < 3):
            raise ValueError("rotary_apply: x must be a [..., heads, D] CUDA tensor")
    lead, shape = q.shape[:-2], positions.shape
    if k is not None and (k.shape[:-2] != lead or k.shape[-1] != q.shape[-1]):
        raise ValueError("rotary_apply: q and k must agree in tokens and head size")
    if positions.is_floating_point():
        raise ValueError("rotary_apply: positions must be whole numbers")
    if shape == lead:
        axes = 1
    elif shape[:-1] == lead:
        axes = shape[-1]
    else:
        raise ValueError("rotary_apply: positions must have x's leading shape, with or without "
                         "a dimension of axes behind it")
    out = _ops.overload("pkv_rotary_apply")(q, k, positions, axes, inv_freq, axis,
                                            layout == "half", scale)
    return out[0] if k is None else out
