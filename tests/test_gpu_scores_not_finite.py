"""Scores that are NaN, infinite or far below their row's maximum, at every
place of a step of keys, in every attention kernel.

From the softmax's definition: a NaN score or one of +inf makes its rows NaN
(inf - inf); a score of -inf has weight 0; so has one that is 200 powers of two
below the row's maximum, to well under half a bf16 step of any output.  Rows
whose scores are all -inf give zeros in the block-sparse kernels, as rows
without keys do.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_sparse import BF, U

pytestmark = pytest.mark.gpu

N = 256   # keys of a segment: full steps only (of 64 and of 128 keys)


def _heads(cuda, H, R, D, seed):
    """One segment a head, first query elements positive."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(R, H, D, generator=g)
    q[..., 0] = q[..., 0].abs() + 0.5
    k, v = (torch.randn(H * N, D, generator=g) for _ in range(2))
    k[:, 0] = 0.0
    cu = torch.arange(0, H * N + 1, N, dtype=torch.int32)
    return [t.to(cuda, BF) for t in (q, k, v)] + [cu.to(cuda)]


def _attend(kernel, q, k, v, cu, D, lists=None):
    from pyramidkv import _ops
    from pyramidkv.sparse import block_attention
    R, H = q.shape[:2]
    if kernel == "dense":
        return _ops.ops().pkv_attention(q, k, v, cu, 1, R, D ** -0.5)
    every = torch.arange(N // 64, dtype=torch.int32, device=q.device)
    return block_attention(q, k, v, cu, 1, R, every.expand(H, -(-R // 128), -1).contiguous())


# (kernel, rows, head size): few rows, tiles, the dense attention
KERNELS = [("sparse", 1, 128), ("sparse", 16, 64), ("sparse", 17, 128), ("sparse", 130, 64),
           ("dense", 130, 128), ("dense", 300, 128)]


@pytest.mark.parametrize("kernel,R,D", KERNELS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_nan_or_infinite_score_makes_its_rows_nan(cuda, kernel, R, D, bad):
    """Head h has the score at key 128 + h % 128."""
    H = 130
    q, k, v, cu = _heads(cuda, H, R, D, 1)
    want = _attend(kernel, q, k, v, cu, D)
    h = torch.arange(0, H - 2, device=cuda)     # the last two heads stay as they were
    k[h * N + 128 + h % 128, 0] = bad
    out = _attend(kernel, q, k, v, cu, D)
    assert torch.isnan(out[:, :H - 2]).all()
    assert torch.equal(out[:, H - 2:], want[:, H - 2:])


@pytest.mark.parametrize("kernel,R,D", KERNELS)
@pytest.mark.parametrize("low", [-float("inf"), -2000.0 * 2.0 ** 7])
def test_a_far_lower_score_has_no_weight(cuda, kernel, R, D, low):
    """Values near bf16's maximum at that key, where any weight would show: the
    other keys' attention, within the bound of test_gpu_sparse."""
    H, scale = 128, D ** -0.5
    q, k, v, cu = _heads(cuda, H, R, D, 2)
    h = torch.arange(0, H, device=cuda)
    at = h * N + 128 + h
    k[at, 0] = low
    v[at] = 3e38
    out = _attend(kernel, q, k, v, cu, D).double()
    keep = torch.ones(H * N, dtype=torch.bool, device=cuda)
    keep[at] = False
    kk, vv = (t[keep].view(H, N - 1, D).double() for t in (k, v))
    qq = q.double().transpose(0, 1)                       # [H, R, D]
    p = torch.softmax(qq @ kk.mT * scale, dim=-1)
    ds = ((D + 8) * U * scale * (qq.abs() @ kk.abs().mT)).amax(-1, keepdim=True)
    want = p @ vv
    bound = (p @ vv.abs()) * (2.0 ** -8 + 2e-4 + 3 * ds + 2 * N * U) + 2.0 ** -8 * want.abs()
    assert ((out.transpose(0, 1) - want).abs() <= bound).all()


@pytest.mark.parametrize("kernel,R,D", [c for c in KERNELS if c[0] == "sparse"])
def test_rows_of_scores_that_are_all_minus_infinity_give_zeros(cuda, kernel, R, D):
    H = 3
    q, k, v, cu = _heads(cuda, H, R, D, 3)
    k[N:2 * N, 0] = -float("inf")
    out = _attend(kernel, q, k, v, cu, D)
    assert (out[:, 1] == 0).all()
    assert torch.isfinite(out.float()).all() and (out[:, 0] != 0).any() and (out[:, 2] != 0).any()


@pytest.mark.parametrize("kernel,R,D", [c for c in KERNELS if c[0] == "sparse"])
def test_scores_that_pass_the_range_when_scaled_are_not_zeros(cuda, kernel, R, D):
    """Finite scores times a scale past fp32's range: infinite, so NaN, as in
    fp32 operations; a head whose scores stay in range keeps its result."""
    from pyramidkv.sparse import block_attention
    q, k, v, cu = _heads(cuda, 2, R, D, 4)
    q[:, 1], k[N:] = 0.0, 1.0                   # head 1: scores of 0
    every = torch.arange(N // 64, dtype=torch.int32, device=cuda)
    out = block_attention(q, k, v, cu, 1, R, every.expand(2, -(-R // 128), -1).contiguous(),
                          softmax_scale=2e38)
    scores = q[:, 0].float() @ k[:N].float().T * 2e38
    assert torch.isinf(scores.amax(1)).all()
    assert torch.isnan(out[:, 0]).all()
    mean = v[N:].double().mean(0)
    assert ((out[:, 1].double() - mean).abs() <= 2.0 ** -7 * v[N:].double().abs().mean(0)).all()
