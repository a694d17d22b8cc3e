"""Sums behind the block selection where low bits and the range matter: keys and
queries of far exponents, sums that cancel, values near bf16's maximum.

A mean is its float64 sum divided and rounded to fp32 once: off by at most
u |mean|, u = 2^-24, plus the float64 sum's n 2^-53 mean |k| (n <= 128 keys).
The queries below have sums that float64 holds exactly in any order, so the
lists have one answer.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_sparse import BF, U, _exact_lists, _mean_rows, _tc_select

pytestmark = pytest.mark.gpu


def _check_means(k, cu, B):
    from pyramidkv.sparse import block_means
    means = block_means(k, cu, B)
    for s in range(cu.numel() - 1):
        for j, keys in enumerate(_mean_rows(k, cu, s, B)):
            got = means[int(cu[s]) // B + s + j].double()
            want = keys.sum(0) / keys.shape[0]
            bound = U * want.abs() + 2.0 ** -46 * keys.abs().mean(0) + 2.0 ** -150
            assert torch.isfinite(got).all()
            assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [64, 128])
@pytest.mark.parametrize("spread", [1, 300])
def test_block_means_of_far_exponents(cuda, D, B, spread):
    """Keys whose exponents differ by up to 40 and that cancel in part; few
    table rows and many."""
    lens = [1, 64, 200, 1000, 77] * spread
    g = torch.Generator().manual_seed(D + B)
    T = sum(lens)
    k = torch.randn(T, D, generator=g) * 2.0 ** torch.randint(-20, 21, (T, 1), generator=g)
    k[1::2] = -k[:-1:2][:k[1::2].shape[0]] + torch.randn(k[1::2].shape, generator=g) * 2.0 ** -12
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens), 0)
    k, cu = k.to(cuda, BF), cu.to(cuda)
    if spread > 1:   # a few of the segments
        from pyramidkv.sparse import block_means
        means = block_means(k, cu, B)
        for s in (0, 3, 700, 703, len(lens) - 2):
            for j, keys in enumerate(_mean_rows(k, cu, s, B)):
                want = keys.sum(0) / keys.shape[0]
                bound = U * want.abs() + 2.0 ** -46 * keys.abs().mean(0)
                assert ((means[int(cu[s]) // B + s + j].double() - want).abs() <= bound).all()
    else:
        _check_means(k, cu, B)


@pytest.mark.parametrize("n", [64, 50, 128])
def test_block_means_near_the_end_of_the_range(cuda, n):
    """Sums past fp32's range whose means are inside it."""
    g = torch.Generator().manual_seed(n)
    big = torch.finfo(BF).max
    k = big * torch.rand(n, 128, generator=g).to(BF).float()
    k[:, 64:] *= torch.tensor([1.0, -1.0])[torch.randint(0, 2, (n, 64), generator=g)]
    k[:, 0], k[:, 1] = big, -big
    _check_means(k.to(cuda, BF), torch.tensor([0, n], dtype=torch.int32, device=cuda), 128)


def _cancelling(cuda, R, D, size, unit, seed):
    """Rows whose large ones (bf16 multiples of size / 128) cancel exactly and
    whose sum is that of the small ones, whole numbers of `unit`: every partial
    sum fits 53 bits."""
    g = torch.Generator().manual_seed(seed)
    third = R // 3
    big = (torch.randint(128, 216, (third, D), generator=g) * (size / 128)).to(BF)
    small = (torch.randint(-64, 65, (R - 2 * third, D), generator=g) * unit).to(BF)
    rows = torch.cat([big, -big, small])[torch.randperm(R, generator=g)]
    return rows[:, None].contiguous().to(cuda)


@pytest.mark.parametrize("tensor_cores", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size,unit", [(2.0 ** 30, 1.0), (2.0 ** 127, 2.0 ** 90)])
def test_select_blocks_of_cancelling_queries(cuda, tensor_cores, D, size, unit):
    """(2^127: two rows' sum is past fp32's range.)"""
    from pyramidkv.sparse import block_means, select_blocks
    nb, R, top = 700, 256, 9
    g = torch.Generator().manual_seed(D)
    k = torch.randn(nb * 64, D, generator=g).to(cuda, BF)
    cu = torch.tensor([0, nb * 64], dtype=torch.int32, device=cuda)
    q = torch.cat([_cancelling(cuda, 128, D, size, unit, s) for s in (1, 2)])
    assert torch.isfinite(q.float()).all()
    means = block_means(k, cu)
    got = _tc_select(q, means, cu, 1, R, top, 128, 64) if tensor_cores else \
        select_blocks(q, means, cu, nb * 64, 1, R, top)
    assert torch.equal(got, _exact_lists(q, k, cu, 1, R, top, 128, 64))
