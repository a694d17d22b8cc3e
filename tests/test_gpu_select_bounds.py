"""The tensor-core selection at the ends of its error bound: queries and means
whose split into bf16 pairs loses most, and products at the end of fp32's range.
The lists are those of the float64 definition."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sparse import BF, _tc_select

pytestmark = pytest.mark.gpu


def _check(q, means, cu, nb, R, gr, top):
    got = _tc_select(q, means, cu, 1, R, top, gr, 64)[0].cpu()
    sums = q[:, 0].double().view(R // gr, gr, -1).sum(1)
    scores = (sums @ means[:nb].double().T).cpu()
    order = torch.argsort(scores, dim=1, descending=True, stable=True)[:, :top]
    assert torch.equal(got, order.sort(1).values.int())


@pytest.mark.parametrize("D", [64, 128])
def test_products_that_pass_the_range_only_when_rounded(cuda, D):
    """|q| and |mean| below the root of fp32's maximum, so their squares are
    finite, but rounded to bf16 both are 2^64 and their product is 2^128."""
    nb, R, gr = 700, 6, 2
    g = torch.Generator().manual_seed(D)
    q = torch.zeros(R, 1, D)
    q[0::2, 0, 0] = 2.0 ** 64 * (1 - 2.0 ** -8)
    q[1::2, 0, 0] = 2.0 ** 56 * (1 - 2.0 ** -8)        # together 2^64 (1 - 2^-16)
    means = torch.zeros(nb + 1, D)
    means[:, 0] = 2.0 ** 64 - 2.0 ** 47 - 2.0 ** 40 * torch.randint(0, 64, (nb + 1,), generator=g)
    cu = torch.tensor([0, nb * 64], dtype=torch.int32, device=cuda)
    for top in (1, 9, 300, 699):
        _check(q.to(cuda, BF), means.to(cuda), cu, nb, R, gr, top)
        _check(-q.to(cuda, BF), means.to(cuda), cu, nb, R, gr, top)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seed", range(4))
def test_splits_that_lose_most(cuda, D, seed):
    """x = 1 + 2^-8 + 2^-17 + ... leaves 2^-8 of its bf16 rounding and 2^-17 of
    the remainder's: products of two such are 8 * 2^-18 too small, those with
    bf16 means (the odd blocks) a quarter of that.  Scores apart by less."""
    nb, R, gr = 700, 6, 3
    g = torch.Generator().manual_seed(seed)
    sign = torch.tensor([1.0, -1.0])[torch.randint(0, 2, (D,), generator=g)]
    q = torch.stack([torch.full((D,), 1.0), torch.full((D,), 2.0 ** -8),
                     torch.full((D,), 2.0 ** -17 + 2.0 ** -18)]) * sign
    q = torch.cat([q, q.flip(0)])[:, None].contiguous()
    low = torch.randint(0, 2 ** 5, (nb + 1, D), generator=g) * 2.0 ** -23
    means = 1.0 + 2.0 ** -8 + 2.0 ** -17 + low
    short = torch.rand(nb + 1, D, generator=g).argsort(1) % 2 * 2.0 ** -7 + 1.0
    means[1::2] = short[1::2]
    means[:, 0] = (2.0 ** -7 * torch.randn(nb + 1, generator=g)).to(BF).float()
    means *= sign
    cu = torch.tensor([0, nb * 64], dtype=torch.int32, device=cuda)
    for top in (7, 100, 350, 650):
        _check(q.to(cuda, BF), means.to(cuda), cu, nb, R, gr, top)
