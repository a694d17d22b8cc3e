"""The tensor-core selection where many scores lie within the error bound of one
another: padded (zero) query groups, zero or repeated means, one infinite mean.
The lists are those of the float64 definition, equal scores by index, in about
the time of other data."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sparse import BF, _tc_select

pytestmark = pytest.mark.gpu


def _check(q, means, cu, nb, gr, top):
    R = q.shape[0]
    got = _tc_select(q, means, cu, 1, R, top, gr, 64)[0].cpu()
    scores = q[:, 0].double().view(R // gr, gr, -1).sum(1) @ means[:nb].double().T
    # NaN last, behind -inf
    scores = torch.where(torch.isnan(scores), -torch.inf, scores.clamp(min=-1e300)).cpu()
    order = torch.argsort(scores, dim=1, descending=True, stable=True)[:, :top]
    assert torch.equal(got, order.sort(1).values.int())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nb,tops", [(40, (1, 7, 39)), (513, (1, 32, 100, 512)),
                                     (2500, (64, 1024)), (4100, (5, 1000))])
def test_many_near_scores(cuda, D, nb, tops):
    g = torch.Generator().manual_seed(nb + D)
    cu = torch.tensor([0, nb * 64], dtype=torch.int32, device=cuda)
    R, gr = 68, 4
    # values of few bits: every float64 sum is exact in any order
    q = torch.randint(-8, 9, (R, 1, D), generator=g).to(BF)
    q[8:16] = 0                                          # two zero groups among others
    means = torch.randint(-8, 9, (nb + 1, D), generator=g).float()
    kinds = means[torch.randint(0, 5, (nb + 1,), generator=g)]        # five kinds of block
    close = kinds + torch.randint(0, 3, (nb + 1, D), generator=g) * 2.0 ** -18
    some = means.clone()
    some[torch.randperm(nb, generator=g)[:nb // 2]] = 0.0
    odd = means.clone()
    odd[3, 5], odd[nb - 2, 0], odd[nb // 2, 1] = float("inf"), -float("inf"), float("nan")
    for m in (means, kinds, close, some, odd, torch.zeros_like(means)):
        for top in tops:
            _check(q.to(cuda), m.to(cuda), cu, nb, gr, top)


def test_padded_groups_take_about_the_usual_time(cuda):
    """A group of zero queries scores every block alike; ranking all against all
    took 40 times a usual selection."""
    nb, segs, R = 512, 36, 1560
    g = torch.Generator().manual_seed(5)
    q = torch.randn(R, segs, 128, generator=g).to(cuda, BF)
    means = torch.randn(segs * (nb + 1), 128, generator=g).to(cuda)
    cu = torch.arange(0, segs * nb * 64 + 1, nb * 64, dtype=torch.int32, device=cuda)
    padded = q.clone()
    padded[-128:] = 0
    ops = torch.ops.adahead

    def time(x):
        best = 1e9
        for _ in range(12):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            for _ in range(4):
                ops.pkv_select_blocks(x, means, cu, segs * nb * 64, 1, R, 32, 128, 64)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    assert time(padded) < 12 * time(q)
