"""Block-sparse attention (pyramidkv.sparse) against its definition in 64 bits.

Means: keys are added four at a time in fp32, then in float64, and rounded to
fp32 once: off by at most u (|mean| + mean |k|), u = 2^-24.  Lists: equal.
Outputs, with S the exact scores and W = sum p |v| the weighted magnitudes: a
score is a D-term fp32 sum, off by ds = (D + 8) u scale sum |q||k|; a weight is
off relatively by ds, by the exponential (7.5e-5 for the polynomial) and by its
rounding to bf16 (2^-8); sums of n terms by n u; the output by half a bf16
step (2^-8).  So |error| <= W (2^-8 + 2e-4 + 3 ds + 2 n u) + 2^-8 |out|.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = torch.bfloat16


def _case(cuda, lens, C, H, R, D, seed=0, spare=13, kv_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q = torch.randn(C * R, H, D, generator=g).to(cuda, BF)
    drift = torch.randn(T // 48 + 2, D, generator=g).repeat_interleave(48, 0)[:T + spare]
    drift = torch.cat([drift, torch.zeros(T + spare - drift.shape[0], D)])
    k = ((torch.randn(T + spare, D, generator=g) + 0.7 * drift) * kv_scale).to(cuda, BF)
    v = torch.randn(T + spare, D, generator=g).to(cuda, BF)
    cu = torch.zeros(C * H + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens), 0)
    return q, k, v, cu.to(cuda)


def _mean_rows(k, cu, s, B):
    a, b = int(cu[s]), int(cu[s + 1])
    return [k[i:min(i + B, b)].double() for i in range(a, b, B)]


def _exact_lists(q, k, cu, C, R, top, gr, B):
    H = q.shape[1]
    G = -(-R // gr)
    out = torch.full((C * H, G, top), -1, dtype=torch.int32)
    for s in range(C * H):
        blocks = _mean_rows(k, cu, s, B)
        if not blocks:
            continue
        m = torch.stack([b.mean(0).float().double() for b in blocks])
        for g in range(G):
            rows = q[s // H * R + g * gr: s // H * R + min(R, (g + 1) * gr), s % H].double()
            order = torch.argsort(m @ rows.sum(0), descending=True, stable=True)[:top]
            out[s, g, :order.numel()] = order.sort().values.int().cpu()
    return out.to(q.device)


def _exact_out(q, k, v, cu, C, R, lists, gr, B, scale):
    """(value, bound) of block_attention over given lists."""
    H, D = q.shape[1:]
    val = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(val)
    lists = lists.cpu()
    for s in range(C * H):
        a, n = int(cu[s]), int(cu[s + 1]) - int(cu[s])
        for g in range(lists.shape[1]):
            idx = [j for e in lists[s, g].tolist() if 0 <= e * B < n and e >= 0
                   for j in range(e * B, min(n, (e + 1) * B))]
            if not idx:
                continue
            rows = slice(s // H * R + g * gr, s // H * R + min(R, (g + 1) * gr))
            i = torch.tensor(idx, device=q.device) + a
            qq, kk, vv = q[rows, s % H].double(), k[i].double(), v[i].double()
            p = torch.softmax(qq @ kk.T * scale, dim=-1)
            ds = ((D + 8) * U * scale * (qq.abs() @ kk.abs().T)).amax(-1, keepdim=True)
            o = p @ vv
            val[rows, s % H] = o
            err[rows, s % H] = (p @ vv.abs()) * (2.0 ** -8 + 2e-4 + 3 * ds + 2 * len(idx) * U) \
                + 2.0 ** -8 * o.abs()
    return val, err


def _within(out, want):
    value, bound = want
    assert torch.isfinite(out.float()).all()
    off = ((out.double() - value).abs() - bound).max().item()
    assert off <= 1e-37, f"over its bound by {off:.3e}"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [64, 128])
def test_block_means(cuda, D, B):
    from pyramidkv.sparse import block_means
    lens = [1, 0, 63, 64, 65, 0, 127, 128, 129, 1000, 5]
    _, k, _, cu = _case(cuda, lens, 1, len(lens), 1, D, seed=D + B)
    means = block_means(k, cu, B)
    assert means.shape == (k.shape[0] // B + len(lens), D) and means.dtype == torch.float32
    used = set()
    for s in range(len(lens)):
        for j, keys in enumerate(_mean_rows(k, cu, s, B)):
            row = int(cu[s]) // B + s + j
            assert row not in used
            used.add(row)
            want = keys.mean(0)
            assert ((means[row].double() - want).abs()
                    <= U * (want.abs() + keys.abs().mean(0))).all()
    rest = [r for r in range(means.shape[0]) if r not in used]
    assert (means[rest] == 0).all()


SELECT = [
    # segment lengths, chunks, heads, rows, D, top, query_block, block
    ([700, 0, 64, 3001], 2, 2, 300, 128, 5, 128, 64),
    ([700, 1, 65, 3001], 1, 4, 130, 64, 7, 64, 128),
    ([9000, 4096], 1, 2, 1, 128, 16, 128, 64),
    ([2000, 1999, 130], 1, 3, 40, 128, 3, 1, 64),       # every row its own blocks
    ([200_001], 1, 1, 3, 64, 20, 16, 64),                # more blocks than one round holds
    ([140_000, 131_000], 1, 2, 1, 64, 1024, 16, 64),     # as many as can be asked for, two rounds
    ([500, 600], 2, 1, 17, 64, 1, 17, 64),
]


@pytest.mark.parametrize("lens,C,H,R,D,top,gr,B", SELECT)
def test_select_blocks(cuda, lens, C, H, R, D, top, gr, B):
    from pyramidkv.sparse import block_means, select_blocks
    q, k, _, cu = _case(cuda, lens, C, H, R, D, seed=len(lens) + R)
    got = select_blocks(q, block_means(k, cu, B), cu, k.shape[0], C, R, top, query_block=gr,
                        block=B)
    assert torch.equal(got, _exact_lists(q, k, cu, C, R, top, gr, B))


def test_select_blocks_ties_zeros_and_nan(cuda):
    """Equal blocks go by index; -0 and 0 are equal; blocks whose score is NaN
    come last, an infinite one first."""
    from pyramidkv.sparse import block_means, select_blocks
    D, B, nb = 128, 64, 40
    g = torch.Generator().manual_seed(3)
    base = torch.randn(3, B, D, generator=g)
    k = base[torch.arange(nb) % 3].reshape(nb * B, D).to(cuda, BF)   # three kinds of block
    cu = torch.tensor([0, nb * B], dtype=torch.int32, device=cuda)
    q = torch.randn(1, 1, D, generator=g).to(cuda, BF)
    means = block_means(k, cu, B)
    for top in (1, 5, 13, 14, 20, 39, 40, 41):
        got = select_blocks(q, means, cu, k.shape[0], 1, 1, top)
        assert torch.equal(got, _exact_lists(q, k, cu, 1, 1, top, 128, B)), top
    zero = select_blocks(torch.zeros_like(q), means, cu, k.shape[0], 1, 1, 4)
    assert zero.flatten().tolist() == [0, 1, 2, 3]
    signed = means.clone()
    signed[::2] = -0.0
    signed[1::2] = 0.0
    assert select_blocks(q.abs(), signed, cu, k.shape[0], 1, 1, 3).flatten().tolist() == [0, 1, 2]
    odd = means.clone()
    odd[:] = -1.0
    odd[4], odd[9] = float("nan"), float("inf")
    ones = torch.ones_like(q)
    assert select_blocks(ones, odd, cu, k.shape[0], 1, 1, 1).item() == 9
    assert 4 not in select_blocks(ones, odd, cu, k.shape[0], 1, 1, 39).flatten().tolist()


@pytest.mark.parametrize("R", [1, 600])
@pytest.mark.parametrize("nb,top", [(40, 7), (300, 20), (2500, 64)])
def test_select_blocks_scores_closer_than_fp32(cuda, R, nb, top):
    """Blocks whose keys differ in one element by one bf16 step: scores apart by
    less than the error of an fp32 sum, many of them equal."""
    from pyramidkv.sparse import block_means, select_blocks
    D, B = 128, 64
    g = torch.Generator().manual_seed(nb + R)
    base = torch.randn(B, D, generator=g)
    base[:, :16] *= 1e-2
    k = base.to(BF).repeat(nb, 1).view(nb, B, D)
    at = torch.randint(0, 16, (nb,), generator=g)
    bits = k[torch.arange(nb), 5, at].view(torch.int16) + torch.randint(-1, 2, (nb,), generator=g).short()
    k[torch.arange(nb), 5, at] = bits.view(BF)
    k = k.reshape(nb * B, D).to(cuda)
    cu = torch.tensor([0, nb * B], dtype=torch.int32, device=cuda)
    q = torch.randn(R, 1, D, generator=g).to(cuda, BF)
    means = block_means(k, cu, B)
    got = select_blocks(q, means, cu, k.shape[0], 1, R, top)
    assert torch.equal(got, _exact_lists(q, k, cu, 1, R, top, 128, B))


def test_select_blocks_huge_and_infinite(cuda):
    """Products past fp32's range, infinite queries and means: the float64
    order, NaN last, equal ones by index."""
    from pyramidkv.sparse import select_blocks
    D, nb = 64, 700
    g = torch.Generator().manual_seed(8)
    q = torch.randn(3, 1, D, generator=g).to(cuda, BF)
    means = torch.randn(nb + 1, D, generator=g).to(cuda)
    cu = torch.tensor([0, nb * 64], dtype=torch.int32, device=cuda)

    def want(q, m, top):
        s = (m[:nb].double() @ q[:, 0].double().sum(0)).cpu()
        s = torch.where(torch.isnan(s), -torch.inf, s)
        return torch.argsort(s, descending=True, stable=True)[:top].sort().values.int().tolist()
    for qs, ms in ((1e30, 1e30), (1e-30, 1e-30), (1.0, 3e38), (1e-38, 1.0)):
        m, qq = means * ms, (q.float() * qs).to(BF)
        got = select_blocks(qq, m, cu, nb * 64, 1, 3, 33)
        assert got.flatten().tolist() == want(qq, m, 33), (qs, ms)
    inf = means.clone()
    inf[5, 3], inf[77, 3], inf[400, 3] = float("inf"), -float("inf"), float("inf")
    ones = q.abs()
    assert select_blocks(ones, inf, cu, nb * 64, 1, 3, 9).flatten().tolist() == want(ones, inf, 9)


def _tc_select(q, means, cu, C, R, top, gr, B):
    """select_blocks with a table of means and a row count as of a far larger
    k: few groups then go over the tensor cores too."""
    from pyramidkv.sparse import select_blocks
    blocks = 17_000                                   # two groups: 34 000 > 220 an SM
    assert -(-R // gr) >= 2
    wide = torch.full((blocks + cu.numel(), means.shape[1]), float("nan"), device=means.device)
    wide[:means.shape[0]] = means
    return select_blocks(q, wide, cu, blocks * B, C, R, top, query_block=gr, block=B)


@pytest.mark.parametrize("lens,C,H,R,D,top,gr,B", [
    ([700, 0, 64, 3001], 2, 2, 300, 128, 5, 128, 64),
    ([700, 1, 65, 3001], 1, 4, 130, 64, 7, 64, 128),
    ([2000, 1999, 130], 1, 3, 40, 128, 3, 1, 64),       # 40 groups: the last 16 rows half full
    ([500, 333] * 12, 2, 12, 17, 64, 1, 9, 64),          # clusters of four
    ([70_000], 1, 1, 400, 64, 20, 1, 64),                # two rounds
    ([70_000, 140_000], 1, 2, 10, 128, 1024, 5, 64),     # as many as can be asked for, three
    ([66_000, 70_000], 1, 2, 33, 128, 700, 2, 64),
])
def test_select_blocks_on_tensor_cores(cuda, lens, C, H, R, D, top, gr, B):
    from pyramidkv.sparse import block_means
    q, k, _, cu = _case(cuda, lens, C, H, R, D, seed=len(lens) + R)
    got = _tc_select(q, block_means(k, cu, B), cu, C, R, top, gr, B)
    assert torch.equal(got, _exact_lists(q, k, cu, C, R, top, gr, B))


def test_select_blocks_on_tensor_cores_ties_and_extremes(cuda):
    """Equal scores by index, -0 equal to 0, NaN last, infinities and products
    past fp32's range in order; one group's infinite query leaves the others'."""
    D, nb = 128, 700
    g = torch.Generator().manual_seed(21)
    cu = torch.tensor([0, nb * 64], dtype=torch.int32, device=cuda)

    def check(q, m, top):
        got = _tc_select(q, m, cu, 1, q.shape[0], top, 1, 64)
        s = (q[:, 0].double() @ m[:nb].double().T).cpu()
        s = torch.where(torch.isnan(s), -torch.inf, s)
        want = torch.argsort(s, dim=1, descending=True, stable=True)[:, :top].sort(1).values.int()
        assert torch.equal(got[0].cpu(), want)
    q = torch.randn(3, 1, D, generator=g).to(cuda, BF)
    kinds = torch.randn(3, D, generator=g)[torch.arange(nb + 1) % 3].to(cuda)
    for top in (1, 5, 233, 234, 300, 699):
        check(q, kinds, top)
    check(torch.zeros_like(q), kinds, 4)
    signed = torch.zeros(nb + 1, D, device=cuda)
    signed[::2] = -0.0
    check(q.abs(), signed, 3)
    means = torch.randn(nb + 1, D, generator=g).to(cuda)
    for qs, ms in ((1e30, 1e30), (1e-30, 1e-30), (1.0, 3e38), (1e-38, 1.0), (1e38, 1.0)):
        check((q.float() * qs).to(BF), means * ms, 33)
    odd = means.clone()
    odd[5, 3], odd[77, 3], odd[400, 3] = float("inf"), -float("inf"), float("nan")
    check(q.abs(), odd, 9)
    big = q.abs()
    big[1, 0, 7] = float("inf")
    check(big, means, 9)


@pytest.mark.parametrize("nb,top", [(40, 7), (300, 20), (2500, 64)])
def test_select_blocks_on_tensor_cores_scores_closer_than_fp32(cuda, nb, top):
    from pyramidkv.sparse import block_means
    D, B, R = 128, 64, 600
    g = torch.Generator().manual_seed(nb)
    base = torch.randn(B, D, generator=g)
    base[:, :16] *= 1e-2
    k = base.to(BF).repeat(nb, 1).view(nb, B, D)
    at = torch.randint(0, 16, (nb,), generator=g)
    step = torch.randint(-1, 2, (nb,), generator=g).short()
    k[torch.arange(nb), 5, at] = (k[torch.arange(nb), 5, at].view(torch.int16) + step).view(BF)
    k = k.reshape(nb * B, D).to(cuda)
    cu = torch.tensor([0, nb * B], dtype=torch.int32, device=cuda)
    q = torch.randn(R, 1, D, generator=g).to(cuda, BF)
    got = _tc_select(q, block_means(k, cu, B), cu, 1, R, top, 128, B)
    assert torch.equal(got, _exact_lists(q, k, cu, 1, R, top, 128, B))


ATTEND = [
    # segment lengths, chunks, heads, rows, D, query_block, block: few rows ...
    ([700, 0, 64, 3001], 1, 4, 1, 128, 128, 64),
    ([700, 1, 65, 3001], 2, 2, 16, 64, 16, 128),
    ([333, 2000], 1, 2, 37, 128, 8, 64),
    ([333, 2000, 90], 1, 3, 50, 128, 1, 64),
    # ... and tiles of up to 128
    ([700, 0, 64, 3001], 2, 2, 300, 128, 128, 64),
    ([700, 1, 65, 3001], 1, 4, 130, 64, 64, 128),
    ([129, 3000], 1, 2, 17, 128, 128, 128),
    ([1560, 4680, 390], 1, 3, 1560, 128, 100, 64),
    ([63, 200], 2, 1, 129, 64, 128, 64),
]


@pytest.mark.parametrize("lens,C,H,R,D,gr,B", ATTEND)
@pytest.mark.parametrize("top", [1, 2, 7, 40])
def test_block_attention_given_lists(cuda, lens, C, H, R, D, gr, B, top):
    """Lists in any order, with holes (-1), entries behind the segment and
    repeated blocks; rows behind a segment's last key hold NaN."""
    from pyramidkv.sparse import block_attention
    q, k, v, cu = _case(cuda, lens, C, H, R, D, seed=R + top, kv_scale=1.5)
    k[sum(lens):], v[sum(lens):] = float("nan"), float("nan")
    g = torch.Generator().manual_seed(top)
    G = -(-R // gr)
    nb = max(-(-n // B) for n in lens)
    lists = torch.randint(-2, nb + 2, (C * H, G, top), generator=g).int()
    lists[torch.rand(lists.shape, generator=g) < 0.1] = 2 ** 31 - 1
    lists = lists.to(cuda)
    scale = D ** -0.5
    out = block_attention(q, k, v, cu, C, R, lists, query_block=gr, block=B)
    _within(out, _exact_out(q, k, v, cu, C, R, lists, gr, B, scale))
    assert torch.equal(out, block_attention(q, k, v, cu, C, R, lists, query_block=gr, block=B))


@pytest.mark.parametrize("R,gr", [(1, 128), (300, 128)])
def test_neighbours_and_unselected_blocks_do_not_leak(cuda, R, gr):
    """NaN and infinities in the next segment's keys and in blocks that are not
    listed: the same bits as without them."""
    from pyramidkv.sparse import block_attention
    lens, H, D = [1000, 700], 2, 128
    q, k, v, cu = _case(cuda, lens, 1, H, R, D, seed=4)
    G = -(-R // gr)
    lists = torch.tensor([[0, 3, 15], [1, 10, -1]], dtype=torch.int32, device=cuda)
    lists = lists[:, None].expand(H, G, 3).contiguous()
    clean = block_attention(q, k, v, cu, 1, R, lists, query_block=gr)
    listed = torch.zeros(k.shape[0], dtype=torch.bool, device=cuda)
    for s, js in ((0, (0, 3, 15)), (1, (1, 10))):
        a, b = int(cu[s]), int(cu[s + 1])
        for j in js:
            listed[a + j * 64:min(b, a + (j + 1) * 64)] = True
    k[~listed], v[~listed] = float("inf"), float("nan")
    assert torch.equal(block_attention(q, k, v, cu, 1, R, lists, query_block=gr), clean)


@pytest.mark.parametrize("R", [1, 200])
def test_growing_maxima_and_extreme_scores(cuda, R):
    """Row maxima that jump from block to block by 2^8 to 2^60 and more, in
    both directions, and scores near the end of the range."""
    from pyramidkv.sparse import block_attention
    D, n = 128, 64 * 12
    q, k, v, cu = _case(cuda, [n], 1, 1, R, D, seed=9)
    for ramp in (torch.linspace(0.05, 12.0, 12), torch.linspace(12.0, 0.05, 12),
                 torch.tensor([1, 30, 1, 60, 2, 90, 1, 1, 120, 1, 5, 1.0])):
        kk = (k.float() * torch.cat([ramp.repeat_interleave(64), torch.ones(13)]).to(cuda)[:, None]
              ).to(BF)
        lists = torch.arange(12, dtype=torch.int32, device=cuda).expand(1, -(-R // 128), 12)
        out = block_attention(q, kk, v, cu, 1, R, lists.contiguous())
        _within(out, _exact_out(q, kk, v, cu, 1, R, lists, 128, 64, D ** -0.5))


def test_all_blocks_are_the_dense_attention(cuda):
    """With top_k beyond the number of blocks every block is listed: the
    library's dense attention, each within its own rounding."""
    from pyramidkv import _ops
    from pyramidkv.sparse import sparse_attention
    C, H, R, D = 2, 3, 333, 128
    lens = [1560, 0, 777, 3120, 64, 390]
    q, k, v, cu = _case(cuda, lens, C, H, R, D, seed=2)
    out, lists = sparse_attention(q, k, v, cu, C, R, 60)
    want = _exact_out(q, k, v, cu, C, R, lists, 128, 64, D ** -0.5)
    _within(out, want)
    dense = _ops.ops().pkv_attention(q, k, v, cu, C, R, D ** -0.5)
    assert ((out.double() - dense.double()).abs() <= 2 * want[1]).all()


@pytest.mark.parametrize("R", [1, 70])
def test_offsets_past_32_bits(cuda, R):
    """Keys whose element offset passes 2^31 and whose byte offset passes 2^32."""
    from pyramidkv.sparse import sparse_attention
    D, n = 128, 5000
    rows = (1 << 24) + 70_000          # 2^31 elements and more
    k = torch.zeros(rows, D, dtype=BF, device=cuda)
    q, tail, _, _ = _case(cuda, [n], 1, 1, R, D, seed=6, spare=0)
    k[-n:] = tail
    cu = torch.tensor([0, rows - n, rows], dtype=torch.int32, device=cuda)
    qq = q.expand(R, 2, D).contiguous()
    out, lists = sparse_attention(qq, k, k, cu, 1, R, 9)
    sub = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    want_lists = _exact_lists(q, tail, sub, 1, R, 9, 128, 64)
    assert torch.equal(lists[1], want_lists[0])
    _within(out[:, 1:], _exact_out(q, tail, tail, sub, 1, R, want_lists, 128, 64, D ** -0.5))
    assert (out[:, 0] == 0).all()


def test_strided_queries_and_kept_means(cuda):
    """Queries as slices of a fused projection, odd strides and offsets (copied
    inside), expanded heads; a table of means made once; a longer cu_seqlens."""
    from pyramidkv.sparse import block_means, sparse_attention
    C, H, R, D = 1, 3, 150, 64
    lens = [2000, 300, 1111]
    q, k, v, cu = _case(cuda, lens, C, H, R, D, seed=8)
    want, lists = sparse_attention(q, k, v, cu, C, R, 6)
    wide = torch.zeros(R, 3 * H * D, dtype=BF, device=cuda)
    wide[:, H * D:2 * H * D] = q.flatten(1)
    odd = torch.zeros(R, H * D + 3, dtype=BF, device=cuda)
    odd[:, 3:] = q.flatten(1)
    longer = torch.cat([cu, cu[-1:] + 13])
    for qq, c in ((wide[:, H * D:2 * H * D].unflatten(1, (H, D)), cu),
                  (odd[:, 3:].unflatten(1, (H, D)), cu),
                  (q.transpose(0, 1).contiguous().transpose(0, 1), longer)):
        out, got = sparse_attention(qq, k, v, c, C, R, 6, means=block_means(k, cu))
        assert torch.equal(got, lists) and torch.equal(out, want)
    one = q[:, :1].expand(R, H, D)
    out, got = sparse_attention(one, k, v, cu, C, R, 6)
    again, _ = sparse_attention(one.contiguous(), k, v, cu, C, R, 6)
    assert torch.equal(out, again)
    shifted = torch.zeros(k.numel() + 1, dtype=BF, device=cuda)
    shifted[1:] = k.flatten()
    out, got = sparse_attention(q, shifted[1:].view_as(k), v, cu, C, R, 6)
    assert torch.equal(got, lists) and torch.equal(out, want)


def test_no_keys_no_rows(cuda):
    from pyramidkv.sparse import sparse_attention
    for R in (1, 40):
        q = torch.randn(R, 2, 128, device=cuda).to(BF)
        none = torch.empty(0, 128, dtype=BF, device=cuda)
        out, lists = sparse_attention(q, none, none, torch.zeros(3, dtype=torch.int32, device=cuda),
                                      1, R, 4)
        assert (out == 0).all() and (lists == -1).all()
    q, k, v, cu = _case(cuda, [100, 50], 1, 2, 1, 128)
    out, lists = sparse_attention(q[:0], k, v, cu, 1, 0, 4)
    assert out.shape == (0, 2, 128) and lists.shape == (2, 0, 4)


def test_streams_and_graph_replay(cuda):
    """Two calls at once on two streams; one captured step replayed with other
    queries, keys and segment lengths."""
    from pyramidkv.sparse import sparse_attention
    C, H, R, D = 1, 4, 260, 128
    a = _case(cuda, [3000, 100, 1500, 900], C, H, R, D, seed=1)
    b = _case(cuda, [64, 2500, 2400, 536], C, H, R, D, seed=2)
    want = [sparse_attention(*x, C, R, 8) for x in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        g1 = sparse_attention(*a, C, R, 8)
    with torch.cuda.stream(s2):
        g2 = sparse_attention(*b, C, R, 8)
    torch.cuda.synchronize()
    for got, ref in zip((g1, g2), want):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    bufs = [t.clone() for t in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = sparse_attention(*bufs, C, R, 8)
    for x, ref in zip((b, a), (want[1], want[0])):
        for dst, src in zip(bufs, x):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(res[0], ref[0]) and torch.equal(res[1], ref[1])


def test_refusals(cuda):
    from pyramidkv.sparse import block_attention, block_means, select_blocks, sparse_attention
    q, k, v, cu = _case(cuda, [100, 50], 1, 2, 3, 128)
    means = block_means(k, cu)
    ok = dict(num_chunks=1, rows_per_chunk=3, top_k=2)
    for bad in (dict(top_k=0), dict(top_k=1025), dict(query_block=0), dict(query_block=129),
                dict(block=32), dict(rows_per_chunk=4), dict(num_chunks=2)):
        with pytest.raises(RuntimeError, match="pkv_"):
            sparse_attention(q, k, v, cu, **{**ok, **bad})
    for args in ((q.float(), k, v, cu), (q, k.half(), v, cu), (q, k, v, cu.long()),
                 (q, k, v, cu[:2]), (q, k, v[:-1], cu), (q, k.cpu(), v, cu), (q.cpu(), k, v, cu),
                 (q[..., :96], k, v, cu)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            sparse_attention(*args, **ok, means=means)
    with pytest.raises(RuntimeError, match="means"):
        select_blocks(q, means[:1], cu, k.shape[0], 1, 3, 2)
    lists = torch.zeros(2, 1, 2, dtype=torch.int32, device=cuda)
    for bad in (lists.long(), lists[:1], lists[0], lists.expand(2, 2, 2)):
        with pytest.raises(RuntimeError, match="blocks"):
            block_attention(q, k, v, cu, 1, 3, bad)
    with pytest.raises(RuntimeError, match="no gradient"):
        sparse_attention(q.clone().requires_grad_(True), k, v, cu, 1, 3, 2)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        block_attention(q, k, v, cu, 1, 3, lists, softmax_scale=-1.0)


def test_megacache_attend_with_top_blocks(cuda):
    """MegaCache.attend(top_blocks=) over a cache after some blocks: all blocks
    give the dense attend; few give the definition over the packed cache, also
    with other group and block sizes and from a captured graph."""
    import numpy as np
    from causal_dit.model import rope_table
    from pyramidkv import _mega_cache, policy
    H, D, W, Hg, F_ = 4, 128, 13, 8, 3
    FSEQ = W * Hg
    caches = _mega_cache.build_mega_caches(
        1, H, D, FSEQ, 3, 24, 4, policy.compositions_from_labels(np.array([[-1, 1, 2, 2]])),
        device="cuda:0", sink_time_mapping_mode="window_clamp", sink_time_clamp_min=18,
        sink_time_clamp_max=21, spatial_width=W, spatial_height=Hg, freqs=rope_table(D))
    cache, mgr = caches[0], caches[0].ctx.mgr
    g = torch.Generator().manual_seed(0)
    for blk in range(6):
        start = blk * F_ * FSEQ
        k, v, q = (torch.randn(1, F_ * FSEQ, H, D, generator=g).to(cuda, BF) for _ in range(3))
        cache.update(k, v, start, cache_update_mode="clean")
    dense = cache.attend(q, start)
    cu = mgr.cu_seqlens_k()[:F_ * H + 1].clone()
    kf, vf = (t.view(-1, D)[:int(cu[-1])].clone() for t in (mgr.k_flat_out(), mgr.v_flat_out()))
    every = torch.arange(64, dtype=torch.int32).expand(F_ * H, 1, 64)
    bound = _exact_out(q[0], kf, vf, cu, F_, FSEQ, every, 128, 64, D ** -0.5)
    _within(cache.attend(q, start, top_blocks=64)[0], bound)
    _within(dense[0], bound)
    for top, gr, B in ((4, 128, 64), (3, 64, 128), (5, 8, 64)):
        out = cache.attend(q, start, top_blocks=top, query_block=gr, key_block=B)
        lists = _exact_lists(q[0], kf, cu, F_, FSEQ, top, gr, B)
        _within(out[0], _exact_out(q[0], kf, vf, cu, F_, FSEQ, lists, gr, B, D ** -0.5))
    eager = cache.attend(q, start, top_blocks=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, start, top_blocks=4)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    assert cache.ctx.check_status() == 0
