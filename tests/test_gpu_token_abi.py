"""What the header allows of the token-path entry points beyond the torch ops:
results in their inputs' memory, table rows left as they were, axes clamped."""
from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

I64, INT, PTR, FLT = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_float
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
CODE = {BF: 0, HF: 1, FP: 2}


@pytest.fixture(scope="module")
def lib():
    from pyramidkv import _scatter_ext
    _scatter_ext.load_library()
    return ctypes.CDLL(_scatter_ext.KERNEL_PATH)


def _at(t):
    return PTR(t.data_ptr())


def _stream():
    return PTR(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("D,P,dt", [(128, 64, BF), (128, 32, HF), (90, 31, BF), (12, 2, FP),
                                    (64, 0, BF), (6, 3, HF)])
def test_rotary_in_place(cuda, lib, half, D, P, dt):
    g = torch.Generator().manual_seed(D + P)
    T, H, HK = 321, 5, 2
    q, k = (torch.randn(T, h, D, generator=g).to(cuda, dt) for h in (H, HK))
    pos = torch.randint(-9000, 9000, (T, 2), generator=g).to(cuda)
    inv = torch.rand(P, generator=g, dtype=torch.float64).to(cuda)
    axis = torch.randint(0, 2, (P,), generator=g).int().to(cuda)
    want = torch.ops.adahead.pkv_rotary(q, k, pos, inv, axis, half, 1.25, False)
    a = [(x, I64(x.stride(0)), I64(x.stride(1))) for x in (q.clone(), k.clone())]
    rc = lib.pkv_rotary(_at(a[0][0]), a[0][1], a[0][2], INT(H), _at(a[0][0]), a[0][1], a[0][2],
                        _at(a[1][0]), a[1][1], a[1][2], INT(HK), _at(a[1][0]), a[1][1], a[1][2],
                        INT(CODE[dt]), I64(T), INT(D), _at(pos), INT(2), _at(inv), _at(axis),
                        INT(P), INT(half), FLT(1.25), INT(0), _stream())
    torch.cuda.synchronize()
    assert rc == 0
    for (got, *_), ref in zip(a, want):
        assert torch.equal(got, ref)


def test_rotary_axes_are_clamped(cuda):
    q = torch.randn(40, 2, 16, generator=torch.Generator().manual_seed(1)).to(cuda)
    pos = torch.arange(120, device=cuda).view(40, 3)
    inv = torch.linspace(0.1, 1.0, 8, dtype=torch.float64, device=cuda)
    wild = torch.tensor([-5, 0, 1, 2, 3, 9, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=cuda)
    ops = torch.ops.adahead
    got, _ = ops.pkv_rotary(q, None, pos, inv, wild, True, 1.0, False)
    want, _ = ops.pkv_rotary(q, None, pos, inv, wild.clamp(0, 2), True, 1.0, False)
    assert torch.equal(got, want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spread", [1, 40])
def test_block_means_leave_other_rows(cuda, lib, D, spread):
    """zero_rest = 0: rows that no block has keep what was there; a table longer
    than the keys need, few rows and many."""
    lens = [130, 0, 1, 64, 2000] * spread
    total = sum(lens)
    g = torch.Generator().manual_seed(D)
    k = torch.randn(total, D, generator=g).to(cuda, BF)
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens), 0)
    cu = cu.to(cuda)
    full = torch.ops.adahead.pkv_block_means(k, cu, 64, True)
    table = torch.full((full.shape[0] + 9, D), 7.0, device=cuda)
    rc = lib.pkv_block_means(_at(k), I64(total), INT(D), _at(cu), INT(len(lens)), INT(64),
                             _at(table), I64(table.shape[0]), INT(0), _stream())
    torch.cuda.synchronize()
    assert rc == 0
    own = torch.zeros(table.shape[0], dtype=torch.bool)
    for s, n in enumerate(lens):
        first = int(cu[s]) // 64 + s
        own[first:first + -(-n // 64)] = True
    own = own.to(cuda)
    assert torch.equal(table[own], full[own[:full.shape[0]]])
    assert (table[~own] == 7.0).all()


@pytest.mark.parametrize("rows,cols,dt", [(2500, 1535, BF), (40, 1535, HF), (2500, 24, BF),
                                          (600, 777, FP), (2500, 1534, BF)])
def test_layer_norm_backward_in_place_of_odd_widths(cuda, lib, rows, cols, dt):
    ops = torch.ops.adahead
    g = torch.Generator().manual_seed(rows + cols)
    x, dy = (torch.randn(rows, cols, generator=g).to(cuda, dt) for _ in range(2))
    w = torch.randn(1, cols, generator=g).to(cuda)
    _, mean, rstd = ops.pkv_layer_norm(x, w, None, 1e-6, False, True)
    want = ops.pkv_layer_norm_backward(dy, x, w, None, mean, rstd, False, True, True, False)
    lib.pkv_layer_norm_workspace_bytes.restype = I64
    need = lib.pkv_layer_norm_workspace_bytes(I64(rows), I64(cols), I64(1))
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    both, dw = dy.clone(), torch.empty_like(w)
    rc = lib.pkv_layer_norm_backward(
        _at(both), I64(cols), _at(x), I64(cols), _at(w), _at(mean), _at(rstd), INT(CODE[dt]),
        INT(2), I64(rows), I64(cols), I64(1), INT(0), _at(both), I64(cols), _at(dw), None,
        _at(ws), I64(need), _stream())
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(both, want[0]) and torch.equal(dw, want[1])
