"""Host side of the token-path operators, without a GPU: the frequency tables,
the argument checks of the Python entry points and of the C ABI (an error code
before anything is launched)."""
from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from conftest import ROOT

EINVAL, EUNSUPPORTED = 1, 4
LIB = os.path.join(ROOT, "pyramid-forcing_b200", "pyramidkv", "lib", "libpkv.so")
I64, INT, PTR, FLT = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(LIB)


def test_frequency_tables():
    from pyramidkv.rope import axial_frequencies, rotary_frequencies
    inv, s = rotary_frequencies(8)
    assert s == 1.0 and torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001],
                                                         dtype=torch.float64))
    lin, _ = rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.equal(lin, inv / 4)
    ntk, _ = rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(inv[-1]) / 4, rel_tol=1e-12)
    yarn, s = rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=2048)
    full = rotary_frequencies(64)[0]
    turns = 2048 * full / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], full[turns >= 32])
    assert torch.allclose(yarn[turns <= 1], full[turns <= 1] / 4, rtol=1e-15)
    between = (turns < 32) & (turns > 1)
    assert between.any() and ((yarn < full) & (yarn > full / 4))[between].all()
    assert math.isclose(s, 0.1 * math.log(4) + 1)
    inv, axis = axial_frequencies((44, 42, 42))
    assert inv.numel() == 64 and axis.tolist() == [0] * 22 + [1] * 21 + [2] * 21
    assert inv[22] == inv[43] == 1.0 and axis.dtype == torch.int32
    for bad in (dict(dim=7), dict(dim=8, scaling="other"), dict(dim=8, factor=0.5)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_python_entry_points_refuse_cpu_tensors():
    from pyramidkv.norm import layer_norm
    from pyramidkv.rope import rotary_apply
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="CUDA"):
        rotary_apply(torch.zeros(2, 1, 4), torch.zeros(2, dtype=torch.int64),
                     torch.ones(2, dtype=torch.float64))


def test_layer_norm_abi_checks(lib):
    p = PTR(256)  # never dereferenced: every call below is refused

    def fwd(x=p, rs=8, dt=0, wt=0, rows=4, cols=8, groups=1, eps=1e-6, y=p):
        return lib.pkv_layer_norm(x, I64(rs), p, p, INT(dt), INT(wt), I64(rows), I64(cols),
                                  I64(groups), FLT(eps), INT(0), y, I64(8), None, None, None)
    for bad in (dict(rows=-1), dict(cols=0), dict(groups=0), dict(groups=3), dict(dt=3),
                dict(dt=2, wt=0), dict(dt=0, wt=1), dict(x=None), dict(y=None), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert fwd(**bad) == EINVAL, bad
    assert fwd(cols=(1 << 20) + 1) == EUNSUPPORTED
    assert fwd(rows=0) == 0

    lib.pkv_layer_norm_workspace_bytes.restype = I64
    need = lib.pkv_layer_norm_workspace_bytes(I64(16), I64(8), I64(2))
    assert need == 2 * 2 * 2 * 8 * 4           # eight rows a group: two parts
    # two rows a group: one part, whose sums need no second pass up to 8192 columns
    assert lib.pkv_layer_norm_workspace_bytes(I64(4), I64(8192), I64(2)) == 0
    assert lib.pkv_layer_norm_workspace_bytes(I64(4), I64(8193), I64(2)) == 2 * 1 * 2 * 8193 * 4
    assert lib.pkv_layer_norm_workspace_bytes(I64(4), I64(8), I64(3)) == 0

    def bwd(dy=p, x=p, mean=p, dt=0, wt=0, rows=16, cols=8, groups=2, dw=p, ws=p, size=need):
        return lib.pkv_layer_norm_backward(
            dy, I64(8), x, I64(8), p, mean, p, INT(dt), INT(wt), I64(rows), I64(cols),
            I64(groups), INT(0), p, I64(8), dw, None, ws, I64(size), None)
    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rows=0), dict(groups=3),
                dict(ws=None), dict(size=need - 1), dict(ws=PTR(258)), dict(wt=1)):
        assert bwd(**bad) == EINVAL, bad


def test_rotary_abi_checks(lib):
    p = PTR(256)

    def call(q=p, qh=2, k=p, kh=2, dt=0, tokens=4, dim=8, pos=p, axes=1, inv=p, axis=p, pairs=4):
        return lib.pkv_rotary(q, I64(16), I64(8), INT(qh), p, I64(16), I64(8), k, I64(16), I64(8),
                              INT(kh), p, I64(16), I64(8), INT(dt), I64(tokens), INT(dim), pos,
                              INT(axes), inv, axis, INT(pairs), INT(0), FLT(1.0), INT(0), None)
    for bad in (dict(q=None), dict(k=None), dict(qh=-1), dict(dt=3), dict(tokens=-1), dict(dim=0),
                dict(pairs=5), dict(pairs=-1), dict(axes=0), dict(axes=5), dict(pos=None),
                dict(inv=None), dict(axes=2, axis=None)):
        assert call(**bad) == EINVAL, bad
    assert call(dim=8192, pairs=2049) == EUNSUPPORTED
    assert call(tokens=0) == 0 and call(qh=0, kh=0) == 0


def test_sparse_abi_checks(lib):
    p = PTR(256)
    lib.pkv_block_rows.restype = I64
    assert lib.pkv_block_rows(I64(1000), INT(3), INT(64)) == 18
    assert lib.pkv_block_rows(I64(1000), INT(3), INT(32)) == 0

    def means(k=p, rows=100, dim=128, cu=p, segs=2, block=64, out=p, n=4):
        return lib.pkv_block_means(k, I64(rows), INT(dim), cu, INT(segs), INT(block), out, I64(n),
                                   INT(1), None)
    for bad in (dict(k=None), dict(rows=-1), dict(cu=None), dict(segs=-1), dict(block=96),
                dict(out=None), dict(n=-1)):
        assert means(**bad) == EINVAL, bad
    for bad in (dict(dim=96), dict(rows=1 << 31), dict(k=PTR(258)), dict(out=PTR(264))):
        assert means(**bad) == EUNSUPPORTED, bad
    assert means(segs=0) == 0 and means(n=0) == 0

    def select(q=p, qs=256, mean=p, cu=p, C=1, H=2, R=3, dim=128, gr=128, block=64, top=4, out=p):
        return lib.pkv_select_blocks(q, I64(qs), I64(128), mean, I64(4), cu, I64(100), INT(C),
                                     INT(H), INT(R), INT(dim), INT(gr), INT(block), INT(top), out,
                                     None)
    for bad in (dict(q=None), dict(mean=None), dict(cu=None), dict(out=None), dict(C=-1),
                dict(H=-1), dict(R=-1), dict(gr=0), dict(gr=129), dict(block=16), dict(top=0)):
        assert select(**bad) == EINVAL, bad
    assert select(top=1025) == 3   # PKV_ECAPACITY
    for bad in (dict(dim=80), dict(q=PTR(264)), dict(qs=257), dict(mean=PTR(260))):
        assert select(**bad) == EUNSUPPORTED, bad
    assert select(R=0) == 0 and select(C=0) == 0

    def attend(q=p, qs=256, hs=128, k=p, v=p, rows=100, R=3, dim=128, scale=0.1, lst=p, gr=128,
               block=64, top=4, out=p, os_=256):
        return lib.pkv_block_attention(q, I64(qs), I64(hs), k, v, I64(rows), p, INT(1), INT(2),
                                       INT(R), INT(dim), FLT(scale), lst, INT(gr), INT(block),
                                       INT(top), out, I64(os_), I64(128), None, None)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(lst=None), dict(out=None),
                dict(scale=0.0), dict(scale=float("nan")), dict(rows=-1), dict(gr=0),
                dict(block=1), dict(top=0)):
        assert attend(**bad) == EINVAL, bad
    assert attend(top=1025) == 3
    for bad in (dict(dim=96), dict(rows=1 << 31), dict(q=PTR(258)), dict(k=PTR(258)),
                dict(qs=12), dict(hs=0), dict(qs=0), dict(os_=4), dict(out=PTR(264))):
        assert attend(**bad) == EUNSUPPORTED, bad
    assert attend(R=0) == 0


def test_meta_shapes():
    from pyramidkv import _scatter_ext
    _scatter_ext.load_library()
    ops = torch.ops.adahead
    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")
    assert ops.pkv_norm(meta(2, 3, 8), meta(8), None, 1e-6, True).shape == (2, 3, 8)
    q, k = ops.pkv_rotary_apply(meta(5, 4, 8), meta(5, 2, 8), meta(5, dtype=torch.int64), 1,
                                meta(4, dtype=torch.float64), None, True, 1.0)
    assert q.shape == (5, 4, 8) and k.shape == (5, 2, 8)
    cu = meta(7, dtype=torch.int32)
    assert ops.pkv_block_means(meta(1000, 128), cu, 64, True).shape == (1000 // 64 + 6, 128)
    out, blocks = ops.pkv_sparse_attention(meta(300, 2, 128), meta(1000, 128), meta(1000, 128), cu,
                                           3, 100, 5, 64, 64, None, None, None)
    assert out.shape == (300, 2, 128) and blocks.shape == (6, 2, 5)
    assert blocks.dtype == torch.int32


def test_selection_refuses_counts_past_32_bits(lib):
    p = PTR(256)

    def select(rows=100, C=1, R=3, gr=128):
        return lib.pkv_select_blocks(p, I64(256), I64(128), p, I64(4), p, I64(rows), INT(C), INT(2),
                                     INT(R), INT(128), INT(gr), INT(64), INT(4), p, None)
    for bad in (dict(rows=1 << 31), dict(rows=(1 << 63) - 1), dict(C=1 << 16, R=1 << 16),
                dict(R=(1 << 31) - 1)):
        assert select(**bad) == EUNSUPPORTED, bad
