"""The token-path ops on fake CUDA tensors, without a GPU: shapes, types and
strides of every op, with gradients wanted too, and what a shape alone can refuse.
(A backward pass needs the device: test_gpu_token_transforms.)"""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


@pytest.fixture
def fake():
    from pyramidkv import _scatter_ext
    _scatter_ext.load_library()
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.float32, grad=False: torch.empty(
            *shape, dtype=dtype, device="cuda", requires_grad=grad)


def _is(t, shape, dtype=torch.float32):
    assert tuple(t.shape) == shape and t.dtype == dtype and t.device.type == "cuda"
    assert t.is_contiguous()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("shape", [(6, 8), (2, 3, 8), (8,)])
def test_norm(fake, grad, shape):
    ops = torch.ops.adahead
    x, w, b = fake(*shape, dtype=BF, grad=grad), fake(8, grad=grad), fake(8, grad=grad)
    y = ops.pkv_norm(x, w, b, 1e-6, True)
    _is(y, shape, BF)
    assert y.requires_grad == grad


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_rotary(fake, grad, lead):
    ops = torch.ops.adahead
    q, k = fake(*lead, 4, 16, grad=grad), fake(*lead, 2, 16, grad=grad)
    pos, inv = fake(*lead, dtype=torch.int64), fake(8, dtype=torch.float64)
    a, b = ops.pkv_rotary_apply(q, k, pos, 1, inv, None, True, 1.0)
    _is(a, lead + (4, 16))
    _is(b, lead + (2, 16))
    assert a.requires_grad == b.requires_grad == grad
    one = ops.pkv_rotary_apply(q, None, pos, 1, inv, None, True, 1.0)
    _is(one[0], lead + (4, 16))
    assert one[1] is None


def test_plain_ops(fake):
    ops = torch.ops.adahead
    x, w = fake(6, 8, dtype=BF), fake(2, 8)
    y, mean, rstd = ops.pkv_layer_norm(x, w, None, 1e-6, True, True)
    _is(y, (6, 8), BF)
    _is(mean, (6,))
    _is(rstd, (6,))
    dx, dw, db = ops.pkv_layer_norm_backward(x, x, w, None, mean, rstd, True, True, True, False)
    _is(dx, (6, 8), BF)
    _is(dw, (2, 8))
    assert db is None and ops.pkv_layer_norm(x, w, None, 1e-6, True, False)[1] is None
    q = fake(6, 4, 16)
    a, b = ops.pkv_rotary(q, q[:, :1], fake(6, 2, dtype=torch.int64),
                          fake(8, dtype=torch.float64), fake(8, dtype=torch.int32), True, 1.0, True)
    _is(a, (6, 4, 16))
    _is(b, (6, 1, 16))


def test_sparse_ops(fake):
    from pyramidkv import sparse  # noqa: F401  (the ops' public module imports without a GPU)
    ops = torch.ops.adahead
    q, k = fake(300, 2, 128, dtype=BF), fake(1000, 128, dtype=BF)
    cu = fake(7, dtype=torch.int32)
    means = ops.pkv_block_means(k, cu, 64, True)
    _is(means, (1000 // 64 + 6, 128))
    lists = ops.pkv_select_blocks(q, means, cu, 1000, 3, 100, 5, 64, 64)
    _is(lists, (6, 2, 5), torch.int32)
    _is(ops.pkv_block_attention(q, k, k, cu, 3, 100, lists, 64, 64, 0.1, None), (300, 2, 128), BF)
    out, again = ops.pkv_sparse_attention(q, k, k, cu, 3, 100, 5, 64, 64, None, means, None)
    _is(out, (300, 2, 128), BF)
    _is(again, (6, 2, 5), torch.int32)


def test_shapes_alone_refuse(fake):
    """A size that would divide by zero, or a gradient of nothing, is an error."""
    ops = torch.ops.adahead
    q, k = fake(6, 2, 64, dtype=BF), fake(300, 64, dtype=BF)
    cu = fake(3, dtype=torch.int32)
    x = fake(6, 8)
    for call in (lambda: ops.pkv_block_means(k, cu, 0, True),
                 lambda: ops.pkv_block_means(k[:, :0], cu, 64, True),
                 lambda: ops.pkv_select_blocks(q, fake(6, 64), cu, 300, 1, 6, 2, 0, 64),
                 lambda: ops.pkv_sparse_attention(q, k, k, cu, 1, 6, 2, 0, 64, None, None, None),
                 lambda: ops.pkv_layer_norm_backward(x, x, None, None, x[:, 0], x[:, 0], False,
                                                     True, True, False)):
        with pytest.raises(RuntimeError):
            call()
