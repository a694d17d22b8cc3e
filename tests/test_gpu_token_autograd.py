"""Layer norm, rotary positions and the block-sparse ops under torch's
transforms: results changed in place, forward-mode derivatives, vmap, tracing."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _rotary_inputs(cuda, dtype=torch.float32, T=30, H=3, D=64):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(T, h, D, generator=g).to(cuda, dtype) for h in (H, 1))
    pos = torch.randint(0, 500, (T,), generator=g).to(cuda)
    inv = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).to(cuda)
    return q, k, pos, inv


@pytest.mark.parametrize("shape", [(20, 64), (2, 10, 64), (64,)])
def test_layer_norm_result_changed_in_place(cuda, shape):
    """What the call returns is a tensor of its own, as a torch op's is."""
    from pyramidkv.norm import layer_norm
    g = torch.Generator().manual_seed(0)
    x = torch.randn(*shape, generator=g).to(cuda).requires_grad_(True)
    w = torch.randn(64, generator=g).to(cuda).requires_grad_(True)
    dy = torch.randn(*shape, generator=g).to(cuda)
    want = torch.autograd.grad(layer_norm(x, w) * 3.0, (x, w), dy)
    y = layer_norm(x, w)
    y.mul_(3.0)
    got = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("lead", [(30,), (5, 6)])
def test_rotary_result_changed_in_place(cuda, lead):
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv = _rotary_inputs(cuda)
    q, k, pos = q.view(*lead, 3, 64), k.view(*lead, 1, 64), pos.view(lead)
    q.requires_grad_(True)
    k.requires_grad_(True)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    a, b = rotary_apply((q, k), pos, inv)
    want = torch.autograd.grad((a * 2.0, b + 1.0), (q, k), (dq, dk))
    a, b = rotary_apply((q, k), pos, inv)
    a.mul_(2.0)
    b.add_(1.0)
    got = torch.autograd.grad((a, b), (q, k), (dq, dk))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
