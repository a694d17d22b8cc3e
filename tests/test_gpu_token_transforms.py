"""The token-path ops under torch's dispatch modes, tracing and vmap: the eager
bits.  Forward-mode derivatives are refused, not dropped."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.utils._python_dispatch import TorchDispatchMode

from test_gpu_token_autograd import BF, _rotary_inputs

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused(cuda):
    """A dual tensor's tangent is not dropped."""
    from pyramidkv import sparse
    from pyramidkv.norm import layer_norm
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv = _rotary_inputs(cuda)
    x, w = torch.randn(6, 64, device=cuda), torch.randn(64, device=cuda)
    sq = torch.randn(3, 2, 64, device=cuda).to(BF)
    sk = torch.randn(300, 64, device=cuda).to(BF)
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=cuda)
    lists = torch.zeros(2, 1, 2, dtype=torch.int32, device=cuda)
    with fwAD.dual_level():
        def dual(t):
            return fwAD.make_dual(t, torch.ones_like(t))
        for call in (lambda: layer_norm(dual(x)), lambda: layer_norm(x, dual(w)),
                     lambda: layer_norm(x, w, dual(w)),
                     lambda: rotary_apply(dual(q), pos, inv),
                     lambda: rotary_apply((q, dual(k)), pos, inv),
                     lambda: rotary_apply(q, pos, dual(inv)),
                     lambda: sparse.block_means(dual(sk), cu),
                     lambda: sparse.block_attention(sq, dual(sk), sk, cu, 1, 3, lists),
                     lambda: sparse.sparse_attention(dual(sq), sk, sk, cu, 1, 3, 2)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError,
                                                                 match="forward|gradient"):
                    call()
        with pytest.raises(RuntimeError, match="forward"):
            torch.func.jvp(layer_norm, (x,), (x,))
        # no dual tensor among the inputs: as ever
        assert torch.equal(layer_norm(x, w), layer_norm(x.clone(), w))
        rotary_apply(q, pos, inv)
        sparse.sparse_attention(sq, sk, sk, cu, 1, 3, 2)


class _Names(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.add(func.name())
        return func(*args, **(kwargs or {}))


def test_dispatch_modes_see_the_calls(cuda):
    from pyramidkv.norm import layer_norm
    from pyramidkv.rope import rotary_apply
    q, k, pos, inv = _rotary_inputs(cuda)
    x, w = torch.randn(6, 64, device=cuda), torch.randn(64, device=cuda)
    with _Names() as plain:
        layer_norm(x, w)
        rotary_apply((q, k), pos, inv)
    assert {"adahead::pkv_norm", "adahead::pkv_rotary_apply"} <= plain.seen
    x.requires_grad_(True)
    q.requires_grad_(True)
    with _Names() as train:
        y = layer_norm(x, w)
        a, b = rotary_apply((q, k), pos, inv)
        torch.autograd.grad((y, a), (x, q), (torch.ones_like(y), torch.ones_like(a)))
    assert {"adahead::pkv_layer_norm", "adahead::pkv_layer_norm_backward",
            "adahead::pkv_rotary"} <= train.seen


def test_traced_step_gives_the_eager_bits(cuda):
    """A forward and backward step through make_fx, run on other inputs."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from pyramidkv.norm import layer_norm
    from pyramidkv.rope import rotary_apply
    inv = _rotary_inputs(cuda)[3]

    def step(x, w, b, pos, inv):
        x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
        y = layer_norm(x, w, b, one_plus=True)
        a, c = rotary_apply((y.view(12, 3, 64), y.view(12, 3, 64)[:, :1]), pos, inv,
                            layout="half")
        loss = (a * a * a).sum() + (c * c).sum()
        return (y, a, c) + torch.autograd.grad(loss, (x, w, b))

    g = torch.Generator().manual_seed(3)
    sets = [[torch.randn(12, 192, generator=g).to(cuda), torch.randn(192, generator=g).to(cuda),
             torch.randn(192, generator=g).to(cuda),
             torch.randint(0, 99, (12,), generator=g).to(cuda), inv] for _ in range(2)]
    for mode in ("real", "fake"):
        traced = make_fx(step, tracing_mode=mode)(*sets[0])
        for args in sets:
            for got, want in zip(traced(*args), step(*args)):
                assert torch.equal(got, want)


def test_opcheck(cuda):
    """Schemas, fake kernels, autograd registration and tracing of every op."""
    from torch.library import opcheck
    from pyramidkv import _ops
    ops = _ops.ops()
    q, k, pos, inv = _rotary_inputs(cuda)
    x = torch.randn(6, 64, device=cuda)
    w, b = torch.randn(2, 64, device=cuda), torch.randn(2, 64, device=cuda)
    opcheck(ops.pkv_norm.default, (x, w, b, 1e-6, True))
    opcheck(ops.pkv_norm.default, (x.clone().requires_grad_(True), None, None, 1e-6, False))
    opcheck(ops.pkv_norm.default, tuple(t.clone().requires_grad_(True) for t in (x, w, b))
            + (1e-6, True))
    opcheck(ops.pkv_rotary_apply.default, (q, k, pos, 1, inv, None, True, 1.5))
    opcheck(ops.pkv_rotary_apply.default,
            (q.clone().requires_grad_(True), k.clone().requires_grad_(True), pos, 1, inv, None,
             False, 1.0))
    opcheck(ops.pkv_layer_norm.default, (x, w, b, 1e-6, True, True))
    mean, rstd = ops.pkv_layer_norm(x, w, b, 1e-6, True, True)[1:]
    opcheck(ops.pkv_layer_norm_backward.default,
            (x.flip(0), x, w, b, mean, rstd, True, True, True, True))
    opcheck(ops.pkv_rotary.default, (q, k, pos[:, None], inv, None, False, 1.0, True))
    sq = torch.randn(6, 2, 64, device=cuda).to(BF)
    sk = torch.randn(300, 64, device=cuda).to(BF)
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=cuda)
    means = ops.pkv_block_means(sk, cu, 64, True)
    lists = ops.pkv_select_blocks(sq, means, cu, 300, 1, 6, 2, 4, 64)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    opcheck(ops.pkv_block_means.default, (sk, cu, 64, True))
    opcheck(ops.pkv_select_blocks.default, (sq, means, cu, 300, 1, 6, 2, 4, 64))
    opcheck(ops.pkv_block_attention.default, (sq, sk, sk, cu, 1, 6, lists, 4, 64, 0.1, None))
    opcheck(ops.pkv_block_attention.default, (sq, sk, sk, cu, 1, 6, lists, 4, 64, 0.1, status))
    opcheck(ops.pkv_sparse_attention.default, (sq, sk, sk, cu, 1, 6, 2, 4, 64, None, None, None))


@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_step_gives_the_eager_bits(cuda, dynamic):
    """Through torch.compile's graph capture and its split into a forward and a
    backward graph (backend "aot_eager": the captured ops run as they are)."""
    from pyramidkv.norm import layer_norm
    from pyramidkv.rope import rotary_apply
    _, _, _, inv = _rotary_inputs(cuda)

    def step(x, w, pos):
        y = layer_norm(x, w, one_plus=True)
        return rotary_apply(y.unflatten(-1, (3, 64)), pos, inv, layout="half")

    compiled = torch.compile(step, backend="aot_eager", dynamic=dynamic)
    g = torch.Generator().manual_seed(4)
    for T in (12, 20):
        x, w = torch.randn(T, 192, generator=g).to(cuda), torch.randn(192, generator=g).to(cuda)
        pos, dy = torch.arange(T, device=cuda), torch.randn(T, 3, 64, generator=g).to(cuda)
        for t in (x, w):
            t.requires_grad_(True)
        got, want = compiled(x, w, pos), step(x, w, pos)
        assert torch.equal(got, want)
        for a, b in zip(torch.autograd.grad(got, (x, w), dy),
                        torch.autograd.grad(want, (x, w), dy)):
            assert torch.equal(a, b)


def test_vmap_gives_the_bits_of_a_loop(cuda):
    from pyramidkv.norm import layer_norm
    x, w = torch.randn(3, 6, 64, device=cuda), torch.randn(64, device=cuda)
    got = torch.vmap(lambda t: layer_norm(t, w))(x)
    assert torch.equal(got, torch.stack([layer_norm(t, w) for t in x]))
