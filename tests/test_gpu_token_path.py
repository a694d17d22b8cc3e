"""The token-path operators together, as a DiT block uses them.

* Training: modulated norm -> Q and K projections -> rotary positions ->
  softmax(q k^T) weights, and the gradients of its input, modulation and
  projections.  The reference is the same graph in 64 bits; the bound is the
  error that the graph has in plain fp32 torch operations on the same inputs
  (its roundings are of the same kind and number; twice that, for another order
  of sums) plus four fp32 steps of the gradient's norm.
* Serving: the random-init DiT with fused norms and block-sparse
  self-attention over its cache, through the few-step loop; and one forward
  pass whose kept blocks are all of the cache against the dense one.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain_norm(x, w, b, groups):
    d = x - x.mean(-1, keepdim=True)
    xh = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-6)
    N, C = x.shape
    return (xh.view(groups, N // groups, C) * (1 + w)[:, None] + b[:, None]).view(N, C)


def _plain_rotary(x, pos, inv, axis):
    ang = pos.double()[:, axis.long()] * inv
    c, s = ang.cos().to(x.dtype)[:, None], ang.sin().to(x.dtype)[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _loss(x, w, b, wq, wk, pos, inv, axis, probe, norm, rotary):
    y = norm(x, w, b)
    N, H, D = x.shape[0], probe.shape[0], inv.numel() * 2
    q, k = rotary((y @ wq).view(N, H, D), (y @ wk).view(N, H, D))
    p = torch.softmax(q.transpose(0, 1) @ k.permute(1, 2, 0) * D ** -0.5, dim=-1)
    return (p * probe).sum()


def test_training_block_gradients(cuda):
    from pyramidkv.norm import layer_norm
    from pyramidkv.rope import axial_frequencies, rotary_apply
    F_, Hh, Ww, H, D, C = 2, 5, 6, 3, 64, 96
    N = F_ * Hh * Ww
    g = torch.Generator().manual_seed(0)
    inv, axis = axial_frequencies((24, 20, 20), device=cuda)
    i = torch.arange(N, device=cuda)
    pos = torch.stack([7 + i // (Hh * Ww), i // Ww % Hh, i % Ww], dim=1)
    ins = [torch.randn(N, C, generator=g), 0.3 * torch.randn(F_, C, generator=g),
           torch.randn(F_, C, generator=g), torch.randn(C, H * D, generator=g) * C ** -0.5,
           torch.randn(C, H * D, generator=g) * C ** -0.5]
    probe = torch.randn(H, N, N, generator=g).to(cuda)

    def grads(dtype, norm, rotary):
        leaves = [t.to(cuda, dtype).requires_grad_(True) for t in ins]
        loss = _loss(*leaves, pos, inv, axis, probe.to(dtype), norm, rotary)
        return torch.autograd.grad(loss, leaves)

    plain = (lambda x, w, b: _plain_norm(x, w, b, F_),
             lambda q, k: (_plain_rotary(q, pos, inv, axis), _plain_rotary(k, pos, inv, axis)))
    exact = grads(torch.float64, *plain)
    fp32 = grads(torch.float32, *plain)
    own = grads(torch.float32, lambda x, w, b: layer_norm(x, w, b, one_plus=True),
                lambda q, k: rotary_apply((q, k), pos, inv, axis))
    for e, f, o in zip(exact, fp32, own):
        assert o.dtype == torch.float32
        off, base = (o.double() - e).norm(), (f.double() - e).norm()
        assert off <= 2 * base + 4 * 2.0 ** -24 * e.norm(), (off / e.norm(), base / e.norm())


def _model(cuda, **kw):
    from causal_dit import CausalWanDiT, WanConfig
    from pyramidkv import _mega_cache, policy
    cfg = WanConfig(dim=256, ffn_dim=512, freq_dim=32, text_dim=64, num_heads=2, num_layers=2,
                    text_len=16, **kw)
    model = CausalWanDiT(cfg, cuda, seed=3)
    caches = _mega_cache.build_mega_caches(
        2, 2, 128, 128, 3, 24, 4, policy.compositions_from_labels(np.array([[-1, 1], [2, -1]])),
        device="cuda:0", sink_time_mapping_mode="window_clamp", sink_time_clamp_min=18,
        sink_time_clamp_max=21, spatial_width=16, spatial_height=8, freqs=model.freqs)
    return model, caches


def test_dit_with_fused_norm_and_sparse_attention(cuda):
    from causal_dit import generate_video
    outs = []
    for _ in range(2):
        model, caches = _model(cuda, fused_norm=True, top_blocks=4)
        g = torch.Generator(device=cuda).manual_seed(5)
        text = torch.randn(1, 16, 64, generator=g, device=cuda)
        noise = torch.randn(1, 16, 6, 16, 32, generator=g, device=cuda, dtype=torch.bfloat16)
        outs.append(generate_video(model, caches, noise, text, generator=g))
        assert caches[0].ctx.check_status() == 0
    assert outs[0].shape == (1, 16, 6, 16, 32) and torch.isfinite(outs[0].float()).all()
    assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))


def test_dit_forward_with_every_block_kept(cuda):
    """One pass of the self-attention's first layer over a cache of 6 frames:
    768 keys a head are at most 12 blocks, so 16 keep all of them, and the
    sparse attend is the dense one: each side is off by the bf16 rounding of P
    (2^-8 of the weighted magnitudes of V), of the output (2^-8 of it) and less
    than 1e-3 of V for the exponentials and sums; all at most max |v|."""
    model, caches = _model(cuda)
    g = torch.Generator(device=cuda).manual_seed(6)
    cache = caches[0]
    for blk in range(2):
        k, v, q = (torch.randn(1, 384, 2, 128, generator=g, device=cuda, dtype=torch.bfloat16)
                   for _ in range(3))
        cache.update(k, v, blk * 384, cache_update_mode="clean")
    dense = cache.attend(q, 384).double()
    sparse = cache.attend(q, 384, top_blocks=16).double()
    vmax = cache.ctx.mgr.v_flat_out().abs().max().double()
    assert ((dense - sparse).abs() <= 2 * (2 * 2.0 ** -8 + 1e-3) * vmax).all()
    assert cache.ctx.check_status() == 0
