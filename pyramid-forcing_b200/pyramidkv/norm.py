"""Layer norm with the modulation a DiT block applies, forward and backward.

``layer_norm`` normalises over the last dimension and applies a weight and a
bias that may differ between groups of rows (frames, videos), optionally as
``1 + weight``: the ``LN(x) * (1 + scale) + shift`` of a DiT block is one
launch.  Differentiable in ``x``, ``weight`` and ``bias``
(``torch.ops.adahead.pkv_layer_norm`` / ``pkv_layer_norm_backward``).  The
reference leaves this to torch (wan/modules/causal_model.py:335-360).
"""
from __future__ import annotations

import torch

from . import _ops


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, one_plus):
        y, mean, rstd = _ops.ops().pkv_layer_norm(x, weight, bias, eps, one_plus,
                                                  any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.one_plus = one_plus
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        dx, dw, db = _ops.ops().pkv_layer_norm_backward(dy, x, weight, bias, mean, rstd,
                                                        ctx.one_plus, *need)
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None,
                None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-6, *,
               one_plus: bool = False) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * w + bias over the last dimension of x.

    x: CUDA bf16, fp16 or fp32, any leading shape; w is ``weight``, or
    ``1 + weight`` with ``one_plus``.  weight / bias: [C], or [G, C] where G
    divides the number N of rows and row r uses row r // (N // G); x's type or
    fp32.  Statistics and sums are fp32; the result has x's type, the
    gradients their inputs' types.
    """
    if not x.is_cuda:
        raise ValueError("layer_norm: x must be a CUDA tensor")
    if x.dim() == 0:
        raise ValueError("layer_norm: x needs a last dimension to normalise")
    if weight is not None and bias is not None:
        if weight.dtype != bias.dtype:
            raise ValueError("layer_norm: weight and bias must have one type")
        if weight.shape != bias.shape:
            weight, bias = torch.broadcast_tensors(weight, bias)
    rows = x.reshape(x.numel() // x.shape[-1], x.shape[-1]) if x.shape[-1] else x.view(0, 0)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, weight, bias)):
        y = _LayerNorm.apply(rows, weight, bias, float(eps), bool(one_plus))
    else:
        y = _ops.ops().pkv_layer_norm(rows, weight, bias, float(eps), bool(one_plus), False)[0]
    return y.view(x.shape)
