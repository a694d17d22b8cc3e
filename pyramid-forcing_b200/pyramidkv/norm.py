"""Layer norm with the modulation a DiT block applies, forward and backward.

``layer_norm`` normalises over the last dimension and applies a weight and a
bias that may differ between groups of rows (frames, videos), optionally as
``1 + weight``: the ``LN(x) * (1 + scale) + shift`` of a DiT block is one
launch.  Differentiable (once) in ``x``, ``weight`` and ``bias``
(``torch.ops.adahead.pkv_norm`` over ``pkv_layer_norm`` and
``pkv_layer_norm_backward``).  The reference leaves this to torch (wan/modules/causal_model.py:335-360).
"""
from __future__ import annotations

import torch

from . import _ops


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
    if weight is not None and bias is not None:
        if weight.dtype != bias.dtype:
            raise ValueError("layer_norm: weight and bias must have one type")
        if weight.shape != bias.shape:
            weight, bias = torch.broadcast_tensors(weight, bias)
    return _ops.overload("pkv_norm")(x, weight, bias, eps, one_plus)
