"""Block-sparse attention over the ragged K/V layout of ``pkv_attention``.

The keys of every (chunk, head) segment are cut into blocks; every group of
query rows keeps the ``top_k`` blocks whose mean key scores highest against the
group's queries and attends those blocks only:

    means  = block_means(k, cu_seqlens_k)                  # one pass over K
    blocks = select_blocks(q, means, cu_seqlens_k, ...)    # int32 lists
    out    = block_attention(q, k, v, cu_seqlens_k, ..., blocks)

or ``sparse_attention`` for the three.  A program whose cache stands (many
queries on the same keys) keeps ``means`` and passes them in.  Inference only:
the ops have no gradients.  ``MegaCache.attend(..., top_blocks=k)`` is this over
the packed cache.  The reference attends the whole cache
(pyramidkv/_mega_cache.py:529-569).
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _ops


def _no_tangent(*tensors) -> None:
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("block-sparse attention has no forward-mode derivative")


def _no_grad(*tensors) -> None:
    _no_tangent(*tensors)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("block-sparse attention has no gradient: call it under "
                           "torch.no_grad()")


def block_means(k: torch.Tensor, cu_seqlens_k: torch.Tensor, block: int = 64) -> torch.Tensor:
    """Mean key of every block, fp32 [rows // block + segments, D].

    k: bf16 [rows, D] (D 64 or 128); segment s holds keys cu_seqlens_k[s] to
    cu_seqlens_k[s + 1], its block j the row cu_seqlens_k[s] // block + s + j
    of the table.  Rows between segments and behind the last are zero.
    """
    _no_tangent(k)
    return _ops.overload("pkv_block_means")(k, cu_seqlens_k, int(block), True)


def select_blocks(q: torch.Tensor, means: torch.Tensor, cu_seqlens_k: torch.Tensor, kv_rows: int,
                  num_chunks: int, rows_per_chunk: int, top_k: int, *, query_block: int = 128,
                  block: int = 64) -> torch.Tensor:
    """int32 [num_chunks * H, ceil(rows_per_chunk / query_block), top_k]: for
    every group of query rows its top_k blocks by score (the group's queries
    summed, times the block's mean), equal scores by index, listed ascending,
    -1 behind the last.  kv_rows: rows of the k that ``means`` was made from."""
    return _ops.overload("pkv_select_blocks")(q, means, cu_seqlens_k, int(kv_rows), int(num_chunks),
                                        int(rows_per_chunk), int(top_k), int(query_block),
                                        int(block))


def block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    cu_seqlens_k: torch.Tensor, num_chunks: int, rows_per_chunk: int,
                    blocks: torch.Tensor, *, query_block: int = 128, block: int = 64,
                    softmax_scale: float | None = None,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """``pkv_attention`` over the listed blocks: q bf16 [num_chunks *
    rows_per_chunk, H, D], k / v bf16 [rows, D].  Entries of ``blocks`` outside
    a segment are skipped, a block listed twice counts twice, a row with no
    keys gives zeros."""
    _no_grad(q, k, v)
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else float(softmax_scale)
    return _ops.overload("pkv_block_attention")(q, k, v, cu_seqlens_k, int(num_chunks),
                                          int(rows_per_chunk), blocks, int(query_block),
                                          int(block), scale, status)


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     cu_seqlens_k: torch.Tensor, num_chunks: int, rows_per_chunk: int,
                     top_k: int, *, query_block: int = 128, block: int = 64,
                     softmax_scale: float | None = None, means: torch.Tensor | None = None,
                     status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(output, blocks): select_blocks and block_attention, and block_means
    where the caller does not keep the table, in one call."""
    _no_grad(q, k, v)
    return _ops.overload("pkv_sparse_attention")(q, k, v, cu_seqlens_k, num_chunks,
                                                 rows_per_chunk, top_k, query_block, block,
                                                 softmax_scale, means, status)
