"""Causal grouped-query attention of new tokens over the paged per-head cache (``gqa_cache``): a prefill chunk, a decode step of
a batch, or both in one call -- ``flash_paged_mla`` for heads that are not compressed."""
from __future__ import annotations

import torch

from . import _lib
from .gqa_cache import _check_metadata, _check_pages, _check_rows
from .kernel import _call, _require_cuda, _stream


def flash_paged_gqa(query: torch.Tensor, kv_pages: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                    seq_lens: torch.Tensor, output: torch.Tensor, lse: torch.Tensor | None = None, *, kv_heads: int,
                    scale: float | None = None) -> None:
    """query bf16 [tokens, heads, head_dim] (tokens may be further apart than their heads take), head_dim 64 or 128, heads a
    multiple of kv_heads and at most 128: query head h reads kv head h // (heads // kv_heads).  kv_pages, block_table,
    cu_seqlens, seq_lens as ``gqa_cache`` describes them, the tokens' own keys written before.  A token at position p sees the
    keys 0 .. p of its sequence; ``output`` bf16 [tokens, heads, head_dim] and, when given, ``lse`` fp32 [tokens, heads] (ln of
    the sum of exp of its scores) are filled, with 0 and -inf for a token that sees no key.  ``scale`` is the softmax
    scale, head_dim ** -0.5 unless given; positive, and finite times log2(e).

    Scores, statistics and sums are fp32.  The weights are multiplied with the values in 16 bits, or, in a batch with more than
    32 rows (tokens times heads // kv_heads; 64 with head_dim 64) a sequence in the mean, in bf16's 8 bits, which takes the
    result's rms error from 0.0017 to 0.0023 of it: the same token may have either, alone or beside a chunk.  Within a call a
    row follows from its query and the keys that it sees, whatever the other rows hold; how its sum is split follows from
    the batch's sizes and lengths."""
    name = "flash_paged_gqa"
    query_stride = _check_rows(name, "query", query)
    tokens, heads, head_dim = query.shape
    n_pages = _check_pages(name, kv_pages, kv_heads, head_dim)
    if not 1 <= heads <= 128 or heads % kv_heads:
        raise ValueError(f"{name}: unsupported heads {heads} over kv_heads {kv_heads}")
    n, max_pages = _check_metadata(name, block_table, seq_lens, cu_seqlens)
    if output.dtype != torch.bfloat16 or output.shape != query.shape or not output.is_contiguous():
        raise ValueError(f"{name}: output must be a contiguous bfloat16 tensor of query's shape")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (tokens, heads) or not lse.is_contiguous()):
        raise ValueError(f"{name}: lse must be a contiguous float32 [{tokens}, {heads}] tensor")
    _require_cuda(name, query, kv_pages, block_table, cu_seqlens, seq_lens, output, lse)
    nbytes = _lib.query("tl_flash_paged_gqa_workspace_bytes", n, tokens, heads, kv_heads, head_dim, max_pages)
    # taken from the allocator call by call: its memory is ordered on the stream, and a captured graph's is its own
    ws = query.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(query, "tl_flash_paged_gqa", query.data_ptr(), query_stride, kv_pages.data_ptr(), n_pages,
          block_table.data_ptr(), max_pages, cu_seqlens.data_ptr(), seq_lens.data_ptr(), n, tokens, heads, kv_heads, head_dim,
          float(head_dim ** -0.5 if scale is None else scale), output.data_ptr(), lse.data_ptr() if lse is not None else None,
          ws.data_ptr() if ws is not None else None, nbytes, _stream(query))
