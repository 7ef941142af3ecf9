"""Causal MLA attention of new tokens over the paged latent cache (``mla_cache``): a prefill chunk, a decode step of a
batch, or both in one call -- the dense counterpart of ``flash_sparse_mla``, whose scores, scale and absorbed
512 + 64 wide queries it shares (FlashSparseMLACombine.golden_forward, ops/flash_sparse_mla.py:152-196, with every
position up to the token's own selected)."""
from __future__ import annotations

import torch

from . import _lib
from .flash_sparse_mla import softmax_scale
from .kernel import _call, _require_cuda, _stream
from .mla_cache import LATENT, ROPE, _check_batch

_SCALES: dict[str, float] = {}


def flash_paged_mla(query: torch.Tensor, query_pe: torch.Tensor, kv_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, output: torch.Tensor,
                    lse: torch.Tensor | None = None, profile_logs: torch.Tensor | None = None,
                    compute_kernel_type: str = "bf16mma", *, model_arch: str, scale: float | None = None) -> None:
    """query bf16 [.., heads, 512] and query_pe bf16 [.., heads, 64], heads <= 128, one pair of rows a token; kv_pages,
    block_table, cu_seqlens, seq_lens as ``mla_cache`` describes them, the tokens' own keys written before.  A token at
    position p sees the keys 0 .. p of its sequence; ``output`` bf16 [.., heads, 512] and, when given, ``lse`` fp32
    [.., heads] (ln of the sum of exp of its scores) are filled, with 0 and -inf for a token that sees no key.
    Keys outside the table, or in a page outside the pool, are not seen.  ``scale`` overrides the model's softmax
    scale."""
    n = _check_batch("flash_paged_mla", kv_pages, block_table, cu_seqlens, seq_lens)
    if compute_kernel_type != "bf16mma":
        raise ValueError(f"unsupported compute_kernel_type {compute_kernel_type!r}")
    if query.dtype != torch.bfloat16 or query_pe.dtype != torch.bfloat16 or output.dtype != torch.bfloat16:
        raise ValueError("flash_paged_mla: query, query_pe and output must be bfloat16 tensors")
    if query.dim() < 2 or query.shape[-1] != LATENT or query_pe.shape[-1] != ROPE:
        raise ValueError("flash_paged_mla expects a 512-wide latent and 64-wide rope part")
    if not query.is_contiguous() or not query_pe.is_contiguous() or not output.is_contiguous():
        raise ValueError("flash_paged_mla: query, query_pe and output must be contiguous")
    heads = query.shape[-2]
    if not 1 <= heads <= 128:
        raise ValueError(f"Unsupported heads: {heads}")
    if query_pe.shape[:-1] != query.shape[:-1] or output.shape != query.shape:
        raise ValueError("flash_paged_mla: query_pe must have query's tokens and heads, output query's shape")
    rows = query.numel() // LATENT
    if lse is not None and (lse.dtype != torch.float32 or lse.numel() != rows or not lse.is_contiguous()):
        raise ValueError("flash_paged_mla: lse must be a contiguous float32 [.., heads] tensor")
    _require_cuda("flash_paged_mla", query, query_pe, kv_pages, block_table, cu_seqlens, seq_lens, output, lse)
    if scale is None:
        scale = _SCALES.get(model_arch)
        if scale is None:
            scale = _SCALES[model_arch] = softmax_scale(model_arch)
    st = _stream(query)
    tokens = rows // heads
    nbytes = _lib.query("tl_flash_paged_mla_workspace_bytes", n, tokens, heads, block_table.shape[1])
    # taken from the allocator call by call: its memory is ordered on the stream, and a captured graph's is its own
    ws = query.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(query, "tl_flash_paged_mla", query.data_ptr(), query_pe.data_ptr(), kv_pages.data_ptr(), kv_pages.shape[0],
          block_table.data_ptr(), block_table.shape[1], cu_seqlens.data_ptr(), seq_lens.data_ptr(), n, tokens, heads,
          float(scale), output.data_ptr(), lse.data_ptr() if lse is not None else None,
          ws.data_ptr() if ws is not None else None, nbytes, st)
