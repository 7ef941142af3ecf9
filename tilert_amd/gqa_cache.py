"""The paged per-head cache of grouped-query attention: pages of 64 keys, for each kv head the keys' and the values' e4m3fn
codes with one fp32 scale each a page, a power of two.  It stands beside the latent cache (``mla_cache``) for layers whose
heads are not compressed: ``gqa_cache_write`` normalises and rotates the new tokens' queries and keys head by head and
writes keys and values into the pages, ``flash_paged_gqa`` attends over them, ``gqa_cache_weights`` sums the attention
weights that each key gathers, and ``gqa_cache_evict`` keeps a sequence's heaviest and latest keys.

``kv_pages`` is uint8 [n_pages, gqa_page_bytes(kv_heads, head_dim)]; for each kv head 64 x head_dim key codes, then
head_dim x 64 value codes (a dim is a row), and behind all heads the scales [kv_heads, 2].  A batch's ``block_table``,
``cu_seqlens`` and ``seq_lens`` are those of ``mla_cache``, read on the device, so a captured graph follows changes of them;
rows behind cu_seqlens[B] are left as they are, and rows and keys whose position the table does not hold (below 0,
past it, or a page outside the pool) are not written and not seen.  A position is a place in the cache: after an eviction
the rotation's angles, which a call gets row by row, go on from the token's own place in its text.
"""
from __future__ import annotations

import torch

from .kernel import _call, _require_cuda, _stream

GQA_PAGE_KEYS = 64
GQA_HEAD_DIMS = (64, 128)
EPS = 1e-6


def gqa_page_bytes(kv_heads: int, head_dim: int) -> int:
    """Bytes of a page: codes of keys and values, and two scales a head padded to 128 bytes."""
    return kv_heads * 2 * GQA_PAGE_KEYS * head_dim + -(-kv_heads * 8 // 128) * 128


def _check_pages(name: str, kv_pages, kv_heads: int, head_dim: int) -> int:
    """The number of pages."""
    if head_dim not in GQA_HEAD_DIMS:
        raise ValueError(f"{name}: unsupported head_dim {head_dim} (one of {GQA_HEAD_DIMS})")
    if not 1 <= kv_heads <= 128:
        raise ValueError(f"{name}: unsupported kv_heads {kv_heads}")
    size, shape = gqa_page_bytes(kv_heads, head_dim), kv_pages.shape
    if kv_pages.dtype != torch.uint8 or len(shape) != 2 or shape[1] != size or not kv_pages.is_contiguous():
        raise ValueError(f"{name}: kv_pages must be a contiguous uint8 [n_pages, {size}] tensor")
    return shape[0]


def _check_metadata(name: str, block_table, seq_lens, cu_seqlens=None) -> tuple[int, int]:
    """The numbers of sequences and of a table's pages."""
    i32 = torch.int32
    if block_table.dtype != i32 or seq_lens.dtype != i32 or (cu_seqlens is not None and cu_seqlens.dtype != i32):
        raise ValueError(f"{name}: block_table, cu_seqlens and seq_lens must be int32 tensors")
    shape = block_table.shape
    if len(shape) != 2 or not block_table.is_contiguous() or not seq_lens.is_contiguous() \
            or (cu_seqlens is not None and not cu_seqlens.is_contiguous()):
        raise ValueError(f"{name}: block_table must be a contiguous [sequences, max_pages] tensor, cu_seqlens and seq_lens "
                         "contiguous")
    n = shape[0]
    if seq_lens.numel() != n or (cu_seqlens is not None and cu_seqlens.numel() != n + 1):
        raise ValueError(f"{name}: {n} sequences take {n + 1} cu_seqlens and {n} seq_lens")
    return n, shape[1]


def _check_rows(name: str, what: str, t, tokens: int | None = None, heads: int | None = None, head_dim: int | None = None) -> int:
    """bf16 [tokens, heads, head_dim] whose heads are contiguous; tokens may be further apart (views of a joint projection).
    Returns a token's stride."""
    shape = t.shape
    if t.dtype != torch.bfloat16 or len(shape) != 3:
        raise ValueError(f"{name}: {what} must be a bfloat16 [tokens, heads, head_dim] tensor")
    n, h, d = shape
    if (tokens is not None and n != tokens) or (heads is not None and h != heads) or (head_dim is not None and d != head_dim):
        raise ValueError(f"{name}: {what} is {tuple(shape)}, not "
                         f"[{tokens}, {'heads' if heads is None else heads}, {'head_dim' if head_dim is None else head_dim}]")
    per_token, per_head, per_dim = t.stride()
    if n <= 1:
        per_token = h * d
    if n * h * d and (per_dim != 1 or (h > 1 and per_head != d) or per_token % 8 or per_token < h * d):
        raise ValueError(f"{name}: a token's heads in {what} must be contiguous, and tokens a multiple of 8 elements apart "
                         f"(strides {t.stride()})")
    return per_token


def _check_key_weights(name: str, key_weights, n_pages: int, kv_heads: int) -> None:
    if key_weights.dtype != torch.float32 or key_weights.shape != (n_pages, kv_heads, GQA_PAGE_KEYS) or not key_weights.is_contiguous():
        raise ValueError(f"{name}: key_weights must be a contiguous float32 [{n_pages}, {kv_heads}, {GQA_PAGE_KEYS}] tensor")


def gqa_cache_write(key: torch.Tensor, value: torch.Tensor, kv_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, gamma_k: torch.Tensor | None = None,
                    freqs_cis: torch.Tensor | None = None, *, query: torch.Tensor | None = None,
                    gamma_q: torch.Tensor | None = None, query_out: torch.Tensor | None = None,
                    key_weights: torch.Tensor | None = None, interleaved: bool = False, eps: float = EPS) -> None:
    """Write the batch's new keys and values into ``kv_pages`` and, in the same pass, its queries into ``query_out``.

    key, value bf16 [tokens, kv_heads, head_dim] and query bf16 [tokens, heads, head_dim]: views whose tokens are further apart
    (of a joint projection's output) are taken as they are; query_out is contiguous.  Each head's row of key and query is
    normalised by RMSNorm with ``gamma_k`` / ``gamma_q`` (fp32 [head_dim]) when it is given, then its first dims are turned
    by the token's row of ``freqs_cis`` (fp32 [tokens, 1, rope_dim], cos and sin interleaved, rope_dim a multiple of 16) when
    it is given: dims i and i + rope_dim / 2 are a pair, or 2i and 2i + 1 with ``interleaved``.

    Keys and values are quantised by page and head, with the least power of two that holds the block's new rows; a block with
    older keys keeps a larger scale, or moves their codes to the larger new one, and older keys under a scale that is none
    (NaN to all that see them) stay NaN.  A key that holds a NaN or an infinity,
    in its key or its value row, is NaN to the rows that see it and touches nothing else.  ``key_weights`` (fp32 [n_pages,
    kv_heads, 64]) is set to 0 for the keys written.  A page that is written to belongs to one place of one sequence."""
    name = "gqa_cache_write"
    key_stride = _check_rows(name, "key", key)
    tokens, kv_heads, head_dim = key.shape
    value_stride = _check_rows(name, "value", value, tokens, kv_heads, head_dim)
    n_pages = _check_pages(name, kv_pages, kv_heads, head_dim)
    n, max_pages = _check_metadata(name, block_table, seq_lens, cu_seqlens)
    if (query is None) != (query_out is None) or (query is None and gamma_q is not None):
        raise ValueError(f"{name}: query and query_out go together, and gamma_q with them")
    heads = query_stride = 0
    if query is not None:
        query_stride = _check_rows(name, "query", query, tokens, None, head_dim)
        heads = query.shape[1]
        if not 1 <= heads <= 128 or heads % kv_heads:
            raise ValueError(f"{name}: unsupported heads {heads} over kv_heads {kv_heads}")
        if query_out.dtype != torch.bfloat16 or query_out.shape != query.shape or not query_out.is_contiguous():
            raise ValueError(f"{name}: query_out must be a contiguous bfloat16 tensor of query's shape")
    rope_dim = 0
    if freqs_cis is not None:
        rope_dim = freqs_cis.shape[-1] if freqs_cis.dim() else 0
        if freqs_cis.dtype != torch.float32 or not freqs_cis.is_contiguous() or rope_dim % 16 or not 16 <= rope_dim <= head_dim \
                or freqs_cis.numel() != tokens * rope_dim:
            raise ValueError(f"{name}: freqs_cis must be a contiguous float32 [{tokens}, 1, rope_dim] tensor, rope_dim a multiple of "
                             f"16 up to {head_dim}")
    for what, t in (("gamma_k", gamma_k), ("gamma_q", gamma_q)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != head_dim or not t.is_contiguous()):
            raise ValueError(f"{name}: {what} must be a contiguous float32 tensor of {head_dim} values")
    if key_weights is not None:
        _check_key_weights(name, key_weights, n_pages, kv_heads)
    _require_cuda(name, key, value, kv_pages, block_table, cu_seqlens, seq_lens, gamma_k, freqs_cis, query, gamma_q, query_out,
                  key_weights)
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    _call(key, "tl_gqa_cache_write", key.data_ptr(), key_stride, value.data_ptr(), value_stride, kv_pages.data_ptr(),
          n_pages, block_table.data_ptr(), max_pages, cu_seqlens.data_ptr(), seq_lens.data_ptr(), n, tokens,
          kv_heads, head_dim, ptr(gamma_k), ptr(freqs_cis), rope_dim, ptr(query), query_stride, heads, ptr(gamma_q), ptr(query_out), ptr(key_weights), float(eps), int(interleaved), _stream(key))


def gqa_cache_weights(query: torch.Tensor, lse: torch.Tensor, kv_pages: torch.Tensor, block_table: torch.Tensor,
                      cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, key_weights: torch.Tensor, *, accumulate: bool = True,
                      scale: float | None = None) -> None:
    """The attention weights that each key gathers from the batch's tokens, by kv head: for every key of a sequence with new
    tokens, up to the last one's own, the sum over the tokens that see it and the query heads of its group of
    exp(score - lse), with ``query`` and ``lse`` as ``flash_paged_gqa`` took and gave them.  It is added to ``key_weights``
    (fp32 [n_pages, kv_heads, 64], at the key's page and row), or takes its place with ``accumulate=False``.  A batch of a
    prompt's last tokens alone (their own cu_seqlens) gives the weights of that window.  Sequences must not share pages, and a
    sequence's table names a page once: a key's sum is one wave's."""
    name = "gqa_cache_weights"
    query_stride = _check_rows(name, "query", query)
    tokens, heads, head_dim = query.shape
    kv_heads = key_weights.shape[1] if key_weights.dim() == 3 else 0
    if not 1 <= kv_heads <= 128 or not 1 <= heads <= 128 or heads % kv_heads:
        raise ValueError(f"{name}: unsupported heads {heads} over kv_heads {kv_heads}")
    n_pages = _check_pages(name, kv_pages, kv_heads, head_dim)
    _check_key_weights(name, key_weights, n_pages, kv_heads)
    n, max_pages = _check_metadata(name, block_table, seq_lens, cu_seqlens)
    if lse.dtype != torch.float32 or lse.shape != (tokens, heads) or not lse.is_contiguous():
        raise ValueError(f"{name}: lse must be a contiguous float32 [{tokens}, {heads}] tensor")
    _require_cuda(name, query, lse, kv_pages, block_table, cu_seqlens, seq_lens, key_weights)
    _call(query, "tl_gqa_cache_weights", query.data_ptr(), query_stride, lse.data_ptr(), kv_pages.data_ptr(), n_pages,
          block_table.data_ptr(), max_pages, cu_seqlens.data_ptr(), seq_lens.data_ptr(), n, tokens, heads, kv_heads, head_dim,
          float(head_dim ** -0.5 if scale is None else scale), int(accumulate), key_weights.data_ptr(), _stream(query))


def gqa_cache_evict(kv_pages: torch.Tensor, key_weights: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    keep_lens: torch.Tensor, kept_table: torch.Tensor, kept_lens: torch.Tensor,
                    kept_slots: torch.Tensor | None = None, *, head_dim: int, recent: int = 0) -> None:
    """Bring each sequence down to its keep_lens[b] keys, for each kv head on its own: the last ``recent`` positions stay, and
    of the others those of the largest ``key_weights`` (equal ones: the lowest position; NaN counts as the largest).  They
    go in ascending order, codes, scales and weights, into the pages of ``kept_table`` (int32 [sequences, pages], of the
    same pool); the sequences' own pages are left as they are, and may be given back afterwards.  ``kept_lens`` (int32
    [sequences], not in seq_lens' memory; it may be keep_lens itself, but not overlap it) receives the new lengths -- keep_lens, but no more than there are keys
    or kept_table has room for -- and ``kept_slots`` (int32 [sequences, kv_heads, 64 * pages]) the positions that were kept,
    -1 behind them.  kept_table names a page once, and none of the tables'; one outside the pool is not written."""
    name = "gqa_cache_evict"
    kv_heads = key_weights.shape[1] if key_weights.dim() == 3 else 0
    n_pages = _check_pages(name, kv_pages, kv_heads, head_dim)
    _check_key_weights(name, key_weights, n_pages, kv_heads)
    n, max_pages = _check_metadata(name, block_table, seq_lens)
    for what, t in (("keep_lens", keep_lens), ("kept_lens", kept_lens)):
        if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be a contiguous int32 tensor of {n} values")
    if kept_table.dtype != torch.int32 or kept_table.dim() != 2 or kept_table.shape[0] != n or not kept_table.is_contiguous():
        raise ValueError(f"{name}: kept_table must be a contiguous int32 [{n}, pages] tensor")
    pages = kept_table.shape[1]
    if kept_slots is not None and (kept_slots.dtype != torch.int32 or kept_slots.shape != (n, kv_heads, pages * GQA_PAGE_KEYS)
                                   or not kept_slots.is_contiguous()):
        raise ValueError(f"{name}: kept_slots must be a contiguous int32 [{n}, {kv_heads}, {pages * GQA_PAGE_KEYS}] tensor")
    if recent < 0:
        raise ValueError(f"{name}: recent must not be negative (got {recent})")
    _require_cuda(name, kv_pages, key_weights, block_table, seq_lens, keep_lens, kept_table, kept_lens, kept_slots)
    if kept_slots is None:
        kept_slots = kept_table.new_empty(n, kv_heads, pages * GQA_PAGE_KEYS)
    _call(kv_pages, "tl_gqa_cache_evict", kv_pages.data_ptr(), key_weights.data_ptr(), n_pages, block_table.data_ptr(),
          max_pages, seq_lens.data_ptr(), keep_lens.data_ptr(), n, kv_heads, head_dim, recent, kept_table.data_ptr(), pages,
          kept_lens.data_ptr(), kept_slots.data_ptr(), _stream(kv_pages))
