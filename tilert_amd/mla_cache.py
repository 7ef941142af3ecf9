"""The paged MLA latent cache: pages of 64 keys, each key 512 e4m3fn codes with one fp32 scale and a 64-wide bf16
rope part (the KI pages' layout, ``sparse_index.KI_PAGE_BYTES``, with a rope block).  ``mla_cache_write`` turns the
down-projection's output into keys of it (rmsnorm_kv_op and the key half of qkv_rope_op, ops/rmsnorm_kv.py:20-43,
ops/qkv_rope.py:42-50, with the quantisation the reference keeps for its wire format); ``mla_cache_read`` brings keys
back in the flat bf16 form that ``flash_sparse_mla`` takes; ``flash_paged_mla`` attends over the pages.

The three share a batch's metadata, int32 on the device: ``block_table`` [B, max_pages] (the pages of each sequence's
cache), ``cu_seqlens`` [B + 1] (sequence b owns rows cu_seqlens[b] .. cu_seqlens[b+1]-1 of the call's tensors) and
``seq_lens`` [B] (the cache's length with those rows): row t of sequence b is the key at position
seq_lens[b] - (cu_seqlens[b+1] - cu_seqlens[b]) + t - cu_seqlens[b], the newest keys of the cache.  It is read by the
kernels, so a captured graph follows changes of it.  Rows behind cu_seqlens[B] are left as they are, and so are
rows whose position the table does not hold (below 0, past it, or a page outside the pool).
"""
from __future__ import annotations

import torch

from .kernel import SCALE_MODES, _call, _require_cuda, _stream

LATENT, ROPE = 512, 64
KV_PAGE_KEYS = 64
KV_PAGE_BYTES = KV_PAGE_KEYS * (LATENT + 4 + 2 * ROPE)  # 41216
EPS = 1e-6


def _check_batch(name: str, kv_pages, block_table, cu_seqlens, seq_lens) -> int:
    """The batch's checks, common to the three operators; the number of sequences."""
    if kv_pages.dtype != torch.uint8 or kv_pages.dim() != 2 or kv_pages.shape[1] != KV_PAGE_BYTES \
            or not kv_pages.is_contiguous():
        raise ValueError(f"{name}: kv_pages must be a contiguous uint8 [n_pages, {KV_PAGE_BYTES}] tensor")
    if block_table.dtype != torch.int32 or cu_seqlens.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError(f"{name}: block_table, cu_seqlens and seq_lens must be int32 tensors")
    if block_table.dim() != 2 or not block_table.is_contiguous() or not cu_seqlens.is_contiguous() \
            or not seq_lens.is_contiguous():
        raise ValueError(f"{name}: block_table must be a contiguous [sequences, max_pages] tensor, cu_seqlens and seq_lens "
                         "contiguous")
    n = block_table.shape[0]
    if cu_seqlens.numel() != n + 1 or seq_lens.numel() != n:
        raise ValueError(f"{name}: {n} sequences take {n + 1} cu_seqlens and {n} seq_lens "
                         f"(got {cu_seqlens.numel()} and {seq_lens.numel()})")
    return n


def _check_rows(name: str, kv, pe) -> int:
    """bf16 [.., 512] and [.., 64] of as many rows; their number."""
    if kv.dtype != torch.bfloat16 or pe.dtype != torch.bfloat16:
        raise ValueError(f"{name}: the latent and rope rows must be bfloat16 tensors")
    if kv.shape[-1] != LATENT or pe.shape[-1] != ROPE or not kv.is_contiguous() or not pe.is_contiguous():
        raise ValueError(f"{name}: expects contiguous [.., {LATENT}] latent and [.., {ROPE}] rope rows")
    n = kv.numel() // LATENT
    if pe.numel() != n * ROPE:
        raise ValueError(f"{name}: as many rope rows as latent rows ({pe.numel() // ROPE} vs {n})")
    return n


def mla_cache_write(kv_in: torch.Tensor, pe_in: torch.Tensor, kv_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, gamma: torch.Tensor | None = None,
                    freqs_cis: torch.Tensor | None = None, *, scale_fmt: str | None = "div", interleaved: bool = True,
                    eps: float = EPS) -> None:
    """Write the batch's new keys into ``kv_pages``: kv_in bf16 [.., 512], normalised by RMSNorm with ``gamma`` (fp32
    [512]) when it is given, quantised with one scale a key (``scale_fmt`` as in ``act_quant``) from the fp32
    values; pe_in bf16 [.., 64], turned by its row of ``freqs_cis`` (fp32 [rows, 1, 64], cos and sin interleaved as
    ``layernorm_rope_rotate`` takes them) when it is given: dims 2i and 2i + 1 are a pair, or i and i + 32 with
    ``interleaved=False``.  A key that holds a NaN or an infinity reads back as NaN.  Sequences must not share the pages
    that are written to."""
    n = _check_batch("mla_cache_write", kv_pages, block_table, cu_seqlens, seq_lens)
    rows = _check_rows("mla_cache_write", kv_in, pe_in)
    for what, t, size in (("gamma", gamma, LATENT), ("freqs_cis", freqs_cis, rows * ROPE)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != size or not t.is_contiguous()):
            raise ValueError(f"mla_cache_write: {what} must be a contiguous float32 tensor of {size} values")
    _require_cuda("mla_cache_write", kv_in, pe_in, kv_pages, block_table, cu_seqlens, seq_lens, gamma, freqs_cis)
    _call(kv_in, "tl_mla_cache_write", kv_in.data_ptr(), pe_in.data_ptr(), kv_pages.data_ptr(), kv_pages.shape[0],
              block_table.data_ptr(), block_table.shape[1], cu_seqlens.data_ptr(), seq_lens.data_ptr(), n, rows,
              gamma.data_ptr() if gamma is not None else None, freqs_cis.data_ptr() if freqs_cis is not None else None,
              float(eps), int(interleaved), SCALE_MODES.get(scale_fmt, 1), _stream(kv_in))


def mla_cache_read(kv_pages: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor,
                   kv_out: torch.Tensor, pe_out: torch.Tensor) -> None:
    """Read the batch's keys back: kv_out bf16 [.., 512] = bf16(code * scale), pe_out bf16 [.., 64]; with
    cu_seqlens the running sum of seq_lens, whole caches one behind another.  (MlaNsaProfile.convert's bf16 caches,
    pd_vllm/profiles/mla_nsa.py:150-185.)"""
    n = _check_batch("mla_cache_read", kv_pages, block_table, cu_seqlens, seq_lens)
    rows = _check_rows("mla_cache_read", kv_out, pe_out)
    _require_cuda("mla_cache_read", kv_pages, block_table, cu_seqlens, seq_lens, kv_out, pe_out)
    _call(kv_pages, "tl_mla_cache_read", kv_pages.data_ptr(), kv_pages.shape[0], block_table.data_ptr(), block_table.shape[1],
              cu_seqlens.data_ptr(), seq_lens.data_ptr(), n, rows, kv_out.data_ptr(), pe_out.data_ptr(), _stream(kv_out))
