// A batch of sequences over the paged latent cache: what the kernels of mla_cache.hip and paged_mla.hip share.
//
// KV page, kKvPageBytes = 41216 bytes, 64 keys: their e4m3fn codes [64][512], their fp32 scales [64], their rope
// parts bf16 [64][64].  A key's latent is code * scale.
//
// Sequence b owns the batch's tokens cu[b] .. cu[b+1]-1, its newest; its cache holds lens[b] keys with them, so token t
// stands at position lens[b] - (cu[b+1] - cu[b]) + t - cu[b].  The key at position p is row p % 64 of page
// table[b][p / 64].  All of it is read on the device and none of it is trusted: a position below 0 or past the
// table, and a page outside the pool, name no key.
#pragma once

#include "common.h"

namespace tl {

constexpr int kKvLatent = 512;  // kv_lora_rank
constexpr int kKvRope = 64;     // qk_rope_head_dim
constexpr int kKvPageKeys = 64;
constexpr int kKvScaleAt = kKvPageKeys * kKvLatent;
constexpr int kKvRopeAt = kKvScaleAt + kKvPageKeys * 4;
constexpr int kKvPageBytes = kKvRopeAt + kKvPageKeys * kKvRope * 2;  // 41216

struct PagedBatch {
  const int32_t* table;  // [n_seqs][max_pages]
  const int32_t* cu;     // [n_seqs + 1]
  const int32_t* lens;   // [n_seqs]
  int n_seqs, max_pages, n_pages, n_tokens;
};

// The last index i of 0 .. n_seqs for which upto(i) holds, a wave-uniform predicate that holds up to some index (-1: for
// none).  64 indices a round, so one round up to 63 sequences, two up to 4095.  Whatever upto says, it is asked about
// 0 .. n_seqs only and the result is in [-1, n_seqs].
template <class F>
__device__ inline int last_seq(int n_seqs, F upto) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = n_seqs + 1;  // the first index for which it does not hold is in [lo, lo + n]
  while (n > 64) {
    const int step = (n + 63) >> 6, i = lane * step;
    const int c = __popcll(__ballot(i < n && upto(lo + i)));
    if (c == 0) return lo - 1;
    const int from = (c - 1) * step + 1;
    n = min(n, c * step) - from;
    lo += from;
  }
  return lo + __popcll(__ballot(lane < n && upto(lo + lane))) - 1;
}
// The sequence of token t (wave-uniform; -1 or n_seqs: none; empty sequences are passed over).
__device__ inline int find_seq(const int32_t* __restrict__ cu, int n_seqs, int t) {
  return last_seq(n_seqs, [&](int b) { return cu[b] <= t; });
}

// The place of token t of sequence b (any lane, any value): its page and row in the pool; page < 0: there is none.
struct KeyPlace {
  int page, row;
};
__device__ inline KeyPlace key_place(const PagedBatch& p, int b, int t) {
  if (b < 0 || b >= p.n_seqs) return {-1, 0};
  const int64_t first = p.cu[b], end = p.cu[b + 1];
  if (t < first || t >= end) return {-1, 0};
  const int64_t pos = p.lens[b] - end + t;
  if (pos < 0 || pos >= static_cast<int64_t>(p.max_pages) * kKvPageKeys) return {-1, 0};
  const int page = p.table[static_cast<int64_t>(b) * p.max_pages + (pos >> 6)];
  return {page >= 0 && page < p.n_pages ? page : -1, static_cast<int>(pos & 63)};
}

// The host's checks of a batch; `who` names the entry point.
inline int check_batch(const char* who, const void* pages, int64_t n_pages, const int32_t* table, int64_t max_pages,
                       const int32_t* cu, const int32_t* lens, int64_t n_seqs, int64_t n_tokens) {
  // (a launch has fewer than 2^32 threads: a wave a token, four tokens a workgroup)
  if (n_seqs < 0 || n_tokens < 0 || n_seqs >= (1ll << 24) || n_tokens > (1ll << 26) - 4) {
    set_error("%s: %lld sequences, %lld tokens: out of range", who, (long long)n_seqs, (long long)n_tokens);
    return kErrArg;
  }
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (max_pages < 1 || max_pages > (1ll << 25) - 1 || n_pages < 1 || n_pages >= (1ll << 31)) {
    set_error("%s: max_pages=%lld must be in [1, 2^25), n_pages=%lld in [1, 2^31)", who, (long long)max_pages, (long long)n_pages);
    return kErrArg;
  }
  if (!pages || !table || !cu || !lens) { set_error("%s: null pointer", who); return kErrArg; }
  if (reinterpret_cast<uintptr_t>(pages) & 15) { set_error("%s: the pages must be 16-byte aligned", who); return kErrArg; }
  return kOk;
}

}  // namespace tl
