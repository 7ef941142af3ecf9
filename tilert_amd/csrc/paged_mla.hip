// Causal MLA attention of a batch's new tokens over the paged latent cache (paged.h).  For token t of sequence b, at
// position p, and head h, over the keys j <= p:
//   s[j] = (q_nope[t,h] . latent[j] + q_pe[t,h] . rope[j]) * softmax_scale
//   out[t,h] = sum_j softmax(s)[j] latent[j],  lse[t,h] = ln sum_j e^s[j]      (0 and -inf where no key is seen)
#include <math.h>

#include "paged.h"
#include "../../include/tilert_amd.h"

namespace tl {

typedef uint32_t u32x4p __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2p __attribute__((ext_vector_type(2)));

// One wave a row (token, head): 8 latent dims and one rope dim a lane, key after key, with the running
// maximum and sum.
__global__ __launch_bounds__(256) void paged_mla_rows_kernel(const uint16_t* __restrict__ q_nope, const uint16_t* __restrict__ q_pe,
                                                             const uint8_t* __restrict__ pages, PagedBatch p, int heads,
                                                             float scale, uint16_t* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = static_cast<int>(r / heads);
  if (t >= p.n_tokens) return;
  const int b = find_seq(p.cu, p.n_seqs, t);
  if (b < 0 || b >= p.n_seqs) return;
  const int64_t first = p.cu[b], end = p.cu[b + 1];
  if (t < first || t >= end) return;
  const int64_t seen = min(p.lens[b] - end + t + 1, static_cast<int64_t>(p.max_pages) * kKvPageKeys);
  float q[8], o[8], qp = bf16_to_f32(q_pe[r * kKvRope + lane]);
  const u32x4p raw = reinterpret_cast<const u32x4p*>(q_nope + r * kKvLatent)[lane];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = __uint_as_float(i & 1 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < seen; ++j) {
    const int pg = p.table[static_cast<int64_t>(b) * p.max_pages + (j >> 6)];
    if (pg < 0 || pg >= p.n_pages) continue;
    const int row = static_cast<int>(j & 63);
    const uint8_t* page = pages + static_cast<int64_t>(pg) * kKvPageBytes;
    const uint2 code = reinterpret_cast<const uint2*>(page + row * kKvLatent)[lane];
    const float ks = *reinterpret_cast<const float*>(page + kKvScaleAt + row * 4);
    float k[8];
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(code.x, false), c = __builtin_amdgcn_cvt_pk_f32_fp8(code.x, true);
    const v2f d = __builtin_amdgcn_cvt_pk_f32_fp8(code.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8(code.y, true);
    k[0] = a.x; k[1] = a.y; k[2] = c.x; k[3] = c.y; k[4] = d.x; k[5] = d.y; k[6] = e.x; k[7] = e.y;
    float dot = qp * bf16_to_f32(reinterpret_cast<const uint16_t*>(page + kKvRopeAt)[row * kKvRope + lane]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      k[i] *= ks;
      dot = __builtin_fmaf(q[i], k[i], dot);
    }
    const float s = wave_sum_f32(dot) * scale;
    const float mn = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(s - mn);
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * keep + w * k[i];
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  u32x4p w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = bf16x2_bits(v2f{o[2 * i] * inv, o[2 * i + 1] * inv});
  reinterpret_cast<u32x4p*>(out + r * kKvLatent)[lane] = w;
  if (lse && lane == 0) lse[r] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace tl

using namespace tl;

extern "C" int tl_flash_paged_mla(const void* q_nope_bf16, const void* q_pe_bf16, const void* kv_pages, int64_t n_pages,
                                  const int32_t* block_table, int64_t max_pages, const int32_t* cu_seqlens,
                                  const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens, int64_t heads,
                                  float softmax_scale, void* out_bf16, float* lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_batch("flash_paged_mla", kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (heads < 1 || heads > 128) { set_error("flash_paged_mla: heads=%lld must be in [1, 128]", (long long)heads); return kErrUnsupported; }
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (n_tokens * heads >= (1ll << 31)) { set_error("flash_paged_mla: %lld tokens x %lld heads: too many rows", (long long)n_tokens, (long long)heads); return kErrUnsupported; }
  if (!q_nope_bf16 || !q_pe_bf16 || !out_bf16) { set_error("flash_paged_mla: null pointer"); return kErrArg; }
  if ((reinterpret_cast<uintptr_t>(q_nope_bf16) | reinterpret_cast<uintptr_t>(q_pe_bf16) | reinterpret_cast<uintptr_t>(out_bf16)) & 15) {
    set_error("flash_paged_mla: q and out must be 16-byte aligned");
    return kErrArg;
  }
  const PagedBatch p{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens};
  hipLaunchKernelGGL(paged_mla_rows_kernel, dim3(cdiv(n_tokens * heads, 4)), dim3(256), 0, (hipStream_t)stream,
                     (const uint16_t*)q_nope_bf16, (const uint16_t*)q_pe_bf16, (const uint8_t*)kv_pages, p, (int)heads,
                     softmax_scale, (uint16_t*)out_bf16, lse);
  return check_launch("flash_paged_mla");
}

extern "C" size_t tl_flash_paged_mla_workspace_bytes(int64_t n_seqs, int64_t n_tokens, int64_t heads) {
  return 0;
}
