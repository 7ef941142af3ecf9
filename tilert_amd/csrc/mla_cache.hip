// The paged latent cache (paged.h): writing the new tokens' keys, quantised, and reading keys back as bf16.
#include "paged.h"
#include "../../include/tilert_amd.h"

namespace tl {

typedef uint32_t u32x4c __attribute__((ext_vector_type(4)));

// One wave a token, 8 latent values a lane:
//   n = kv * rsqrt(mean(kv^2) + eps) * gamma   (NORM; n = kv without)
//   s = group_scale(max |n|), code = e4m3(clamp(n / s)), all from the fp32 n
// and the rope part turned by its token's angles (lanes 0 .. 31, a pair each).  A key that holds a
// NaN or an infinity gets the scale NaN: its codes are finite whatever it held, so only rows of an attention that see
// the key are touched by it.
// A wave needs no other's values: no LDS, no barrier, and the row's loads are all under way before the token's place
// is known.  Bound by the round trips one behind another (cu_seqlens, lengths, table, store) in small calls and by
// bytes (1408 read and 644 written a token) in large ones: one token 2.6 us, 4000 tokens of 5 sequences 5.7 us,
// 1.5 TB/s, where a launch that does nothing takes 2.
template <bool NORM>
__global__ __launch_bounds__(256) void mla_cache_write_kernel(const uint16_t* __restrict__ kv, const uint16_t* __restrict__ pe,
                                                              uint8_t* __restrict__ pages, PagedBatch p,
                                                              const float* __restrict__ gamma, const float* __restrict__ freqs,
                                                              float eps, int interleaved, int scale_mode) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.n_tokens) return;
  const u32x4c raw = reinterpret_cast<const u32x4c*>(kv + static_cast<int64_t>(t) * kKvLatent)[lane];
  float g[8];
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = gamma[lane * 8 + i];
  }
  const int pair = lane & 31;
  const int at0 = interleaved ? 2 * pair : pair, at1 = interleaved ? 2 * pair + 1 : pair + 32;
  const uint16_t* pr = pe + static_cast<int64_t>(t) * kKvRope;
  float z0 = bf16_to_f32(pr[at0]), z1 = bf16_to_f32(pr[at1]);
  if (freqs) {
    const float c = freqs[static_cast<int64_t>(t) * kKvRope + 2 * pair], s = freqs[static_cast<int64_t>(t) * kKvRope + 2 * pair + 1];
    const float a = z0 * c - z1 * s;
    z1 = z0 * s + z1 * c;
    z0 = a;
  }
  const KeyPlace to = key_place(p, find_seq(p.cu, p.n_seqs, t), t);
  if (to.page < 0) return;
  float n[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    n[2 * i] = __uint_as_float(raw[i] << 16);
    n[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
  }
  if constexpr (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(n[i], n[i], ss);
    const float r = 1.0f / __builtin_sqrtf(wave_sum_f32(ss) / kKvLatent + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = n[i] * r * g[i];
  }
  float amax = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax = fmaxf(amax, __builtin_fabsf(n[i]));
    finite = finite && __builtin_fabsf(n[i]) < INFINITY;
  }
  const float s = __all(finite) ? group_scale(wave_max_f32(amax), scale_mode) : __builtin_nanf("");
  uint8_t* page = pages + static_cast<int64_t>(to.page) * kKvPageBytes;
  reinterpret_cast<uint2*>(page + to.row * kKvLatent)[lane] = quant8_e4m3(n, s);
  if (lane == 0) *reinterpret_cast<float*>(page + kKvScaleAt + to.row * 4) = s;
  if (lane < 32) {
    uint16_t* rope = reinterpret_cast<uint16_t*>(page + kKvRopeAt) + to.row * kKvRope;
    rope[at0] = f32_to_bf16(z0);
    rope[at1] = f32_to_bf16(z1);
  }
}

// One wave a key: its latent as bf16(code * scale), its rope part as it is.  Bound by bytes, 644 read and 1152 written a
// key: 143 thousand keys of 9 sequences, 257 MB, 40 us (6.4 TB/s) where the Infinity Cache holds part of them, 59 us a
// call (4.4 TB/s; a large copy 4.7) over caches that it does not; 2100 keys 3.2 us.
__global__ __launch_bounds__(256) void mla_cache_read_kernel(const uint8_t* __restrict__ pages, PagedBatch p,
                                                             uint16_t* __restrict__ kv, uint16_t* __restrict__ pe) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= p.n_tokens) return;
  const KeyPlace at = key_place(p, find_seq(p.cu, p.n_seqs, t), t);
  if (at.page < 0) return;
  const uint8_t* page = pages + static_cast<int64_t>(at.page) * kKvPageBytes;
  const uint2 code = reinterpret_cast<const uint2*>(page + at.row * kKvLatent)[lane];
  const float s = *reinterpret_cast<const float*>(page + kKvScaleAt + at.row * 4);
  const v8bf v = dequant8_bf16(code.x, code.y, s);
  reinterpret_cast<u32x4c*>(kv + static_cast<int64_t>(t) * kKvLatent)[lane] = __builtin_bit_cast(u32x4c, v);
  pe[static_cast<int64_t>(t) * kKvRope + lane] = reinterpret_cast<const uint16_t*>(page + kKvRopeAt)[at.row * kKvRope + lane];
}

}  // namespace tl

using namespace tl;

extern "C" int tl_mla_cache_write(const void* kv_bf16, const void* pe_bf16, void* kv_pages, int64_t n_pages,
                                  const int32_t* block_table, int64_t max_pages, const int32_t* cu_seqlens,
                                  const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens, const float* gamma,
                                  const float* freqs, float eps, int interleaved, int scale_mode, void* stream) {
  if (int rc = check_batch("mla_cache_write", kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (scale_mode < 0 || scale_mode > 2) { set_error("mla_cache_write: bad scale_mode %d", scale_mode); return kErrArg; }
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (!kv_bf16 || !pe_bf16) { set_error("mla_cache_write: null pointer"); return kErrArg; }
  if ((reinterpret_cast<uintptr_t>(kv_bf16) | reinterpret_cast<uintptr_t>(gamma)) & 15) {
    set_error("mla_cache_write: kv and gamma must be 16-byte aligned");
    return kErrArg;
  }
  const PagedBatch p{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens};
  const auto kern = gamma ? mla_cache_write_kernel<true> : mla_cache_write_kernel<false>;
  hipLaunchKernelGGL(kern, dim3(cdiv(n_tokens, 4)), dim3(256), 0, (hipStream_t)stream, (const uint16_t*)kv_bf16,
                     (const uint16_t*)pe_bf16, (uint8_t*)kv_pages, p, gamma, freqs, eps, interleaved, scale_mode);
  return check_launch("mla_cache_write");
}

extern "C" int tl_mla_cache_read(const void* kv_pages, int64_t n_pages, const int32_t* block_table, int64_t max_pages,
                                 const int32_t* cu_seqlens, const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens,
                                 void* kv_bf16, void* pe_bf16, void* stream) {
  if (int rc = check_batch("mla_cache_read", kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (!kv_bf16 || !pe_bf16) { set_error("mla_cache_read: null pointer"); return kErrArg; }
  if ((reinterpret_cast<uintptr_t>(kv_bf16) | reinterpret_cast<uintptr_t>(pe_bf16)) & 15) {
    set_error("mla_cache_read: kv and pe must be 16-byte aligned");
    return kErrArg;
  }
  const PagedBatch p{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens};
  hipLaunchKernelGGL(mla_cache_read_kernel, dim3(cdiv(n_tokens, 4)), dim3(256), 0, (hipStream_t)stream,
                     (const uint8_t*)kv_pages, p, (uint16_t*)kv_bf16, (uint16_t*)pe_bf16);
  return check_launch("mla_cache_read");
}
