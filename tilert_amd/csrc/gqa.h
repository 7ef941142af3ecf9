// The paged per-head cache (grouped-query attention): what the kernels of gqa_cache.hip and paged_gqa.hip share.
//
// Page of 64 keys: for each kv head 64 x D e4m3fn key codes, then D x 64 e4m3fn value codes (a dim is a row); behind all heads
// two fp32 scales a head (keys, values), the whole padded to 128 bytes.  A key is code * scale, its head's scale in its page.
//
// * The scales are powers of two, so that code * scale is exact in bf16 and v_cvt_scalef32_pk_bf16_fp8 makes two of them
//   in one instruction, and so that codes move to a larger scale exactly but for those that become subnormal.
// * The values lie transposed: the 16 consecutive keys of a dim that a lane of the second product multiplies are then one
//   16-byte load from the page, and the products need no transposition through LDS.
//
// The batch is paged.h's: its sequences, their tokens and tables, none of it trusted.
#pragma once

#include "paged.h"

namespace tl {

typedef uint32_t u32x4g __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2g __attribute__((ext_vector_type(2)));

constexpr int kGqaKeys = 64;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

__host__ __device__ inline int64_t gqa_page_bytes(int64_t kv_heads, int64_t head_dim) {
  return kv_heads * 2 * kGqaKeys * head_dim + (kv_heads * 8 + 127) / 128 * 128;
}

// One head's block of a page.
struct GqaBlock {
  uint8_t* k;    // [64][D]
  uint8_t* v;    // [D][64]
  float* scale;  // keys, values
};
template <int D>
__device__ inline GqaBlock gqa_block(const uint8_t* pages, int64_t page_bytes, int kv_heads, int page, int head) {
  uint8_t* p = const_cast<uint8_t*>(pages) + page * page_bytes;
  uint8_t* k = p + static_cast<int64_t>(head) * (2 * kGqaKeys * D);
  return {k, k + kGqaKeys * D, reinterpret_cast<float*>(p + static_cast<int64_t>(kv_heads) * (2 * kGqaKeys * D)) + 2 * head};
}

// The least power of two s with max(amax, 1e-4) <= 448 s, from the bits: 448 is 1.75 * 2^8.  At most 2^120.
__device__ inline float gqa_scale(float amax) {
  const uint32_t u = __float_as_uint(fmaxf(amax, 1e-4f));
  const uint32_t e = (u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
  return __uint_as_float(e << 23);
}
// Whether a stored scale is one: positive and finite, no subnormal.
__device__ inline bool gqa_scale_ok(float s) { return s >= 0x1p-126f && s <= 0x1p127f; }

// e4m3 codes of four values over a scale (given as its reciprocal).  At the largest scale the codes end at 240: 256 * 2^120
// is no float.
__device__ inline uint32_t gqa_codes4(float a, float b, float c, float d, float inv, float most) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(a * inv, -most, most), __builtin_amdgcn_fmed3f(b * inv, -most, most), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(c * inv, -most, most), __builtin_amdgcn_fmed3f(d * inv, -most, most), r, true);
  return static_cast<uint32_t>(r);
}
__device__ inline float gqa_most(float scale) { return scale >= 0x1p120f ? 240.f : kE4m3Max; }
// Four codes times a power of two, rounded to codes again (NaN stays NaN: no clamp, and the power is at most 1, or brings
// the block's largest to at most 448).
__device__ inline uint32_t gqa_rescale4(uint32_t x, float ratio) {
  const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, r, true));
}

__device__ inline int gqa_wave_scan(int v) {  // inclusive sum over the wave
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

// The host's checks of heads and dims; `who` names the entry point.
inline int check_gqa(const char* who, int64_t kv_heads, int64_t head_dim) {
  if (head_dim != 64 && head_dim != 128) { set_error("%s: head_dim=%lld must be 64 or 128", who, (long long)head_dim); return kErrUnsupported; }
  if (kv_heads < 1 || kv_heads > 128) { set_error("%s: kv_heads=%lld must be in [1, 128]", who, (long long)kv_heads); return kErrUnsupported; }
  return kOk;
}
inline int check_gqa_heads(const char* who, int64_t heads, int64_t kv_heads) {
  if (heads < 1 || heads > 128 || heads % kv_heads) {
    set_error("%s: heads=%lld must be a multiple of kv_heads=%lld, at most 128", who, (long long)heads, (long long)kv_heads);
    return kErrUnsupported;
  }
  return kOk;
}
// A token's stride in a tensor of [tokens, heads, D] whose heads are contiguous.
inline int check_gqa_rows(const char* who, const char* what, const void* p, int64_t stride, int64_t heads, int64_t head_dim) {
  if (!p) { set_error("%s: null pointer (%s)", who, what); return kErrArg; }
  if ((reinterpret_cast<uintptr_t>(p) & 15) || stride % 8 || stride < heads * head_dim || stride >= (1ll << 40)) {
    set_error("%s: %s must be 16-byte aligned, its token stride (%lld) a multiple of 8 and no less than its heads", who, what, (long long)stride);
    return kErrArg;
  }
  return kOk;
}

}  // namespace tl
