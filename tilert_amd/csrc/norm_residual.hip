// RMSNorm of a residual sum, with its quantisation (RMSNorm.forward with a residual, tilert/models/common.py:92-133,
// and act_quant behind it):
//   h = x + residual (fp32), sum_out = bf16(h)
//   n = h * rsqrt(mean(h^2) + eps) * gamma, y = bf16(n)
//   per 128 columns s = group_scale(max |n|), code = e4m3(clamp(n / s))
// The norm is the unrounded sum's, and the codes are the unrounded norm's: one rounding each.  (rmsnorm_quant's codes
// are those of its bf16 output.)  A group that holds a NaN or an infinity gets the scale NaN; its codes are finite
// whatever it held.
#include <type_traits>

#include "common.h"
#include "../../include/tilert_amd.h"

namespace tl {

typedef uint32_t u32x4r __attribute__((ext_vector_type(4)));

constexpr int kAddNormMaxDim = 16384;

// One workgroup a row, held in registers as h: thread t has the chunks (8 columns) t, t + NT, ...; 16 consecutive lanes
// hold a 128-column group.  sum_out may be x's or the residual's memory: every thread reads its chunks before it
// writes them, and no other thread uses them (those behind the row's end read its last chunk and drop it).
// Bound by bytes, 9 an element, in large calls: 4096 x 7168, 265 MB, 40 us (6.6 TB/s) where the Infinity Cache holds
// part of them, 50 us a call (5.3 TB/s) where it does not; by its two round trips and the reduction in small ones:
// 4 x 7168 3.5 us.  One chunk a thread, up to 8192 columns of 1024 threads: a row is read in one round of loads (4 x 7168
// in a graph 3.0 us, 3.4 with 512 threads, 4.4 with 256; 4096 x 7168 49.2, 50.4, 52.7); up to 2048 columns 256
// threads, where 1024 would leave three quarters of them without one (4096 x 2048 13.4 us, 22.8 with 1024).
template <int NT, int NC>
__global__ __launch_bounds__(NT) void add_rmsnorm_quant_kernel(const uint16_t* x, const uint16_t* residual,
                                                               const float* __restrict__ gamma, float eps, int dim,
                                                               uint16_t* sum_out, uint16_t* __restrict__ y,
                                                               uint8_t* __restrict__ y8, float* __restrict__ ys, int scale_mode) {
  __shared__ float part[NT / 64];
  const int tid = threadIdx.x, nch = dim / 8;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * dim;
  u32x4r a[NC], b[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = min(tid + j * NT, nch - 1);
    a[j] = reinterpret_cast<const u32x4r*>(x + row)[c];
    b[j] = reinterpret_cast<const u32x4r*>(residual + row)[c];
  }
  float h[NC][8], ss = 0.f;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    u32x4r sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[j][2 * i] = __uint_as_float(a[j][i] << 16) + __uint_as_float(b[j][i] << 16);
      h[j][2 * i + 1] = __uint_as_float(a[j][i] & 0xffff0000u) + __uint_as_float(b[j][i] & 0xffff0000u);
      sum[i] = bf16x2_bits(v2f{h[j][2 * i], h[j][2 * i + 1]});
    }
    const int c = tid + j * NT;
    if (c < nch) {
      reinterpret_cast<u32x4r*>(sum_out + row)[c] = sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(h[j][i], h[j][i], ss);
    }
  }
  ss = wave_sum_f32(ss);
  if ((tid & 63) == 0) part[tid >> 6] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) tot += part[w];
  const float r = 1.0f / __builtin_sqrtf(tot / static_cast<float>(dim) + eps);
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = tid + j * NT, cc = min(c, nch - 1);
    const v4f g0 = reinterpret_cast<const v4f*>(gamma)[2 * cc], g1 = reinterpret_cast<const v4f*>(gamma)[2 * cc + 1];
    float n[8];
    uint32_t most = 0;  // the largest magnitude's bits: a NaN's are above an infinity's
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      n[i] = h[j][i] * r * (i < 4 ? g0[i & 3] : g1[i & 3]);
      most = max(most, __float_as_uint(n[i]) & 0x7fffffffu);
    }
    if (y && c < nch) {
      u32x4r v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = bf16x2_bits(v2f{n[2 * i], n[2 * i + 1]});
      reinterpret_cast<u32x4r*>(y + row)[c] = v;
    }
    if (y8) {
      most = row16_max_u32(most);
      const float s = most < 0x7f800000u ? group_scale(__uint_as_float(most), scale_mode) : __builtin_nanf("");
      const uint2 code = quant8_e4m3(n, s);
      if (c < nch) {
        reinterpret_cast<uint2*>(y8 + row)[c] = code;
        if ((c & 15) == 0) ys[row / kBlock + (c >> 4)] = s;
      }
    }
  }
}

}  // namespace tl

using namespace tl;

extern "C" int tl_add_rmsnorm_quant(const void* x_bf16, const void* residual_bf16, const float* gamma, float eps,
                                    int64_t rows, int64_t dim, void* sum_bf16, void* y_bf16, void* y_fp8, float* y_scale,
                                    int scale_mode, void* stream) {
  if (rows < 0 || dim <= 0 || dim % kBlock || dim > kAddNormMaxDim) {
    set_error("add_rmsnorm_quant: dim=%lld must be a positive multiple of 128, at most %d (rows=%lld)", (long long)dim,
              kAddNormMaxDim, (long long)rows);
    return kErrArg;
  }
  if (scale_mode < 0 || scale_mode > 2) { set_error("add_rmsnorm_quant: bad scale_mode %d", scale_mode); return kErrArg; }
  if (rows == 0) return kOk;
  if (rows >= (dim <= 2048 ? 1ll << 24 : 1ll << 22)) {  // a launch has fewer than 2^32 threads
    set_error("add_rmsnorm_quant: %lld rows: at most 2^24 - 1 up to 2048 columns, 2^22 - 1 behind", (long long)rows);
    return kErrUnsupported;
  }
  if (!x_bf16 || !residual_bf16 || !gamma || !sum_bf16 || (!y_fp8) != (!y_scale) || (!y_bf16 && !y_fp8)) {
    set_error("add_rmsnorm_quant: null pointer (y_fp8 and y_scale are given together; y_bf16 may be left out beside them)");
    return kErrArg;
  }
  if ((reinterpret_cast<uintptr_t>(x_bf16) | reinterpret_cast<uintptr_t>(residual_bf16) | reinterpret_cast<uintptr_t>(gamma) |
       reinterpret_cast<uintptr_t>(sum_bf16) | reinterpret_cast<uintptr_t>(y_bf16) | reinterpret_cast<uintptr_t>(y_fp8)) & 15) {
    set_error("add_rmsnorm_quant: pointers must be 16-byte aligned");
    return kErrArg;
  }
  auto launch = [&](auto nt, auto nc) {
    hipLaunchKernelGGL((add_rmsnorm_quant_kernel<decltype(nt)::value, decltype(nc)::value>), dim3(static_cast<unsigned>(rows)),
                       dim3(decltype(nt)::value), 0, (hipStream_t)stream, (const uint16_t*)x_bf16, (const uint16_t*)residual_bf16,
                       gamma, eps, (int)dim, (uint16_t*)sum_bf16, (uint16_t*)y_bf16, (uint8_t*)y_fp8, y_scale, scale_mode);
  };
  if (dim <= 2048) launch(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  else if (dim <= 8192) launch(std::integral_constant<int, 1024>{}, std::integral_constant<int, 1>{});
  else launch(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
  return check_launch("add_rmsnorm_quant");
}
