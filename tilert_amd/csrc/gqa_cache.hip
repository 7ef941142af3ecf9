// The paged per-head cache (gqa.h): writing new tokens with their heads' norms and rotation, and eviction by weight.
#include <type_traits>

#include "gqa.h"
#include "../../include/tilert_amd.h"

namespace tl {

// ------------------------------------------------------------------------------------------------------ writing
// For a head's row x (a query, a key; a value is taken as it is):
//   n = x * rsqrt(mean(x^2) + eps) * gamma        (fp32; n = x without gamma)
//   y = n with its first `rope` dims turned pair by pair by the token's angles (n without)
// A query row leaves as bf16(y).  Keys and values are quantised by block, the new rows of one page and head:
//   s = the least power of two with max |y| <= 448 s; a block that holds older keys keeps its scale if it is larger, and
//   if not its older codes are brought to the new one;  code = e4m3(y / s).  Older keys of a block of which a scale is none
//   are NaN; they become NaN codes.
// A key with a NaN or an infinity in its key or value row gets NaN key codes and value codes 0, and does not count for
// the scales: its scores are NaN for the rows that see it, and nothing reaches a row that does not.
struct GqaWriteArgs {
  const uint16_t *k, *v, *q;
  int64_t k_stride, v_stride, q_stride;
  uint8_t* pages;
  int64_t page_bytes;
  PagedBatch p;
  int kv_heads, heads, rope, interleaved, page_slots;
  const float *gamma_k, *gamma_q, *freqs;
  float eps;
  uint16_t* q_out;
  float* key_weights;
  uint64_t per_heads;  // ceil(2^34 / heads): x / heads = x * per_heads >> 34 for x < 2^27, heads <= 128
};

template <int LANES, bool MAX = false>  // sum / max over 8 or 16 consecutive lanes, in all of them
__device__ inline float row_sum(float v) {
  v = dpp_combine<0xb1, MAX>(v);
  v = dpp_combine<0x4e, MAX>(v);
  v = dpp_combine<0x141, MAX>(v);
  return LANES == 16 ? dpp_combine<0x140, MAX>(v) : v;
}

__device__ inline void unpack8(u32x4g raw, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(raw[i] << 16);
    x[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
  }
}

// Eight floats, for which 16-byte alignment is not known, in as few loads as there can be.
typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ inline void load8(const float* p, float (&x)[8]) {
  const v4u a = *reinterpret_cast<const v4u*>(p), b = *reinterpret_cast<const v4u*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = a[i];
    x[4 + i] = b[i];
  }
}

// A lane's angles for a row of its token, cosines and sines of its dims' pairs: lane `part` of the row's D / 8 has the dims 8
// part .. + 7, so eight pairs, or four where a pair's dims are neighbours.
struct Angles {
  float x[8], y[8];
};
__device__ inline Angles load_angles(const float* freqs, int part, int rope, int interleaved) {
  Angles r = {};
  if (part * 8 >= rope) return r;
  if (interleaved) {
    load8(freqs + part * 8, r.x);
  } else {
    const int half = rope / 16, pair = part >= half ? part - half : part;
    load8(freqs + pair * 16, r.x);
    load8(freqs + pair * 16 + 8, r.y);
  }
  return r;
}

// The row's norm and rotation, all lanes of a row together.
template <int D>
__device__ inline void norm_rope(float (&x)[8], int part, bool norm, const float (&gamma)[8], const float* freqs, const Angles& w,
                                 int rope, int interleaved, float eps) {
  constexpr int LANES = D / 8;
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
    float mean = row_sum<LANES>(ss) * (1.0f / D) + eps;
    // Where the squares pass fp32 (elements from some 2^60 on) or are lost below it (with an eps that is as small), the row and
    // eps are brought by a power of two to where the larger of them, the row's largest or sqrt(eps), is in [1, 2).
    const bool far = !(mean >= 0x1p-100f && mean < INFINITY);
    if (__any(far)) {
      float top = __builtin_sqrtf(eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, __builtin_fabsf(x[i]));
      top = row_sum<LANES, true>(top);
      const int by = far && top > 0.f && top < INFINITY ? 1 - __builtin_amdgcn_frexp_expf(top) : 0;
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_ldexpf(x[i], by);
        ss = __builtin_fmaf(x[i], x[i], ss);
      }
      const float scaled = row_sum<LANES>(ss) * (1.0f / D) + __builtin_ldexpf(eps, 2 * by);
      mean = far ? scaled : mean;
    }
    const float r = __builtin_amdgcn_rsqf(mean);  // (within 2^-23)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * gamma[i];
  }
  if (!freqs) return;
  const bool turned = part * 8 < rope;
  if (interleaved) {
    if (!turned) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = w.x[2 * i], s = w.x[2 * i + 1], a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * c - b * s;
      x[2 * i + 1] = a * s + b * c;
    }
    return;
  }
  const int half = rope / 16;  // lanes of half the turned dims
  const bool upper = part >= half;
  const int lane = threadIdx.x & 63, from = 4 * (turned ? lane + (upper ? -half : half) : lane);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float other = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(x[i])));
    const float c = i < 4 ? w.x[2 * i] : w.y[2 * i - 8], s = i < 4 ? w.x[2 * i + 1] : w.y[2 * i - 7];
    const float y = x[i] * c + other * (upper ? s : -s);
    x[i] = turned ? y : x[i];
  }
}

// A workgroup takes one page of a sequence's new keys and one kv head (its scales need all of the block's rows), or, behind
// those, 64 query rows; 8 or 16 lanes a row, 16 bytes each.  Values are transposed through LDS.  Bound by bytes and the loads'
// latency, as a workgroup's work is one round of them: 4040 tokens, 32 heads over 8 of 128 dims, 92 MB, 25 us, 3.7 TB/s,
// vector instructions busy for 60 % of it (27 us with angles loaded row by row and for dims that are not turned).
template <int D>
__global__ __launch_bounds__(256) void gqa_write_kernel(const GqaWriteArgs A) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES, STEPS = kGqaKeys / ROWS;
  __shared__ __attribute__((aligned(16))) uint8_t vt[D][kGqaKeys + 16];
  __shared__ float amax_w[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = tid % LANES, sub = tid / LANES;
  const PagedBatch& p = A.p;
  const int page_wgs = A.page_slots * A.kv_heads;
  const bool query = static_cast<int>(blockIdx.x) >= page_wgs;
  const float* gamma_at = query ? A.gamma_q : A.gamma_k;
  float gamma[8] = {};
  if (gamma_at) load8(gamma_at + part * 8, gamma);
  auto angles = [&](int64_t t) { return A.freqs ? load_angles(A.freqs + t * A.rope, part, A.rope, A.interleaved) : Angles{}; };
  if (query) {  // ---- query rows; all loads first
    const int64_t end = static_cast<int64_t>(min(max(p.cu[p.n_seqs], 0), p.n_tokens)) * A.heads;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x - page_wgs) * kGqaKeys;
    if (row0 >= end) return;
    u32x4g raw[STEPS];
    Angles w[STEPS];
    int before = -1;  // (heads of one token have its angles in common)
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int64_t row = row0 + i * ROWS + sub, r = row < end ? row : end - 1;
      const int t = static_cast<int>(static_cast<uint64_t>(r) * A.per_heads >> 34), h = static_cast<int>(r - static_cast<int64_t>(t) * A.heads);
      raw[i] = *reinterpret_cast<const u32x4g*>(A.q + t * A.q_stride + h * D + part * 8);
      if (i > 0 && __all(t == before)) w[i] = w[i - 1];
      else w[i] = angles(t);
      before = t;
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int64_t row = row0 + i * ROWS + sub;
      float x[8];
      unpack8(raw[i], x);
      norm_rope<D>(x, part, gamma_at != nullptr, gamma, A.freqs, w[i], A.rope, A.interleaved, A.eps);
      if (row < end) *reinterpret_cast<u32x4g*>(A.q_out + row * D + part * 8) = u32x4g{bf16x2_bits(v2f{x[0], x[1]}), bf16x2_bits(v2f{x[2], x[3]}),
                                                                                     bf16x2_bits(v2f{x[4], x[5]}), bf16x2_bits(v2f{x[6], x[7]})};
    }
    return;
  }
  // ---- a page: sequence b's are the slots from before(b) on, which leaves it as many as its tokens can touch
  const int slot = blockIdx.x / A.kv_heads, head = blockIdx.x % A.kv_heads;
  auto before = [&](int b) { return min(max(p.cu[b], 0), p.n_tokens) / kGqaKeys + 2 * b; };
  const int b = last_seq(p.n_seqs, [&](int i) { return before(i) <= slot; });
  if (b < 0 || b >= p.n_seqs || slot < before(b)) return;  // (below it where cu_seqlens does not ascend)
  const int c0 = p.cu[b], c1 = p.cu[b + 1];
  const int first = min(max(c0, 0), p.n_tokens), n = min(max(c1, first), p.n_tokens) - first;
  const int64_t base = static_cast<int64_t>(p.lens[b]) - c1 + first;  // position of the first token
  if (n <= 0) return;
  const int64_t pg = (base >> 6) + (slot - before(b));
  if (pg < 0 || pg >= p.max_pages || pg > (base + n - 1) >> 6) return;
  const int page = p.table[static_cast<int64_t>(b) * p.max_pages + pg];
  if (page < 0 || page >= p.n_pages) return;
  // rows r0 .. r1 - 1 of the page are tokens first + pg * 64 - base + row
  const int64_t shift = pg * kGqaKeys - base;
  const int r0 = static_cast<int>(shift < 0 ? -shift : 0), r1 = static_cast<int>(n - shift < kGqaKeys ? n - shift : kGqaKeys);
  const GqaBlock blk = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, page, head);
  const float old_k = blk.scale[0], old_v = blk.scale[1];
  float y[STEPS][8], z[STEPS][8];
  bool fine[STEPS];
  float amax_k = 0.f, amax_v = 0.f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int row = i * ROWS + sub;
    const bool live = row >= r0 && row < r1;
    const int64_t t = first + shift + (live ? row : r0);
    unpack8(*reinterpret_cast<const u32x4g*>(A.k + t * A.k_stride + head * D + part * 8), y[i]);
    unpack8(*reinterpret_cast<const u32x4g*>(A.v + t * A.v_stride + head * D + part * 8), z[i]);
    norm_rope<D>(y[i], part, gamma_at != nullptr, gamma, A.freqs, angles(t), A.rope, A.interleaved, A.eps);
    float bad = 0.f, mk = 0.f, mv = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad = __builtin_fmaf(z[i][j], 0.f, __builtin_fmaf(y[i][j], 0.f, bad));  // (NaN where one is not finite)
      mk = fmaxf(mk, __builtin_fabsf(y[i][j]));
      mv = fmaxf(mv, __builtin_fabsf(z[i][j]));
    }
    fine[i] = row_sum<LANES>(bad) == 0.f;
    if (live && fine[i]) {
      amax_k = fmaxf(amax_k, mk);
      amax_v = fmaxf(amax_v, mv);
    }
  }
  amax_k = wave_max_f32(amax_k);
  amax_v = wave_max_f32(amax_v);
  if (lane == 0) {
    amax_w[0][wave] = amax_k;
    amax_w[1][wave] = amax_v;
  }
  __syncthreads();
  float s_k = gqa_scale(fmaxf(fmaxf(amax_w[0][0], amax_w[0][1]), fmaxf(amax_w[0][2], amax_w[0][3])));
  float s_v = gqa_scale(fmaxf(fmaxf(amax_w[1][0], amax_w[1][1]), fmaxf(amax_w[1][2], amax_w[1][3])));
  if (r0 > 0 && gqa_scale_ok(old_k) && gqa_scale_ok(old_v)) {  // older keys in front
    if (old_k >= s_k) {
      s_k = old_k;
    } else {
      const float ratio = old_k / s_k;
      for (int i = tid; i < r0 * (D / 16); i += 256) {
        u32x4g x = reinterpret_cast<u32x4g*>(blk.k)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = gqa_rescale4(x[j], ratio);
        reinterpret_cast<u32x4g*>(blk.k)[i] = x;
      }
    }
    if (old_v >= s_v) {
      s_v = old_v;
    } else {
      const float ratio = old_v / s_v;
      for (int i = tid; i < D * kGqaKeys / 4; i += 256) {  // four keys of a dim; those behind r0 - 1 are written below
        uint32_t* at = reinterpret_cast<uint32_t*>(blk.v) + i;
        if (i % (kGqaKeys / 4) * 4 < r0) *at = gqa_rescale4(*at, ratio);
      }
    }
  } else if (r0 > 0) {  // older keys that are NaN, as one of their scales is none: under the new scales their codes say so
    for (int i = tid; i < r0 * (D / 16); i += 256) reinterpret_cast<u32x4g*>(blk.k)[i] = u32x4g{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
    for (int i = tid; i < D * kGqaKeys / 4; i += 256)
      if (i % (kGqaKeys / 4) * 4 < r0) reinterpret_cast<uint32_t*>(blk.v)[i] = 0x7f7f7f7fu;
  }
  const float inv_k = 1.0f / s_k, inv_v = 1.0f / s_v, most_k = gqa_most(s_k), most_v = gqa_most(s_v);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int row = i * ROWS + sub;
    if (row < r0 || row >= r1) continue;
    u32x2g c = u32x2g{0x7f7f7f7fu, 0x7f7f7f7fu}, d = u32x2g{0, 0};
    if (fine[i]) {
      c = u32x2g{gqa_codes4(y[i][0], y[i][1], y[i][2], y[i][3], inv_k, most_k), gqa_codes4(y[i][4], y[i][5], y[i][6], y[i][7], inv_k, most_k)};
      d = u32x2g{gqa_codes4(z[i][0], z[i][1], z[i][2], z[i][3], inv_v, most_v), gqa_codes4(z[i][4], z[i][5], z[i][6], z[i][7], inv_v, most_v)};
    }
    reinterpret_cast<u32x2g*>(blk.k + row * D)[part] = c;
#pragma unroll
    for (int j = 0; j < 8; ++j) vt[part * 8 + j][row] = static_cast<uint8_t>(d[j / 4] >> (8 * (j % 4)));
  }
  __syncthreads();  // (and the older codes are where they go: the stores of this workgroup are in order from here)
  for (int i = tid; i < D * 4; i += 256) {
    const int dim = i >> 2, q = i & 3, lo = max(r0, 16 * q), hi = min(r1, 16 * q + 16);
    uint8_t* to = blk.v + dim * kGqaKeys;
    if (hi - lo == 16) *reinterpret_cast<u32x4g*>(to + 16 * q) = *reinterpret_cast<const u32x4g*>(&vt[dim][16 * q]);
    else
      for (int r = lo; r < hi; ++r) to[r] = vt[dim][r];
  }
  if (tid == 0) {
    blk.scale[0] = s_k;
    blk.scale[1] = s_v;
  }
  if (A.key_weights && tid >= r0 && tid < r1) A.key_weights[(static_cast<int64_t>(page) * A.kv_heads + head) * kGqaKeys + tid] = 0.f;
}

// ----------------------------------------------------------------------------------------------------- eviction
struct GqaEvictArgs {
  uint8_t* pages;
  int64_t page_bytes;
  float* weights;  // [n_pages][kv_heads][64]
  const int32_t* table;
  const int32_t* lens;
  const int32_t* keep;
  int n_pages, max_pages, kv_heads, recent;
  const int32_t* kept_table;
  int kept_pages;
  int32_t* kept_lens;
  int32_t* slots;  // [n_seqs][kv_heads][kept_pages * 64]
};

// A weight as a number that ascends with it; -0 is 0 and a NaN the largest.
__device__ inline uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Which keys of one sequence and head stay: the last `recent`, and the heaviest of the others, k in all, in ascending
// order; equal weights: the lowest position.  The k-th largest weight is found digit by digit (11, 11 and 10 bits) from
// histograms in LDS, then every wave counts and writes its own stretch of the positions.
// A workgroup a head; each of its 16 waves goes through its own stretch of pages, four pages at a time, four keys a lane, once
// for each digit and once to mark the keys that stay, two bits each in LDS, from which their places are counted.  Bound by
// vector instructions, some 10 a key and pass: 65536 keys 55 us, 64 with every key's place looked at and 115 with a page at a
// time and the marking done twice; 4000 keys 12.6 us.  (The keys kept in LDS, or only those of the first digit's bin, were no
// faster: 68 and 13.0; nor the histogram in four or eight copies, 64 and 67.)
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kSelBins = 2048, kSelBatch = 4;
constexpr int kSelBlock = 1024;  // pages that are marked at a time
__global__ __launch_bounds__(kSelThreads) void gqa_select_kernel(const GqaEvictArgs A) {
  __shared__ int hist[kSelBins];
  __shared__ uint8_t marks[kSelBlock * kGqaKeys / 4];  // of four keys: bits 0 .. 3, which stay; 4 .. 7, which equal the threshold
  __shared__ int wave_sum[kSelWaves], wave_eq[kSelWaves];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / A.kv_heads, h = blockIdx.x % A.kv_heads;
  const int32_t* table = A.table + static_cast<int64_t>(b) * A.max_pages;
  const int width = A.kept_pages * kGqaKeys;
  int32_t* out = A.slots + (static_cast<int64_t>(b) * A.kv_heads + h) * width;
  const int64_t most = static_cast<int64_t>(A.max_pages) * kGqaKeys;
  const int n = static_cast<int>(A.lens[b] < 0 ? 0 : (A.lens[b] < most ? A.lens[b] : most));
  const int n_pages = (n + kGqaKeys - 1) / kGqaKeys;
  auto there = [&](int id) { return id >= 0 && id < A.n_pages; };
  auto all_waves = [&](int mine) {  // a sum over the workgroup
    for (int o = 32; o; o >>= 1) mine += __shfl_xor(mine, o);
    __syncthreads();
    if (lane == 0) wave_sum[wave] = mine;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kSelWaves; ++w) total += wave_sum[w];
    return total;
  };
  // keys that there are from position `from` on
  auto count = [&](int from) {
    int mine = 0;
    for (int pg = from / kGqaKeys + tid; pg < n_pages; pg += kSelThreads)
      mine += there(table[pg]) ? min(n - pg * kGqaKeys, kGqaKeys) - max(from - pg * kGqaKeys, 0) : 0;
    return all_waves(mine);
  };
  const int total = count(0), k = min(min(max(A.keep[b], 0), total), width);
  const int last0 = n - min(A.recent, k);  // positions from here on stay
  int need = k - count(last0);             // of the others
  // f(position of a lane's four keys, their sort keys, low) for the wave's stretch of pages page0 .. page1 - 1, in order; sort
  // key 0, which no weight has: none is there; low: the wave's keys are all there and below last0
  auto pages = [&](int page0, int page1, auto f) __attribute__((always_inline)) {
    const int quads = (page1 - page0 + 3) / 4, per = (quads + kSelWaves - 1) / kSelWaves;
    const int q0 = wave * per, q1 = min(q0 + per, quads);
    for (int first = q0; first < q1; first += kSelBatch) {
      v4u w[kSelBatch];
      int id[kSelBatch];
#pragma unroll
      for (int i = 0; i < kSelBatch; ++i) id[i] = table[min(page0 + 4 * min(first + i, q1 - 1) + (lane >> 4), page1 - 1)];
#pragma unroll
      for (int i = 0; i < kSelBatch; ++i)
        w[i] = reinterpret_cast<const v4u*>(A.weights + (static_cast<int64_t>(there(id[i]) ? id[i] : 0) * A.kv_heads + h) * kGqaKeys)[lane & 15];
#pragma unroll
      for (int i = 0; i < kSelBatch; ++i) {
        if (first + i >= q1) break;
        const int pos = (page0 + 4 * (first + i)) * kGqaKeys + 4 * lane, here = there(id[i]) ? n - pos : 0;
        uint32_t key[4] = {weight_key(w[i].x), weight_key(w[i].y), weight_key(w[i].z), weight_key(w[i].w)};
        const bool low = __all(here > 3) && (page0 + 4 * (first + i) + 4) * kGqaKeys <= last0;
        if (!low)
#pragma unroll
          for (int j = 0; j < 4; ++j) key[j] = here > j ? key[j] : 0u;
        f(pos, key, low);
      }
    }
  };
  // the need-th largest key of the positions below last0, and how many equal to it stay
  uint32_t prefix = 0;
  auto digit = [&](auto high, auto bits) __attribute__((always_inline)) {  // the digit of `bits` bits below bit `high`
    constexpr int HIGH = decltype(high)::value, SHIFT = HIGH - decltype(bits)::value, BINS = 1 << decltype(bits)::value;
    for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    auto add = [&](uint32_t key) __attribute__((always_inline)) {
      if (HIGH == 32 || (key ^ prefix) >> (HIGH % 32) == 0) atomicAdd(&hist[(key >> SHIFT) & (BINS - 1)], 1);
    };
    pages(0, n_pages, [&](int pos, const uint32_t (&key)[4], bool low) __attribute__((always_inline)) {
      if (low) {
#pragma unroll
        for (int j = 0; j < 4; ++j) add(key[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key[j] != 0 && pos + j < last0) add(key[j]);
      }
    });
    __syncthreads();
    // from the largest digit down: thread t has the bins 2047 - 2 t and 2046 - 2 t
    const int hi = hist[kSelBins - 1 - 2 * tid], lo = hist[kSelBins - 2 - 2 * tid];
    int up = gqa_wave_scan(hi + lo);
    if (lane == 63) wave_sum[wave] = up;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) up += w < wave ? wave_sum[w] : 0;
    const int above = up - hi - lo;
    if (above < need && up >= need) {
      found[0] = above + hi >= need ? kSelBins - 1 - 2 * tid : kSelBins - 2 - 2 * tid;
      found[1] = above + hi >= need ? above : above + hi;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[0]) << SHIFT;
    need -= found[1];
    __syncthreads();
  };
  if (need > 0) {
    using std::integral_constant;
    digit(integral_constant<int, 32>{}, integral_constant<int, 11>{});
    digit(integral_constant<int, 21>{}, integral_constant<int, 11>{});
    digit(integral_constant<int, 10>{}, integral_constant<int, 10>{});
  }
  const uint64_t below = (1ull << lane) - 1;
  int at0 = 0, eq0 = 0;  // kept ones, and equal ones, in the blocks in front
  for (int page0 = 0; page0 < n_pages; page0 += kSelBlock) {
    const int page1 = min(page0 + kSelBlock, n_pages), pos0 = page0 * kGqaKeys;
    int sures = 0, equals = 0;
    const uint32_t over = need > 0 ? prefix : 0xffffffffu;  // (without a threshold nothing is over it)
    pages(page0, page1, [&](int pos, const uint32_t (&key)[4], bool low) __attribute__((always_inline)) {
      int sure = 0, equal = 0;
      if (low) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sure |= key[j] > over ? 1 << j : 0;
          equal |= key[j] == over ? 1 << j : 0;
        }
        equal = need > 0 ? equal : 0;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool last = pos + j >= last0;
          sure |= key[j] != 0 && (last || key[j] > over) ? 1 << j : 0;
          equal |= key[j] != 0 && !last && need > 0 && key[j] == over ? 1 << j : 0;
        }
      }
      sures += __popc(sure);
      equals += __popc(equal);
      marks[(pos - pos0) / 4] = static_cast<uint8_t>(sure | equal << 4);
    });
    for (int o = 32; o; o >>= 1) {
      sures += __shfl_xor(sures, o);
      equals += __shfl_xor(equals, o);
    }
    __syncthreads();
    if (lane == 0) {
      wave_sum[wave] = sures;
      wave_eq[wave] = equals;
    }
    __syncthreads();
    int at = at0, eq = eq0;
    for (int w = 0; w < kSelWaves; ++w) {
      if (w == wave) {
        at = at0;
        eq = eq0;
      }
      at0 += wave_sum[w] + max(0, min(wave_eq[w], need - eq0));
      eq0 += wave_eq[w];
    }
    // (the stretch that this wave has marked)
    const int quads = (page1 - page0 + 3) / 4, per = (quads + kSelWaves - 1) / kSelWaves, q1 = min((wave + 1) * per, quads);
    for (int q = wave * per; q < q1; ++q) {
      const int mark = marks[q * 64 + lane], equal = mark >> 4;
      int e_before = 0, before = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) e_before += __popcll(__ballot(equal >> j & 1) & below);
      int stays = mark & 15, e = eq + e_before;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (equal >> j & 1) stays |= e++ < need ? 1 << j : 0;
      int all = 0, all_eq = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t m = __ballot(stays >> j & 1);
        before += __popcll(m & below);
        all += __popcll(m);
        all_eq += __popcll(__ballot(equal >> j & 1));
      }
      int to = at + before;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (stays >> j & 1) {
          if (to < width) out[to] = pos0 + q * 256 + 4 * lane + j;
          ++to;
        }
      at += all;
      eq += all_eq;
    }
    __syncthreads();  // (the next block's marks)
  }
  for (int i = k + tid; i < width; i += kSelThreads) out[i] = -1;
  if (h == 0 && tid == 0) A.kept_lens[b] = k;
}

// A workgroup gathers the keys of one new page and head: their codes under the least common scale, and their weights.  A key's
// row is loads of 16 bytes; a value is a column of its page's block, a byte a lane, so that the blocks of all pages with a
// kept key come whole.  Bound by those bytes: 9 sequences of up to 65536 keys brought down to 8192, 594 MB, 122 us, 4.9 TB/s
// (the blocks through LDS by loads of 16 bytes: 125).
template <int D>
__global__ __launch_bounds__(256) void gqa_gather_kernel(const GqaEvictArgs A) {
  constexpr int CH = D / 16, ROWS = 256 / CH, STEPS = kGqaKeys / ROWS, DIMS = D / 4;
  __shared__ int src_page[kGqaKeys], src_row[kGqaKeys];
  __shared__ float src_k[kGqaKeys], src_v[kGqaKeys];
  __shared__ float amax_w[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % A.kv_heads, slot = blockIdx.x / A.kv_heads, b = slot / A.kept_pages, pg = slot % A.kept_pages;
  const int to = A.kept_table[static_cast<int64_t>(b) * A.kept_pages + pg];
  if (to < 0 || to >= A.n_pages) return;
  const int32_t* list = A.slots + ((static_cast<int64_t>(b) * A.kv_heads + h) * A.kept_pages + pg) * kGqaKeys;
  if (list[0] < 0) return;
  if (tid < kGqaKeys) {
    const int pos = list[tid];
    int page = -1;
    float sk = 0.f, sv = 0.f;
    if (pos >= 0) {
      page = A.table[static_cast<int64_t>(b) * A.max_pages + (pos >> 6)];
      const GqaBlock s = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, page, h);
      sk = s.scale[0];
      sv = s.scale[1];
      if (!gqa_scale_ok(sk) || !gqa_scale_ok(sv)) sk = sv = __builtin_nanf("");  // (either: its keys are NaN, and their codes will say so)
      A.weights[(static_cast<int64_t>(to) * A.kv_heads + h) * kGqaKeys + tid] = A.weights[(static_cast<int64_t>(page) * A.kv_heads + h) * kGqaKeys + (pos & 63)];
    }
    src_page[tid] = page;
    src_row[tid] = pos & 63;
    src_k[tid] = sk;
    src_v[tid] = sv;
  }
  __syncthreads();
  u32x4g kc[STEPS];
  float amax_k = 0.f, amax_v = 0.f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int row = i * ROWS + tid / CH, page = src_page[row];
    kc[i] = u32x4g{0, 0, 0, 0};
    if (page >= 0) {
      kc[i] = reinterpret_cast<const u32x4g*>(gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, page, h).k + src_row[row] * D)[tid % CH];
      const float s = src_k[row];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(kc[i][j], false), c = __builtin_amdgcn_cvt_pk_f32_fp8(kc[i][j], true);
        amax_k = fmaxf(amax_k, fmaxf(fmaxf(__builtin_fabsf(a[0]), __builtin_fabsf(a[1])), fmaxf(__builtin_fabsf(c[0]), __builtin_fabsf(c[1]))) * s);
      }
    }
  }
  // values: lane = key, a wave a quarter of the dims
  uint32_t vc[DIMS / 4];
  const int vpage = src_page[lane];
  const float sv = src_v[lane];
  if (vpage >= 0) {
    const uint8_t* from = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, vpage, h).v + wave * DIMS * kGqaKeys + src_row[lane];
#pragma unroll
    for (int i = 0; i < DIMS / 4; ++i)
      vc[i] = from[(4 * i) * kGqaKeys] | from[(4 * i + 1) * kGqaKeys] << 8 | from[(4 * i + 2) * kGqaKeys] << 16 |
              static_cast<uint32_t>(from[(4 * i + 3) * kGqaKeys]) << 24;
#pragma unroll
    for (int i = 0; i < DIMS / 4; ++i) {
      const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(vc[i], false), c = __builtin_amdgcn_cvt_pk_f32_fp8(vc[i], true);
      amax_v = fmaxf(amax_v, fmaxf(fmaxf(__builtin_fabsf(a[0]), __builtin_fabsf(a[1])), fmaxf(__builtin_fabsf(c[0]), __builtin_fabsf(c[1]))) * sv);
    }
  }
  amax_k = wave_max_f32(amax_k);
  amax_v = wave_max_f32(amax_v);
  if (lane == 0) {
    amax_w[0][wave] = amax_k;
    amax_w[1][wave] = amax_v;
  }
  __syncthreads();
  const float s_k = gqa_scale(fmaxf(fmaxf(amax_w[0][0], amax_w[0][1]), fmaxf(amax_w[0][2], amax_w[0][3])));
  const float s_v = gqa_scale(fmaxf(fmaxf(amax_w[1][0], amax_w[1][1]), fmaxf(amax_w[1][2], amax_w[1][3])));
  const GqaBlock dst = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, to, h);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int row = i * ROWS + tid / CH;
    if (src_page[row] < 0) continue;
    const float ratio = src_k[row] / s_k;
#pragma unroll
    for (int j = 0; j < 4; ++j) kc[i][j] = gqa_rescale4(kc[i][j], ratio);
    reinterpret_cast<u32x4g*>(dst.k + row * D)[tid % CH] = kc[i];
  }
  if (vpage >= 0) {
    const float ratio = sv / s_v;
    uint8_t* into = dst.v + wave * DIMS * kGqaKeys + lane;
#pragma unroll
    for (int i = 0; i < DIMS / 4; ++i) {
      const uint32_t x = gqa_rescale4(vc[i], ratio);
      into[(4 * i) * kGqaKeys] = static_cast<uint8_t>(x);
      into[(4 * i + 1) * kGqaKeys] = static_cast<uint8_t>(x >> 8);
      into[(4 * i + 2) * kGqaKeys] = static_cast<uint8_t>(x >> 16);
      into[(4 * i + 3) * kGqaKeys] = static_cast<uint8_t>(x >> 24);
    }
  }
  if (tid == 0) {
    dst.scale[0] = s_k;
    dst.scale[1] = s_v;
  }
}

}  // namespace tl

using namespace tl;

extern "C" int tl_gqa_cache_write(const void* k_bf16, int64_t k_stride, const void* v_bf16, int64_t v_stride, void* kv_pages,
                                  int64_t n_pages, const int32_t* block_table, int64_t max_pages, const int32_t* cu_seqlens,
                                  const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens, int64_t kv_heads, int64_t head_dim,
                                  const float* gamma_k, const float* freqs, int64_t rope_dim, const void* q_bf16, int64_t q_stride,
                                  int64_t heads, const float* gamma_q, void* q_out_bf16, float* key_weights, float eps,
                                  int interleaved, void* stream) {
  const char* who = "gqa_cache_write";
  if (int rc = check_batch(who, kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (int rc = check_gqa(who, kv_heads, head_dim)) return rc;
  if (freqs && (rope_dim < 16 || rope_dim > head_dim || rope_dim % 16)) {
    set_error("%s: rope_dim=%lld must be a multiple of 16 in [16, %lld]", who, (long long)rope_dim, (long long)head_dim);
    return kErrUnsupported;
  }
  if (q_bf16) {
    if (int rc = check_gqa_heads(who, heads, kv_heads)) return rc;
    if (n_tokens * heads >= (1ll << 27)) { set_error("%s: %lld tokens x %lld heads: fewer than 2^27 rows", who, (long long)n_tokens, (long long)heads); return kErrUnsupported; }
  }
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (int rc = check_gqa_rows(who, "key", k_bf16, k_stride, kv_heads, head_dim)) return rc;
  if (int rc = check_gqa_rows(who, "value", v_bf16, v_stride, kv_heads, head_dim)) return rc;
  if (q_bf16) {
    if (int rc = check_gqa_rows(who, "query", q_bf16, q_stride, heads, head_dim)) return rc;
    if (int rc = check_gqa_rows(who, "query_out", q_out_bf16, heads * head_dim, heads, head_dim)) return rc;
  }
  const int64_t slots = n_tokens / kGqaKeys + 2 * n_seqs;
  const int64_t wgs = slots * kv_heads + (q_bf16 ? cdiv(n_tokens * heads, kGqaKeys) : 0);
  if (wgs >= (1ll << 24)) {  // 256 threads each, fewer than 2^32
    set_error("%s: %lld tokens, %lld sequences: more than a launch has room for", who, (long long)n_tokens, (long long)n_seqs);
    return kErrUnsupported;
  }
  const GqaWriteArgs args{(const uint16_t*)k_bf16, (const uint16_t*)v_bf16, (const uint16_t*)q_bf16, k_stride, v_stride, q_stride,
                          (uint8_t*)kv_pages, gqa_page_bytes(kv_heads, head_dim),
                          PagedBatch{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens},
                          (int)kv_heads, (int)heads, (int)rope_dim, interleaved, (int)slots, gamma_k, gamma_q, freqs, eps,
                          (uint16_t*)q_out_bf16, key_weights, q_bf16 ? ((1ull << 34) + heads - 1) / heads : 0};
  hipLaunchKernelGGL(head_dim == 64 ? gqa_write_kernel<64> : gqa_write_kernel<128>, dim3(wgs), dim3(256), 0, (hipStream_t)stream, args);
  return check_launch(who);
}

extern "C" int tl_gqa_cache_evict(void* kv_pages, float* key_weights, int64_t n_pages, const int32_t* block_table, int64_t max_pages,
                                  const int32_t* seq_lens, const int32_t* keep_lens, int64_t n_seqs, int64_t kv_heads,
                                  int64_t head_dim, int64_t recent, const int32_t* kept_table, int64_t kept_pages,
                                  int32_t* kept_lens, int32_t* kept_slots, void* stream) {
  const char* who = "gqa_cache_evict";
  if (int rc = check_batch(who, kv_pages, n_pages, block_table, max_pages, keep_lens, seq_lens, n_seqs, n_seqs)) return rc;
  if (int rc = check_gqa(who, kv_heads, head_dim)) return rc;
  if (recent < 0 || recent > INT32_MAX) { set_error("%s: recent=%lld is out of range", who, (long long)recent); return kErrArg; }
  if (n_seqs == 0) return kOk;
  if (kept_pages < 1 || kept_pages > (1ll << 25) - 1) { set_error("%s: kept_pages=%lld must be in [1, 2^25)", who, (long long)kept_pages); return kErrArg; }
  if (!key_weights || !kept_table || !kept_lens || !kept_slots) { set_error("%s: null pointer", who); return kErrArg; }
  if (n_seqs * kv_heads * kept_pages >= (1ll << 24) || n_seqs * kv_heads >= (1ll << 22)) {  // 256 and 1024 threads each, fewer than 2^32
    set_error("%s: %lld sequences of %lld kept pages: more than a launch has room for", who, (long long)n_seqs, (long long)kept_pages);
    return kErrUnsupported;
  }
  // (a head's workgroup may read its sequence's length, or another sequence's its count, when another's has written the new length;
  // a sequence's own count in its place does no harm, as the new length brings out itself)
  const uintptr_t to = reinterpret_cast<uintptr_t>(kept_lens);
  auto overlaps = [&](const int32_t* p) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p);
    return (from < to ? to - from : from - to) < static_cast<uintptr_t>(n_seqs) * 4;
  };
  if (overlaps(seq_lens) || (keep_lens != kept_lens && overlaps(keep_lens))) {
    set_error("%s: kept_lens must not be the memory of seq_lens, nor a part of keep_lens'", who);
    return kErrArg;
  }
  const GqaEvictArgs args{(uint8_t*)kv_pages, gqa_page_bytes(kv_heads, head_dim), key_weights, block_table, seq_lens, keep_lens,
                          (int)n_pages, (int)max_pages, (int)kv_heads, (int)recent, kept_table, (int)kept_pages, kept_lens, kept_slots};
  hipLaunchKernelGGL(gqa_select_kernel, dim3(n_seqs * kv_heads), dim3(kSelThreads), 0, (hipStream_t)stream, args);
  if (int rc = check_launch(who)) return rc;
  hipLaunchKernelGGL(head_dim == 64 ? gqa_gather_kernel<64> : gqa_gather_kernel<128>, dim3(n_seqs * kv_heads * kept_pages), dim3(256), 0,
                     (hipStream_t)stream, args);
  return check_launch(who);
}
