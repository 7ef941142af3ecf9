// Causal grouped-query attention of a batch's new tokens over the paged per-head cache (gqa.h), and the attention weights
// that its keys gather.  For token t of a sequence, at position p, and query head h of kv head h / G, over the keys j <= p:
//   s[j] = q[t,h] . k[j] * softmax_scale
//   out[t,h] = sum_j softmax(s)[j] v[j],  lse[t,h] = ln sum_j e^s[j]      (0 and -inf where no key is seen)
//   w[j] (+)= sum over t, h of the group of e^(s[j] - lse[t,h])             (the second operator)
//
// A kv head's rows of a sequence are its (token, head of the group) pairs, token-major; tiles of 16 RT of them go through the
// sequence's pages.  Both products take the cached side as A: S^T = K Q^T and O^T = V^T P^T on the bf16 MFMA, so that a
// row is a lane's column, its statistics one register, and a lane's weights are the second product's operand as they
// stand: score tile t of a page holds the keys 16 g + 4 t + j (g: the lane's group of 16, j: its four results), a lane then
// has 16 consecutive keys of its row, and a dim of the transposed values is one 16-byte load.  No operand passes
// through LDS.  Codes become bf16 two an instruction, scale and all, exactly.
#include <math.h>

#include <type_traits>

#include "gqa.h"
#include "../../include/tilert_amd.h"

namespace tl {

typedef const __attribute__((address_space(4))) int32_t* gqa_const_i32;  // scalar loads

struct GqaArgs {
  const uint16_t* q;
  int64_t q_stride;
  const uint8_t* pages;
  int64_t page_bytes;
  PagedBatch p;
  int heads, kv_heads, group;
  float scale;  // softmax_scale * log2 e
  uint16_t* out;
  float* lse;
  int chunk, splits;  // pages a workgroup, workgroups a tile
  float2* part_ml;    // [tile slots][kv_heads][splits][BM]
  float* part_o;      // [tile slots][kv_heads][splits][BM * D]
};

// A sequence's rows of one kv head and what they see, from untrusted metadata.
struct GqaSeq {
  int first, rows, group;
  int64_t base, most;  // position of the first token; keys that the table has room for
  __device__ inline GqaSeq(const PagedBatch& p, int group_, int b) : group(group_) {
    const int c0 = p.cu[b], c1 = p.cu[b + 1];
    first = min(max(c0, 0), p.n_tokens);
    rows = (min(max(c1, first), p.n_tokens) - first) * group;
    base = static_cast<int64_t>(p.lens[b]) - c1 + first;
    most = static_cast<int64_t>(p.max_pages) * kGqaKeys;
  }
  // keys that a row sees
  __device__ inline int seen(int row) const {
    const int64_t n = base + row / group + 1;
    return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
  }
};

// Tiles of BM rows: sequence b's are the slots from before(b) on, which leaves it as many as it can have.
template <int BM>
__device__ inline bool gqa_tile(const PagedBatch& p, int group, int slot, int& b, int& tile) {
  auto before = [&](int i) { return min(max(p.cu[i], 0), p.n_tokens) * group / BM + i; };
  b = last_seq(p.n_seqs, [&](int i) { return before(i) <= slot; });
  if (b < 0 || b >= p.n_seqs) return false;
  tile = slot - before(b);
  return tile >= 0;
}
inline int64_t gqa_slots(int64_t n_tokens, int64_t group, int64_t n_seqs, int bm) { return n_tokens * group / bm + n_seqs; }

__device__ inline v8bf bf16_of(u32x4g x) { return __builtin_bit_cast(v8bf, x); }
// Eight codes times a power of two.
__device__ inline v8bf codes8_bf16(uint32_t a, uint32_t b, float scale) {
  u32x4g r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true));
  return bf16_of(r);
}
__device__ inline v4f mfma_bf16(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Max / sum over the lanes i, i ^ 16, i ^ 32, i ^ 48, in all of them.
template <bool MAX>
__device__ inline float four_lanes(float v) {
  const u32x2g a = __builtin_bit_cast(u32x2g, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float a0 = __uint_as_float(a[0]), a1 = __uint_as_float(a[1]), x = MAX ? fmaxf(a0, a1) : a0 + a1;
  const u32x2g b = __builtin_bit_cast(u32x2g, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
  const float b0 = __uint_as_float(b[0]), b1 = __uint_as_float(b[1]);
  return MAX ? fmaxf(b0, b1) : b0 + b1;
}

// Bytes that are a NaN code, as 0x80 each.
__device__ inline uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The query rows of a tile as the first product's B operand: lane (c, g) holds of row c the dims 64 i + 16 g + 8 e .. + 7, the
// order in which a 16-byte load gives it a key's codes.
template <int D>
struct GqaQuery {
  v8bf x[D / 64][2];
};
template <int D>
__device__ inline GqaQuery<D> load_query(const uint16_t* q, int64_t stride, const GqaSeq& s, int head0, int row, int g) {
  GqaQuery<D> r;
  const bool live = row < s.rows;
  const int at = live ? row : 0;
  const uint16_t* from = q + (s.first + at / s.group) * stride + (head0 + at % s.group) * D + 16 * g;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      u32x4g x = *reinterpret_cast<const u32x4g*>(from + 64 * i + 8 * e);
      if (!live) x = u32x4g{0, 0, 0, 0};
      r.x[i][e] = bf16_of(x);
    }
  return r;
}

// A page's keys or values of one head, as loaded.
template <int D>
struct GqaKeys {
  u32x4g k[4][D / 64];
};
template <int D>
struct GqaValues {
  u32x4g v[D / 16];
};
template <int D>
__device__ inline GqaKeys<D> load_keys(const uint8_t* k, int lane) {
  GqaKeys<D> r;
  const int c = lane & 15, g = lane >> 4;
  const uint8_t* from = k + (16 * (c >> 2) + (c & 3)) * D + 16 * g;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) r.k[t][i] = *reinterpret_cast<const u32x4g*>(from + 4 * t * D + 64 * i);
  return r;
}
template <int D>
__device__ inline GqaValues<D> load_values(const uint8_t* v, int lane) {
  GqaValues<D> r;
  const uint8_t* from = v + (lane & 15) * kGqaKeys + 16 * (lane >> 4);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) r.v[d] = *reinterpret_cast<const u32x4g*>(from + d * 16 * kGqaKeys);
  return r;
}

// One tile of 16 RT rows and one kv head over `chunk` pages; the four waves take every fourth of them, each with its own
// statistics, and are joined in LDS.  Weights go into the second product as hi + lo in bf16, 16 bits of them.
// Weights are relative to 2^24 times the row's largest: their sums of values then stay inside fp32 whatever the values.
constexpr float kGqaHead = 24.f;
template <int D, int RT>
__global__ __launch_bounds__(256, 2) void gqa_attend_kernel(const GqaArgs A) {
  constexpr int BM = 16 * RT, DT = D / 16, KI = D / 64;
  __shared__ v4f sum_o[4][DT][64];
  __shared__ float sum_m[4][BM], sum_l[4][BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / A.kv_heads, head = blockIdx.x % A.kv_heads, split = blockIdx.y;
  int b, tile;
  if (!gqa_tile<BM>(A.p, A.group, slot, b, tile)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  const GqaSeq s(A.p, A.group, b);
  const int row0 = tile * BM, rows = min(s.rows - row0, BM);
  if (rows <= 0) return;
  const int least = s.seen(row0), n_pages = (s.seen(row0 + rows - 1) + kGqaKeys - 1) / kGqaKeys;
  const int pg0 = split * A.chunk, pg1 = min(pg0 + A.chunk, n_pages);
  if (split > 0 && pg0 >= n_pages) return;
  const gqa_const_i32 table = (gqa_const_i32)(A.p.table + static_cast<int64_t>(b) * A.p.max_pages);
  GqaQuery<D> q[RT];
  int seen[RT];
  float m[RT], l[RT];
  v4f o[RT][DT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    q[r] = load_query<D>(A.q, A.q_stride, s, head * A.group, row0 + r * 16 + c, g);
    seen[r] = s.seen(row0 + min(r * 16 + c, rows - 1));
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[r][d] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  for (int pg = pg0 + wave; pg < pg1; pg += 4) {
    const int id = __builtin_amdgcn_readfirstlane(table[pg]);
    if (id < 0 || id >= A.p.n_pages) continue;
    const GqaBlock blk = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, id, head);
    const GqaKeys<D> kc = load_keys<D>(blk.k, lane);
    GqaValues<D> vc = load_values<D>(blk.v, lane);
    const bool ok = gqa_scale_ok(blk.scale[0]) && gqa_scale_ok(blk.scale[1]);
    const float sk = ok ? blk.scale[0] : 1.f, sv = ok ? blk.scale[1] : 1.f, unit = ok ? A.scale : __builtin_nanf("");
    const int key0 = pg * kGqaKeys;
    const bool masked = key0 + kGqaKeys > least;
    // ---- scores
    v4f x[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int r = 0; r < RT; ++r) x[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const v8bf a = codes8_bf16(kc.k[t][i][2 * e], kc.k[t][i][2 * e + 1], sk);
#pragma unroll
          for (int r = 0; r < RT; ++r) x[r][t] = mfma_bf16(a, q[r].x[i][e], x[r][t]);
        }
    }
    // ---- weights
    v8bf hi[RT][2], lo[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int my = seen[r] - key0 - 16 * g;  // of this lane's 16 keys, the row sees this many
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[r][t][j] *= unit;
          if (masked && 4 * t + j >= my) x[r][t][j] = -INFINITY;
          top = fmaxf(top, x[r][t][j]);
        }
      top = fmaxf(m[r], four_lanes<true>(top));
      if (__any(top > m[r])) {
        const float by = m[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - top);  // (before the first key all is 0, or NaN)
        m[r] = top;
        l[r] *= by;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= by;
      }
      const float from = m[r] == -INFINITY ? 0.f : m[r] + kGqaHead;
      float p[16];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[4 * t + j] = __builtin_amdgcn_exp2f(x[r][t][j] - from);
          l[r] += p[4 * t + j];
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x4g h, w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = p[8 * e + 2 * i], p1 = p[8 * e + 2 * i + 1];
          h[i] = bf16x2_bits(v2f{p0, p1});
          w[i] = bf16x2_bits(v2f{p0 - __uint_as_float(h[i] << 16), p1 - __uint_as_float(h[i] & 0xffff0000u)});
        }
        hi[r][e] = bf16_of(h);
        lo[r][e] = bf16_of(w);
      }
    }
    // ---- values; on a page with keys that some row does not see, codes that are NaN are taken apart
    uint32_t bad[DT][4] = {};
    bool any_bad = false;
    if (masked) {
      uint32_t all = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t n = nan_codes(vc.v[d][i]);
          all |= n;
          bad[d][i] = n;
          vc.v[d][i] &= ~(n | (n - (n >> 7)));
        }
      any_bad = __any(all != 0);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const v8bf a = codes8_bf16(vc.v[d][2 * e], vc.v[d][2 * e + 1], sv);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          o[r][d] = mfma_bf16(a, hi[r][e], o[r][d]);
          o[r][d] = mfma_bf16(a, lo[r][e], o[r][d]);
        }
      }
    if (any_bad) {  // how many NaN values a row sees
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int my = seen[r] - key0 - 16 * g;
        v8bf sees[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          u32x4g w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = (8 * e + 2 * i < my ? 0x3f80u : 0u) | (8 * e + 2 * i + 1 < my ? 0x3f800000u : 0u);
          sees[e] = bf16_of(w);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          v4f n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 2; ++e) n = mfma_bf16(codes8_bf16(bad[d][2 * e] >> 1, bad[d][2 * e + 1] >> 1, 1.f), sees[e], n);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[r][d][j] = n[j] > 0.f ? __builtin_nanf("") : o[r][d][j];
        }
      }
    }
  }
  // ---- the four waves together
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] = four_lanes<false>(l[r]);
    if (g == 0) {
      sum_m[wave][r * 16 + c] = m[r];
      sum_l[wave][r * 16 + c] = l[r];
    }
  }
  __syncthreads();
  const bool whole = n_pages <= A.chunk;
  const int64_t part = (static_cast<int64_t>(slot) * A.kv_heads + head) * A.splits + split;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sum_m[w][r * 16 + c]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = sum_m[w][r * 16 + c];
      total += sum_l[w][r * 16 + c] * (mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - top));
    }
    const float by = m[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - top);
    if (r) __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) sum_o[wave][d][lane] = o[r][d] * by;
    __syncthreads();
    const int row = row0 + r * 16 + c;
    const int64_t at = (static_cast<int64_t>(s.first + row / A.group) * A.heads + head * A.group + row % A.group);
    const bool live = r * 16 + c < rows;
    const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < DT / 4; ++i) {
      const int d = 4 * i + wave;
      const v4f v = sum_o[0][d][lane] + sum_o[1][d][lane] + sum_o[2][d][lane] + sum_o[3][d][lane];
      if (whole) {
        if (live) *reinterpret_cast<u32x2g*>(A.out + at * D + 16 * d + 4 * g) = u32x2g{bf16x2_bits(v2f{v[0] * inv, v[1] * inv}), bf16x2_bits(v2f{v[2] * inv, v[3] * inv})};
      } else if (live) {
        reinterpret_cast<v4f*>(A.part_o + part * (BM * D))[(r * DT + d) * 64 + lane] = v;
      }
    }
    if (wave == 0 && g == 0 && live) {
      if (!whole) A.part_ml[part * BM + r * 16 + c] = float2{top, total};
      else if (A.lse) A.lse[at] = total == 0.f ? -INFINITY : (top + kGqaHead + log2f(total)) * kLn2;
    }
  }
}

// The parts of split tiles joined in a fixed order: a workgroup takes 16 rows x 16 dims of a tile, its eight waves every eighth
// part, joined in LDS.
template <int D, int RT>
__global__ __launch_bounds__(512) void gqa_join_kernel(const GqaArgs A) {
  constexpr int BM = 16 * RT, DT = D / 16, WAVES = 8;
  __shared__ v4f sum_o[WAVES][64];
  __shared__ float sum_l[WAVES][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / A.kv_heads, head = blockIdx.x % A.kv_heads, r = blockIdx.y / DT, d = blockIdx.y % DT;
  int b, tile;
  if (!gqa_tile<BM>(A.p, A.group, slot, b, tile)) return;
  const GqaSeq s(A.p, A.group, b);
  const int row0 = tile * BM, rows = min(s.rows - row0, BM);
  if (rows <= r * 16) return;
  const int n_pages = (s.seen(row0 + rows - 1) + kGqaKeys - 1) / kGqaKeys, parts = (n_pages + A.chunk - 1) / A.chunk;
  if (parts <= 1) return;
  const int64_t part0 = (static_cast<int64_t>(slot) * A.kv_heads + head) * A.splits;
  const bool live = r * 16 + c < rows;
  const int row = r * 16 + (live ? c : 0);  // (rows that are not there have no parts)
  const int at = (r * DT + d) * 64 + (live ? lane : 16 * g);
  float top = -INFINITY;
  for (int i = g; i < parts; i += 4) top = fmaxf(top, A.part_ml[(part0 + i) * BM + row].x);
  top = four_lanes<true>(top);
  float l = 0.f;
  v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = wave; i < parts; i += WAVES) {
    const float2 ml = A.part_ml[(part0 + i) * BM + row];
    const v4f x = reinterpret_cast<const v4f*>(A.part_o + (part0 + i) * (BM * D))[at];
    const float by = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
    l += ml.y * by;
    o += x * by;
  }
  sum_o[wave][lane] = o;
  if (g == 0) sum_l[wave][c] = l;
  __syncthreads();
  if (wave > 0 || !live) return;
  l = sum_l[0][c];
  for (int w = 1; w < WAVES; ++w) {
    o += sum_o[w][lane];
    l += sum_l[w][c];
  }
  const int64_t to = static_cast<int64_t>(s.first + (row0 + row) / A.group) * A.heads + head * A.group + (row0 + row) % A.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<u32x2g*>(A.out + to * D + 16 * d + 4 * g) = u32x2g{bf16x2_bits(v2f{o[0] * inv, o[1] * inv}), bf16x2_bits(v2f{o[2] * inv, o[3] * inv})};
  if (A.lse && d == 0 && g == 0) A.lse[to] = l == 0.f ? -INFINITY : (top + kGqaHead + log2f(l)) * kLn2;
}

// The launch: rows a tile, pages a workgroup, and the workspace.
struct GqaPlan {
  int rt;
  int64_t slots, chunk, splits;
  size_t o_at, bytes;
};
constexpr int kGqaChunks = 2048;  // workgroups of a split launch, about
constexpr int kGqaFew = 8;        // pages that are not split
inline GqaPlan gqa_plan(int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_pages) {
  GqaPlan d{};
  const int64_t group = heads / kv_heads, each = cdiv(n_tokens * group, n_seqs);
  d.rt = each <= 16 ? 1 : 2;
  d.slots = gqa_slots(n_tokens, group, n_seqs, 16 * d.rt);
  const int64_t tiles = d.slots * kv_heads;
  d.chunk = cdiv(tiles * max_pages, kGqaChunks);
  if (d.chunk < kGqaFew) d.chunk = kGqaFew;
  if (d.chunk > max_pages) d.chunk = max_pages;
  d.splits = cdiv(max_pages, d.chunk);
  if (d.splits > 1) {
    d.o_at = static_cast<size_t>((tiles * d.splits * 16 * d.rt * sizeof(float2) + 255) / 256 * 256);
    d.bytes = d.o_at + static_cast<size_t>(tiles * d.splits) * 16 * d.rt * head_dim * sizeof(float);
  }
  return d;
}

// ------------------------------------------------------------------------------------ the weights that keys gather
struct GqaSumArgs {
  const uint16_t* q;
  int64_t q_stride;
  const float* lse;
  const uint8_t* pages;
  int64_t page_bytes;
  PagedBatch p;
  int heads, kv_heads, group, accumulate;
  float scale;  // softmax_scale * log2 e
  float* weights;
  int64_t units;  // sequences x groups of pages x kv heads
  int page_groups;
};

// One page and kv head at a time: its keys stay in registers, the rows that see them come by in tiles of 16, and every lane
// sums its keys' weights over its column of rows.  SPLIT: the four waves of a workgroup share a page, each with every
// fourth tile of rows, and are joined in LDS; else each has a page of its own.
template <int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void gqa_sum_kernel(const GqaSumArgs A) {
  constexpr int KI = D / 64;
  __shared__ float part[4][kGqaKeys];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  for (int64_t u = blockIdx.x; u < A.units; u += gridDim.x) {
    const int head = static_cast<int>(u % A.kv_heads);
    const int64_t v = u / A.kv_heads;
    const int b = static_cast<int>(v / A.page_groups), pg = static_cast<int>(v % A.page_groups) * (SPLIT ? 1 : 4) + (SPLIT ? 0 : wave);
    const GqaSeq s(A.p, A.group, b);
    const int n_keys = s.rows > 0 ? s.seen(s.rows - 1) : 0, key0 = pg * kGqaKeys;
    int id = -1;
    if (key0 < n_keys) id = A.p.table[static_cast<int64_t>(b) * A.p.max_pages + pg];
    id = __builtin_amdgcn_readfirstlane(id);
    const bool there = id >= 0 && id < A.p.n_pages;
    float w[4][4] = {};
    if (there) {
      const GqaBlock blk = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, id, head);
      const GqaKeys<D> kc = load_keys<D>(blk.k, lane);
      const bool ok = gqa_scale_ok(blk.scale[0]);
      const float sk = ok ? blk.scale[0] : 1.f, unit = ok ? A.scale : __builtin_nanf("");
      v8bf k[4][KI][2];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < KI; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) k[t][i][e] = codes8_bf16(kc.k[t][i][2 * e], kc.k[t][i][2 * e + 1], sk);
      // the first row that sees a key of the page
      const int64_t row_first = max(static_cast<int64_t>(0), key0 - s.base) * A.group;
      for (int row0 = static_cast<int>(row_first / 16) * 16 + (SPLIT ? 16 * wave : 0); row0 < s.rows; row0 += SPLIT ? 64 : 16) {
        const int row = row0 + c;
        const GqaQuery<D> q = load_query<D>(A.q, A.q_stride, s, head * A.group, row, g);
        const int at = min(row, s.rows - 1);
        const float lse2 = A.lse[(static_cast<int64_t>(s.first) + at / A.group) * A.heads + head * A.group + at % A.group] * kLog2e;
        const int my = row < s.rows ? s.seen(row) - key0 - 16 * g : 0;
        const bool masked = __any(my < 16);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < KI; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) x = mfma_bf16(k[t][i][e], q.x[i][e], x);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], unit, -lse2));
            if (masked && 4 * t + j >= my) p = 0.f;
            w[t][j] += p;
          }
        }
      }
    }
    // over the 16 rows of a column: lane (c, g) keeps key 16 g + c
    float mine = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = row16_reduce<false>(w[t][j]);
        mine = c == 4 * t + j ? x : mine;
      }
    if constexpr (SPLIT) {
      part[wave][lane] = mine;
      __syncthreads();
      mine = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
      __syncthreads();
    }
    if (there && (!SPLIT || wave == 0) && key0 + lane < n_keys) {
      float* to = A.weights + (static_cast<int64_t>(id) * A.kv_heads + head) * kGqaKeys + lane;
      *to = A.accumulate ? *to + mine : mine;
    }
  }
}

}  // namespace tl

using namespace tl;

constexpr int64_t kGqaMaxRows = 1 << 27;  // (token, head) rows, fewer than this

static int check_gqa_batch(const char* who, int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t max_pages, float softmax_scale) {
  if (n_tokens * heads >= kGqaMaxRows || n_seqs > (1ll << 16) || max_pages > (1ll << 20)) {
    set_error("%s: %lld tokens x %lld heads, %lld sequences, %lld pages a sequence: fewer than 2^27 rows, up to 2^16 sequences and "
              "2^20 pages", who, (long long)n_tokens, (long long)heads, (long long)n_seqs, (long long)max_pages);
    return kErrUnsupported;
  }
  if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY)) { set_error("%s: softmax_scale must be positive and finite", who); return kErrArg; }
  return kOk;
}

extern "C" size_t tl_flash_paged_gqa_workspace_bytes(int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_pages) {
  if (n_seqs < 1 || n_tokens < 1 || kv_heads < 1 || heads < 1 || heads > 128 || heads % kv_heads || max_pages < 1 || n_seqs > (1ll << 16) ||
      max_pages > (1ll << 20) || n_tokens * heads >= kGqaMaxRows || (head_dim != 64 && head_dim != 128)) return 0;
  return gqa_plan(n_seqs, n_tokens, heads, kv_heads, head_dim, max_pages).bytes;
}

extern "C" int tl_flash_paged_gqa(const void* q_bf16, int64_t q_stride, const void* kv_pages, int64_t n_pages,
                                  const int32_t* block_table, int64_t max_pages, const int32_t* cu_seqlens,
                                  const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t kv_heads,
                                  int64_t head_dim, float softmax_scale, void* out_bf16, float* lse, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* who = "flash_paged_gqa";
  if (int rc = check_batch(who, kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (int rc = check_gqa(who, kv_heads, head_dim)) return rc;
  if (int rc = check_gqa_heads(who, heads, kv_heads)) return rc;
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (int rc = check_gqa_batch(who, n_seqs, n_tokens, heads, max_pages, softmax_scale)) return rc;
  if (int rc = check_gqa_rows(who, "query", q_bf16, q_stride, heads, head_dim)) return rc;
  if (int rc = check_gqa_rows(who, "output", out_bf16, heads * head_dim, heads, head_dim)) return rc;
  const GqaPlan d = gqa_plan(n_seqs, n_tokens, heads, kv_heads, head_dim, max_pages);
  if (d.bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < d.bytes)) {
    set_error("%s: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", who, d.bytes, workspace_bytes);
    return kErrArg;
  }
  if (d.slots * kv_heads * d.splits >= (1ll << 24)) {
    set_error("%s: %lld tokens, %lld sequences: more than a launch has room for", who, (long long)n_tokens, (long long)n_seqs);
    return kErrUnsupported;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const GqaArgs args{(const uint16_t*)q_bf16, q_stride, (const uint8_t*)kv_pages, gqa_page_bytes(kv_heads, head_dim),
                     PagedBatch{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens},
                     (int)heads, (int)kv_heads, (int)(heads / kv_heads), softmax_scale * kLog2e, (uint16_t*)out_bf16, lse,
                     (int)d.chunk, (int)d.splits, reinterpret_cast<float2*>(ws), reinterpret_cast<float*>(ws + d.o_at)};
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto dim, auto rt) -> int {
    constexpr int D = decltype(dim)::value, RT = decltype(rt)::value;
    hipLaunchKernelGGL((gqa_attend_kernel<D, RT>), dim3(d.slots * kv_heads, d.splits), dim3(256), 0, st, args);
    if (int rc = check_launch(who)) return rc;
    if (d.splits == 1) return kOk;
    hipLaunchKernelGGL((gqa_join_kernel<D, RT>), dim3(d.slots * kv_heads, RT * D / 16), dim3(512), 0, st, args);
    return check_launch(who);
  };
  using std::integral_constant;
  if (head_dim == 64) return d.rt == 1 ? launch(integral_constant<int, 64>{}, integral_constant<int, 1>{}) : launch(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  return d.rt == 1 ? launch(integral_constant<int, 128>{}, integral_constant<int, 1>{}) : launch(integral_constant<int, 128>{}, integral_constant<int, 2>{});
}

extern "C" int tl_gqa_cache_weights(const void* q_bf16, int64_t q_stride, const float* lse, const void* kv_pages, int64_t n_pages,
                                    const int32_t* block_table, int64_t max_pages, const int32_t* cu_seqlens,
                                    const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t kv_heads,
                                    int64_t head_dim, float softmax_scale, int accumulate, float* key_weights, void* stream) {
  const char* who = "gqa_cache_weights";
  if (int rc = check_batch(who, kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (int rc = check_gqa(who, kv_heads, head_dim)) return rc;
  if (int rc = check_gqa_heads(who, heads, kv_heads)) return rc;
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (int rc = check_gqa_batch(who, n_seqs, n_tokens, heads, max_pages, softmax_scale)) return rc;
  if (int rc = check_gqa_rows(who, "query", q_bf16, q_stride, heads, head_dim)) return rc;
  if (!lse || !key_weights) { set_error("%s: null pointer", who); return kErrArg; }
  const bool split = n_tokens * (heads / kv_heads) >= 64 * n_seqs;
  const int64_t groups = split ? max_pages : cdiv(max_pages, 4), units = n_seqs * groups * kv_heads;
  const GqaSumArgs args{(const uint16_t*)q_bf16, q_stride, lse, (const uint8_t*)kv_pages, gqa_page_bytes(kv_heads, head_dim),
                        PagedBatch{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens},
                        (int)heads, (int)kv_heads, (int)(heads / kv_heads), accumulate, softmax_scale * kLog2e, key_weights, units, (int)groups};
  const auto kern = head_dim == 64 ? (split ? gqa_sum_kernel<64, true> : gqa_sum_kernel<64, false>)
                                   : (split ? gqa_sum_kernel<128, true> : gqa_sum_kernel<128, false>);
  hipLaunchKernelGGL(kern, dim3(units < (1 << 16) ? units : (1 << 16)), dim3(256), 0, (hipStream_t)stream, args);
  return check_launch(who);
}
