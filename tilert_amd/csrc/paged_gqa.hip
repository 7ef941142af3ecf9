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

typedef float v16f __attribute__((ext_vector_type(16)));
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
  int target;       // pieces that the pages of all tiles are cut into at most, about; 0: one workgroup a tile
  int at_once;      // workgroups that run at a time
  int2* tile_parts;  // [tile slots]: a tile's first part and its parts (heads: `kv_heads` of them side by side)
  float2* part_ml;   // [parts][BM]
  float* part_o;     // [parts][BM * D]
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
  __device__ inline GqaSeq(const PagedBatch& p, int group_, int first_, int rows_, int64_t base_)
      : first(first_), rows(rows_), group(group_), base(base_), most(static_cast<int64_t>(p.max_pages) * kGqaKeys) {}
  // keys that a row sees, and their pages
  __device__ inline int seen(int row) const {
    const int64_t n = base + row / group + 1;
    return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
  }
  __device__ inline int pages(int row) const { return (seen(row) + kGqaKeys - 1) / kGqaKeys; }
};

// Tiles of BM rows: sequence b's have the slots from gqa_slot0(b) on, which leaves it as many as it can have.
__device__ inline int gqa_slot0(const PagedBatch& p, int group, int b, int bm) { return min(max(p.cu[b], 0), p.n_tokens) * group / bm + b; }
__device__ inline bool gqa_tile(const PagedBatch& p, int group, int slot, int bm, int& b, int& tile) {
  b = __builtin_amdgcn_readfirstlane(last_seq(p.n_seqs, [&](int i) { return gqa_slot0(p, group, i, bm) <= slot; }));
  if (b < 0 || b >= p.n_seqs) return false;
  tile = slot - gqa_slot0(p, group, b, bm);
  return tile >= 0;
}
inline int64_t gqa_slots(int64_t n_tokens, int64_t group, int64_t n_seqs, int bm) { return n_tokens * group / bm + n_seqs; }

// Max / sum over the lanes i, i ^ 16, i ^ 32, i ^ 48, in all of them.
template <bool MAX>
__device__ inline float four_lanes(float v) {
  const u32x2g a = __builtin_bit_cast(u32x2g, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float a0 = __uint_as_float(a[0]), a1 = __uint_as_float(a[1]), x = MAX ? fmaxf(a0, a1) : a0 + a1;
  const u32x2g b = __builtin_bit_cast(u32x2g, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
  const float b0 = __uint_as_float(b[0]), b1 = __uint_as_float(b[1]);
  return MAX ? fmaxf(b0, b1) : b0 + b1;
}

// What a workgroup works on: a tile of one kv head, and its pages pg0 .. pg1 - 1; the tile's parts and which of them this is.
struct GqaItem {
  int b, tile, pg0, pg1, parts;
  int64_t part;
};
// Every workgroup plans the launch for itself, from the metadata on the device: the pages of all tiles are cut into pieces of
// at most `chunk`, at least kGqaFew; a tile's pieces are of one size.  Where a tile has several, they have a place each in
// the workspace: at most 2 * target of them, as such a tile has more than `chunk` pages, and `chunk` is no less than the
// target-th part of all.
// SEARCH: of kGqaPlans sizes from that part on, up to four times of it, the one that should be done first.  Pieces that run all at
// once are done with the longest; where they are more, they follow one another as workgroups end: all of them, and half of the
// longest.  A piece costs kGqaPiece pages beside its own.  (With a fixed number of pieces wanted, 7 sequences of 2 to 700 new
// tokens over 324 to 5000 keys took 57 us with 120, 53 with 330, 50 with 384 and 55 with 780; with the search 45.  32 sequences of
// 1024 keys, 256 tiles of 32 rows: 33 uncut, as the search has it, and 52 with 512 pieces.)
// Sequences that a launch plans for; with more, a workgroup takes a tile.  In us with one sequence of 32768 keys among 512 and 513 of
// 1024, 64 heads over 8, head_dim 128: attention 357 / 424, key weights 176 / 599.
constexpr int kGqaPlanSeqs = 512;
constexpr int kGqaFew = 8;         // pages that are not cut
constexpr int kGqaPlans = 16;
constexpr float kGqaPiece = 9.f;
struct GqaPlanLds {
  int end[kGqaPlanSeqs];   // pieces up to sequence b and with it
  int part[kGqaPlanSeqs];  // of them, those of tiles with several, before sequence b
  int splits[kGqaPlanSeqs], rows[kGqaPlanSeqs], first[kGqaPlanSeqs];
  int64_t base[kGqaPlanSeqs];
  int scan[2][8];
  float sum[8];
  float pieces[8][kGqaPlans], longest[8][kGqaPlans];
};
template <int THREADS, int BM, bool SEARCH, class Args>
__device__ inline bool gqa_plan_item(const Args& A, GqaPlanLds& L, int v, GqaItem& it, int& first, int& rows, int64_t& base) {
  constexpr int WAVES = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float units = 0.f;
  for (int b = tid; b < A.p.n_seqs; b += THREADS) {
    const GqaSeq s(A.p, A.group, b);
    const int n = s.rows > 0 ? s.pages(s.rows - 1) : 0, tiles = (s.rows + BM - 1) / BM;
    L.first[b] = s.first;
    L.rows[b] = s.rows;
    L.base[b] = s.base;
    L.splits[b] = n;
    units += static_cast<float>(tiles) * static_cast<float>(n);
  }
  units = wave_sum_f32(units);
  if (lane == 0) L.sum[wave] = units;
  __syncthreads();
  units = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) units += L.sum[w];
  // (a little more than their share, so that the sum's rounding leaves no piece over)
  units *= A.kv_heads;
  auto size = [&](float by) { return max(kGqaFew, static_cast<int>(fminf(units / A.target * 1.001f * by, 2e6f)) + 1); };  // (2^20 pages a sequence at most)
  int chunk = size(1.f);
  if constexpr (SEARCH) {
    auto plan = [](int i) { return __builtin_amdgcn_exp2f(2.f / (kGqaPlans - 1) * i); };
    static_assert(kGqaPlans == 16, "a plan is a lane of 16");
    const int mine = lane & 15;
    const float by = 1.0f / size(plan(mine));
    float pieces = 0.f, longest = 0.f;
    for (int b = tid >> 4; b < A.p.n_seqs; b += THREADS / 16) {
      const int tiles = (L.rows[b] + BM - 1) / BM;
      const float n = static_cast<float>(L.splits[b]), cut = fmaxf(1.f, __builtin_ceilf(n * by));
      pieces += tiles * cut;
      longest = fmaxf(longest, tiles ? n / cut : 0.f);
    }
    pieces = four_lanes<false>(pieces);
    longest = four_lanes<true>(longest);
    if (lane < 16) {
      L.pieces[wave][lane] = pieces;
      L.longest[wave][lane] = longest;
    }
    __syncthreads();
    pieces = longest = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      pieces += L.pieces[w][mine];
      longest = fmaxf(longest, L.longest[w][mine]);
    }
    pieces *= A.kv_heads;
    longest += kGqaPiece;
    const float time = pieces <= A.at_once ? longest : (units + pieces * kGqaPiece) / A.at_once + 0.5f * longest;
    float best = time;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) best = fminf(best, __shfl_xor(best, o));
    chunk = size(plan(63 - __builtin_clzll(__ballot(lane < 16 && time == best) | 1)));
    chunk = __builtin_amdgcn_readfirstlane(chunk);
  }
  int ends = 0, parts = 0;
  for (int b0 = 0; b0 < A.p.n_seqs; b0 += THREADS) {
    const int b = b0 + tid;
    int pieces = 0, cut = 0;
    if (b < A.p.n_seqs) {
      const int tiles = (L.rows[b] + BM - 1) / BM, n = max(1, (L.splits[b] + chunk - 1) / chunk);
      L.splits[b] = n;
      pieces = tiles * n;
      cut = n > 1 ? pieces : 0;
    }
    const int e = gqa_wave_scan(pieces), p = gqa_wave_scan(cut);
    if (lane == 63) {
      L.scan[0][wave] = e;
      L.scan[1][wave] = p;
    }
    __syncthreads();
    int before_e = ends, before_p = parts;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int x = L.scan[0][w], y = L.scan[1][w];
      before_e += w < wave ? x : 0;
      before_p += w < wave ? y : 0;
      ends += x;
      parts += y;
    }
    if (b < A.p.n_seqs) {
      L.end[b] = before_e + e;
      L.part[b] = before_p + p - cut;
    }
    __syncthreads();
  }
  if (v >= ends) return false;
  const int b = __builtin_amdgcn_readfirstlane(last_seq(A.p.n_seqs, [&](int i) { return (i ? L.end[i - 1] : 0) <= v; }));
  if (b < 0 || b >= A.p.n_seqs) return false;
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  first = uniform(L.first[b]);
  rows = uniform(L.rows[b]);
  base = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(L.base[b] >> 32)))) << 32 |
                              static_cast<uint32_t>(uniform(static_cast<int>(L.base[b]))));
  const int at = uniform(v - (b ? L.end[b - 1] : 0));
  it.b = b;
  it.parts = uniform(L.splits[b]);
  it.tile = at / it.parts;
  it.part = static_cast<int64_t>(uniform(L.part[b])) + at;
  it.pg0 = at % it.parts;  // (in pieces yet)
  return at >= 0 && it.tile < (rows + BM - 1) / BM;  // (cu_seqlens that does not ascend)
}

// The workgroup's item; false: it has none.
template <int THREADS, int BM>
__device__ inline bool gqa_item(const GqaArgs& A, GqaPlanLds& L, int v, GqaItem& it, int& first, int& rows, int64_t& base) {
  if (A.target) {
    if (!gqa_plan_item<THREADS, BM, true>(A, L, v, it, first, rows, base)) return false;
  } else {
    if (!gqa_tile(A.p, A.group, v, BM, it.b, it.tile)) return false;
    const GqaSeq s(A.p, A.group, it.b);
    first = s.first;
    rows = s.rows;
    base = s.base;
    if (it.tile >= (rows + BM - 1) / BM) return false;
    it.parts = 1;
    it.pg0 = 0;
    it.part = 0;
  }
  const GqaSeq s(A.p, A.group, first, rows, base);
  const int n = s.pages(min((it.tile + 1) * BM, rows) - 1), each = (n + it.parts - 1) / it.parts, piece = it.pg0;
  it.pg0 = piece * each;
  it.pg1 = min(it.pg0 + each, n);
  // (tile_parts: by slot, as a join's workgroups find their tiles)
  if (A.target && piece == 0 && threadIdx.x == 0 && blockIdx.x % A.kv_heads == 0)
    A.tile_parts[gqa_slot0(A.p, A.group, it.b, BM) + it.tile] = int2{static_cast<int>(it.part), it.parts};
  return true;
}

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

// Bytes that are no number in bf16 under a block's scale, as 0x80 each: NaN codes, and from 2^120 on those that it takes past the
// largest (a page's earlier use may have left them behind its last key; a key that a row does not see has weight 0, and 0 times an
// infinity is NaN).  `from`, of the scale: what brings the least of them to 0x80.
__device__ inline uint32_t bad_codes_from(float scale) {
  return 0x01010101u * static_cast<uint32_t>(max(1, (static_cast<int>(__float_as_uint(scale) >> 23) - 246) * 8));
}
__device__ inline uint32_t bad_codes(uint32_t x, uint32_t from) { return ((x & 0x7f7f7f7fu) + from) & 0x80808080u; }

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
template <int D, bool ONCE>  // ONCE: no other wave reads them
__device__ inline GqaValues<D> load_values(const uint8_t* v, int lane) {
  GqaValues<D> r;
  const uint8_t* from = v + (lane & 15) * kGqaKeys + 16 * (lane >> 4);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const u32x4g* at = reinterpret_cast<const u32x4g*>(from + d * 16 * kGqaKeys);
    r.v[d] = ONCE ? __builtin_nontemporal_load(at) : *at;
  }
  return r;
}

__device__ inline float2 load_scales(const float* s) { return float2{load_f32_vector(s), load_f32_vector(s + 1)}; }

// One tile of 16 RT rows and one kv head over a piece's pages; the four waves take every fourth of them (RT = 4: two by two every
// second), each with its own statistics, and are joined in LDS.  A wave has up to 32 rows, so that the codes, 128 conversions
// of two a page and lane, are turned for all of them (16 rows a wave, two waves on the same pages: 4 tokens of 8 heads over
// 131072 keys 76 us, 59 so).  Weights go into the second product as hi + lo in bf16, 16 bits of them.
// Weights are relative to 2^24 times the row's largest: their sums of values then stay inside fp32 whatever the values, for up to
// 2^24 keys as heavy as the heaviest.
// Bound by bytes, two pages a wave on their way: 60 sequences of 2048 to 32768 keys, 1.42 GB, 238 us, 6.0 TB/s; 131072 keys, 268 MB,
// 55 us and 6 to join, where a copy's rate takes 52.  One token over a table of up to 8 pages, which is not planned, is bound by
// latency: 1 to 64 keys 5.6 us, loads one behind another (token ranges and lengths, table, page), the products, the waves' join;
// 256, a page each for the four waves, 6.8; 500, two one behind another, 8.4.
constexpr float kGqaHead = 24.f;
template <int D, int RT>
__global__ __launch_bounds__(256, D == 128 && RT > 1 ? 1 : 2) void gqa_attend_kernel(const GqaArgs A) {
  constexpr int BM = 16 * RT, DT = D / 16, KI = D / 64, TW = RT < 2 ? 1 : 2, RG = RT / TW, PW = 4 / RG;  // TW: row tiles of a wave; PW: waves that share their pages
  __shared__ union {
    GqaPlanLds plan;
    v4f sum_o[4][DT][64];
  } L;
  __shared__ float sum_m[TW][4][16], sum_l[TW][4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4, rg = wave % RG, pw = wave / RG, rt0 = rg * TW;
  const int head = blockIdx.x % A.kv_heads;
  GqaItem it;
  int first, rows_all;
  int64_t base;
  if (!gqa_item<256, BM>(A, L.plan, blockIdx.x / A.kv_heads, it, first, rows_all, base)) return;
  const GqaSeq s(A.p, A.group, first, rows_all, base);
  const int row0 = it.tile * BM, rows = min(s.rows - row0, BM);
  const int least = s.seen(row0 + min(16 * rt0, rows - 1));
  const gqa_const_i32 table = (gqa_const_i32)(A.p.table + static_cast<int64_t>(it.b) * A.p.max_pages);
  GqaQuery<D> q[TW];
  int seen[TW];
  float m[TW], l[TW];
  v4f o[TW][DT];
#pragma unroll
  for (int r = 0; r < TW; ++r) {
    q[r] = load_query<D>(A.q, A.q_stride, s, head * A.group, row0 + (rt0 + r) * 16 + c, g);
    seen[r] = s.seen(row0 + min((rt0 + r) * 16 + c, rows - 1));
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[r][d] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // A page's scores, weights and sums.  Its keys are there already; its values are under way while the scores are made, and
  // the next page's keys behind them.
  auto step = [&](int pg, bool there, const GqaKeys<D>& kc, GqaValues<D>& vc, float2 scales) __attribute__((always_inline)) {
    const bool ok = gqa_scale_ok(scales.x) && gqa_scale_ok(scales.y);
    const float sk = ok ? scales.x : 1.f, sv = ok ? scales.y : 1.f;
    const int key0 = pg * kGqaKeys;
    const bool masked = !there || !__all(ok) || key0 + kGqaKeys > least;
    // ---- scores
    v4f x[TW][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int r = 0; r < TW; ++r) x[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const v8bf k = codes8_bf16(kc.k[t][i][2 * e], kc.k[t][i][2 * e + 1], sk);
#pragma unroll
          for (int r = 0; r < TW; ++r) x[r][t] = mfma_bf16(k, q[r].x[i][e], x[r][t]);
        }
    }
    // ---- weights
    v8bf hi[TW][2], lo[TW][2];
    int my[TW];  // of this lane's 16 keys, the row sees this many
#pragma unroll
    for (int r = 0; r < TW; ++r) {
      my[r] = there ? seen[r] - key0 - 16 * g : 0;
      if (masked) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[r][t][j] = 4 * t + j >= my[r] ? -INFINITY : (ok ? x[r][t][j] : __builtin_nanf(""));
      }
      float top = x[r][0][0];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, x[r][t][j]);
      top = fmaxf(m[r], four_lanes<true>(top) * A.scale);
      if (__any(top > m[r])) {
        const float by = m[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - top);  // (before the first key all is 0, or NaN)
        m[r] = top;
        l[r] *= by;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= by;
      }
      const float from = m[r] == -INFINITY ? 0.f : m[r] + kGqaHead;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x4g h, w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4f y = x[r][2 * e + i / 2];
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * (i & 1)], A.scale, -from));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * (i & 1) + 1], A.scale, -from));
          l[r] += p0 + p1;
          h[i] = bf16x2_bits(v2f{p0, p1});
          w[i] = bf16x2_bits(v2f{p0 - __uint_as_float(h[i] << 16), p1 - __uint_as_float(h[i] & 0xffff0000u)});
        }
        hi[r][e] = bf16_of(h);
        lo[r][e] = bf16_of(w);
      }
    }
    // ---- values; on a page with keys that some row does not see, codes that are no number are taken apart
    if (masked) {
      const uint32_t bad_from = bad_codes_from(sv);
      uint32_t all = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) all |= bad_codes(vc.v[d][i], bad_from);
      if (__any(all != 0)) {  // how many of them a row sees
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
          for (int r = 0; r < TW; ++r) {
            v4f n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              u32x4g w;
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = (8 * e + 2 * i < my[r] ? 0x3f80u : 0u) | (8 * e + 2 * i + 1 < my[r] ? 0x3f800000u : 0u);
              n = mfma_bf16(codes8_bf16(bad_codes(vc.v[d][2 * e], bad_from) >> 1, bad_codes(vc.v[d][2 * e + 1], bad_from) >> 1, 1.f), bf16_of(w), n);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) o[r][d][j] = n[j] > 0.f ? __builtin_nanf("") : o[r][d][j];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t bad = bad_codes(vc.v[d][i], bad_from);
            vc.v[d][i] &= ~(bad | (bad - (bad >> 7)));
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const v8bf a = codes8_bf16(vc.v[d][2 * e], vc.v[d][2 * e + 1], sv);
#pragma unroll
        for (int r = 0; r < TW; ++r) {
          o[r][d] = mfma_bf16(a, hi[r][e], o[r][d]);
          o[r][d] = mfma_bf16(a, lo[r][e], o[r][d]);
        }
      }
  };
  // pages pg0 + pw, + PW, ..; one outside the pool is read as page 0 and seen by no row
  auto page_id = [&](int pg) { return __builtin_amdgcn_readfirstlane(table[min(pg, it.pg1 - 1)]); };
  auto there = [&](int id) { return id >= 0 && id < A.p.n_pages; };
  auto block = [&](int id) { return gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, there(id) ? id : 0, head); };
  int pg = it.pg0 + pw;
  if (pg < it.pg1 && rt0 * 16 < rows) {
    GqaKeys<D> ka, kb;
    GqaValues<D> va, vb;
    float2 sa, sb;
    int id = page_id(pg), next = page_id(pg + PW);
    ka = load_keys<D>(block(id).k, lane);
    va = load_values<D, RG == 1>(block(id).v, lane);
    sa = load_scales(block(id).scale);
    // (two buffers by turns: one copied into the other would wait for its loads)
    auto half = [&](const GqaKeys<D>& k_now, GqaValues<D>& v_now, float2 s_now, GqaKeys<D>& k_then, GqaValues<D>& v_then, float2& s_then) __attribute__((always_inline)) {
      k_then = load_keys<D>(block(next).k, lane);
      v_then = load_values<D, RG == 1>(block(next).v, lane);
      s_then = load_scales(block(next).scale);
      const bool is = there(id);
      id = next;
      next = page_id(pg + 2 * PW);
      step(pg, is, k_now, v_now, s_now);
      pg += PW;
    };
    while (true) {
      half(ka, va, sa, kb, vb, sb);
      if (pg >= it.pg1) break;
      half(kb, vb, sb, ka, va, sa);
      if (pg >= it.pg1) break;
    }
  }
  // ---- the waves of the same rows together
  float top[TW], total[TW];
#pragma unroll
  for (int r = 0; r < TW; ++r) {
    l[r] = four_lanes<false>(l[r]);
    if (g == 0) {
      sum_m[r][wave][c] = m[r];
      sum_l[r][wave][c] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < TW; ++r) {
    top[r] = -INFINITY;
    total[r] = 0.f;
#pragma unroll
    for (int w = 0; w < PW; ++w) top[r] = fmaxf(top[r], sum_m[r][rg + RG * w][c]);
#pragma unroll
    for (int w = 0; w < PW; ++w) {
      const float mw = sum_m[r][rg + RG * w][c];
      total[r] += sum_l[r][rg + RG * w][c] * (mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - top[r]));
    }
  }
  const bool whole = it.parts == 1;
  const int64_t part = it.part * A.kv_heads + head;
#pragma unroll
  for (int r = 0; r < TW; ++r) {
    const int rt = rt0 + r;
    const float by = m[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - top[r]);
    if (r) __syncthreads();  // (the tile in front is read)
#pragma unroll
    for (int d = 0; d < DT; ++d) L.sum_o[wave][d][lane] = o[r][d] * by;
    __syncthreads();
    const bool live = rt * 16 + c < rows;
    const int row = row0 + rt * 16 + c;
    const int64_t at = static_cast<int64_t>(s.first + row / A.group) * A.heads + head * A.group + row % A.group;
    const float inv = total[r] == 0.f ? 0.f : 1.0f / total[r];
#pragma unroll
    for (int i = 0; i < DT / PW; ++i) {
      const int d = PW * i + pw;
      v4f v = L.sum_o[rg][d][lane];
#pragma unroll
      for (int w = 1; w < PW; ++w) v += L.sum_o[rg + RG * w][d][lane];
      if (!live) continue;
      if (whole) *reinterpret_cast<u32x2g*>(A.out + at * D + 16 * d + 4 * g) = u32x2g{bf16x2_bits(v2f{v[0] * inv, v[1] * inv}), bf16x2_bits(v2f{v[2] * inv, v[3] * inv})};
      else reinterpret_cast<v4f*>(A.part_o + part * (BM * D))[(rt * DT + d) * 64 + lane] = v;
    }
    if (pw == 0 && g == 0 && live) {
      if (!whole) A.part_ml[part * BM + rt * 16 + c] = float2{top[r], total[r]};
      else if (A.lse) A.lse[at] = total[r] == 0.f ? -INFINITY : (top[r] + kGqaHead + log2f(total[r])) * kLn2;
    }
  }
}

// ---- many rows: the waves of a workgroup go through the pages together
// A page's codes are turned into bf16 once, by the wave that loaded them, and lie in LDS as the products' operands, fragment
// by fragment in lane order; each wave multiplies them with its own 32 rows.  Weights go into the second product in
// bf16, 8 bits: the result's rms error is 0.0023 of it, 0.0017 with the 16 bits that few rows have, of which the result's own rounding
// to bf16 is the most; a second product for the other 8 would be half of the matrix pipe's work again.
// A row's reference m is set anew only where a score of its own passes it by 2^8: hardly a page rescales anything.
//
// The two waves of a SIMD are a third of a page apart: between two barriers waves 0 .. 3 make scores, weights and sums of page k,
// waves 4 .. 7 weights and sums of page k - 1 and scores of page k, so that one's products run while the other makes
// weights.  (At the same place of the page, 532 us for 2048 tokens over 16384 keys, 482 so: 1.07 PFLOP/s, the matrix pipe busy
// 53 % of the cycles at 2.15 GHz; bound by the issue of vector instructions beside it.)  Values are multiplied up to a page
// later than keys, so they have three buffers and keys two.
constexpr float kGqaLag = 8.f;
constexpr int kChunkWaves = 8, kChunkRows = 32 * kChunkWaves;
template <int D>
struct GqaChunkLds {
  static constexpr int KF = D / 16, VT = D / 32;  // fragments of 32 keys; 32-dim tiles of the values
  union {
    GqaPlanLds plan;
    struct {
      u32x4g k[2][2][KF][64];     // [t][f]: 32 keys x 16 dims
      u32x4g v[3][VT][2][2][64];  // [d][t][e]: 32 dims x 16 keys
      u32x4g bad[3][VT][2][64];   // [d][t]: where values of a page that is not seen by all rows are no number
    };
  };
  int odd[3];  // the page of a buffer that has such values
};
__device__ inline v16f mfma32_bf16(v8bf a, v8bf b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
template <bool MAX>
__device__ inline float two_halves(float v) {  // of lanes i, i ^ 32, in both
  const u32x2g b = __builtin_bit_cast(u32x2g, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float b0 = __uint_as_float(b[0]), b1 = __uint_as_float(b[1]);
  return MAX ? fmaxf(b0, b1) : b0 + b1;
}
// Row i of a 32-key fragment of tile t is the page's key 32 (i / 4 % 2) + 16 t + 4 (i / 8) + i % 4, so that a lane's sixteen
// results are the keys 32 h + 16 t .. + 15 of its row, as a 16-byte load of a dim's values has them (h: the lane's half).
template <int D>
__global__ __launch_bounds__(64 * kChunkWaves, 2) void gqa_chunk_kernel(const GqaArgs A) {
  constexpr int NW = kChunkWaves, BM = kChunkRows, KI = D / 64, KP = 4 * KI, MINE = (KP + D / 16) / NW, KF = D / 16, VT = D / 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t gqa_smem[];
  GqaChunkLds<D>& L = *reinterpret_cast<GqaChunkLds<D>*>(gqa_smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5, late = wave >> 2;
  const int head = blockIdx.x % A.kv_heads;
  GqaItem it;
  int first, rows_all;
  int64_t base;
  if (!gqa_item<64 * NW, BM>(A, L.plan, blockIdx.x / A.kv_heads, it, first, rows_all, base)) return;
  const GqaSeq s(A.p, A.group, first, rows_all, base);
  const int row0 = it.tile * BM + wave * 32, last = s.rows - 1;  // this wave's rows
  const bool any = row0 <= last;
  const int least = s.seen(min(row0, last)), least_all = s.seen(it.tile * BM);
  const gqa_const_i32 table = (gqa_const_i32)(A.p.table + static_cast<int64_t>(it.b) * A.p.max_pages);
  // the query rows as the first product's B operand: lane (c, h) has of row c the dims 64 i + 32 j + 16 h + 8 e .. + 7 for
  // fragment 4 i + 2 j + e, as a 16-byte load gives it a key's codes
  v8bf q[KF];
  {
    const bool live = row0 + c <= last;
    const int at = live ? row0 + c : 0;
    const uint16_t* from = A.q + (s.first + at / A.group) * A.q_stride + (head * A.group + at % A.group) * D + 16 * h;
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      u32x4g v = *reinterpret_cast<const u32x4g*>(from + 32 * (f / 2) + 8 * (f % 2));
      if (!live) v = u32x4g{0, 0, 0, 0};
      q[f] = bf16_of(v);
    }
  }
  const int seen = s.seen(min(row0 + c, last));
  float m = -INFINITY, l = 0.f;
  v16f o[VT], x[2];
  v8bf p[2][2];
#pragma unroll
  for (int d = 0; d < VT; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[d][j] = 0.f;
  const int n = it.pg1 - it.pg0;
  auto page_id = [&](int k) { return __builtin_amdgcn_readfirstlane(table[it.pg0 + min(k, n - 1)]); };
  auto there = [&](int id) { return id >= 0 && id < A.p.n_pages; };
  auto unseen = [&](int k) { return (it.pg0 + k + 1) * kGqaKeys > least_all; };  // some row of the tile does not see all of the page
  auto fine = [&](float2 v) { return static_cast<bool>(__all(gqa_scale_ok(v.x) && gqa_scale_ok(v.y))); };
  struct Codes {
    u32x4g x[MINE];
    float2 s;
    bool is;
  };
  // This wave's pieces of a page, 1 KB each: 16 keys x 64 dims, then 16 dims x 64 keys; lane (r, b) has 16 bytes b of row r
  const int r16 = lane & 15, b16 = lane >> 4;
  auto fetch = [&](int id) __attribute__((always_inline)) {
    const GqaBlock blk = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, there(id) ? id : 0, head);
    Codes r;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int piece = wave + NW * j, rows = piece / KI;  // of keys: t = rows / 2, fragment rows 16 (rows % 2) ..
      const int i = 16 * (rows & 1) + r16;
      const uint8_t* k = blk.k + (32 * (i >> 2 & 1) + 16 * (rows >> 1) + 4 * (i >> 3) + (i & 3)) * D + 64 * (piece % KI) + 16 * b16;
      const uint8_t* v = blk.v + ((piece - KP) * 16 + r16) * kGqaKeys + 16 * b16;
      r.x[j] = *reinterpret_cast<const u32x4g*>(piece < KP ? k : v);
    }
    r.s = load_scales(blk.scale);
    r.is = there(id);
    return r;
  };
  auto stage = [&](const Codes& r, bool ok, int k, int kb, int vb) __attribute__((always_inline)) {
    const bool masked = unseen(k) || !r.is;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int piece = wave + NW * j;
      const float by = ok ? (piece < KP ? r.s.x : r.s.y) : 1.f;
      u32x4g x = r.x[j];
      u32x4g* to;  // the fragment of the piece's even 8 bytes; that of the odd ones is the next
      if (piece < KP) {
        const int rows = piece / KI;
        to = &L.k[kb][rows >> 1][4 * (piece % KI) + 2 * (b16 >> 1)][32 * (b16 & 1) + 16 * (rows & 1) + r16];
      } else {
        const int d = piece - KP, at = 32 * (b16 >> 1) + 16 * (d & 1) + r16;
        if (masked) {  // on a page with keys that some row does not see, values that are no number are taken apart
          const uint32_t bad_from = bad_codes_from(by);
          u32x4g bad;
#pragma unroll
          for (int i = 0; i < 4; ++i) bad[i] = bad_codes(x[i], bad_from);
          if (__any((bad[0] | bad[1] | bad[2] | bad[3]) != 0) && lane == 0) L.odd[vb] = it.pg0 + k;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] &= ~(bad[i] | (bad[i] - (bad[i] >> 7)));
            bad[i] >>= 1;  // the code of 2
          }
          L.bad[vb][d >> 1][b16 & 1][at] = bad;
        }
        to = &L.v[vb][d >> 1][b16 & 1][0][at];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) to[64 * e] = __builtin_bit_cast(u32x4g, codes8_bf16(x[2 * e], x[2 * e + 1], by));
    }
  };
  // (operands are read four fragments ahead of the products, by hand: left to itself the compiler waits for each)
  auto scores = [&](int kb) __attribute__((always_inline)) {
    if (!any) return;
    v8bf f[2][4];
    auto load = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[i & 1][j] = bf16_of(L.k[kb][i / (KF / 4)][i % (KF / 4) * 4 + j][lane]);
    };
    load(0);
#pragma unroll
    for (int i = 0; i < KF / 2; ++i) {
      const int t = i / (KF / 4);
      if (i + 1 < KF / 2) load(i + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (i % (KF / 4) == 0)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[t][j] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[t] = mfma32_bf16(f[i & 1][j], q[i % (KF / 4) * 4 + j], x[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto values = [&](int k, bool is, int vb) __attribute__((always_inline)) {
    if ((unseen(k) || !is) && L.odd[vb] == it.pg0 + k) {  // how many of them a row sees
      const int my = is ? seen - (it.pg0 + k) * kGqaKeys - 32 * h : 0;
#pragma unroll
      for (int d = 0; d < VT; ++d) {
        v16f z;
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const u32x4g w = L.bad[vb][d][t][lane];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u32x4g sees;
#pragma unroll
            for (int i = 0; i < 4; ++i) sees[i] = (16 * t + 8 * e + 2 * i < my ? 0x3f80u : 0u) | (16 * t + 8 * e + 2 * i + 1 < my ? 0x3f800000u : 0u);
            z = mfma32_bf16(codes8_bf16(w[2 * e], w[2 * e + 1], 1.f), bf16_of(sees), z);
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] = z[j] > 0.f ? __builtin_nanf("") : o[d][j];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    v8bf f[2][VT];
    auto load = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < VT; ++d) f[i & 1][d] = bf16_of(L.v[vb][d][i >> 1][i & 1][lane]);
    };
    load(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < 3) load(i + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < VT; ++d) o[d] = mfma32_bf16(f[i & 1][d], p[i >> 1][i & 1], o[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto weights = [&](int pg, bool is, bool ok) __attribute__((always_inline)) {
    const int key0 = pg * kGqaKeys;
    if (!is || !ok || key0 + kGqaKeys > least) {
      const int my = is ? seen - key0 - 32 * h : 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[t][j] = 16 * t + j >= my ? -INFINITY : (ok ? x[t][j] : __builtin_nanf(""));
    }
    float top = x[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, x[t][j]);
    top *= A.scale;
    if (__any(top > m + kGqaLag)) {  // (row by row: one that stays is multiplied by 1, and owes nothing to its neighbours)
      const float high = two_halves<true>(top), now = high > m + kGqaLag ? high : m;
      const float by = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= by;
#pragma unroll
      for (int d = 0; d < VT; ++d) o[d] *= by;
    }
    const float from = m == -INFINITY ? 0.f : m + kGqaHead;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x4g w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][8 * e + 2 * i], A.scale, -from));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][8 * e + 2 * i + 1], A.scale, -from));
          l += p0 + p1;
          w[i] = bf16x2_bits(v2f{p0, p1});
        }
        p[t][e] = bf16_of(w);
      }
  };
  // Of two waves that could issue, the hardware takes the older one, and waves 4 .. 7, with their weights first and both
  // products behind, would come last to every barrier: 510 us, 482 with their priority raised.
  if (late) __builtin_amdgcn_s_setprio(1);
  __syncthreads();  // (the plan's memory is free)
  if (tid < 3) L.odd[tid] = -1;
  __syncthreads();
  if (n > 0) {
    // of page k and the one before: whether its scales are fine, and whether it is there; the codes of the two pages behind it,
    // by turns in ca and cb
    int vb = 0;
    Codes ca = fetch(page_id(0)), cb;
    bool ok = fine(ca.s), is = ca.is, ok_before = ok, was = is;
    stage(ca, ok, 0, 0, 0);
    cb = fetch(page_id(1));
    ca = fetch(page_id(2));
    __syncthreads();
    auto ahead = [&](int k, int kb, Codes& codes) __attribute__((always_inline)) {  // page k + 1 into its buffers, page k + 3 on its way
      const int to = vb == 2 ? 0 : vb + 1;
      ok_before = ok;
      was = is;
      ok = fine(codes.s);
      is = codes.is;
      if (k + 1 < n) stage(codes, ok, k + 1, kb ^ 1, to);
      codes = fetch(page_id(k + 3));
      vb = to;
      __syncthreads();
    };
    auto earlier = [&](int k) __attribute__((always_inline)) {
      if (!any) return;
      weights(it.pg0 + k - 1, was, ok_before);
      values(k - 1, was, vb == 0 ? 2 : vb - 1);
    };
    if (late) {
      scores(0);
      ahead(0, 0, cb);
      int k = 1;
#pragma unroll 1
      for (; k + 1 < n; k += 2) {
        earlier(k);
        scores(1);
        ahead(k, 1, ca);
        earlier(k + 1);
        scores(0);
        ahead(k + 1, 0, cb);
      }
      if (k < n) {
        earlier(k);
        scores(1);
        ahead(k, 1, ca);
      }
      earlier(n);
    } else {
      auto page = [&](int k, int kb, Codes& codes) __attribute__((always_inline)) {
        scores(kb);
        if (any) {
          weights(it.pg0 + k, is, ok);
          values(k, is, vb);
        }
        ahead(k, kb, codes);
      };
      int k = 0;
#pragma unroll 1
      for (; k + 1 < n; k += 2) {
        page(k, 0, cb);
        page(k + 1, 1, ca);
      }
      if (k < n) page(k, 0, cb);
    }
  }
  l = two_halves<false>(l);
  if (row0 + c > last) return;
  const bool whole = it.parts == 1;
  const int64_t part = it.part * A.kv_heads + head;
  const int64_t at = static_cast<int64_t>(s.first + (row0 + c) / A.group) * A.heads + head * A.group + (row0 + c) % A.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int d = 0; d < VT; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // dims 32 d + 8 j + 4 h .. + 3
      const v4f v = {o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
      if (whole) *reinterpret_cast<u32x2g*>(A.out + at * D + 32 * d + 8 * j + 4 * h) = u32x2g{bf16x2_bits(v2f{v[0] * inv, v[1] * inv}), bf16x2_bits(v2f{v[2] * inv, v[3] * inv})};
      else reinterpret_cast<v4f*>(A.part_o + part * (BM * D))[((wave * 2 + (c >> 4)) * (D / 16) + 2 * d + (j >> 1)) * 64 + (2 * (j & 1) + h) * 16 + (c & 15)] = v;
    }
  if (h == 0) {
    if (!whole) A.part_ml[part * BM + wave * 32 + c] = float2{m, l};
    else if (A.lse) A.lse[at] = l == 0.f ? -INFINITY : (m + kGqaHead + log2f(l)) * kLn2;
  }
}

// The parts of cut tiles joined in a fixed order, 16 rows of a tile at a time.  DEEP: a workgroup takes 16 dims of them, its eight
// waves every eighth part, joined in LDS (few tiles of many parts); else its waves take 16 dims each.  Bound by latency: 8 tiles of
// 32 parts, 8 MB in all, 5.9 us.
constexpr int kJoinWaves = 8;
template <int D, int BM, bool DEEP>
__global__ __launch_bounds__(64 * kJoinWaves) void gqa_join_kernel(const GqaArgs A) {
  constexpr int DT = D / 16, PER = DEEP ? DT : (DT + kJoinWaves - 1) / kJoinWaves, STEP = DEEP ? kJoinWaves : 1;
  __shared__ v4f sum_o[kJoinWaves][64];
  __shared__ float sum_l[kJoinWaves][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / A.kv_heads, head = blockIdx.x % A.kv_heads, r = blockIdx.y / PER;
  const int d = DEEP ? blockIdx.y % PER : blockIdx.y % PER * kJoinWaves + wave;
  if (!DEEP && d >= DT) return;
  int b, tile;
  const int2 mine = A.tile_parts[slot];
  if (!gqa_tile(A.p, A.group, slot, BM, b, tile)) return;
  const GqaSeq s(A.p, A.group, b);
  const int row0 = tile * BM, rows = min(s.rows - row0, BM), parts = mine.y;
  // A tile that is there has told its parts; where cu_seqlens does not ascend, one may be found here that has not, and
  // nothing outside the workspace is read for it.
  if (rows <= r * 16 || parts <= 1 || parts > 2 * A.target || mine.x < 0 || mine.x > 2 * A.target) return;
  if ((static_cast<int64_t>(mine.x) + parts) * A.kv_heads > 2 * A.target) return;
  const bool live = r * 16 + c < rows;
  const int row = r * 16 + (live ? c : 0);  // (rows that are not there have no parts)
  const int at = (r * DT + d) * 64 + (live ? lane : 16 * g);
  auto part = [&](int i) { return static_cast<int64_t>(mine.x + i) * A.kv_heads + head; };
  float top = -INFINITY;
  for (int i = g; i < parts; i += 4) top = fmaxf(top, A.part_ml[part(i) * BM + row].x);
  top = four_lanes<true>(top);
  float l = 0.f;
  v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = DEEP ? wave : 0; i < parts; i += STEP) {
    const float2 ml = A.part_ml[part(i) * BM + row];
    const v4f x = reinterpret_cast<const v4f*>(A.part_o + part(i) * (BM * D))[at];
    const float by = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
    l += ml.y * by;
    o += x * by;
  }
  if constexpr (DEEP) {
    sum_o[wave][lane] = o;
    if (g == 0) sum_l[wave][c] = l;
    __syncthreads();
    if (wave > 0) return;
    l = sum_l[0][c];
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) {
      o += sum_o[w][lane];
      l += sum_l[w][c];
    }
  }
  if (!live) return;
  const int64_t to = static_cast<int64_t>(s.first + (row0 + row) / A.group) * A.heads + head * A.group + (row0 + row) % A.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<u32x2g*>(A.out + to * D + 16 * d + 4 * g) = u32x2g{bf16x2_bits(v2f{o[0] * inv, o[1] * inv}), bf16x2_bits(v2f{o[2] * inv, o[3] * inv})};
  if (A.lse && d == 0 && g == 0) A.lse[to] = l == 0.f ? -INFINITY : (top + kGqaHead + log2f(l)) * kLn2;
}

// The launch: rows a tile, workgroups, and the workspace.
struct GqaLaunch {
  int bm;
  int64_t slots, target, at_once, wgs;
  size_t ml_at, o_at, bytes;
};
inline GqaLaunch gqa_launch(int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_pages) {
  GqaLaunch d{};
  const int64_t group = heads / kv_heads, each = cdiv(n_tokens * group, n_seqs);
  // Tiles of 16 rows a wave, or 32 (64 in two waves where a head's 64 dims leave the registers), and beyond them kChunkRows.  In
  // us with 32-row, 64-row / kChunkRows tiles, 64 heads over 8, head_dim 128: 32 rows of 1 sequence over 131072 keys 66 / 95, of 8
  // over 4096 29 / 32, of 64 over 4096 142 / 184; 64 rows 91 / 98, 42 / 34, 204 / 191.  head_dim 64: 32 rows 35 / 73, 18 / 26,
  // 66 / 140; 64 rows 55 / 76, 26 / 27, 105 / 147; 96 rows of 8 over 4096 34 / 27.
  // The rule goes by the batch's mean, so a batch of unlike sequences pays for it: 60 sequences of one token over 1000 to 8000 keys
  // (119 us) and a chunk of 512 over 4096 (82) take 328 in one call, 64 heads over 8; 200 of one token over 200 to 2000 keys (113)
  // and a prompt of 800 (30) 241, with one of 100 (12) 116, 32 heads over 8.
  d.bm = each <= 16 ? 16 : (each <= 32 ? 32 : (each <= 64 && head_dim == 64 ? 64 : kChunkRows));
  d.slots = gqa_slots(n_tokens, group, n_seqs, d.bm);
  d.at_once = d.bm == kChunkRows || (head_dim == 128 && d.bm > 16) ? 256 : 512;  // (by registers one workgroup a CU, or two)
  // More pieces than run at once even out tiles of unlike lengths where those are about as many; elsewhere they are work to join,
  // and workgroups without any.  In us with at_once / 2 at_once: 60 sequences of 2048 to 32768 keys (480 tiles) 282 / 273; 200 of 94 to
  // 1500 (1600) 90 / 95; 4 tokens over 131072 (8) 66 / 75.
  const int64_t tiles = d.slots * kv_heads;
  if (n_seqs <= kGqaPlanSeqs && max_pages > kGqaFew) d.target = 2 * tiles <= d.at_once || tiles >= 2 * d.at_once ? d.at_once : d.at_once * 2;
  d.wgs = d.slots * kv_heads + d.target;
  if (d.target) {
    d.ml_at = (d.slots * sizeof(int2) + 255) / 256 * 256;
    d.o_at = d.ml_at + static_cast<size_t>(2 * d.target) * d.bm * sizeof(float2);
    d.bytes = d.o_at + static_cast<size_t>(2 * d.target) * d.bm * head_dim * sizeof(float);
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
  int target;       // few rows: as in GqaArgs
  int64_t units;    // sequences x groups of pages x kv heads
  int page_groups;  // of a sequence
  uint64_t per_group;  // ceil(2^34 / group): x / group = x * per_group >> 34 for x < 2^27, group <= 128
};
// Unit u: its kv head, sequence and group of pages (a head's units are kv_heads apart: with 8 heads, on one XCD and its L2).
struct GqaUnit {
  int head, b, pages;
  __device__ inline GqaUnit(const GqaSumArgs& A, int64_t u) {
    head = static_cast<int>(u % A.kv_heads);
    const int64_t v = u / A.kv_heads;
    b = static_cast<int>(v / A.page_groups);
    pages = static_cast<int>(v % A.page_groups);
  }
};

// Few rows (a decode step): a wave takes every fourth page of a piece, one behind another, the next two's keys on their way;
// their rows, RT tiles of 16 as a rule, stay in registers (a sequence's more of them are loaded page by page: 200 sequences of one token
// and a prompt of 800, 32 heads over 8, 70 and 30 us in a call each, 628 in one).  Scores as in the
// attention's first product, S^T = K Q^T: a lane sums its keys' weights over its column of rows.  A weight is e^(s - lse) as
// 2^(s' - lse'), lse' = lse log2 e rounded to fp32, which costs it up to 2^-24 lse': the sums' rms error is 2.0e-7, the
// plain form's in fp32 1.2e-7.  Bound by bytes: 60
// sequences of 2048 to 32768 keys, 730 MB, 157 us, 4.6 TB/s.  Pieces as the attention plans them (in groups of kSumPages
// pages by the table's width they took 170 us).  Two tiles against the kernel for many rows below: 4 tokens of 8 heads over
// 131072 keys 34 / 59 us, over 8192 keys of 40 sequences 90 / 147; four tiles, 8 tokens, 75 / 66.
constexpr int kSumPages = 32;  // pages of a piece where nothing is planned
template <int D, int RT>
__global__ __launch_bounds__(256, 2) void gqa_sum_few_kernel(const GqaSumArgs A) {
  __shared__ GqaPlanLds plan;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  for (int64_t u = blockIdx.x; u < A.units; u += gridDim.x) {
    GqaUnit unit(A, u);
    int pg0, pg1, first, rows_all;
    int64_t base;
    if (A.target) {  // (one unit a workgroup)
      GqaItem it;
      if (!gqa_plan_item<256, 1 << 30, false>(A, plan, static_cast<int>(u / A.kv_heads), it, first, rows_all, base)) return;
      unit.b = it.b;
      unit.pages = it.pg0;
      pg0 = it.parts;
    } else {
      const GqaSeq s(A.p, A.group, unit.b);
      first = s.first;
      rows_all = s.rows;
      base = s.base;
      pg0 = 0;
    }
    const GqaSeq s(A.p, A.group, first, rows_all, base);
    const int n_keys = s.rows > 0 ? s.seen(s.rows - 1) : 0, n_pages = (n_keys + kGqaKeys - 1) / kGqaKeys;
    const int each = A.target ? (n_pages + pg0 - 1) / pg0 : kSumPages;
    pg0 = unit.pages * each + wave;
    pg1 = min((unit.pages + 1) * each, n_pages);
    if (pg0 >= pg1) continue;
    const gqa_const_i32 table = (gqa_const_i32)(A.p.table + static_cast<int64_t>(unit.b) * A.p.max_pages);
    auto page_id = [&](int pg) { return __builtin_amdgcn_readfirstlane(table[min(pg, pg1 - 1)]); };
    auto there = [&](int id) { return id >= 0 && id < A.p.n_pages; };
    auto block = [&](int id) { return gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, there(id) ? id : 0, unit.head); };
    GqaQuery<D> q[RT];
    float lse2[RT];
    int seen[RT];
    auto rows = [&](int row0) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int row = row0 + 16 * r + c, at = min(row, s.rows - 1);
        q[r] = load_query<D>(A.q, A.q_stride, s, unit.head * A.group, row, g);
        lse2[r] = A.lse[(static_cast<int64_t>(s.first) + at / A.group) * A.heads + unit.head * A.group + at % A.group] * kLog2e;
        seen[r] = row < s.rows ? s.seen(row) : 0;
      }
    };
    rows(0);
    int pg = pg0;
    auto page = [&](const GqaKeys<D>& kc, float2 scales, bool is, int id) __attribute__((always_inline)) {
      const bool ok = gqa_scale_ok(scales.x) && gqa_scale_ok(scales.y);
      const float by = ok ? scales.x : 1.f, scale = ok ? A.scale : __builtin_nanf("");
      const int key0 = pg * kGqaKeys;
      float w[4][4] = {};
      for (int row0 = 0; row0 < s.rows; row0 += 16 * RT) {
        if (s.rows > 16 * RT) rows(row0);
        bool masked[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) masked[r] = __any(seen[r] - key0 - 16 * g < 16);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          v4f x[RT] = {};
#pragma unroll
          for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const v8bf k = codes8_bf16(kc.k[t][i][2 * e], kc.k[t][i][2 * e + 1], by);
#pragma unroll
              for (int r = 0; r < RT; ++r) x[r] = mfma_bf16(k, q[r].x[i][e], x[r]);
            }
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r][j], scale, -lse2[r]));
              w[t][j] += masked[r] && 4 * t + j >= seen[r] - key0 - 16 * g ? 0.f : p;
            }
        }
      }
      float mine = 0.f;  // over the 16 rows of a column: lane (c, g) keeps key 16 g + c
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = row16_reduce<false>(w[t][j]);
          mine = c == 4 * t + j ? x : mine;
        }
      if (is && key0 + lane < n_keys) {
        float* to = A.weights + (static_cast<int64_t>(id) * A.kv_heads + unit.head) * kGqaKeys + lane;
        *to = A.accumulate ? *to + mine : mine;
      }
    };
    // Two pages' keys on their way behind the one at work, 128 KB a CU.  (Three buffers by turns: one copied into another would
    // wait for its loads.)
    GqaKeys<D> k0, k1, k2;
    float2 s0, s1, s2;
    int id = page_id(pg), id1 = page_id(pg + 4), id2 = page_id(pg + 8);
    k0 = load_keys<D>(block(id).k, lane);
    s0 = load_scales(block(id).scale);
    k1 = load_keys<D>(block(id1).k, lane);
    s1 = load_scales(block(id1).scale);
    auto turn = [&](const GqaKeys<D>& now, float2 s_now, GqaKeys<D>& then, float2& s_then) __attribute__((always_inline)) {
      then = load_keys<D>(block(id2).k, lane);
      s_then = load_scales(block(id2).scale);
      page(now, s_now, there(id), id);
      id = id1;
      id1 = id2;
      id2 = page_id(pg + 12);
      pg += 4;
      return pg < pg1;
    };
    while (turn(k0, s0, k2, s2) && turn(k1, s1, k0, s0) && turn(k2, s2, k1, s1)) {
    }
  }
}

// Many rows: eight waves share PW pages of a head, each with a page's keys in registers as bf16, and 8 / PW tiles of 32 rows a
// step, which go through LDS as the product's operand (32 x 32 scores an instruction).  Waves of the same page are added
// at the end, in a fixed order.  Bound by vector instructions: a score takes a multiply-add, an exponential and a sum,
// 21 cycles a wave of 64 lanes, and 8 of the matrix pipe's: 2048 tokens over 16384 keys, 32 heads over 8 of 128 dims, 272 us.
constexpr int kSumWaves = 8;
template <int D, int PW>
struct GqaSumLds {
  static constexpr int KF = D / 16, RS = kSumWaves / PW;
  u32x4g q[2][RS][KF][64];
  float lse[2][RS][32];
  float part[kSumWaves][kGqaKeys];
};
template <int D, int PW>
__global__ __launch_bounds__(64 * kSumWaves, 2) void gqa_sum_kernel(const GqaSumArgs A) {
  constexpr int KF = D / 16, RS = kSumWaves / PW, CH = D / 8, ALL = RS * 32 * CH;      // 16-byte pieces of a row, and of a step
  constexpr int PIECES = (ALL + 64 * kSumWaves - 1) / (64 * kSumWaves);                // that a thread loads
  extern __shared__ __attribute__((aligned(16))) uint8_t gqa_smem[];
  GqaSumLds<D, PW>& L = *reinterpret_cast<GqaSumLds<D, PW>*>(gqa_smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5, pw = wave % PW, rs = wave / PW;
  for (int64_t u = blockIdx.x; u < A.units; u += gridDim.x) {
    const GqaUnit unit(A, u);
    const GqaSeq s(A.p, A.group, unit.b);
    const int n_keys = s.rows > 0 ? s.seen(s.rows - 1) : 0, first = unit.pages * PW * kGqaKeys;
    if (first >= n_keys) continue;  // (the whole workgroup)
    const int pg = unit.pages * PW + pw, key0 = pg * kGqaKeys;
    int id = -1;
    if (key0 < n_keys) id = __builtin_amdgcn_readfirstlane(A.p.table[static_cast<int64_t>(unit.b) * A.p.max_pages + pg]);
    const bool there = id >= 0 && id < A.p.n_pages;
    const GqaBlock blk = gqa_block<D>(A.pages, A.page_bytes, A.kv_heads, there ? id : 0, unit.head);
    const bool ok = gqa_scale_ok(blk.scale[0]) && gqa_scale_ok(blk.scale[1]);
    const float sk = ok ? blk.scale[0] : 1.f, scale = ok ? A.scale : __builtin_nanf("");
    // keys: fragment f of tile t, row c of it the key 32 (c / 4 % 2) + 16 t + 4 (c / 8) + c % 4, dims 64 i + 32 j + 16 h + 8 e .. + 7
    // for f = 4 i + 2 j + e; the queries' fragments are the same
    v8bf k[2][KF];
    {
      const uint8_t* from = blk.k + (32 * (c >> 2 & 1) + 4 * (c >> 3) + (c & 3)) * D + 16 * h;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int f = 0; f < KF / 2; ++f) {
          const u32x4g x = *reinterpret_cast<const u32x4g*>(from + 16 * t * D + 32 * f);
          k[t][2 * f] = codes8_bf16(x[0], x[1], sk);
          k[t][2 * f + 1] = codes8_bf16(x[2], x[3], sk);
        }
    }
    // rows below `none` see none of this wave's page, rows from `full` on all of it
    auto row_of = [&](int64_t pos) { const int64_t n = pos - s.base; return static_cast<int>(n <= 0 ? 0 : (n * s.group < s.rows ? n * s.group : s.rows)); };
    const int none = there ? row_of(key0) : s.rows, full = row_of(static_cast<int64_t>(key0) + kGqaKeys - 1);
    const int start = row_of(first) / (32 * RS) * (32 * RS), steps = (s.rows - start + 32 * RS - 1) / (32 * RS);
    auto token_of = [&](int row) { return static_cast<int>(row * A.per_group >> 34); };  // (a division is 30 instructions)
    float w[2][16] = {}, lse2 = 0.f;
    v16f x[2];
    auto row_at = [&](int step) { return start + step * 32 * RS + 32 * rs; };
    auto idle = [&](int row0) { return row0 + 32 <= none || row0 >= s.rows; };
    auto weights = [&](int row0) __attribute__((always_inline)) {
      if (row0 < full || row0 + 32 > s.rows) {
        const int row = row0 + c, my = row < s.rows ? s.seen(row) - key0 - 32 * h : 0;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][j], scale, -lse2));
            w[t][j] += 16 * t + j >= my ? 0.f : p;
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) w[t][j] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][j], scale, -lse2));
      }
    };
    struct Rows {
      u32x4g x[PIECES];
      float lse;
    };
    auto fetch = [&](int step) __attribute__((always_inline)) {
      Rows r;
      const int row0 = start + min(step, steps - 1) * 32 * RS;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int piece = i * 64 * kSumWaves + tid, at = min(row0 + piece / CH, s.rows - 1), t = token_of(at);
        r.x[i] = *reinterpret_cast<const u32x4g*>(A.q + (s.first + t) * A.q_stride + (unit.head * s.group + at - t * s.group) * D + piece % CH * 8);
      }
      r.lse = 0.f;
      if (tid < 32 * RS) {
        const int at = min(row0 + tid, s.rows - 1), t = token_of(at);
        r.lse = A.lse[(static_cast<int64_t>(s.first) + t) * A.heads + unit.head * s.group + at - t * s.group];
      }
      return r;
    };
    // (a piece's place is its row, turned by its fragment and half, so that a row's pieces are in different banks)
    auto stage = [&](const Rows& r, int buf) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int piece = i * 64 * kSumWaves + tid, row = piece / CH, j = piece % CH, f = 2 * (j >> 2) + (j & 1), half = j >> 1 & 1;
        if (ALL % (64 * kSumWaves) == 0 || piece < ALL) L.q[buf][row >> 5][f][32 * half + ((row & 31) ^ (2 * f + half))] = r.x[i];
      }
      if (tid < 32 * RS) L.lse[buf][tid >> 5][tid & 31] = r.lse * kLog2e;
    };
    auto tile = [&](int step, int buf) __attribute__((always_inline)) {
      if (idle(row_at(step))) return;
      lse2 = L.lse[buf][rs][c];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[0][j] = x[1][j] = 0.f;
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        const v8bf q = bf16_of(L.q[buf][rs][f][32 * h + (c ^ (2 * f + h))]);
        x[0] = mfma32_bf16(k[0][f], q, x[0]);
        x[1] = mfma32_bf16(k[1][f], q, x[1]);
      }
      weights(row_at(step));
    };
    // rows on their way for two steps (281 us for 2048 tokens over 16384 keys, 295 with one), or, where a step's take many
    // registers, for one
    Rows ra = fetch(0), rb;
    stage(ra, 0);
    if constexpr (RS <= 2) {
      rb = fetch(1);
      ra = fetch(2);
      __syncthreads();
#pragma unroll 1
      for (int step = 0; step < steps; step += 2) {
        tile(step, 0);
        stage(rb, 1);
        rb = fetch(step + 3);
        __syncthreads();
        if (step + 1 < steps) tile(step + 1, 1);
        stage(ra, 0);
        ra = fetch(step + 4);
        __syncthreads();
      }
    } else {
      ra = fetch(1);
      __syncthreads();
#pragma unroll 1
      for (int step = 0; step < steps; ++step) {
        tile(step, step & 1);
        stage(ra, (step & 1) ^ 1);
        ra = fetch(step + 2);
        __syncthreads();
      }
    }
    // over a half's 32 rows: lane (c, h) keeps key 32 h + c
    float mine = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float y = row16_reduce<false>(w[t][j]);
        const u32x2g z = __builtin_bit_cast(u32x2g, __builtin_amdgcn_permlane16_swap(__float_as_uint(y), __float_as_uint(y), false, false));
        const float sum = __uint_as_float(z[0]) + __uint_as_float(z[1]);
        mine = c == 16 * t + j ? sum : mine;
      }
    if constexpr (RS > 1) {
      L.part[wave][lane] = mine;
      __syncthreads();
      mine = L.part[pw][lane];
#pragma unroll
      for (int i = 1; i < RS; ++i) mine += L.part[pw + PW * i][lane];
    }
    if (there && rs == 0 && key0 + lane < n_keys) {
      float* to = A.weights + (static_cast<int64_t>(id) * A.kv_heads + unit.head) * kGqaKeys + lane;
      *to = A.accumulate ? *to + mine : mine;
    }
    __syncthreads();  // (the next unit's rows)
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
  if (!(softmax_scale > 0.f) || !(softmax_scale * kLog2e < INFINITY)) {  // (the kernels take it times log2 e; infinite, it makes a score of 0 NaN)
    set_error("%s: softmax_scale must be positive, and finite times log2(e)", who);
    return kErrArg;
  }
  return kOk;
}

extern "C" size_t tl_flash_paged_gqa_workspace_bytes(int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_pages) {
  if (n_seqs < 1 || n_tokens < 1 || kv_heads < 1 || heads < 1 || heads > 128 || heads % kv_heads || max_pages < 1 || n_seqs > (1ll << 16) ||
      max_pages > (1ll << 20) || n_tokens * heads >= kGqaMaxRows || (head_dim != 64 && head_dim != 128)) return 0;
  return gqa_launch(n_seqs, n_tokens, heads, kv_heads, head_dim, max_pages).bytes;
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
  const GqaLaunch d = gqa_launch(n_seqs, n_tokens, heads, kv_heads, head_dim, max_pages);
  if (d.bytes && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < d.bytes)) {
    set_error("%s: needs a workspace of %zu bytes, 16-byte aligned (got %zu)", who, d.bytes, workspace_bytes);
    return kErrArg;
  }
  if (d.wgs >= (1ll << 24)) {
    set_error("%s: %lld tokens, %lld sequences: more than a launch has room for", who, (long long)n_tokens, (long long)n_seqs);
    return kErrUnsupported;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const GqaArgs args{(const uint16_t*)q_bf16, q_stride, (const uint8_t*)kv_pages, gqa_page_bytes(kv_heads, head_dim),
                     PagedBatch{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens},
                     (int)heads, (int)kv_heads, (int)(heads / kv_heads), softmax_scale * kLog2e, (uint16_t*)out_bf16, lse,
                     (int)d.target, (int)d.at_once, reinterpret_cast<int2*>(ws), reinterpret_cast<float2*>(ws + d.ml_at), reinterpret_cast<float*>(ws + d.o_at)};
  const hipStream_t st = (hipStream_t)stream;
  auto join = [&](auto dim, auto bm, auto deep) -> int {
    constexpr int D = decltype(dim)::value, BM = decltype(bm)::value, DT = D / 16;
    if (!d.target) return kOk;
    hipLaunchKernelGGL((gqa_join_kernel<D, BM, decltype(deep)::value>), dim3(d.slots * kv_heads, BM / 16 * (decltype(deep)::value ? DT : cdiv(DT, kJoinWaves))),
                       dim3(64 * kJoinWaves), 0, st, args);
    return check_launch(who);
  };
  using std::integral_constant;
  auto few = [&](auto dim, auto rt) -> int {
    constexpr int D = decltype(dim)::value, RT = decltype(rt)::value;
    hipLaunchKernelGGL((gqa_attend_kernel<D, RT>), dim3(d.wgs), dim3(256), 0, st, args);
    if (int rc = check_launch(who)) return rc;
    return join(dim, integral_constant<int, 16 * RT>{}, std::true_type{});
  };
  auto many = [&](auto dim) -> int {
    constexpr int D = decltype(dim)::value, bytes = sizeof(GqaChunkLds<D>);
    const auto kern = gqa_chunk_kernel<D>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kern), bytes, who)) return rc;
    hipLaunchKernelGGL(kern, dim3(d.wgs), dim3(64 * kChunkWaves), bytes, st, args);
    if (int rc = check_launch(who)) return rc;
    return join(dim, integral_constant<int, kChunkRows>{}, std::false_type{});
  };
  auto by_rows = [&](auto dim) -> int {
    if constexpr (decltype(dim)::value == 64)
      if (d.bm == 64) return few(dim, integral_constant<int, 4>{});
    return d.bm == 16 ? few(dim, integral_constant<int, 1>{}) : (d.bm == 32 ? few(dim, integral_constant<int, 2>{}) : many(dim));
  };
  return head_dim == 64 ? by_rows(std::integral_constant<int, 64>{}) : by_rows(std::integral_constant<int, 128>{});
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
  const int64_t each = cdiv(n_tokens * (heads / kv_heads), n_seqs);
  const bool few = each <= 32;
  // Pages a workgroup: as many as leave most CUs one, by the table's width, which of many sequences fewer fill.  In us with 1, 2, 4
  // and 8, all with 64 heads over 8 of 128 dims: 32 tokens each of 2 sequences of 1500 keys 19 11 12 17; 2048 of 1 of 16384 928 709
  // 575 528; 1000 of 1 of 1000 63 93 152 264; 9 to 300 of 16 of 125 to 2000 98 68 72 91.  (The bound was set between these four.)
  int pw = 8;
  while (pw > 1 && cdiv(max_pages, pw) * kv_heads * n_seqs < std::min<int64_t>(128 + 32 * n_seqs, 768)) pw /= 2;
  // Pieces that few rows' pages are cut into: as many as run at once, or, where more than a few tiles may be of unlike
  // lengths, more.  In us with 512 / 1536: 1 sequence of 131072 keys 30 / 39, 8 of 4096 15 / 17, 16 of 1024 to 16384 33 / 38; 60 of 2048 to
  // 32768 183 / 161, with 4 heads of 64 dims 56 / 50.
  const int64_t target = few && n_seqs <= kGqaPlanSeqs ? (n_seqs * kv_heads <= 128 ? 512 : 1536) : 0;
  const int64_t groups = cdiv(max_pages, few ? kSumPages : pw), units = target ? target + n_seqs * kv_heads : n_seqs * groups * kv_heads;
  const GqaSumArgs args{(const uint16_t*)q_bf16, q_stride, lse, (const uint8_t*)kv_pages, gqa_page_bytes(kv_heads, head_dim),
                        PagedBatch{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens},
                        (int)heads, (int)kv_heads, (int)(heads / kv_heads), accumulate, softmax_scale * kLog2e, key_weights, (int)target, units, (int)groups,
                        ((1ull << 34) + heads / kv_heads - 1) / (heads / kv_heads)};
  const dim3 grid(target || units < (1 << 16) ? units : (1 << 16));  // (a workgroup goes on with another unit)
  const hipStream_t st = (hipStream_t)stream;
  if (few) {
    const auto kern = head_dim == 64 ? (each <= 16 ? gqa_sum_few_kernel<64, 1> : gqa_sum_few_kernel<64, 2>) :
                                       (each <= 16 ? gqa_sum_few_kernel<128, 1> : gqa_sum_few_kernel<128, 2>);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, args);
    return check_launch(who);
  }
  auto many = [&](auto dim, auto pages) -> int {
    constexpr int D = decltype(dim)::value, PW = decltype(pages)::value, bytes = sizeof(GqaSumLds<D, PW>);
    const auto kern = gqa_sum_kernel<D, PW>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kern), bytes, who)) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(64 * kSumWaves), bytes, st, args);
    return check_launch(who);
  };
  using std::integral_constant;
  auto by_pages = [&](auto dim) -> int {
    return pw == 8 ? many(dim, integral_constant<int, 8>{}) : (pw == 4 ? many(dim, integral_constant<int, 4>{}) :
           (pw == 2 ? many(dim, integral_constant<int, 2>{}) : many(dim, integral_constant<int, 1>{})));
  };
  return head_dim == 64 ? by_pages(integral_constant<int, 64>{}) : by_pages(integral_constant<int, 128>{});
}
