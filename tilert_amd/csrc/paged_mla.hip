// Causal MLA attention of a batch's new tokens over the paged latent cache (paged.h).  For token t of sequence b, at
// position p, and head h, over the keys j <= p:
//   s[j] = (q_nope[t,h] . latent[j] + q_pe[t,h] . rope[j]) * softmax_scale
//   out[t,h] = sum_j softmax(s)[j] latent[j],  lse[t,h] = ln sum_j e^s[j]      (0 and -inf where no key is seen)
//
// A sequence's rows (token, head), token-major, are cut into tiles of BM; a workgroup takes a tile through the
// sequence's pages, 64 keys a step.  The latents go into both products as the codes they are stored as, on the fp8
// MFMA; the other operand is split into two e4m3 numbers, x = hi + lo / 32:
//   q / sigma (sigma: a power of two that brings the row's largest magnitude into [128, 256)): exact for
//     values down to 2^-14 of the row's largest, below that within 2^-22 of it;
//   p * scale_j over a power of two that brings the largest of the row's 32 keys (one half of a page) into [128, 256), the
//     scale of that operand in the MFMA: within 2^-8 of the value, as bf16, down to 2^-14 of the largest, below that
//     within 2^-22 of it.  Nothing else sets that power: not the row's other keys, and no other row.
// Two fp8 products take the time of one in bf16, and no code is converted: with codes turned into bf16 the
// conversions alone (64 a page and wave for each product and 32 rows) would take as long as the products.
// Scores are U = scale_j * (codes . q / sigma) + (q_pe / sigma) . rope (bf16 MFMA), the exponent U * (sigma *
// softmax_scale * log2 e) - m; maxima, l and O are fp32.  Inside one instruction the fp8 MFMA adds eight consecutive products
// at a time, aligned to the largest and cut 13 bits below it, and those sums in fp32 (measured): a score's codes . q is
// within 2^-10 of the sum of each eight's largest product (512 random codes: 2^-16 of all products' magnitudes, rms; the lse's
// 1e-6 comes from it), and a page's part of O within 2^-10 of each eight keys' largest, beside the 2^-8 of P.
#include <math.h>

#include <type_traits>

#include "paged.h"
#include "../../include/tilert_amd.h"

namespace tl {

typedef uint32_t u32x4p __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2p __attribute__((ext_vector_type(2)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef short v2s __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef const __attribute__((address_space(4))) int32_t* const_i32;  // scalar loads

constexpr int kPagedWgs = 256;        // workgroups of a split launch: one per CU
// Tiles (and sequences) that a split launch plans in LDS; with more, a workgroup takes one and the last round of them is
// short against the others.  273 tiles, ragged: 177 us split, 230 not; 512 tiles of 225 to 256 pages, two for every
// workgroup: 979 split, 903 not; 1040 tiles (4160 tokens over 32768 keys), a few more than four: 3.97 ms split, 4.38 not.
constexpr int kPagedMaxTiles = 2048;
constexpr int64_t kPagedMaxRows = 1 << 27;  // (token, head) rows, fewer than this (PagedArgs::per_head)
// Pages that a sequence can have (a table's width), up to which no tile is split: one token, 16 heads, 500 keys take
// 13.6 us in one workgroup and 8.6 + 5.3 us over eight and with the join (14.0 and 15.5 us a call, and the second launch
// costs the host 4); from there on the page loop, 1.0 us a page, decides.
constexpr int kPagedFew = 8;
// Pages' time that a tile is counted for besides its pages, where a launch has many tiles: its queries' way into registers,
// the first scores, its results (18 thousand cycles at 64 rows, a page 3.4 thousand), rounded up for the tile that is cut in
// two.  Seven sequences of 2 to 700 new tokens, 273 tiles of 6 to 79 pages: 234 us without, 179 with 5, 175 with 10, 170
// with 18.  32 tiles of 25 to 256 pages (1 token, 128 heads, 8 sequences): 36.3 without, 33.3, 31.8, 32.4; 60 tiles: 101.2,
// 98.6, 101.7, 103.2.  A launch of at most kPagedWgs / 16 tiles has few workgroups with two of them, and does without: 2
// tiles of one sequence (4 tokens over 131072 keys) are 39.7 us, 43.9 with it, as the workgroups on the same pages of both
// are then no longer a multiple of 8, an XCD's L2, apart.
constexpr int kPagedStart = 10;
constexpr int kSlotBytes = kKvPageKeys * (kKvLatent + 2 * kKvRope);  // a page in LDS, its scales apart
constexpr int kSlots = 3;
constexpr int kPStride = 80;        // bytes of a P row of 64 codes: 8 rows' 16-byte pieces are in different banks
// A weight times key scale, in units of 1 / r (the row's largest when m and r were set, below 2 then), and a lane's sum of
// weights on a page, until m and r are set again: sums of 2^26 such times a code are far inside fp32's range.  The second is
// for keys whose scale is 0, or far below the row's others.
constexpr float kPMost = 0x1p40f;
constexpr int kScaleOne = 0x7f7f7f7f, kScaleLo = 0x7a7a7a7a;  // E8M0: 1, 2^-5

// Eight waves, two on a SIMD: 0 .. 3 score, 4 .. 7 multiply.  Scoring wave w takes the 16 rows of group w / KG against the
// 16 KT keys w % KG of a page and writes P; multiplying wave w takes P of all rows with 128 of the latent's dims.
// A SIMD's MFMA pipe always has the other wave's products while one wave turns scores into weights or waits for LDS, and
// either wave's registers (queries 72, or sums up to 128) fit without the other's.  With every wave doing both, the two
// waves of a SIMD stood at the same place of the step most of the time.
template <int BM_>
struct PagedCfg {
  static constexpr int BM = BM_;
  static constexpr int RG = BM / 16, KG = 4 / RG, KT = 4 / KG;
  static constexpr int RT2 = (BM + 31) / 32;     // 32-row tiles of the second product
  static constexpr int PR = RT2 * 32;            // rows of P in LDS
  // Keys of a P row that share a power of two: 32, a block of the MFMA.  With 16-row tiles a scoring wave has 16 keys and
  // would have to wait for another's, so its odd 16 keys take the P row 16 behind, which has no other use: each P row holds
  // every other 16 keys, with zeros between, and the two rows' sums are added at the end.
  static constexpr bool kTwoRows = BM == 16;
  static constexpr int BT = KT < 2 ? KT : 2;     // 16-key tiles of a block in a scoring wave
  static constexpr int SCALE_OFF = kSlots * kSlotBytes;
  static constexpr int P_OFF = SCALE_OFF + kSlots * kKvPageKeys * 4;
  static constexpr int P_BYTES = PR * kPStride;  // one of hi, lo of one buffer
  static constexpr int POW_OFF = P_OFF + 4 * P_BYTES;       // [2][32][2] u32: E8M0 of hi, lo of P rows n, n + 32; block
  static constexpr int STAT_OFF = POW_OFF + 2 * 32 * 2 * 4; // [3][KG][BM] f32
  static constexpr int ALPHA_OFF = STAT_OFF + 3 * KG * BM * 4;  // [BM] f32
  static constexpr int ROWL_OFF = ALPHA_OFF + BM * 4;       // [BM] f32
  static constexpr int UNIT_OFF = ROWL_OFF + BM * 4;        // [BM] f32
  static constexpr int FLAG_OFF = UNIT_OFF + BM * 4;        // [4] i32
  static constexpr int SCAN_OFF = FLAG_OFF + 16;            // [24] i32
  static constexpr int SEQ_OFF = SCAN_OFF + 96;             // [kPagedMaxTiles] i32: tiles up to sequence b and with it
  static constexpr int TILE_OFF = SEQ_OFF + kPagedMaxTiles * 4;  // [kPagedMaxTiles] i32: pages up to tile t and with it
  static constexpr int BYTES = TILE_OFF + kPagedMaxTiles * 4;
  static constexpr size_t kPartFloats = static_cast<size_t>(PR) * kKvLatent;
};
constexpr int kPagedThreads = 512;

// What bounds it.  Decode: bytes; 60 sequences, 60 to 32768 keys, 447 MB of pages and rows: 101 us a call, 4.4 TB/s (a large
// copy 4.7), 96 + 7.9 us in the two kernels.  Chunks: 2048 tokens, 16 heads over 16384 keys, 1.10 TFLOP: 0.95 to 0.98 ms,
// 1.12 to 1.16 PFLOP/s; a large bf16 product of the library reaches 1.39.  A step of 64 rows x 64 keys takes 3900 cycles, in
// which a SIMD's matrix pipe works for 2176.  Of 976 us a call 682 are left without the scoring waves' reads of the codes,
// 769 without the second product, 936 without turning the weights into P, 925 without fetches, partly by a higher
// clock, which gives way to the power drawn.  (Scoring waves of 32 rows would halve the reads; their queries' 144 registers
// leave too few: with reloads from scratch memory 1.8 ms.)  Small calls: the latency of plan, queries, pages and join, one
// behind another; 1 token over 500 keys 13.6 us in one kernel, of which seven pages' steps are 7.5.
// 32 rows' queries on their way into registers, in slot 2: hi codes [32][512], lo codes, rope parts bf16 [32][64]
constexpr int kQueryLo = 32 * kKvLatent, kQueryRope = 2 * kQueryLo;
static_assert(kQueryRope + 32 * kKvRope * 2 <= kSlotBytes, "");

// What a split launch leaves for the combine kernel, in the workspace: for every workgroup the tile that it
// continues, if it is the second on it; two slots of partial results a workgroup (0: of the tile that it continues, 1: of
// the tile that another one goes on with): (m, l) and the mean of the latents, whose sum may pass fp32's range.
struct SplitTile {
  int64_t row0;
  int rows, parts;
};

struct PagedArgs {
  const uint16_t* q_nope;
  const uint16_t* q_pe;
  const uint8_t* pages;
  PagedBatch p;
  int heads;
  uint64_t per_head;  // ceil(2^34 / heads): x / heads = x * per_head >> 34 for x < 2^34 / heads
  float scale;  // softmax_scale * log2 e
  uint16_t* out;
  float* lse;
  SplitTile* split;  // [kPagedWgs]; null: one workgroup a tile
  float2* part_ml;   // [2 kPagedWgs][PR]
  float* part_o;     // [2 kPagedWgs][kPartFloats]
  int tile_cap;      // tiles that the launch makes room for
  int start;         // pages' time that a tile takes before its first
};

// A sequence's row tiles and what they see, from untrusted metadata.
struct SeqRows {
  int first, n_rows;  // token, (token, head) rows
  int64_t base;       // position of the first token
  __device__ inline SeqRows(const PagedArgs& A, int b) {
    const int c0 = A.p.cu[b], c1 = A.p.cu[b + 1];
    first = min(max(c0, 0), A.p.n_tokens);
    n_rows = (min(max(c1, first), A.p.n_tokens) - first) * A.heads;
    base = static_cast<int64_t>(A.p.lens[b]) - c1 + first;
  }
  __device__ inline int tiles(int bm) const { return (n_rows + bm - 1) / bm; }
  // keys that the row'th row of the sequence sees
  __device__ inline int seen(const PagedArgs& A, int row) const {
    const int64_t n = base + static_cast<int>(row * A.per_head >> 34) + 1, most = static_cast<int64_t>(A.p.max_pages) * kKvPageKeys;  // <= 2^26
    return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
  }
  __device__ inline int pages(const PagedArgs& A, int tile, int bm) const {
    return (seen(A, min(n_rows, (tile + 1) * bm) - 1) + kKvPageKeys - 1) / kKvPageKeys;
  }
};

// Inclusive sum over the wave (row shifts, then the broadcasts of lanes 15 and 31).
__device__ inline int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}
// Inclusive sum over the workgroup's threads, and the total of all; `part` holds one int a wave.
__device__ inline int block_scan(int v, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  if (lane == 63) part[wave] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPagedThreads / 64; ++w) {
    const int x = part[w];
    before += w < wave ? x : 0;
    total += x;
  }
  __syncthreads();
  return v + before;
}

// Inclusive sums of two values at once and their totals; whether `no` is false everywhere.
__device__ inline bool block_scan2(int& a, int& b, bool no, int* part, int& total_a, int& total_b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  a = wave_scan(a);
  b = wave_scan(b);
  const bool any = __any(no);
  if (lane == 63) {
    part[wave] = a;
    part[8 + wave] = b;
    part[16 + wave] = any;
  }
  __syncthreads();
  int before_a = 0, before_b = 0, bad = 0;
  total_a = total_b = 0;
#pragma unroll
  for (int w = 0; w < kPagedThreads / 64; ++w) {
    const int x = part[w], y = part[8 + w];
    before_a += w < wave ? x : 0;
    before_b += w < wave ? y : 0;
    total_a += x;
    total_b += y;
    bad |= part[16 + w];
  }
  a += before_a;
  b += before_b;
  return !bad;
}

// The first index of an ascending array that is > x.
__device__ inline int upper(const int* a, int n, int x) {
  int lo = 0;
  while (n > 0) {
    const int h = n >> 1;
    if (a[lo + h] <= x) { lo += h + 1; n -= h + 1; }
    else n = h;
  }
  return lo;
}

// Max over the lanes i, i ^ 16, i ^ 32, i ^ 48, in all of them; the sums of lanes i and i ^ 16: a's in the lower of the two, b's
// in the upper.
__device__ inline float four_max(float v) {
  const u32x2p a = __builtin_bit_cast(u32x2p, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2p b = __builtin_bit_cast(u32x2p, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float pair_sum(float a, float b) {
  const u32x2p x = __builtin_bit_cast(u32x2p, __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false));
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

__device__ inline v4f mfma16_fp8(const v8i& a, const v8i& b, v4f c, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, kScaleOne, 0, scale_b);
}
// scale_b: byte SEL of the scale of b's column n, for the first 16 bytes of lanes n and n + 32 in lane n, for the others in lane
// n + 32.
template <int SEL>
__device__ inline v16f mfma32_fp8(const v8i& a, const v8i& b, v16f c, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, kScaleOne, SEL, scale_b);
}
__device__ inline v8i two_v4i(v4i a, v4i b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// N copies of 1 KB to LDS at `lds` and behind, from base + off[i] + 1024 i: lane l's 16 bytes go to its place in
// piece i.  The offset field moves both addresses, so m0 is written once; the copy of the base gives m0 its wait
// state, and the copies a base that no vector instruction has just written.
template <int N>
__device__ inline void dma_pieces(const uint8_t* base, const uint32_t (&off)[N], uint32_t lds) {
  static_assert(N == 2 || N == 4, "");
  uint32_t saved;
  uint64_t from;
  if constexpr (N == 4)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_mov_b64 %1, %3\n\tglobal_load_lds_dwordx4 %4, %1\n\t"
        "global_load_lds_dwordx4 %5, %1 offset:0x400\n\tglobal_load_lds_dwordx4 %6, %1 offset:0x800\n\t"
        "global_load_lds_dwordx4 %7, %1 offset:0xc00\n\ts_mov_b32 m0, %0"
        : "=&s"(saved), "=&s"(from) : "s"(lds), "s"(base), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]) : "memory");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_mov_b64 %1, %3\n\tglobal_load_lds_dwordx4 %4, %1\n\t"
        "global_load_lds_dwordx4 %5, %1 offset:0x400\n\ts_mov_b32 m0, %0"
        : "=&s"(saved), "=&s"(from) : "s"(lds), "s"(base), "v"(off[0]), "v"(off[1]) : "memory");
}
__device__ inline void dma_words(const uint8_t* base, uint32_t off, uint32_t lds) {  // 4 bytes a lane
  uint32_t saved;
  uint64_t from;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_mov_b64 %1, %3\n\tglobal_load_lds_dword %4, %1\n\ts_mov_b32 m0, %0"
               : "=&s"(saved), "=&s"(from) : "s"(lds), "s"(base), "v"(off) : "memory");
}

// Four values over a power of two as hi + lo / 32, four codes each; to_lo = the power / 32.
__device__ inline void split4(const float (&x)[4], float power, float to_lo, int& hi, int& lo) {
  v2s h = {0, 0}, l = {0, 0};
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, x[0], x[1], power, false);
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, x[2], x[3], power, true);
  hi = __builtin_bit_cast(int, h);
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, power, true);
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, x[0] - a[0], x[1] - a[1], to_lo, false);
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, x[2] - b[0], x[3] - b[1], to_lo, true);
  lo = __builtin_bit_cast(int, l);
}

// Four values (finite, <= 256 in magnitude, or NaN) as hi + lo / 32, four codes each.
__device__ inline void split4(const float (&x)[4], int& hi, int& lo) {
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], hi, true);
  const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 32.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 32.0f, true);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_fmaf(x[0], 32.0f, -a[0]), __builtin_fmaf(x[1], 32.0f, -a[1]), 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_fmaf(x[2], 32.0f, -b[0]), __builtin_fmaf(x[3], 32.0f, -b[1]), lo, true);
}

template <int BM>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_mla_kernel(const PagedArgs A) {
  using C = PagedCfg<BM>;
  constexpr int KG = C::KG, KT = C::KT, BT = C::BT, RT2 = C::RT2, DT = 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PagedBatch& p = A.p;
  int* seq_end = reinterpret_cast<int*>(smem + C::SEQ_OFF);
  int* unit_end = reinterpret_cast<int*>(smem + C::TILE_OFF);
  int* scan = reinterpret_cast<int*>(smem + C::SCAN_OFF);
  float* stat = reinterpret_cast<float*>(smem + C::STAT_OFF);
  float* alpha_l = reinterpret_cast<float*>(smem + C::ALPHA_OFF);
  float* rowl = reinterpret_cast<float*>(smem + C::ROWL_OFF);
  float* unit_l = reinterpret_cast<float*>(smem + C::UNIT_OFF);
  int* flag = reinterpret_cast<int*>(smem + C::FLAG_OFF);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8_ptr)smem));
  const int w = blockIdx.x;

  if constexpr (C::kTwoRows)  // the keys between a P row's own
    for (int i = tid; i < 4 * C::P_BYTES / 16; i += kPagedThreads) reinterpret_cast<v4i*>(smem + C::P_OFF)[i] = v4i{0, 0, 0, 0};

  // ---- the work of this workgroup
  int n_tiles = 0, u = 0, u_end = 1, quota = 1, tile = 0, seq = 0, seq_tile0 = 0;
  if (A.split) {
    // units are pages of tiles (a tile that sees nothing counts one) and A.start more a tile, in front of its pages; every
    // workgroup takes `quota` of them in a row
    int units;
    bool done = false;
    if (p.n_seqs <= kPagedThreads) {  // a decode step: where no sequence has two tiles, one pass does
      int tiles = 0, pages = 0;
      if (tid < p.n_seqs) {
        const SeqRows s(A, tid);
        tiles = min(s.tiles(BM), A.tile_cap);
        pages = tiles ? max(1, s.pages(A, 0, BM)) + A.start : 0;
      }
      int t = tiles, q = pages;
      done = block_scan2(t, q, tiles > 1, scan, n_tiles, units);
      n_tiles = min(n_tiles, A.tile_cap);
      if (tid < p.n_seqs) {
        seq_end[tid] = min(t, A.tile_cap);
        if (done && tiles && t <= A.tile_cap) unit_end[t - 1] = q;
      }
    } else {
      for (int b0 = 0; b0 < p.n_seqs; b0 += kPagedThreads) {
        const int b = b0 + tid;
        int total;
        const int t = block_scan(b < p.n_seqs ? min(SeqRows(A, b).tiles(BM), A.tile_cap) : 0, scan, total);
        if (b < p.n_seqs) seq_end[b] = min(n_tiles + t, A.tile_cap);
        n_tiles = min(n_tiles + total, A.tile_cap);
      }
    }
    __syncthreads();
    if (!done) {
      const int per = (n_tiles + kPagedThreads - 1) / kPagedThreads, t0 = tid * per, t1 = min(t0 + per, n_tiles);
      int sum = 0;
      if (t0 < t1) {
        int b = upper(seq_end, p.n_seqs, t0);
        SeqRows s(A, b);
        for (int t = t0; t < t1; ++t) {
          while (t >= seq_end[b]) s = SeqRows(A, ++b);
          sum += max(1, s.pages(A, t - (b ? seq_end[b - 1] : 0), BM)) + A.start;
          unit_end[t] = sum;
        }
      }
      const int before = block_scan(sum, scan, units) - sum;
      for (int t = t0; t < t1; ++t) unit_end[t] += before;
      __syncthreads();
    }
    if (done) units = n_tiles ? unit_end[n_tiles - 1] : 0;  // (as many tiles as there is room for)
    units = __builtin_amdgcn_readfirstlane(units);
    quota = max(1, (units + kPagedWgs - 1) / kPagedWgs);
    // the units at which the workgroup before, this one and the next begin: lanes 0, 1, 2
    int at = min((w - 1 + min(tid & 63, 2)) * quota, units);
    const int in = upper(unit_end, n_tiles, at);
    if (in < n_tiles) {
      const int first = in ? unit_end[in - 1] : 0;
      if (at <= first + A.start) at = first;  // all its pages
    }
    const int u_before = __builtin_amdgcn_readlane(at, 0);
    u = __builtin_amdgcn_readlane(at, 1);
    u_end = __builtin_amdgcn_readlane(at, 2);
    tile = __builtin_amdgcn_readlane(in, 1);
    if (tid == 0) {
      SplitTile info{0, 0, 0};
      if (u < u_end) {
        const int before = tile ? unit_end[tile - 1] : 0;
        if (before < u && u_before <= before) {  // the second workgroup on its first tile
          const int b = upper(seq_end, p.n_seqs, tile);
          const SeqRows s(A, b);
          const int j = tile - (b ? seq_end[b - 1] : 0);
          info.row0 = static_cast<int64_t>(s.first) * A.heads + static_cast<int64_t>(j) * BM;
          info.rows = min(BM, s.n_rows - j * BM);
          info.parts = (unit_end[tile] - 1) / quota - w + 2;  // those that begin inside it, and one
        }
      }
      A.split[w] = info;
    }
  } else {
    // one workgroup a tile: sequence b's are the workgroups from `before(b)` on, which leaves it as many as it has tiles
    auto before = [&](int b) { return min(max(p.cu[b], 0), p.n_tokens) * A.heads / BM + b; };
    seq = last_seq(p.n_seqs, [&](int b) { return before(b) <= w; });
    if (seq < 0 || seq >= p.n_seqs) return;
    seq_tile0 = before(seq);
    const int j = w - seq_tile0, last = SeqRows(A, seq).tiles(BM) - 1;
    if (j < 0 || j > last) return;  // (below 0 where cu_seqlens does not ascend)
    tile = seq_tile0 + last - j;  // the last tile, which sees the most, first
  }

  while (u < u_end) {
    // what follows from the lane is computed anew for each tile: taken out of this loop, it would fill the registers that
    // the products need
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int n16 = lane & 15, g = lane >> 4;
    const int n32 = lane & 31, half = lane >> 5;
    // ---- the tile: rows row0 .. row0 + rows - 1 of the call's (token, head) rows, pages pg0 .. pg0 + n - 1
    int tile_u0 = 0, tile_u1 = 1;
    if (A.split) {
      seq = upper(seq_end, p.n_seqs, tile);
      seq_tile0 = seq ? seq_end[seq - 1] : 0;
      tile_u0 = __builtin_amdgcn_readfirstlane(tile ? unit_end[tile - 1] : 0) + A.start;
      tile_u1 = __builtin_amdgcn_readfirstlane(unit_end[tile]);
      u = max(u, tile_u0);
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    seq_tile0 = __builtin_amdgcn_readfirstlane(seq_tile0);
    const SeqRows s(A, seq);
    const int j = tile - seq_tile0;
    const int in_seq = j * BM;
    const int64_t row0 = static_cast<int64_t>(s.first) * A.heads + in_seq;
    const int rows = min(BM, s.n_rows - in_seq);
    const int n_pages = s.pages(A, j, BM);
    const int seen_first = s.seen(A, in_seq);             // every row sees these
    const int pg0 = u - tile_u0;
    const int n = min(A.split ? min(tile_u1, u_end) - u : n_pages, n_pages - pg0);
    const const_i32 table = (const_i32)(p.table + static_cast<int64_t>(seq) * p.max_pages + pg0);

    // the page `id` into a slot, by the multiplying waves, in 1 KB pieces: 32 of codes, four at a time, and 8 of rope
    // parts; each also fetches the scales, all of them the same.  LDS has 64 banks of 4 bytes, 16 chunks of 16 bytes.  A row's
    // chunk c of codes is kept at c ^ turn(row), turn = (row & 7) << 1 | (row >> 3 & 1): 16 rows' chunk c is then in 16
    // places (a read of the scores), and so are the chunks 2 c and 2 c + 1 of 8 rows (a read of the values).  A chunk of a
    // rope part, two rows to the 64 banks, is kept at c ^ (row >> 1 & 7).
    auto valid = [&](int id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(p.n_pages); };
    auto fetch = [&](int id, int slot) {
      if (!valid(id)) id = 0;  // its keys are masked
      int at = lane;  // what follows from it is computed anew for each page: the products need the registers
      asm volatile("" : "+v"(at));
      const uint8_t* page = A.pages + static_cast<int64_t>(id) * kKvPageBytes;
      const uint32_t to = lds0 + slot * kSlotBytes;
      const int piece = (wave - 4) * 8;
      const uint32_t code = (at >> 5) * 512 + ((at & 31) ^ (at >> 5) * 2) * 16;  // rows 2 i, 2 i + 1 of piece i
      const uint32_t off[4] = {code, code ^ 64, code ^ 128, code ^ 192}, odd[4] = {code ^ 16, code ^ 80, code ^ 144, code ^ 208};
      dma_pieces<4>(page + piece * 1024, off, to + piece * 1024);
      dma_pieces<4>(page + piece * 1024 + 4096, odd, to + piece * 1024 + 4096);
      const uint32_t part = (at >> 3) * 128 + ((at & 7) ^ (at >> 4)) * 16;
      const uint32_t rope[2] = {part, part ^ 64};
      dma_pieces<2>(page + kKvRopeAt + piece * 256, rope, to + kKvPageKeys * kKvLatent + piece * 256);
      dma_words(page + kKvScaleAt, at * 4, lds0 + C::SCALE_OFF + slot * kKvPageKeys * 4);
    };
    // whether some row does not see all of page k; an id that is not valid is one whose keys nobody sees
    auto masked = [&](int k, int id) { return (pg0 + k + 1) * kKvPageKeys > seen_first || !valid(id); };
    auto id_of = [&](int k) { return table[min(k, n - 1)]; };
    // every wave's part of a fetch has arrived, and what it wrote to LDS is there
    auto arrive = [&] {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __syncthreads();
    };
    // a page's codes before a masked step: a NaN code would reach rows that do not see its key through 0 * NaN, so it
    // becomes 0 and the key's scale NaN
    auto clean = [&](int slot) {
      uint8_t* codes = smem + slot * kSlotBytes;
#pragma unroll 1
      for (int i = tid; i < kKvPageKeys * kKvLatent / 16; i += kPagedThreads) {
        v4i x = reinterpret_cast<v4i*>(codes)[i];
        uint32_t found = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          // bytes equal to 0x7f: adding 1 to a 7-bit value carries into bit 7 only from 0x7f
          const uint32_t nan = (((static_cast<uint32_t>(x[c]) & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
          found |= nan;
          x[c] &= ~static_cast<int>(nan * 0xffu);
        }
        if (found) {
          reinterpret_cast<v4i*>(codes)[i] = x;
          reinterpret_cast<float*>(smem + C::SCALE_OFF)[slot * kKvPageKeys + i / (kKvLatent / 16)] = __builtin_nanf("");
        }
      }
      __syncthreads();
    };

    __syncthreads();  // the slots, P and the statistics are free again
    if (tid < 4) flag[tid] = 0;

    // ---- the rows' queries as hi + lo / 32, through slot 2: 16 lanes a row, 32 rows a round.  Their loads are first, as
    // their wait would be for the pages too
    v8i qhi[4], qlo[4];
    v8bf qr[2];
    float f = 0.f;
    const int kg = wave % KG, rg = wave / KG;  // a scoring wave's keys and rows
    const int my_row = rg * 16 + n16;
    u32x4p raws[RT2][5];
    uint32_t largest[RT2];  // a row's largest magnitude's bits (bf16, upper half)
    const int place = wave * 4 + g;
#pragma unroll
    for (int round = 0; round < RT2; ++round) {
      const int r = round * 32 + place;
      const int64_t row = row0 + (r < rows ? r : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) raws[round][i] = reinterpret_cast<const u32x4p*>(A.q_nope + row * kKvLatent)[n16 + 16 * i];
      raws[round][4] = reinterpret_cast<const u32x4p*>(A.q_pe + row * kKvRope)[n16 & 7];
    }
#pragma unroll
    for (int round = 0; round < RT2; ++round) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 5; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) most = max(most, max(raws[round][i][c] & 0x7fff0000u, (raws[round][i][c] << 16) & 0x7fff0000u));
      largest[round] = row16_max_u32(most);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int id0 = n > 0 ? id_of(0) : 0, id1 = n > 0 ? id_of(1) : 0;
    if (wave >= 4) {
      if (n > 0) fetch(id0, 0);
      if (n > 1) fetch(id1, 1);
    }
#pragma unroll
    for (int round = 0; round < RT2; ++round) {
      const int r = round * 32 + place;
      const bool live = r < rows;
      const u32x4p (&raw)[5] = raws[round];
      const uint32_t most = largest[round];
      const bool bad = most >= 0x7f800000u;  // a NaN or an infinity: every output of the row is NaN
      const bool zero = bad || !live;
      const int e = zero ? 0 : max(static_cast<int>(most >> 23) - 127 - 7, -120);  // sigma = 2^e
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      uint8_t* to = smem + 2 * kSlotBytes;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v2i hi, lo;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t x0 = zero ? 0u : raw[i][2 * c], x1 = zero ? 0u : raw[i][2 * c + 1];
          const float v[4] = {__uint_as_float(x0 << 16) * inv, __uint_as_float(x0 & 0xffff0000u) * inv,
                              __uint_as_float(x1 << 16) * inv, __uint_as_float(x1 & 0xffff0000u) * inv};
          int a, b;
          split4(v, a, b);
          hi[c] = a;
          lo[c] = b;
        }
        const int at = place * kKvLatent + (((n16 >> 1) ^ (place & 7)) + 8 * i) * 16 + (n16 & 1) * 8;
        *reinterpret_cast<v2i*>(to + at) = hi;
        *reinterpret_cast<v2i*>(to + kQueryLo + at) = lo;
      }
      if (n16 < 8) {
        u32x4p x;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t y = zero ? 0u : raw[4][c];
          x[c] = bf16x2_bits(v2f{__uint_as_float(y << 16) * inv, __uint_as_float(y & 0xffff0000u) * inv});
        }
        *reinterpret_cast<u32x4p*>(to + kQueryRope + place * 128 + (n16 ^ (place & 7)) * 16) = x;
      }
      // (A bad row's factor is NaN, which makes its sum NaN.  Another's is not 0, which would make a masked score, -inf, NaN:
      // one below fp32's normal numbers stands for scores of 0, and 2^-126 does too.)
      if (n16 == 0 && r < BM)
        rowl[r] = bad && live ? __builtin_nanf("") : fmaxf(__uint_as_float(static_cast<uint32_t>(127 + e) << 23) * A.scale, 0x1p-126f);
      __syncthreads();
      if (wave < 4 && my_row / 32 == round) {
        const int q = my_row & 31;
        const uint8_t* from = smem + 2 * kSlotBytes + q * kKvLatent;
        const int c0 = ((2 * g) ^ (q & 7)) * 16;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          qhi[ks] = two_v4i(*reinterpret_cast<const v4i*>(from + c0 + ks * 128), *reinterpret_cast<const v4i*>(from + (c0 ^ 16) + ks * 128));
          qlo[ks] = two_v4i(*reinterpret_cast<const v4i*>(from + kQueryLo + c0 + ks * 128), *reinterpret_cast<const v4i*>(from + kQueryLo + (c0 ^ 16) + ks * 128));
        }
        const int r0 = kQueryRope + q * 128 + (g ^ (q & 7)) * 16;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) qr[ks] = *reinterpret_cast<const v8bf*>(smem + 2 * kSlotBytes + (r0 ^ (ks * 64)));
        f = rowl[my_row];
      }
      if (round + 1 < RT2) __syncthreads();
    }

    // ---- the pages.  Step k: the scoring waves make P of page k + 1, the others multiply that of page k; one barrier a
    // step, before which page k + 2 has arrived.  P is made with the maxima and s_ref that were set last; where a
    // weight would not fit (flag), every wave goes through settle() before it is used.
    if (wave < 4) {
      const int my_key = kg * KT * 16 + n16;       // and 16, 32, .. behind it
      const int my_quad = kg * KT * 16 + 4 * g;    // the keys of this lane's scores: my_quad .. +3, and 16, 32, ..
      const int at_code = my_key * kKvLatent + ((2 * g) ^ ((n16 & 7) << 1) ^ (n16 >> 3)) * 16;  // dims 32 g .. +15 (^ 16: +16 .. +31, ^ 128: 128 + 32 g ..)
      const int at_rope = kKvPageKeys * kKvLatent + my_key * 128 + (g ^ (n16 >> 1)) * 16;  // rope dims 8 g .. (^ 64: 32 + 8 g ..)
      const int p_row = C::kTwoRows ? my_row + 16 * (kg & 1) : my_row;
      const int put_p = p_row * kPStride + my_quad;
      const int put_pow = C::POW_OFF + ((p_row & 31) * 2 + kg * KT / 2) * 4 + (p_row >> 5) * 2;  // the wave's first block
      const int seen = my_row < rows ? s.seen(A, in_seq + my_row) : 0;
      // Weights are e = exp2(U * f - mk), mk = m: the row's largest U * f when it was last set (-300 where it has none).
      // P is e * scale * r; r = 1 / unit, a power of two of the row's largest e * scale when it was set.  l is the sum of such
      // e, O of P times codes.  m and r are set where the row's first keys are, and where a P or l would pass kPMost: both follow
      // from the row's own keys alone, and where they stay another row's change leaves the row's results as they were.
      float m = -INFINITY, mk = 0.f, l = f == f || seen == 0 ? 0.f : f, psum = 0.f, pmost = 0.f, r = 1.f;
      if (f != f) f = 0.f;
      v4f U[KT];

      auto weights_at = [&](int k) { return smem + C::P_OFF + (k & 1) * 2 * C::P_BYTES + put_p; };
      // A weight, times its key's scale and r, from its score; the largest and the sum so far.  (scale * r may pass fp32's
      // range where e is 0.)
      auto weigh = [&](float score, float scale, float& sum, float& most) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(score, f, -mk));
        sum += e;
        const float x = e * scale * r;
        most = fmaxf(most, __builtin_fabsf(x));
        return x;
      };
      // The P of block `b`'s weights, whose largest in this lane is `most`: over the power of two that brings the block's
      // largest into [128, 256) (2^-114 at least, far below what is left in a sum).
      auto put_block = [&](int k, int b, const float (&x)[BT][4], float most) {
        most = four_max(most);
        pmost = fmaxf(pmost, most);
        const uint32_t top = max(__float_as_uint(most) & 0x7f800000u, 20u << 23);
        uint8_t* P = weights_at(k);
#pragma unroll
        for (int i = 0; i < BT; ++i) {
          int hi, lo;
          split4(x[i], __uint_as_float(top - (7u << 23)), __uint_as_float(top - (12u << 23)), hi, lo);
          *reinterpret_cast<int*>(P + (b * BT + i) * 16) = hi;
          *reinterpret_cast<int*>(P + (b * BT + i) * 16 + C::P_BYTES) = lo;
        }
        const uint32_t e = top >> 23;  // (all four lanes of a row store it: a branch for one of them costs 2 % of a chunk's time)
        *reinterpret_cast<uint16_t*>(smem + put_pow + b * 4 + (k & 1) * 256) = static_cast<uint16_t>(e - 7 | (e - 12) << 8);
      };
      // U of page k, and with WEIGH its weights, whose tile of 16 keys is one behind that of the products: the wave issues
      // the vector instructions of the one while the matrix pipe works on the other.  Whether all weights were <= kPMost.
      // 4 KT items of 128 dims, each item's operand read ahead of its products.
      auto load_key = [&](int slot, int i) {
        const uint8_t* at = smem + slot * kSlotBytes + (i / 4) * 16 * kKvLatent + (i & 2) * 128;
        const int x = at_code ^ ((i & 1) * 128);
        return two_v4i(*reinterpret_cast<const v4i*>(at + x), *reinterpret_cast<const v4i*>(at + (x ^ 16)));
      };
      auto scores = [&](int k, int slot, auto weigh_tag) {
        constexpr bool WEIGH = decltype(weigh_tag)::value;
        constexpr int kItems = 4 * KT, kAhead = kItems < 4 ? kItems : 4;  // (6: 979 -> 990 us at 2048 tokens, 16 heads, 16384 keys)
        float most = 0.f, sum = 0.f;
        pmost = 0.f;
        float w[BT][4];
        v8i a[kItems];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) a[i] = load_key(slot, i);
        __builtin_amdgcn_sched_barrier(0);
        v4f x[KT], part[KT], sk[KT];  // of a tile: codes . q, rope . q, scales
#pragma unroll
        for (int kt = 0; kt <= KT; ++kt) {
          if (kt < KT) {
            sk[kt] = *reinterpret_cast<const v4f*>(smem + C::SCALE_OFF + (slot * kKvPageKeys + my_quad + kt * 16) * 4);
            x[kt] = part[kt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
              part[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  *reinterpret_cast<const v8bf*>(smem + slot * kSlotBytes + (at_rope ^ (ks * 64)) + kt * 16 * 128), qr[ks], part[kt], 0, 0, 0);
          }
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            if (kt < KT) {
              const int i = kt * 4 + ks;
              if (i + kAhead < kItems) a[i + kAhead] = load_key(slot, i + kAhead);
              x[kt] = mfma16_fp8(a[i], qhi[ks], x[kt], kScaleOne);
              x[kt] = mfma16_fp8(a[i], qlo[ks], x[kt], kScaleLo);
            }
            if (kt > 0) {
              // (an infinite scale as NaN: a score of -inf is a masked one)
              const float scale = __builtin_fmaf(sk[kt - 1][ks], 0.f, sk[kt - 1][ks]);
              U[kt - 1][ks] = __builtin_fmaf(x[kt - 1][ks], scale, part[kt - 1][ks]);
              if constexpr (WEIGH) w[(kt - 1) % BT][ks] = weigh(U[kt - 1][ks], scale, sum, most);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (WEIGH)
            if (kt > 0 && kt % BT == 0) {
              put_block(k, kt / BT - 1, w, most);
              most = 0.f;
            }
        }
        psum = sum;
        pmost = fmaxf(pmost, sum);
        return !__any(pmost > kPMost);
      };
      // the scores of page k that the row does not see
      auto mask_scores = [&](int k, int id) {
        const int at = (pg0 + k) * kKvPageKeys + my_quad, end = valid(id) ? seen : 0;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) U[kt][i] = at + kt * 16 + i < end ? U[kt][i] : -INFINITY;
      };

      // A key's scale, 0 where the row does not see it, whatever it holds.
      auto scale_seen = [&](int kt, int slot) {
        v4f sk = *reinterpret_cast<const v4f*>(smem + C::SCALE_OFF + (slot * kKvPageKeys + my_quad + kt * 16) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) sk[i] = U[kt][i] == -INFINITY ? 0.f : sk[i];
        return sk;
      };
      // The weights of page k from U where some are masked (-inf).
      auto weights = [&](int k, int slot) {
        float sum = 0.f;
        pmost = 0.f;
#pragma unroll
        for (int b = 0; b < KT / BT; ++b) {
          float w[BT][4], most = 0.f;
#pragma unroll
          for (int i = 0; i < BT; ++i) {
            const v4f sk = scale_seen(b * BT + i, slot);
#pragma unroll
            for (int c = 0; c < 4; ++c) w[i][c] = weigh(U[b * BT + i][c], sk[c], sum, most);
          }
          put_block(k, b, w, most);
        }
        psum = sum;
        pmost = fmaxf(pmost, sum);
        return !__any(pmost > kPMost);
      };

      auto one_over = [](float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); };
      // New m and r from page k's scores and scales for the rows that need them, O and l brought to them, P again.  Every wave
      // comes here, or none.
      auto settle = [&](int k, int slot) {
        float x = -INFINITY, over = four_max(pmost);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) x = fmaxf(x, fmaxf(fmaxf(U[kt][0], U[kt][1]), fmaxf(U[kt][2], U[kt][3])));
        x = four_max(x);
        if constexpr (KG > 1) {
          if (g == 0) {
            stat[kg * BM + my_row] = x;
            stat[(KG + kg) * BM + my_row] = over;
          }
          __syncthreads();
#pragma unroll
          for (int i = 0; i < KG; ++i) {
            x = fmaxf(x, stat[i * BM + my_row]);
            over = fmaxf(over, stat[(KG + i) * BM + my_row]);
          }
        }
        const bool none = m == -INFINITY, set = none || over > kPMost;
        const float was = mk;
        if (set) {
          m = fmaxf(m, x == -INFINITY ? -INFINITY : x * f);
          mk = m == -INFINITY ? -300.f : m;
        }
        const float alpha = none ? 0.f : __builtin_amdgcn_exp2f(was - mk);
        // the row's largest weight times scale on this page
        float top = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const v4f sk = scale_seen(kt, slot);
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fabsf(__builtin_amdgcn_exp2f(__builtin_fmaf(U[kt][i], f, -mk)) * sk[i]));
        }
        top = four_max(top);
        if constexpr (KG > 1) {
          if (g == 0) stat[(2 * KG + kg) * BM + my_row] = top;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < KG; ++i) top = fmaxf(top, stat[(2 * KG + i) * BM + my_row]);
        }
        const float unit = one_over(r);
        if (set) r = __uint_as_float((254u << 23) - min(max(__float_as_uint(fmaxf(top, alpha * unit)) & 0x7f800000u, 27u << 23), 253u << 23));
        l *= alpha;
        if (kg == 0 && g == 0) alpha_l[my_row] = alpha * r * unit;  // (in this order: no factor of it passes fp32's range)
        weights(k, slot);
        __syncthreads();
      };

      if (n > 0) {
        arrive();
        if (masked(0, id0)) clean(0);
        scores(0, 0, std::false_type{});
        if (masked(0, id0)) mask_scores(0, id0);
        settle(0, 0);
        int next = 1, free = 2, slot = 0, id = id1, id_after = id_of(2);
        bool fresh = !valid(id0);  // no page so far had keys: nothing is set yet
#pragma unroll 1
        for (int k = 0; k + 1 < n; ++k) {  // id: page k + 1's
          l += psum;
          if (tid == 0) flag[(k + 2) & 3] = tid;  // (0, without a register that holds it)
          bool fits;
          if (masked(k + 1, id)) {
            clean(next);
            scores(k + 1, next, std::false_type{});
            mask_scores(k + 1, id);
            fits = weights(k + 1, next);
          } else {
            fits = scores(k + 1, next, std::true_type{});
          }
          if ((!fits || fresh) && lane == 0) flag[(k + 1) & 3] = 1;
          fresh = fresh && !valid(id);
          arrive();
          if (flag[(k + 1) & 3]) settle(k + 1, next);
          id = id_after;
          id_after = id_of(k + 3);
          const int was = slot;
          slot = next;
          next = free;
          free = was;
        }
        l += psum;
      }
      // l over the lanes and waves of a row
      __syncthreads();
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      if (g == 0) {
        stat[kg * BM + my_row] = l;
        if (kg == 0) {
          alpha_l[my_row] = m == -INFINITY ? -INFINITY : mk;
          unit_l[my_row] = one_over(r);
        }
      }
      __syncthreads();
      if (tid < BM) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < KG; ++i) x += stat[i * BM + tid];
        rowl[tid] = x;
      }
      __syncthreads();
    } else {
      const int dw = wave - 4;  // dims 128 dw ..
      const int at_value = (16 * half + (n16 >> 1)) * kKvLatent + (dw & 2) * 128 + (lane & 1) * 8 +
                           ((8 * (dw & 1) + (g & 1)) ^ (n16 & 14)) * 16;  // 32-dim tile d: ^ 32 d; keys 8 .. 15 behind it: ^ 16
      const int at_p = n32 * kPStride + half * 16;
      const int at_pow = C::POW_OFF + (n32 * 2 + half) * 4;
      v16f o[RT2][DT];
#pragma unroll
      for (int a = 0; a < RT2; ++a)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[a][d][i] = 0.f;

      // O^T += latent^T P^T of page k: rows of A are dims, of B the tile's rows, 64 keys in one MFMA, whose two scale blocks are
      // the page's halves: lane (n32, half) holds keys 16 half .. +15 of the one and of the other.  A lane's dim is
      // a column of the key-major codes: ds_read_b64_tr_b8 gives lane i of a 16-lane group byte i % 8 of the 8 bytes at
      // lane 2 j + i / 8's address as its byte j, so lane i addresses key 32 (r / 2) + 16 half + 8 (r % 2) + i / 2, half
      // i % 2 of the group's 16-dim chunk, and receives 8 keys of dim i.
      auto product = [&](int k, int slot) {
        const uint8_t* P = smem + C::P_OFF + (k & 1) * 2 * C::P_BYTES + at_p;
        const int at = slot * kSlotBytes + at_value;  // (a slot's place leaves bits 4 .. 8 alone)
        auto load_value = [&](int d) {
          v8i v;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const v2i x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(smem + (at ^ (32 * d + 16 * (r & 1))) + ((r >> 1) * 32 + (r & 1) * 8) * kKvLatent));
            v[2 * r] = x[0];
            v[2 * r + 1] = x[1];
          }
          return v;
        };
        v8i v[2], ph[RT2], pl[RT2];
        v[0] = load_value(0);
#pragma unroll
        for (int a = 0; a < RT2; ++a) {
          const v4i* hi = reinterpret_cast<const v4i*>(P + a * 32 * kPStride);
          const v4i* lo = reinterpret_cast<const v4i*>(P + a * 32 * kPStride + C::P_BYTES);
          ph[a] = two_v4i(hi[0], hi[2]);
          pl[a] = two_v4i(lo[0], lo[2]);
        }
        const int pow = *reinterpret_cast<const int*>(smem + at_pow + (k & 1) * 256);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (d + 1 < DT) v[(d + 1) & 1] = load_value(d + 1);
          __builtin_amdgcn_sched_barrier(0);
          o[0][d] = mfma32_fp8<0>(v[d & 1], ph[0], o[0][d], pow);
          o[0][d] = mfma32_fp8<1>(v[d & 1], pl[0], o[0][d], pow);
          if constexpr (RT2 > 1) {
            o[1][d] = mfma32_fp8<2>(v[d & 1], ph[1], o[1][d], pow);
            o[1][d] = mfma32_fp8<3>(v[d & 1], pl[1], o[1][d], pow);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto settle = [&](bool first) {
        if constexpr (KG > 1) {
          __syncthreads();
          __syncthreads();
        }
        __syncthreads();
        if (first) return;  // (nothing to bring along)
#pragma unroll
        for (int a = 0; a < RT2; ++a) {
          const float x = alpha_l[(a * 32 + n32) & (BM - 1)];
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[a][d][i] *= x;
        }
      };

      if (n > 0) {
        arrive();
        if (masked(0, id0)) clean(0);
        settle(true);
        int next = 1, free = 2, slot = 0, id = id1, id_after = id_of(2);
#pragma unroll 1
        for (int k = 0; k + 1 < n; ++k) {  // id: page k + 1's
          if (k + 2 < n) fetch(id_after, free);
          if (masked(k + 1, id)) clean(next);
          id = id_after;
          id_after = id_of(k + 3);
          product(k, slot);
          arrive();
          if (flag[(k + 1) & 3]) settle(false);
          const int was = slot;
          slot = next;
          next = free;
          free = was;
        }
        product(n - 1, slot);
        // P rows r and r + 16 together: groups of 8 dims 2 i in lanes n32 = r, 2 i + 1 in lanes r + 16
        if constexpr (C::kTwoRows)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[0][d][i] = pair_sum(o[0][d][i / 4 * 8 + i % 4], o[0][d][i / 4 * 8 + 4 + i % 4]);
      }
      constexpr int kGroups = C::kTwoRows ? 2 : 4;  // of a lane's groups of 8 dims in 32
      const int row_in = C::kTwoRows ? n16 : n32;
      auto group = [&](int i) { return C::kTwoRows ? 2 * i + (g & 1) : i; };
      __syncthreads();
      __syncthreads();
      __syncthreads();

      // ---- the rows' results, or the tile's partial ones
      if (!A.split || (u == tile_u0 && u_end >= tile_u1)) {
        const int t = tid - 256;
        if (A.lse && t < rows) A.lse[row0 + t] = rowl[t] == 0.f ? -INFINITY : (alpha_l[t] + log2f(rowl[t])) * 0.6931471805599453f;
#pragma unroll
        for (int a = 0; a < RT2; ++a) {
          const int r = a * 32 + row_in;
          if (r < rows) {
            const float L = rowl[r], x = L == 0.f ? 0.f : 1.0f / L * unit_l[r];
            uint16_t* dst = A.out + (row0 + r) * kKvLatent + dw * 128 + 4 * half;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int i = 0; i < kGroups; ++i)
                *reinterpret_cast<u32x2p*>(dst + d * 32 + 8 * group(i)) = u32x2p{bf16x2_bits(v2f{o[a][d][4 * i] * x, o[a][d][4 * i + 1] * x}),
                                                                         bf16x2_bits(v2f{o[a][d][4 * i + 2] * x, o[a][d][4 * i + 3] * x})};
          }
        }
      } else {
        const int slot = 2 * w + (u == tile_u0 ? 1 : 0), t = tid - 256;
        if (t < rows) A.part_ml[static_cast<int64_t>(slot) * C::PR + t] = float2{alpha_l[t], rowl[t]};
        v4f* dst = reinterpret_cast<v4f*>(A.part_o + static_cast<int64_t>(slot) * C::kPartFloats);
#pragma unroll
        for (int a = 0; a < RT2; ++a)
          if (a * 32 + row_in < rows) {
            const float L = rowl[a * 32 + row_in], x = L == 0.f ? 0.f : 1.0f / L * unit_l[a * 32 + row_in];
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int i = 0; i < kGroups; ++i)
                dst[((a * 16 + dw * DT + d) * 4 + group(i)) * 64 + half * 32 + row_in] =
                    v4f{o[a][d][4 * i], o[a][d][4 * i + 1], o[a][d][4 * i + 2], o[a][d][4 * i + 3]} * x;
          }
      }
    }
    if (!A.split) return;
    u = min(tile_u1, u_end);
    ++tile;
  }
}

// The split tiles' partial means joined, in a fixed order, each weighted by its share of l.  An item is 32 rows x 64 / G
// dims of a tile: a thread takes one row, 4 dims and every G'th part, so that it has few parts (up to eight, all their
// loads in flight together; a context split over all workgroups: sixteen), and the G half-waves of the same dims are joined
// in LDS.  Bound by round trips (the tiles, then the parts, which other XCDs wrote) where few tiles are split, and by the
// parts' bytes where many are: 256 parts of 32 rows, 17 MB, 9 us; 495 of 64, 65 MB, 21 us.  Four workgroups a CU: 60
// sequences 101.2 us a call, 102.6 with two; sixteen do no better.
constexpr int kCombineWgs = 1024, kCombineThreads = 512, kHalfWaves = kCombineThreads / 32;
__device__ inline int part_groups(int parts) { return parts <= 8 ? 1 : (parts <= 16 ? 2 : (parts <= 32 ? 4 : (parts <= 64 ? 8 : 16))); }
template <int PR>
__global__ __launch_bounds__(kCombineThreads) void paged_mla_combine_kernel(const SplitTile* __restrict__ split,
                                                                            const float2* __restrict__ part_ml,
                                                                            const float* __restrict__ part_o,
                                                                            uint16_t* __restrict__ out, float* __restrict__ lse) {
  __shared__ int item_end[kPagedWgs], count[4];
  __shared__ float top[kHalfWaves][32], sums[kHalfWaves][32];
  __shared__ v4f acc[kHalfWaves][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  static_assert(kPagedWgs == 256, "four waves' scan");
  const int parts = tid < kPagedWgs ? split[tid].parts : 0;
  const int mine = wave_scan(parts < 2 ? 0 : (PR / 32) * 8 * part_groups(parts));
  if (lane == 63 && wave < 4) count[wave] = mine;
  __syncthreads();
  const int e0 = count[0], e1 = e0 + count[1], e2 = e1 + count[2], total = e2 + count[3];
  if (static_cast<int>(blockIdx.x) >= total) return;
  if (wave < 4) item_end[tid] = mine + (wave == 0 ? 0 : (wave == 1 ? e0 : (wave == 2 ? e1 : e2)));
  __syncthreads();
  const int n32 = tid & 31, hw = tid >> 5;
  // part i of the tile that workgroup w continues: workgroup w - 1's slot 1, then the slots 0 of w, w + 1, ...
  auto slot_of = [](int w, int i) -> int64_t { return i ? 2 * (w + i - 1) : 2 * w - 1; };
  auto sums_at = [&](int64_t slot, int a, int d4) {  // dims 4 d4 .. +3: 32-dim tile d4 / 8, group (d4 % 8) / 2 of 8 dims, half d4 % 2
    return reinterpret_cast<const v4f*>(part_o + slot * (static_cast<int64_t>(PR) * kKvLatent))[((a * 16 + d4 / 8) * 4 + (d4 % 8) / 2) * 64 + (d4 & 1) * 32 + n32];
  };
  auto store = [&](int64_t row, int d4, const v4f& o, float l, float mx) {
    *reinterpret_cast<u32x2p*>(out + row * kKvLatent + 4 * d4) = u32x2p{bf16x2_bits(v2f{o[0], o[1]}), bf16x2_bits(v2f{o[2], o[3]})};
    if (lse && d4 == 0) lse[row] = l == 0.f ? -INFINITY : (mx + log2f(l)) * 0.6931471805599453f;
  };
  // N parts i0, i0 + step, .. below `end`, added to (mx, l, o); their loads are all in flight together
  auto add = [&](auto count_tag, int w, int a, int d4, int r, int i0, int step, int end, float& mx, float& l, v4f& o) {
    constexpr int N = decltype(count_tag)::value;
    float2 ml[N];
    v4f x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t slot = slot_of(w, min(i0 + i * step, end - 1));
      ml[i] = part_ml[slot * PR + r];
      x[i] = sums_at(slot, a, d4);
    }
    float top = mx;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, i0 + i * step < end ? ml[i].x : -INFINITY);
    const float kept = mx == -INFINITY ? l : l * __builtin_amdgcn_exp2f(mx - top);  // (0, or a bad row's NaN, before the first)
    float share[N];
    l = kept;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      share[i] = i0 + i * step >= end ? 0.f : (ml[i].x == -INFINITY ? ml[i].y : ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - top));
      l += share[i];
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    o *= kept * inv;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i0 + i * step < end) o += x[i] * (share[i] * inv);
    mx = top;
  };
  for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const int w = upper(item_end, kPagedWgs, item);
    const SplitTile t = split[w];
    const int groups = part_groups(t.parts), dims = kHalfWaves / groups;  // float4s of dims an item
    const int at = item - (w ? item_end[w - 1] : 0), items = 8 * groups;    // items of 32 rows
    const int a = at / items, d4 = at % items * dims + hw % dims, part0 = hw / dims, r = a * 32 + n32;
    const bool live = r < t.rows;
    float mx = -INFINITY, l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
    if (live) {
      const int each = (t.parts + groups - 1) / groups;
      if (each <= 2) add(std::integral_constant<int, 2>{}, w, a, d4, r, part0, groups, t.parts, mx, l, o);
      else if (each <= 4) add(std::integral_constant<int, 4>{}, w, a, d4, r, part0, groups, t.parts, mx, l, o);
      else
#pragma unroll 1
        for (int i = part0; i < t.parts; i += 8 * groups)
          add(std::integral_constant<int, 8>{}, w, a, d4, r, i, groups, t.parts, mx, l, o);
    }
    if (groups > 1) {
      top[hw][n32] = mx;
      sums[hw][n32] = l;
      acc[hw][n32] = o;
      __syncthreads();
      if (part0 == 0 && live) {
        for (int i = hw + dims; i < kHalfWaves; i += dims) mx = fmaxf(mx, top[i][n32]);
        auto share = [&](int i) { return top[i][n32] == -INFINITY ? sums[i][n32] : sums[i][n32] * __builtin_amdgcn_exp2f(top[i][n32] - mx); };
        l = 0.f;
        for (int i = hw; i < kHalfWaves; i += dims) l += share(i);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        o = v4f{0.f, 0.f, 0.f, 0.f};
        for (int i = hw; i < kHalfWaves; i += dims) o += acc[i][n32] * (share(i) * inv);
      }
      __syncthreads();
    }
    if (part0 == 0 && live) store(t.row0 + r, d4, o, l, mx);
  }
}

// The launch: rows a tile, whether tiles are split, and the workspace.  More rows a tile read a page for more rows at
// once, and for 64 rows both 32-row products of a multiplying wave share its read of the page; fewer rows have their
// queries split and their sums written in less time and waste less where a sequence's rows end.  Measured, for the rows
// that a sequence has on average, in us with 16 / 32 / 64 rows a tile:
//   16 rows (1 sequence, 500 keys)                         13.9 / 14.7 / 21.7
//   17 rows (60 sequences of 60 to 32768 keys, padded)     100.9 / 101.4 / 116.5
//   64 rows (4 tokens, 16 heads, 131072 keys)              49.4 / 38.8 / 41.7
//   128 rows (8 sequences of 1589 to 16384 keys)           40.6 / 31.5 / 35.5
//   2471 rows (7 sequences of 2 to 700 new tokens)         322 / 181 / 175
struct PagedPlan {
  int bm, pr;
  int64_t tiles;  // of a split launch, at most
  bool split;
  size_t ml_at, o_at, bytes;
};
inline PagedPlan paged_plan(int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t max_pages) {
  PagedPlan d{};
  const int64_t rows = n_tokens * heads, each = cdiv(rows, n_seqs);
  d.bm = each <= 16 ? 16 : (each <= 128 ? 32 : 64);
  d.pr = d.bm < 32 ? 32 : d.bm;
  d.tiles = rows / d.bm + (n_seqs < n_tokens ? n_seqs : n_tokens);
  // (units and the end of the last workgroup's share of them, up to kPagedWgs behind, are ints)
  d.split = d.tiles <= kPagedMaxTiles && n_seqs <= kPagedMaxTiles && max_pages > kPagedFew &&
            d.tiles * (max_pages + kPagedStart) <= INT32_MAX - kPagedWgs;
  if (d.split) {
    d.ml_at = kPagedWgs * sizeof(SplitTile);
    d.o_at = d.ml_at + static_cast<size_t>(2 * kPagedWgs) * d.pr * sizeof(float2);
    d.bytes = d.o_at + static_cast<size_t>(2 * kPagedWgs) * d.pr * kKvLatent * sizeof(float);
  }
  return d;
}

}  // namespace tl

using namespace tl;

extern "C" size_t tl_flash_paged_mla_workspace_bytes(int64_t n_seqs, int64_t n_tokens, int64_t heads, int64_t max_pages) {
  if (n_seqs < 1 || n_tokens < 1 || heads < 1 || heads > 128 || n_seqs > (1ll << 20) || n_tokens * heads >= kPagedMaxRows) return 0;
  return paged_plan(n_seqs, n_tokens, heads, max_pages).bytes;
}

extern "C" int tl_flash_paged_mla(const void* q_nope_bf16, const void* q_pe_bf16, const void* kv_pages, int64_t n_pages,
                                  const int32_t* block_table, int64_t max_pages, const int32_t* cu_seqlens,
                                  const int32_t* seq_lens, int64_t n_seqs, int64_t n_tokens, int64_t heads,
                                  float softmax_scale, void* out_bf16, float* lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_batch("flash_paged_mla", kv_pages, n_pages, block_table, max_pages, cu_seqlens, seq_lens, n_seqs, n_tokens)) return rc;
  if (heads < 1 || heads > 128) { set_error("flash_paged_mla: heads=%lld must be in [1, 128]", (long long)heads); return kErrUnsupported; }
  if (n_seqs == 0 || n_tokens == 0) return kOk;
  if (n_tokens * heads >= kPagedMaxRows || n_seqs > (1ll << 20) || max_pages > (1ll << 20)) {
    set_error("flash_paged_mla: %lld tokens x %lld heads, %lld sequences, %lld pages a sequence: fewer than 2^27 rows, up to 2^20 "
              "sequences and 2^20 pages", (long long)n_tokens, (long long)heads, (long long)n_seqs, (long long)max_pages);
    return kErrUnsupported;
  }
  if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY)) { set_error("flash_paged_mla: softmax_scale must be positive and finite"); return kErrArg; }
  if (!q_nope_bf16 || !q_pe_bf16 || !out_bf16) { set_error("flash_paged_mla: null pointer"); return kErrArg; }
  if ((reinterpret_cast<uintptr_t>(q_nope_bf16) | reinterpret_cast<uintptr_t>(q_pe_bf16) | reinterpret_cast<uintptr_t>(out_bf16) |
       reinterpret_cast<uintptr_t>(workspace)) & 15) {
    set_error("flash_paged_mla: q, out and workspace must be 16-byte aligned");
    return kErrArg;
  }
  const PagedPlan d = paged_plan(n_seqs, n_tokens, heads, max_pages);
  if (d.bytes && (!workspace || workspace_bytes < d.bytes)) {
    set_error("flash_paged_mla: needs a workspace of %zu bytes (got %zu)", d.bytes, workspace_bytes);
    return kErrArg;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const PagedArgs args{(const uint16_t*)q_nope_bf16, (const uint16_t*)q_pe_bf16, (const uint8_t*)kv_pages,
                       PagedBatch{block_table, cu_seqlens, seq_lens, (int)n_seqs, (int)max_pages, (int)n_pages, (int)n_tokens},
                       (int)heads, ((1ull << 34) + heads - 1) / heads, softmax_scale * 1.4426950408889634f, (uint16_t*)out_bf16, lse,
                       d.split ? reinterpret_cast<SplitTile*>(ws) : nullptr, reinterpret_cast<float2*>(ws + d.ml_at),
                       reinterpret_cast<float*>(ws + d.o_at), (int)(d.split ? d.tiles : 0), d.split && d.tiles > kPagedWgs / 16 ? kPagedStart : 0};
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto bm) -> int {
    using C = PagedCfg<decltype(bm)::value>;
    const auto kern = paged_mla_kernel<decltype(bm)::value>;
    if (int rc = allow_dynamic_lds(reinterpret_cast<const void*>(kern), C::BYTES, "flash_paged_mla")) return rc;
    hipLaunchKernelGGL(kern, dim3(d.split ? kPagedWgs : static_cast<unsigned>(n_tokens * heads / d.bm + n_seqs)), dim3(kPagedThreads), C::BYTES, st, args);
    if (int rc = check_launch("flash_paged_mla")) return rc;
    if (!d.split) return kOk;
    hipLaunchKernelGGL((paged_mla_combine_kernel<C::PR>), dim3(kCombineWgs), dim3(kCombineThreads), 0, st, args.split, args.part_ml, args.part_o, args.out, lse);
    return check_launch("flash_paged_mla");
  };
  using std::integral_constant;
  if (d.bm == 16) return launch(integral_constant<int, 16>{});
  if (d.bm == 32) return launch(integral_constant<int, 32>{});
  return launch(integral_constant<int, 64>{});
}
