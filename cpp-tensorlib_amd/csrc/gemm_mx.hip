// Products of MXFP8 rows over MXFP4 weights, in tiles: prompt chunks, plain, as the parts of a split K, and with the gated activation whose
// result is MXFP8 again (mx_mfma.hpp has the arithmetic).
#include "mx_mfma.hpp"

#include <algorithm>
#include <initializer_list>

namespace tlhip {

// ---- tiles: many rows ---------------------------------------------------------------------------------------------
// WF x WT wavefronts, each NF x NT tiles of 16 features by 16 tokens. A step is 128 k: the rows' bytes and scales go from memory into LDS
// by copies, a step ahead; 16-byte chunks of a row are swizzled on the memory side of the copy, so that the lanes an LDS read
// serves together find different banks. A row's four scale bytes of a step are one word, which a lane shifts down to its own block's.
// WORDS: that word is a whole one in memory, too (K % 128 == 0, so that no step ends past a row); elsewhere it is read
// from wherever it lies.
// Bound by the matrix cores where there are many tiles: each element is multiplied twice, as its large and its small half, so their
// ceiling is half the formats' (about 1.9e15 products and sums a second at the clock that such a load leaves). 2048 x 37888 x 3584 with
// the gate takes 390 us (1.43e15 a second), 512 x 3584 x 18944 66 us (1.05e15, four parts' traffic and their sum in it), but 512 x 4608 x
// 3584, 2.25 tiles of 64 x 64 a CU, 27.7 (0.61e15). The activations straight into registers took 484 us instead of 436; a third stage of LDS
// and raised wave priorities changed nothing.
typedef uint32_t any4 __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t short_row(const uint8_t* row, int nb) {      // the scales of a row that has one to three
  uint32_t v = row[0];
  if (nb > 1) v |= (uint32_t)row[1] << 8;
  if (nb > 2) v |= (uint32_t)row[2] << 16;
  return v;
}
struct MxTiles {
  int tokens, count;       // tiles of tokens, all tiles
  int parts, steps;        // K split: parts of so many steps of 128
  int64_t apart;           // numbers of C from one part to the next
};

template <int WF, int WT, int NF, int NT, int WPE, bool GATED, bool WORDS>
__global__ __launch_bounds__(64 * WF * WT, WPE) void mx_tile_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ sa,
                                                                    const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw, int M, int N, int nb,
                                                                    MxTiles P, float* __restrict__ C, uint8_t* __restrict__ codes,
                                                                    uint8_t* __restrict__ scales) {
  constexpr int kWaves = WF * WT, kThreads = 64 * kWaves, TF = 16 * NF * WF, TT = 16 * NT * WT, kRows = TF + TT;
  constexpr int kWBytes = TF * 64, kElems = kWBytes + TT * 128, kStage = kElems + kRows * 4;
  constexpr int kCopies = kElems / 1024 / kWaves, kRowsEach = (kRows + kThreads - 1) / kThreads;
  static_assert(kElems % (1024 * kWaves) == 0 && kWBytes % (1024 * kWaves) == 0 && kRows % 64 == 0, "whole copies");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wf = wave / WT, wt = wave % WT;
  const BlockPlace at = block_place(P.count, P.parts);
  const int tf = at.tile / P.tokens, tt = at.tile - tf * P.tokens;
  const int all = (nb + 3) / 4, first = at.part * P.steps, steps = min(P.steps, all - first);
  // row of the weight for row i of the tile: with a gate, a wavefront's tiles are gate rows, then the up rows of the same features
  constexpr int kFeatures = GATED ? TF / 2 : TF;
  const auto weight_row = [&](int i) -> int64_t {
    if constexpr (!GATED) return min(tf * TF + i, N - 1);
    const int w = i / (16 * NF), f = i % (16 * NF);
    return min(tf * kFeatures + w * (8 * NF) + f % (8 * NF), N - 1) + (f < 8 * NF ? (int64_t)0 : (int64_t)N);
  };
  const auto token_row = [&](int i) -> int64_t { return min(tt * TT + i, M - 1); };

  // Rows of a wavefront's copies, 16 of the weight or 8 of the activations: the first one's address (uniform) and 32-bit offsets
  const uint8_t* src[kCopies];
  uint32_t off[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; j++) {
    const bool w = j * kWaves * 1024 < kWBytes;
    const int q = j * kWaves + wave - (w ? 0 : kWBytes / 1024), row0 = q * (w ? 16 : 8), row = row0 + (lane >> (w ? 2 : 3));
    const int64_t base = w ? weight_row(row0) : token_row(row0), mine = w ? weight_row(row) : token_row(row);
    src[j] = w ? W + base * nb * 16 : A + base * nb * 32;
    off[j] = (uint32_t)(mine - base) * (uint32_t)nb * (w ? 16u : 32u);
  }
  // the chunk of its row that a lane copies: W's lanes & 3 ^ (-(row >> 2) & 3), A's lane & 7 ^ (row >> 1 & 7), rows of a copy being whole 16s and 8s
  const uint32_t wchunk = ((lane & 3) ^ (-(lane >> 4) & 3)) * 16, achunk = ((lane & 7) ^ (lane >> 4)) * 16;
  const uint8_t* srow[kRowsEach];
  uint32_t sc[kRowsEach];
#pragma unroll
  for (int j = 0; j < kRowsEach; j++) {
    const int i = min(j * kThreads + tid, kRows - 1);
    srow[j] = i < TF ? sw + weight_row(i) * nb : sa + token_row(i - TF) * nb;
  }
  // Scale words that are not whole ones go through registers, two steps ahead, so that nobody waits for them (301 x 4608 x 3648 18.9 us,
  // 26.7 where each step waited; x 3712, whose are words, 17.4)
  const auto ask_scales = [&](int step) {
    if constexpr (!WORDS) {
      if (nb >= 4) {
#pragma unroll
        for (int j = 0; j < kRowsEach; j++) sc[j] = *reinterpret_cast<const any4*>(srow[j] + min((first + step) * 4, nb - 4));
      }
    }
  };
  const auto copy = [&](int step, int stage) {
    char* s = lds + stage * kStage;
#pragma unroll
    for (int j = 0; j < kCopies; j++) {
      const bool w = j * kWaves * 1024 < kWBytes;
      uint32_t k = (uint32_t)(first + step) * (w ? 64u : 128u) + (w ? wchunk : achunk ^ (uint32_t)((j * kWaves + wave - kWBytes / 1024) & 1) * 64u);
      if constexpr (!WORDS) k = min(k, (uint32_t)(w ? nb - 1 : 2 * nb - 1) * 16u);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[j] + (off[j] + k)),
                                       (__attribute__((address_space(3))) void*)(s + (j * kWaves + wave) * 1024), 16, 0, 0);
    }
    if constexpr (WORDS) {
#pragma unroll
      for (int j = 0; j < kRowsEach; j++)
        if (j * kThreads + wave * 64 < kRows)
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(srow[j] + (first + step) * 4),
                                           (__attribute__((address_space(3))) void*)(s + kElems + (j * kThreads + wave * 64) * 4), 4, 0, 0);
    }
  };
  const auto keep_scales = [&](int step, int stage) {      // those asked for last; a row's last word has been read from before its end
    if constexpr (!WORDS) {
      const int past = nb < 4 ? 0 : 8 * max((first + step) * 4 - (nb - 4), 0);
#pragma unroll
      for (int j = 0; j < kRowsEach; j++)
        if (j * kThreads + tid < kRows) *reinterpret_cast<uint32_t*>(lds + stage * kStage + kElems + (j * kThreads + tid) * 4) = sc[j] >> past;
    }
  };

  v4f c[NF][NT];
#pragma unroll
  for (int f = 0; f < NF; f++)
#pragma unroll
    for (int t = 0; t < NT; t++) c[f][t] = v4f{0.f, 0.f, 0.f, 0.f};
  // where my operands lie in a stage
  const int wrow = (wf * 16 * NF + r) * 64 + ((g ^ (-(r >> 2) & 3)) << 4);              // (+ 1024 a tile)
  const int arow = kWBytes + (wt * 16 * NT + r) * 128, ax = r >> 1 & 7;                 // (+ 2048 a tile)
  const int a0 = arow + ((g ^ ax) << 4), a1 = arow + (((4 + g) ^ ax) << 4);
  const int ws = kElems + (wf * 16 * NF + r) * 4, as = kElems + (TF + wt * 16 * NT + r) * 4;   // (+ 64 a tile)

  if constexpr (!WORDS) {
    if (nb < 4) {                                // (one step)
#pragma unroll
      for (int j = 0; j < kRowsEach; j++) sc[j] = short_row(srow[j], nb);
    }
  }
  ask_scales(0);
  copy(0, 0);
  keep_scales(0, 0);
  ask_scales(1);
  for (int i = 0; i < steps; i++) {
    // what was copied a step ago has landed, my reads are done, and so are everybody's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + 1 < steps) {
      keep_scales(i + 1, (i + 1) & 1);
      ask_scales(i + 2);
      copy(i + 1, (i + 1) & 1);
    }
    // LDS is read as vectors of words, never as uint4, which the compiler takes for something that a copy in flight may write
    const char* s = lds + (i & 1) * kStage;
    frag16 w[NF];
    int swv[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) {
      w[f] = *reinterpret_cast<const frag16*>(s + wrow + f * 1024);
      swv[f] = (int)(*reinterpret_cast<const uint32_t*>(s + ws + f * 64) >> (8 * g));
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const frag16 lo = *reinterpret_cast<const frag16*>(s + a0 + t * 2048), hi = *reinterpret_cast<const frag16*>(s + a1 + t * 2048);
      const int sav = (int)(*reinterpret_cast<const uint32_t*>(s + as + t * 64) >> (8 * g));
      v8i large, small;
      split_e4m3(row_operand(lo, hi), large, small);
#pragma unroll
      for (int f = 0; f < NF; f++)
        c[f][t] = mx_mma(weight_operand(w[f]), small, c[f][t], swv[f], sav);
#pragma unroll
      for (int f = 0; f < NF; f++)
        c[f][t] = mx_mma(weight_operand(w[f]), large, c[f][t], swv[f], sav);
    }
  }
#pragma unroll
  for (int f = 0; f < NF; f++)
#pragma unroll
    for (int t = 0; t < NT; t++) mx_done(c[f][t]);

#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int m = tt * TT + (wt * NT + t) * 16 + r;
    if constexpr (!GATED) {
      float* out = C + at.part * P.apart + (int64_t)m * N;
#pragma unroll
      for (int f = 0; f < NF; f++)
        if (m < M) store_features(out, tf * TF + (wf * NF + f) * 16 + 4 * g, N, c[f][t]);
    } else {
#pragma unroll
      for (int p = 0; p < NF / 4; p++) {          // blocks of 32 features: two tiles
        const int n = tf * kFeatures + wf * (8 * NF) + 32 * p;
        store_gated(c[2 * p][t], c[2 * p + 1][t], c[NF / 2 + 2 * p][t], c[NF / 2 + 2 * p + 1][t], g, m < M && n < N,
                    codes + (int64_t)min(m, M - 1) * N + n, scales + (int64_t)min(m, M - 1) * (N / kMxBlock) + n / kMxBlock);
      }
    }
  }
}

// Blocks of a launch, each 256 threads, which a grid's x counts in 32 bits. Results of up to 2^37 numbers are at most 2^23 tiles of the
// largest kind, half as many features with the gate, and those that the ends of its rows and columns add.
constexpr int64_t kMostTiles = ((int64_t)1 << 24) - 1;

template <int WF, int WT, int NF, int NT, int WPE, bool GATED>
static hipError_t launch_tiles(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, int64_t M, int64_t N, int64_t K, int parts,
                               int64_t apart, float* C, uint8_t* codes, uint8_t* scales) {
  constexpr int TF = 16 * NF * WF / (GATED ? 2 : 1), TT = 16 * NT * WT;
  constexpr int lds = 2 * (16 * NF * WF * 68 + TT * 132);
  static_assert(lds <= 160 * 1024, "LDS");
  static_assert(64 * WF * WT == 256, "what kMostTiles counts");
  MxTiles P;
  P.tokens = (int)((M + TT - 1) / TT);
  const int64_t count = (N + TF - 1) / TF * P.tokens;
  if (count > kMostTiles) return hipErrorInvalidValue;
  P.count = (int)count;
  const int all = (int)((K + 127) / 128);
  P.steps = (all + parts - 1) / parts;
  P.parts = (all + P.steps - 1) / P.steps;
  P.apart = apart;
  const int nb = (int)(K / kMxBlock);
  const bool words = nb % 4 == 0 && ((reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sw)) & 3) == 0;
  const auto kernel = words ? mx_tile_kernel<WF, WT, NF, NT, WPE, GATED, true> : mx_tile_kernel<WF, WT, NF, NT, WPE, GATED, false>;
  if (const hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess) return e;
  kernel<<<dim3((unsigned)P.count, (unsigned)P.parts), dim3(64 * WF * WT), lds, ctx().stream>>>(A, sa, W, sw, (int)M, (int)N, nb, P, C, codes,
                                                                                                scales);
  return hipGetLastError();
}

// ---- which tiles --------------------------------------------------------------------------------------------------------
// Features x tokens of a tile. A step takes `one` us plus `more` for each block on a CU, as measured on products of 20 to 2048 rows by 896 x 4864
// to 37888 x 3584; the launch that adds parts up 2.2 us and their traffic at 5.4 TB/s. Over 54 products of those sizes the choice takes 1.01
// times the best one's time in the mean and 1.16 at worst. Both sides: 77 x 896 x 4864 7.6 us in 8 parts of 64 x 64, 8.7 of 128 x 64, 23.9 in
// one; with the result read back (5 us of it) 512 x 18944 gated x 3584 116 us with 128 x 128, 132 with 256 x 128, 137 with 128 x 64, 162 with 64 x 64; 2048 x 37888 x 3584 422 with 256 x 128, 427
// with 128 x 128, 532 with 128 x 64. Numbers of parts that the eight dies do not share evenly are not tried (77 x 3584 x 18944 in 10
// parts 30.4 us, in 8 23.5, in 12 26.2).
struct MxPlan { int variant = 0, parts = 1; double us = 1e30; };
constexpr int kVariants = 4;
static const struct { int features, tokens; double one, more; } kVariant[kVariants] = {
    {64, 64, 0.194, 0.2475}, {128, 64, 0.342, 0.38}, {128, 128, 0.39, 0.72}, {256, 128, 0.8, 1.34}};

static MxPlan plan_tiles(int64_t M, int64_t N, int64_t K, int64_t max_parts, bool gated, bool own_sum) {
  const int64_t cus = cu_count(), steps = (K + 127) / 128;
  MxPlan best;
  for (int v = 0; v < kVariants; v++) {
    const int64_t features = kVariant[v].features / (gated ? 2 : 1);
    const int64_t tiles = (N + features - 1) / features * ((M + kVariant[v].tokens - 1) / kVariant[v].tokens);
    if (tiles > kMostTiles) continue;
    for (const int64_t S : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (S > 1 && (S > max_parts || steps / S < 2)) break;
      const int64_t each = (steps + S - 1) / S, parts = (steps + each - 1) / each;
      const double per_cu = std::max(1.09, (double)(tiles * parts) / (double)cus);
      double us = 2.25 + (double)each * (kVariant[v].one + kVariant[v].more * per_cu);
      if (parts > 1) us += (own_sum ? 2.2 : 0.0) + (double)(2 * parts + 1) * (double)M * (double)N * 4.0 / 5.4e6;
      if (us < best.us) best = MxPlan{v, (int)parts, us};
    }
  }
  return best;
}

// A product without the gate: rows of 16 a block, or tiles
struct MxProduct { bool rows; MxPlan tiles; };
static MxProduct plan_product(int64_t M, int64_t N, int64_t K, int64_t max_parts, bool own_sum) {
  const MxPlan tiles = plan_tiles(M, N, K, max_parts, false, own_sum);
  return MxProduct{mx_few_rows_us(M, N, K) < tiles.us, tiles};
}

// A gated product. apart: the products, then a launch that gates them; of few tiles over a long K, gate and up products in parts
// that it adds up (us so, and in one launch, each with the result read back, 2 to 3 of them: 282 x 32 x 11552
// 12.5, 55.9; 310 x 832 x 8128 26.5, 49.9). Of few rows the products are then those of 16 rows
// a block, or of tiles in parts, as their estimates say; up to 16 rows the one launch has blocks of 32 gate and 32 up rows (12 x 32 x 10368
// 11.5, 16.3; 7 x 1792 x 5440 9.1, 11.7; 16 x 512 x 1536 7.7, 8.1; 1024 7.6, 7.9; 16 x 6144 x 3584, where those fill the CUs, 14.0, 11.3).
// room: for the products.
struct MxGated { bool apart, rows; MxPlan tiles; };
static MxGated plan_gated(int64_t M, int64_t ff, int64_t K, bool room) {
  const bool few = M <= kMxFewRows, fits = few && mx_few_rows_fit(ff, K, true);
  const MxPlan one = plan_tiles(M, ff, K, 1, true, false);
  MxPlan two = plan_tiles(M, 2 * ff, K, 16, false, false);
  const double rows_us = mx_few_rows_us(M, 2 * ff, K), whole = 4.0 * (double)M * (double)ff * 4.0 / 5.4e6;    // (of one part, written and read)
  if (two.parts == 1) two.us += whole;
  const bool rows = rows_us + whole < two.us;
  if (rows) two = MxPlan{0, 1, rows_us + whole};
  const bool apart = few ? !fits || (K >= 1536 && ff / kMxBlock <= cu_count() / 2) : two.us + 2.2 < one.us;
  return apart && room ? MxGated{true, rows, two} : MxGated{false, fits, one};
}

static hipError_t launch_plan(const MxPlan& P, const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, int64_t M, int64_t N,
                              int64_t K, int64_t apart, float* C, uint8_t* codes, uint8_t* scales) {
  if (codes) {
    const auto go = P.variant == 0   ? launch_tiles<1, 4, 4, 1, 4, true>
                    : P.variant == 1 ? launch_tiles<1, 4, 8, 1, 4, true>
                    : P.variant == 2 ? launch_tiles<1, 4, 8, 2, 3, true>
                                     : launch_tiles<2, 2, 8, 4, 2, true>;
    return go(A, sa, W, sw, M, N, K, 1, 0, C, codes, scales);
  }
  const auto go = P.variant == 0   ? launch_tiles<1, 4, 4, 1, 4, false>
                  : P.variant == 1 ? launch_tiles<1, 4, 8, 1, 4, false>
                  : P.variant == 2 ? launch_tiles<1, 4, 8, 2, 3, false>
                                   : launch_tiles<2, 2, 8, 4, 2, false>;
  return go(A, sa, W, sw, M, N, K, P.parts, apart, C, nullptr, nullptr);
}

// ---- a split K's parts ----------------------------------------------------------------------------------------------------
// C = their sum, in their order
__global__ __launch_bounds__(256) void mx_sum_kernel(const float4* __restrict__ part, float* __restrict__ C, int64_t total, int64_t apart4, int S) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (4 * i >= total) return;
  const float4 a = sum_parts(S, [&](int s) { return part[s * apart4 + i]; });
  if (4 * i + 4 <= total) {
    *reinterpret_cast<float4*>(C + 4 * i) = a;
  } else {
    const float v[4] = {a.x, a.y, a.z, a.w};
    for (int k = 0; 4 * i + k < total; k++) C[4 * i + k] = v[k];
  }
}

// The gated activation of the sums, parts [S][M][gate | up], as MXFP8 rows: a lane has four features, eight lanes a block
struct MxGateUp { float4 g, u; };
__device__ __forceinline__ MxGateUp plus(const MxGateUp& a, const MxGateUp& b) { return MxGateUp{plus(a.g, b.g), plus(a.u, b.u)}; }
__global__ __launch_bounds__(256) void mx_gate_sum_kernel(const float4* __restrict__ part, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                          int64_t M, int f4, int S) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * f4) return;                                     // (whole groups of eight lanes)
  const int64_t m = i / f4, at = m * f4 + i, apart4 = M * 2 * f4;
  const MxGateUp gu = sum_parts(S, [&](int s) { return MxGateUp{part[s * apart4 + at], part[s * apart4 + at + f4]}; });
  float v[4] = {gated_fast(gu.g.x, gu.u.x), gated_fast(gu.g.y, gu.u.y), gated_fast(gu.g.z, gu.u.z), gated_fast(gu.g.w, gu.u.w)};
  uint32_t big = max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3])));
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0xB1, 0xf, 0xf, true));    // quad_perm [1,0,3,2]
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x4E, 0xf, 0xf, true));    // quad_perm [2,3,0,1]
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x141, 0xf, 0xf, true));   // row_half_mirror
  const uint32_t s = mx_scale_of(big, kMx8Exp);
  const float up = mx_up(min(s, 252u));
#pragma unroll
  for (int k = 0; k < 4; k++) v[k] = s == 255u ? 0.f : v[k] * up;
  reinterpret_cast<uint32_t*>(codes)[i] = to_e4m3x4(v[0], v[1], v[2], v[3]);
  if ((i & 7) == 0) scales[i >> 3] = (uint8_t)s;
}

}  // namespace tlhip

using namespace tlhip;

static const uint8_t* bytes(const void* p) { return static_cast<const uint8_t*>(p); }

extern "C" {

int tlhip_gemm_mxfp4_nt_parts(const void* acodes, const void* ascales, const void* codes, const void* scales, void* parts, int64_t parts_bytes,
                              int64_t M, int64_t N, int64_t K, int* n_parts) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemm_mxfp4_nt_parts";
  if (const int rc = check_mx_product(who, acodes, ascales, codes, scales, parts, M, N, K)) return rc;
  if (const int rc = check_mx_apart(who, parts, {acodes, ascales, codes, scales})) return rc;
  if (!n_parts) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (parts_bytes < M * N * 4) return fail(TLHIP_EINVAL, "%s: the parts need M * N * 4 bytes at least", who);
  hipError_t e;
  const MxProduct P = plan_product(M, N, K, parts_bytes / (M * N * 4), false);
  if (P.rows) {
    *n_parts = 1;
    e = launch_mx_few_rows(bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, N, K, static_cast<float*>(parts), nullptr, nullptr);
  } else {
    *n_parts = P.tiles.parts;
    e = launch_plan(P.tiles, bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, N, K, M * N, static_cast<float*>(parts), nullptr, nullptr);
  }
  if (e != hipSuccess) return hip_fail(e, who);
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMM_MXFP4);
}

int tlhip_gemm_mxfp4_nt(const void* acodes, const void* ascales, const void* codes, const void* scales, void* C, int64_t M, int64_t N,
                        int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemm_mxfp4_nt";
  if (const int rc = check_mx_product(who, acodes, ascales, codes, scales, C, M, N, K)) return rc;
  if (const int rc = check_mx_apart(who, C, {acodes, ascales, codes, scales})) return rc;
  hipError_t e;
  const MxProduct product = plan_product(M, N, K, 16, true);
  MxPlan P = product.tiles;
  if (product.rows) {
    e = launch_mx_few_rows(bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, N, K, static_cast<float*>(C), nullptr, nullptr);
  } else {
    const int64_t apart = (M * N + 3) & ~(int64_t)3;
    float* out = static_cast<float*>(C);
    if (P.parts > 1) {
      out = static_cast<float*>(scratch((size_t)P.parts * apart * 4));
      if (!out) {            // (a recording may not grow it)
        P = plan_tiles(M, N, K, 1, false, true);
        out = static_cast<float*>(C);
      }
    }
    e = launch_plan(P, bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, N, K, apart, out, nullptr, nullptr);
    if (e == hipSuccess && P.parts > 1)
      mx_sum_kernel<<<dim3((unsigned)((apart / 4 + 255) / 256)), dim3(256), 0, ctx().stream>>>(reinterpret_cast<const float4*>(out), static_cast<float*>(C),
                                                                                              M * N, apart / 4, P.parts);
  }
  if (e != hipSuccess) return hip_fail(e, who);
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMM_MXFP4);
}

int tlhip_gemm_mxfp4_nt_swiglu(const void* acodes, const void* ascales, const void* codes, const void* scales, void* act_codes,
                               void* act_scales, int64_t M, int64_t ff, int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemm_mxfp4_nt_swiglu";
  if (const int rc = check_mx_product(who, acodes, ascales, codes, scales, act_codes, M, ff, K)) return rc;
  if (!act_scales) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (!mx_row(ff)) return fail(TLHIP_EINVAL, "%s: ff must be a multiple of 32", who);
  if (const int rc = check_mx_apart(who, act_codes, {acodes, ascales, codes, scales, act_scales})) return rc;
  if (const int rc = check_mx_apart(who, act_scales, {acodes, ascales, codes, scales})) return rc;
  uint8_t *qc = static_cast<uint8_t*>(act_codes), *qs = static_cast<uint8_t*>(act_scales);
  MxGated P = plan_gated(M, ff, K, true);
  float* const parts = P.apart ? static_cast<float*>(scratch((size_t)P.tiles.parts * M * 2 * ff * 4)) : nullptr;
  if (P.apart && !parts) P = plan_gated(M, ff, K, false);       // (a recording may not grow it)
  hipError_t e;
  if (P.apart) {
    e = P.rows ? launch_mx_few_rows(bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, 2 * ff, K, parts, nullptr, nullptr)
               : launch_plan(P.tiles, bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, 2 * ff, K, M * 2 * ff, parts, nullptr, nullptr);
    if (e == hipSuccess)
      mx_gate_sum_kernel<<<dim3((unsigned)((M * (ff / 4) + 255) / 256)), dim3(256), 0, ctx().stream>>>(reinterpret_cast<const float4*>(parts), qc, qs, M,
                                                                                                       (int)(ff / 4), P.tiles.parts);
  } else if (P.rows) {
    e = launch_mx_few_rows(bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, ff, K, nullptr, qc, qs);
  } else {
    e = launch_plan(P.tiles, bytes(acodes), bytes(ascales), bytes(codes), bytes(scales), M, ff, K, 0, nullptr, qc, qs);
  }
  if (e != hipSuccess) return hip_fail(e, who);
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMM_MXFP4);
}

int tlhip_plan_gemm_mxfp4(int64_t M, int64_t N, int64_t K, int gated, int parts, int plan[5]) {
  const char* who = "tlhip_plan_gemm_mxfp4";
  if (!plan || M <= 0 || N <= 0 || !mx_row(K) || parts < 0 || (gated && (parts || !mx_row(N)))) return fail(TLHIP_EINVAL, "%s: bad arguments", who);
  if (M > (1 << 20) || N > (1 << 24) || K > kMxMaxK || M * N > (int64_t)1 << 37) return fail(TLHIP_EUNSUPPORTED, "%s: dimension too large", who);
  const MxGated g = gated ? plan_gated(M, N, K, true) : MxGated{};
  const MxProduct p = gated ? MxProduct{g.rows, g.tiles} : plan_product(M, N, K, parts ? parts : 16, parts == 0);
  plan[0] = p.rows;
  plan[1] = !p.rows ? kVariant[p.tiles.variant].features : gated && !g.apart ? 64 : 16 * mx_few_rows_tiles(M, gated ? 2 * N : N, K);
  plan[2] = p.rows ? 16 : kVariant[p.tiles.variant].tokens;
  plan[3] = p.rows ? 1 : p.tiles.parts;
  plan[4] = g.apart;
  return TLHIP_OK;
}

}  // extern "C"
