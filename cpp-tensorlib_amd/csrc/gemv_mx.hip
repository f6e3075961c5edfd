// Products of few rows over MXFP4 weights: of one f32 row (a decode step's, plain or behind an RMS norm, with or without the gated
// activation) and of MXFP8 rows, 16 to a block. All of it is bound by reading the weight.
#include "mx_mfma.hpp"

#include <algorithm>

namespace tlhip {

// The weight is read once, from memory straight into the registers that the matrix instruction takes it from: a wavefront has 16 NF
// of its rows and every KW-th unit of 256 k (128 bytes of a row). KW wavefronts of a block share rows; their sums are joined in
// LDS, in their order. Features that are left over are the last row's again, and not stored.
//
// kCodes: 16 rows of MXFP8 a block, in two parts each (mx_mfma.hpp).
// kFloat, kNormed: one f32 row (kNormed: rms-normed first), cut into digits that the matrix cores multiply exactly. A number's magnitude,
// over the power of two of its block's largest, is a whole number of 48 bits: twelve digits of four. A byte 0 to 15 is,
// as e4m3, that many times 2^-9, so a digit is its own code; with the number's sign it is one element of a row of the second operand,
// digit p in row p under the scale 16^p. The row's twelve sums, which no product's last bit is missing from, are added up at the end. A
// number keeps all of its 24 bits down to 2^-24 of its block's largest, below that an absolute error of 2^-48 of it. Numbers
// below 2^-81 are cut at 2^-128; a block with an infinity or a NaN is NaN. The sums are of y / 256, so that the largest fit: each of the 192 +
// K / 128 roundings of each of the twelve is 2^-150 at least, 2^-142 of y. Dequantised in the vector unit (1.5 instructions for each
// weight, the conversion of e2m1 alone nearly three times an FMA) the same product was bound by it.
//
// The scales of a block's rows are one run of bytes: copied into LDS whole (a byte loaded by each lane was a request for 16 lines: 70 us
// instead of 60 over 152064 x 3584).
typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(1)));
// (two runs `apart` bytes from each other: both asked for before either is waited for, 4608 x 3584 with the gate 10.2 us one by one)
__host__ __device__ constexpr int whole_16(int bytes) { return (bytes + 15) & ~15; }
template <int RUNS>
__device__ __forceinline__ void put_scales(char* to, const uint8_t* from, int64_t apart, int bytes, int64_t limit, int tid, int threads) {
  for (int i = 16 * tid; i < bytes; i += 16 * threads) {
    if (i + 16 <= limit) {
      any16 v[RUNS];
#pragma unroll
      for (int k = 0; k < RUNS; k++) v[k] = *reinterpret_cast<const any16*>(from + k * apart + i);
#pragma unroll
      for (int k = 0; k < RUNS; k++) *reinterpret_cast<frag16*>(to + k * whole_16(bytes) + i) = v[k];
    } else {
      for (int k = 0; k < RUNS; k++)
        for (int j = 0; j < 16 && i + j < limit; j++) to[k * whole_16(bytes) + i + j] = (char)from[k * apart + i + j];
    }
  }
}
enum { kCodes = 0, kFloat = 1, kNormed = 2, kMerged = 3 };
struct MxRow {               // the f32 row: x (+ delta), its norm weights, and where x + delta goes
  const float *x, *delta, *norm_w;
  float* xout;
  float eps;
  int splits, heads, dim;    // kMerged: x is the attention's partials
};
// Numbers k .. k + 3 of the attention's row from its splits (maxima [heads][S], sums [heads][S], accumulators [heads][S][dim], as
// tlhip_attn_decode_qkv_parts leaves them): sum_s e^(m_s - M) acc_s / sum_s e^(m_s - M) l_s in the order of tlhip_gemv_q4_attn's merge.
// The 16 lanes of a row have numbers of one head (dim is 64 or 128) and the weight of one split each.
struct MergeIn {
  static constexpr int kFirst = 8;             // splits asked for ahead of the weights
  float m, l;
  float4 a[kFirst];
  const float4* acc;
};
__device__ __forceinline__ MergeIn ask_merge(const MxRow& R, int k, int lane) {
  const int S = R.splits, h = k / R.dim, d = k - h * R.dim, s = min(lane & 15, S - 1), hs = R.heads * S;
  MergeIn q;
  q.m = R.x[h * S + s];
  q.l = R.x[hs + h * S + s];
  q.acc = reinterpret_cast<const float4*>(R.x + 2 * hs + (int64_t)h * S * R.dim + d);
#pragma unroll
  for (int i = 0; i < MergeIn::kFirst; i++) q.a[i] = q.acc[min(i, S - 1) * (R.dim / 4)];
  return q;
}
__device__ __forceinline__ float4 merged(const MxRow& R, const MergeIn& q, int lane) {
  const int S = R.splits;
  const float m = q.m, l = q.l;
  float M = fmaxf(m, dpp_read<0x128>(m));      // row_ror:8, 4, 2, 1
  M = fmaxf(M, dpp_read<0x124>(M));
  M = fmaxf(M, dpp_read<0x122>(M));
  M = fmaxf(M, dpp_read<0x121>(M));
  const float w = (lane & 15) < S ? __expf(m - M) : 0.f;
  float L = mul_rn(l, w);
  L = add_rn(L, dpp_read<0x128>(L));
  L += dpp_read<0x124>(L);
  L += dpp_read<0x122>(L);
  L += dpp_read<0x121>(L);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto add = [&](int i, const float4 p) {
    const float f = __shfl(w, (lane & 48) + i);
    v = make_float4(add_rn(v.x, mul_rn(f, p.x)), add_rn(v.y, mul_rn(f, p.y)), add_rn(v.z, mul_rn(f, p.z)), add_rn(v.w, mul_rn(f, p.w)));
  };
#pragma unroll
  for (int i = 0; i < MergeIn::kFirst; i++)
    if (i < S) add(i, q.a[i]);
  for (int i = MergeIn::kFirst; i < S; i++) add(i, q.acc[i * (R.dim / 4)]);
  return make_float4(v.x / L, v.y / L, v.z / L, v.w / L);
}
constexpr int kDigits = 12, kUnitLds = 2 * kDigits * 128 + 16;      // digits of a unit, its eight blocks' exponents

// Numbers 4 lane .. 4 lane + 3 of a unit into LDS: a step's digits [kDigits][128] bytes, then the next one's, then the exponents
__device__ __forceinline__ void put_digits(char* lds, int lane, float4 x) {
  const float v[4] = {x.x, x.y, x.z, x.w};
  uint32_t big = max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3])));
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0xB1, 0xf, 0xf, true));    // quad_perm [1,0,3,2]
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x4E, 0xf, 0xf, true));    // quad_perm [2,3,0,1]
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x141, 0xf, 0xf, true));   // row_half_mirror
  const uint32_t field = max(big >> 23, 46u);
  const float up1 = __uint_as_float((254u - min(field, 253u)) << 23), up2 = field >= 254u ? 1073741824.0f : 2147483648.0f;
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float a = fabsf(v[i]) * up1 * up2;                 // below 2^32: 2^31 over the largest's power of two
    hi[i] = (uint32_t)a;                                     // (towards zero; a whole number from 2^24 on)
    lo[i] = (uint32_t)((a - (float)hi[i]) * 65536.0f);
  }
  // byte b of the four numbers in one word
  const auto plane = [](const uint32_t (&d)[4], int b) {
    const uint32_t s = 0x0c0c0400u + (uint32_t)b * 0x0101u;  // bytes b of a pair, then zeros
    return __builtin_amdgcn_perm(d[1], d[0], s) | __builtin_amdgcn_perm(d[3], d[2], s) << 16;
  };
  const uint32_t f[4] = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  const uint32_t sign = plane(f, 3) & 0x80808080u;
  uint32_t* at = reinterpret_cast<uint32_t*>(lds + (lane >> 5) * (kDigits * 128) + (lane & 31) * 4);
#pragma unroll
  for (int b = 0; b < 6; b++) {
    const uint32_t w = b < 2 ? plane(lo, b) : plane(hi, b - 2);
    at[(2 * b) * 32] = (w & 0x0f0f0f0fu) | sign;
    at[(2 * b + 1) * 32] = (w >> 4 & 0x0f0f0f0fu) | sign;
  }
  if ((lane & 7) == 0) reinterpret_cast<uint8_t*>(lds + 2 * kDigits * 128)[lane >> 3] = (uint8_t)min(field, 255u);
}

__host__ __device__ constexpr int rows_sums(int tiles, int waves) { return waves * (tiles * 1024 + 4); }
// Where the scales of mx_rows_kernel's blocks begin in LDS, 16 bytes of them being put there at a time: behind the sums, or the digits
__host__ __device__ constexpr int rows_scales(int src, int tiles, int waves) {
  const int sums = rows_sums(tiles, waves), digits = src == kCodes ? 0 : waves * kUnitLds;
  return whole_16(sums > digits ? sums : digits);
}
constexpr bool rows_scales_whole() {
  for (int tiles = 1; tiles <= 4; tiles++)
    for (int waves = 1; waves <= 16; waves++)
      if (rows_scales(kCodes, tiles, waves) % 16 || rows_scales(kFloat, tiles, waves) % 16) return false;
  return true;
}
static_assert(rows_scales_whole(), "16-byte stores");

// The sums of a feature's twelve digits, which lie in lanes 0 .. 11 of the sixteen that have it: lane i gets feature i of its four
__device__ __forceinline__ float join_digits(const v4f& c, int r) {
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float v = r < kDigits ? c[i] : 0.f;
    v = dpp_add_f32<0xB1>(v);
    v = dpp_add_f32<0x4E>(v);
    v = dpp_add_f32<0x141>(v);
    v = dpp_add_f32<0x140>(v);
    mine = r == i ? v : mine;
  }
  return mine * 256.0f;
}

// Row r of tile f of a wavefront: a feature, counted from the wavefront's first. With a gate half the tiles are of gate rows,
// the others of the up rows of the same features; one tile alone has eight of each, gate rows first.
struct TileRow { int n; bool up; };
template <int NF, bool GATED>
__device__ __forceinline__ TileRow tile_row(int f, int r) {
  if constexpr (!GATED) return {16 * f + r, false};
  else if constexpr (NF == 1) return {r & 7, r >= 8};
  else return {16 * (f % (NF / 2)) + r, f >= NF / 2};
}

template <int SRC, int NF, bool GATED>
__global__ __launch_bounds__(SRC == kCodes ? 512 : 1024, 2) void mx_rows_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ sa,
                                                         const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw, int M, int N, int nb, int KW,
                                                         int waves, float* __restrict__ C, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                         const MxRow R) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), fw = wave / KW, kw = wave - fw * KW, FW = waves / KW;
  const int units = (nb + 7) / 8, K = nb * kMxBlock;
  constexpr int kTile = GATED ? 8 * NF : 16 * NF;              // features of a wavefront
  const int n0 = (blockIdx.x * FW + fw) * kTile;
  const uint8_t* wrow[NF];
  int wscale[NF];                                              // in the block's run of scales: gate rows first
#pragma unroll
  for (int f = 0; f < NF; f++) {
    const TileRow t = tile_row<NF, GATED>(f, r);
    wrow[f] = W + ((t.up ? (int64_t)N : 0) + min(n0 + t.n, N - 1)) * nb * 16;
    wscale[f] = (fw * kTile + t.n) * nb + (t.up ? whole_16(FW * kTile * nb) : 0);
  }
  const int m = SRC == kCodes ? 16 * blockIdx.y + r : 0;        // my row of the activations
  const uint8_t *arow = A + (int64_t)min(m, M - 1) * nb * 32, *ascale = sa + (int64_t)min(m, M - 1) * nb;
  struct Unit {
    frag16 w[2][NF];
    frag16 lo[2], hi[2];
    uint32_t as[2];
    float4 x, d, nw;
  };
  // Past the end of a row: its last block or numbers again, under scales of 2^-127 on both sides (digits: as zeros)
  const auto ask = [&](Unit& q, int u) {
    MergeIn in;
    if constexpr (SRC == kMerged) in = ask_merge(R, min(256 * u + 4 * lane, K - 4), lane);
    if constexpr (SRC == kFloat || SRC == kNormed) {
      const int k = min(256 * u + 4 * lane, K - 4);
      q.x = *reinterpret_cast<const float4*>(R.x + k);
      if constexpr (SRC == kNormed) {
        if (R.delta) q.d = *reinterpret_cast<const float4*>(R.delta + k);
        q.nw = *reinterpret_cast<const float4*>(R.norm_w + k);
      }
    }
    // (both halves of a row's 128 bytes one after the other, and not past the caches: the second finds the line there)
#pragma unroll
    for (int f = 0; f < NF; f++)
#pragma unroll
      for (int h = 0; h < 2; h++) q.w[h][f] = *reinterpret_cast<const frag16*>(wrow[f] + (int64_t)min(8 * u + 4 * h + g, nb - 1) * 16);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int b = 8 * u + 4 * h + g, at = min(b, nb - 1);
      if constexpr (SRC == kCodes) {
        const int c0 = min(16 * u + 8 * h + g, 2 * nb - 1), c1 = min(16 * u + 8 * h + 4 + g, 2 * nb - 1);
        q.lo[h] = *reinterpret_cast<const frag16*>(arow + (int64_t)c0 * 16);
        q.hi[h] = *reinterpret_cast<const frag16*>(arow + (int64_t)c1 * 16);
        q.as[h] = b < nb ? ascale[at] : 0;
      }
    }
    if constexpr (SRC == kMerged) q.x = merged(R, in, lane);     // (the weights are on their way)
  };
  v4f c[NF];
#pragma unroll
  for (int f = 0; f < NF; f++) c[f] = v4f{0.f, 0.f, 0.f, 0.f};
  float ss = 0.f;
  char* const mine = lds + wave * kUnitLds;
  const uint8_t* const run = reinterpret_cast<const uint8_t*>(lds) + rows_scales(SRC, NF, waves);
  const auto multiply = [&](Unit& q, int u) {
    if constexpr (SRC != kCodes) {
      const bool live = 256 * u + 4 * lane < K;
      float4 x = q.x;
      if constexpr (SRC == kNormed) {
        if (R.delta) x = plus(x, q.d);
        if (live && R.xout && blockIdx.x == 0 && fw == 0) *reinterpret_cast<float4*>(R.xout + 256 * u + 4 * lane) = x;
        ss += live ? (x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w) : 0.f;
        x.x *= q.nw.x; x.y *= q.nw.y; x.z *= q.nw.z; x.w *= q.nw.w;
      }
      if (!live) x = make_float4(0.f, 0.f, 0.f, 0.f);
      asm volatile("" ::: "memory");                           // (the unit before has been read, in LDS's order)
      put_digits(mine, lane, x);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int b = 8 * u + 4 * h + g;
      int ws[NF];
#pragma unroll
      for (int f = 0; f < NF; f++) ws[f] = b < nb ? run[wscale[f] + b] : 0;
      if constexpr (SRC == kCodes) {
        v8i large, small;
        split_e4m3(row_operand(q.lo[h], q.hi[h]), large, small);
#pragma unroll
        for (int f = 0; f < NF; f++) {
          c[f] = mx_mma(weight_operand(q.w[h][f]), small, c[f], ws[f], (int)q.as[h]);
          c[f] = mx_mma(weight_operand(q.w[h][f]), large, c[f], ws[f], (int)q.as[h]);
        }
      } else {
        const int row = min(r, kDigits - 1);
        const char* s = mine + h * (kDigits * 128) + row * 128 + 16 * g;
        const frag16 lo = *reinterpret_cast<const frag16*>(s), hi = *reinterpret_cast<const frag16*>(s + 64);
        const int field = reinterpret_cast<const uint8_t*>(mine + 2 * kDigits * 128)[4 * h + g];
        const int scale = field == 255 ? 255 : field - 46 + 4 * row;
        const v8i a = row_operand(lo, hi);
#pragma unroll
        for (int f = 0; f < NF; f++) c[f] = mx_mma(weight_operand(q.w[h][f]), a, c[f], ws[f], scale);
      }
    }
  };
  Unit one, two;
  if (kw < units) ask(one, kw);
  {
    const int rows = FW * kTile, bytes = rows * nb, first = (int)blockIdx.x * rows;
    char* const to = lds + (reinterpret_cast<const char*>(run) - lds);
    const int64_t left = (int64_t)(N - first) * nb;
    put_scales<GATED ? 2 : 1>(to, sw + (int64_t)first * nb, (int64_t)N * nb, bytes, left, tid, 64 * waves);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  for (int u = kw; u < units; u += 2 * KW) {
    if (u + KW < units) ask(two, u + KW);
    multiply(one, u);
    if (u + KW < units) {
      if (u + 2 * KW < units) ask(one, u + 2 * KW);
      multiply(two, u + KW);
    }
  }
#pragma unroll
  for (int f = 0; f < NF; f++) mx_done(c[f]);

  // the KW wavefronts' sums, added up in their order: tile f by wavefront f % KW, a gated product's all by the first
  float inv = 1.f;
  const auto my_tile = [&](int f) { return GATED ? kw == 0 : f % KW == kw; };
  if (KW > 1 || SRC == kNormed) {
    __syncthreads();
    char* const sums = lds + fw * (KW * NF) * 1024;
    float* const squares = reinterpret_cast<float*>(lds + waves * NF * 1024);
#pragma unroll
    for (int f = 0; f < NF; f++) *reinterpret_cast<v4f*>(sums + (f * KW + kw) * 1024 + lane * 16) = c[f];
    if constexpr (SRC == kNormed) {
      ss = wave_sum(ss);
      if (lane == 0) squares[wave] = ss;
    }
    __syncthreads();
    if constexpr (SRC == kNormed) {
      float total = 0.f;
      for (int k = 0; k < KW; k++) total += squares[fw * KW + k];
      inv = 1.0f / sqrtf(total / (float)K + R.eps);
    }
#pragma unroll
    for (int f = 0; f < NF; f++) {
      if (!my_tile(f)) continue;
      v4f v = *reinterpret_cast<const v4f*>(sums + f * KW * 1024 + lane * 16);
      for (int k = 1; k < KW; k++) v += *reinterpret_cast<const v4f*>(sums + (f * KW + k) * 1024 + lane * 16);
      c[f] = v;
    }
  }
  if constexpr (SRC != kCodes) {
    // a digit's sums lie in one lane of a row of 16; lane i < 4 of them stores feature 4 g + i
    float out[NF];
#pragma unroll
    for (int f = 0; f < NF; f++)
      if (GATED || my_tile(f)) out[f] = join_digits(c[f], r) * inv;
    const int n = n0 + 4 * g + r;
    if constexpr (GATED) {
      if constexpr (NF == 1) {
        const float up = __shfl(out[0], (lane + 32) & 63);
        if (kw == 0 && r < 4 && g < 2 && n < N) C[n] = gated(out[0], up);
      } else {
#pragma unroll
        for (int f = 0; f < NF / 2; f++)
          if (kw == 0 && r < 4 && n + 16 * f < N) C[n + 16 * f] = gated(out[f], out[f + NF / 2]);
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; f++)
        if (my_tile(f) && r < 4 && n + 16 * f < N) C[n + 16 * f] = out[f];
    }
  } else if constexpr (GATED) {
    if (kw != 0) return;
#pragma unroll
    for (int p = 0; p < NF / 4; p++) {
      const int n = n0 + 32 * p;
      const int64_t at = min(m, M - 1);
      store_gated(c[2 * p], c[2 * p + 1], c[NF / 2 + 2 * p], c[NF / 2 + 2 * p + 1], g, m < M && n < N, codes + at * N + n,
                  scales + at * (N / kMxBlock) + n / kMxBlock);
    }
  } else {
#pragma unroll
    for (int f = 0; f < NF; f++)
      if (my_tile(f) && m < M) store_features(C + (int64_t)m * N, n0 + 16 * f + 4 * g, N, c[f]);
  }
}

template <int SRC, int NF, bool GATED>
static hipError_t launch_rows(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, int64_t M, int64_t N, int64_t K, int KW,
                              int waves, float* C, uint8_t* codes, uint8_t* scales, const MxRow& R) {
  constexpr int kTile = GATED ? 8 * NF : 16 * NF;
  const int lds = rows_scales(SRC, NF, waves) + (GATED ? 2 : 1) * whole_16((int)(waves / KW * kTile * (K / kMxBlock)));
  const auto kernel = mx_rows_kernel<SRC, NF, GATED>;
  if (const hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess) return e;
  const int64_t per_block = (int64_t)kTile * (waves / KW);
  kernel<<<dim3((unsigned)((N + per_block - 1) / per_block), SRC == kCodes ? (unsigned)((M + 15) / 16) : 1u), dim3(64 * waves), lds, ctx().stream>>>(
      A, sa, W, sw, (int)M, (int)N, (int)(K / kMxBlock), KW, waves, C, codes, scales, R);
  return hipGetLastError();
}

// The same product where a block has several tiles' worth of rows: the digits of the row, which every tile meets, stay in LDS, the next
// tile's weights and scales are asked for while this one is multiplied, and blocks walk the tiles without a break. UPW:
// units of 256 k a wavefront has (K up to 256 KW UPW).
template <int SRC, int NF, bool GATED, int UPW>
__global__ __launch_bounds__(512, UPW * NF <= 4 ? 4 : 2) void mx_row_tiles_kernel(const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw, int N, int nb, int KW,
                                                              int tiles, float* __restrict__ y, const MxRow R) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), fw = wave / KW, kw = wave - fw * KW, FW = 8 / KW;
  const int K = nb * kMxBlock;
  constexpr int kTile = GATED ? 8 * NF : 16 * NF, kDigitLds = 8 * UPW * kUnitLds;
  const int rows = FW * kTile, run_bytes = rows * nb, run_stage = ((GATED ? 2 : 1) * run_bytes + 15) & ~15;
  char* const mine = lds + wave * UPW * kUnitLds;
  char* const runs = lds + kDigitLds;
  float* const sums = reinterpret_cast<float*>(runs + 2 * run_stage);      // [2][8 wavefronts][NF][16]
  float* const squares = sums + 2 * 8 * NF * 16;
  frag16 q[UPW][2][NF];
  const uint8_t* row[NF];
  const auto rows_of = [&](int tile) {
    const int n0 = min(tile, tiles - 1) * rows + fw * kTile;
#pragma unroll
    for (int f = 0; f < NF; f++) {
      const TileRow t = tile_row<NF, GATED>(f, r);
      row[f] = W + ((t.up ? (int64_t)N : 0) + min(n0 + t.n, N - 1)) * nb * 16;
    }
  };
  // (both halves of a row's 128 bytes one after the other, and not past the caches: the second finds the line there)
  const auto ask = [&](int j, int f) {
#pragma unroll
    for (int h = 0; h < 2; h++) q[j][h][f] = *reinterpret_cast<const frag16*>(row[f] + (uint32_t)min(8 * (kw + j * KW) + 4 * h + g, nb - 1) * 16u);
  };
  const auto ask_all = [&](int tile) {
    rows_of(tile);
#pragma unroll
    for (int j = 0; j < UPW; j++)
#pragma unroll
      for (int f = 0; f < NF; f++) ask(j, f);
  };
  // scales of a tile, 16 bytes a thread (the launcher sees to it that the run is no more than 512 of those, and whole ones: rows * nb % 16 == 0, N % 16 == 0)
  any16 sc[GATED ? 2 : 1];
  const auto ask_scales = [&](int tile) {
    const int64_t total = (int64_t)N * nb, at = min((int64_t)min(tile, tiles - 1) * run_bytes + min(16 * tid, run_bytes - 16), total - 16);
#pragma unroll
    for (int k = 0; k < (GATED ? 2 : 1); k++) sc[k] = *reinterpret_cast<const any16*>(sw + k * total + at);
  };
  const auto keep_scales = [&](int stage) {
#pragma unroll
    for (int k = 0; k < (GATED ? 2 : 1); k++)
      if (16 * tid < run_bytes) *reinterpret_cast<frag16*>(runs + stage * run_stage + k * run_bytes + 16 * tid) = sc[k];
  };
  int tile = blockIdx.x;
  // my units of the row, its digits kept; squares are of the row before the norm's weights
  float4 x[UPW], d[UPW], nw[UPW];
#pragma unroll
  for (int j = 0; j < UPW; j++) {
    const int k = min(256 * (kw + j * KW) + 4 * lane, K - 4);
    x[j] = *reinterpret_cast<const float4*>(R.x + k);
    if constexpr (SRC == kNormed) {
      d[j] = R.delta ? *reinterpret_cast<const float4*>(R.delta + k) : make_float4(0.f, 0.f, 0.f, 0.f);
      nw[j] = *reinterpret_cast<const float4*>(R.norm_w + k);
    }
  }
  ask_scales(tile);
  if (UPW * NF <= 2) ask_all(tile);               // (more than a unit's weights beside the digits' numbers do not fit the registers)
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < UPW; j++) {
    const int k = 256 * (kw + j * KW) + 4 * lane;
    float4 v = x[j];
    if constexpr (SRC == kNormed) {
      if (R.delta) v = plus(v, d[j]);
      if (k < K && R.xout && blockIdx.x == 0 && fw == 0) *reinterpret_cast<float4*>(R.xout + k) = v;
      ss += k < K ? (v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w) : 0.f;
      v.x *= nw[j].x; v.y *= nw[j].y; v.z *= nw[j].z; v.w *= nw[j].w;
    }
    if (k >= K) v = make_float4(0.f, 0.f, 0.f, 0.f);
    put_digits(mine + j * kUnitLds, lane, v);
  }
  if (UPW * NF > 2) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    ask_all(tile);
  }
  if constexpr (SRC == kNormed) {
    ss = wave_sum(ss);
    if (lane == 0) squares[wave] = ss;
  }
  keep_scales(0);
  float inv = 1.f;
  const int digit = min(r, kDigits - 1);
  const auto meet = [] {          // LDS writes only: what is asked for stays in flight
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  meet();
  if constexpr (SRC == kNormed) {
    float total = 0.f;
    for (int k = 0; k < KW; k++) total += squares[fw * KW + k];
    inv = 1.0f / sqrtf(total / (float)K + R.eps);
  }
  for (int stage = 0; tile < tiles; stage ^= 1) {
    const int next = tile + (int)gridDim.x;
    ask_scales(next);
    rows_of(next);
    const uint8_t* run = reinterpret_cast<const uint8_t*>(runs) + stage * run_stage;
    v4f c[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) c[f] = v4f{0.f, 0.f, 0.f, 0.f};
    // a register that has been multiplied is asked for again: the next tile's weights
#pragma unroll
    for (int j = 0; j < UPW; j++) {
      v8i a[2];
      int scale[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const char* s = mine + j * kUnitLds + h * (kDigits * 128) + digit * 128 + 16 * g;
        const frag16 lo = *reinterpret_cast<const frag16*>(s), hi = *reinterpret_cast<const frag16*>(s + 64);
        const int field = reinterpret_cast<const uint8_t*>(mine + j * kUnitLds + 2 * kDigits * 128)[4 * h + g];
        scale[h] = field == 255 ? 255 : field - 46 + 4 * digit;
        a[h] = row_operand(lo, hi);
      }
#pragma unroll
      for (int f = 0; f < NF; f++) {
        const TileRow t = tile_row<NF, GATED>(f, r);
        const int in_run = (t.up ? run_bytes : 0) + (fw * kTile + t.n) * nb;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int b = 8 * (kw + j * KW) + 4 * h + g, ws = b < nb ? run[in_run + b] : 0;
          c[f] = mx_mma(weight_operand(q[j][h][f]), a[h], c[f], ws, scale[h]);
        }
        ask(j, f);
      }
    }
    float* const part = sums + stage * (8 * NF * 16);
#pragma unroll
    for (int f = 0; f < NF; f++) {
      mx_done(c[f]);
      const float v = join_digits(c[f], r);
      if (r < 4) part[(wave * NF + f) * 16 + 4 * g + r] = v;
    }
    keep_scales(stage ^ 1);
    meet();
    // a row's sums over the KW wavefronts, one row a thread
    if (tid < FW * NF * 16) {
      const int w = tid / (NF * 16), f = tid / 16 % NF, i = tid & 15;
      const auto sum = [&](int i) {
        float v = part[(w * KW * NF + f) * 16 + i];
        for (int k = 1; k < KW; k++) v += part[((w * KW + k) * NF + f) * 16 + i];
        return v * inv;
      };
      const int n = tile * rows + w * kTile + 16 * f + i;
      if constexpr (GATED) {
        static_assert(NF == 1, "gate rows in the lower half of a tile");
        if (i < 8 && n < N) y[n] = gated(sum(i), sum(i + 8));
      } else {
        if (n < N) y[n] = sum(i);
      }
    }
    tile = next;
  }
}

template <int SRC, int NF, bool GATED, int UPW>
static hipError_t launch_row_tiles(const uint8_t* W, const uint8_t* sw, int64_t N, int64_t K, int KW, int per_cu, float* y, const MxRow& R) {
  constexpr int kTile = GATED ? 8 * NF : 16 * NF;
  const int nb = (int)(K / kMxBlock), rows = 8 / KW * kTile, run = rows * nb, lds = 8 * UPW * kUnitLds + 2 * (((GATED ? 2 : 1) * run + 15) & ~15) + (2 * 8 * NF * 16 + 8) * 4;
  const int tiles = (int)((N + rows - 1) / rows);
  const auto kernel = mx_row_tiles_kernel<SRC, NF, GATED, UPW>;
  if (const hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess) return e;
  kernel<<<dim3((unsigned)std::min(tiles, per_cu * cu_count())), dim3(512), lds, ctx().stream>>>(W, sw, (int)N, nb, KW, tiles, y, R);
  return hipGetLastError();
}

// The same product where the weight is small, in the vector unit: blocks of few rows, so that all CUs have some, and no digits to make. A
// wavefront has RW rows of the weight (gated: half of them gate rows, and their up rows), 16 numbers of each in a lane, and every KW-th
// 1024 of k. An element is widened times 2^-8 (so that sixteen products of it with any finite number stay in f32), products are
// summed in one chain per lane and scaled by their block's power of two after that, which is exact. A row with an infinity or a
// NaN gives NaN, as its digits do.
// A plain row's numbers are read by each lane for itself (896 x 4864 3.9 us, staged in LDS by the block 4.0, 3584 x 3584 4.1 and 4.6); what
// goes through a norm is three times as much to read, and staged (896 x 4864 4.3, each lane for itself 4.5; 3584 x 3584 5.6, 7.2).
__device__ __forceinline__ int row_place(int i) { return i + (i >> 4); }       // of float4 i: what lanes read together is in different banks
template <int SRC, int RW, bool GATED>
__global__ __launch_bounds__(1024) void mx_row_small_kernel(const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw, int N, int nb, int KW, int FW,
                                                          float* __restrict__ y, const MxRow R) {
  constexpr int kTile = GATED ? RW / 2 : RW;                   // features of a wavefront
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float sums[16][RW + 1];                           // of rows; of the squares, and NaN for a row that is not finite
  float4* const staged = reinterpret_cast<float4*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, threads = 64 * KW * FW;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), fw = wave / KW, kw = wave - fw * KW;
  const int K = nb * kMxBlock, n4 = K / 4, n0 = ((int)blockIdx.x * FW + fw) * kTile;
  const float4 *x4 = reinterpret_cast<const float4*>(R.x), *d4 = reinterpret_cast<const float4*>(R.delta), *w4 = reinterpret_cast<const float4*>(R.norm_w);
  constexpr int kPre = 2;                                      // of the numbers a thread stages, asked for ahead of the weights
  float4 v[4], x[kPre], d[kPre], nw[kPre];
  MergeIn in[kPre];
  if constexpr (SRC == kMerged) {
#pragma unroll
    for (int p = 0; p < kPre; p++) in[p] = ask_merge(R, 4 * min(tid + p * threads, n4 - 1), lane);
  }
  if constexpr (SRC == kNormed) {
#pragma unroll
    for (int p = 0; p < kPre; p++) {
      const int i = min(tid + p * threads, n4 - 1);
      x[p] = x4[i];
      d[p] = d4 ? d4[i] : make_float4(0.f, 0.f, 0.f, 0.f);
      nw[p] = w4[i];
    }
  }
  uint2 w[RW];
  uint32_t s[RW];
  const auto ask = [&](int k) {
    const int at = min(k, K - 16);
    if constexpr (SRC == kFloat) {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = x4[at / 4 + j];
    }
#pragma unroll
    for (int i = 0; i < RW; i++) {
      const int64_t row = min(n0 + i % kTile, N - 1) + (i < kTile ? (int64_t)0 : (int64_t)N);
      w[i] = *reinterpret_cast<const uint2*>(W + row * nb * 16 + at / 2);
      s[i] = sw[row * nb + at / kMxBlock];
    }
  };
  const int first = 1024 * kw + 16 * lane;
  if constexpr (SRC != kFloat) ask(first);                     // (ahead of the row's staging)
  float ss = 0.f, bad = 0.f;
  const auto look = [&](const float4 a) { bad = fmaf(a.x, 0.f, fmaf(a.y, 0.f, fmaf(a.z, 0.f, fmaf(a.w, 0.f, bad)))); };
  if constexpr (SRC == kMerged) {
    const auto stage = [&](int i, const float4 a) {
      look(a);
      staged[row_place(i)] = a;
    };
#pragma unroll
    for (int p = 0; p < kPre; p++)
      if (tid + p * threads < n4) stage(tid + p * threads, merged(R, in[p], lane));
    for (int i = tid + kPre * threads; i < n4; i += threads) stage(i, merged(R, ask_merge(R, 4 * i, lane), lane));
  }
  if constexpr (SRC == kNormed) {
    const auto stage = [&](int i, float4 a, const float4 b, const float4 c) {
      if (d4) a = plus(a, b);
      if (R.xout && blockIdx.x == 0) reinterpret_cast<float4*>(R.xout)[i] = a;
      ss += (a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w);
      a = make_float4(a.x * c.x, a.y * c.y, a.z * c.z, a.w * c.w);
      look(a);
      staged[row_place(i)] = a;
    };
#pragma unroll
    for (int p = 0; p < kPre; p++)
      if (tid + p * threads < n4) stage(tid + p * threads, x[p], d[p], nw[p]);
    for (int i = tid + kPre * threads; i < n4; i += threads) stage(i, x4[i], d4 ? d4[i] : make_float4(0.f, 0.f, 0.f, 0.f), w4[i]);
  }
  if constexpr (SRC != kFloat) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // (the weights stay in flight)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  float total[RW];
#pragma unroll
  for (int i = 0; i < RW; i++) total[i] = 0.f;
  for (int k = first; k - 16 * lane < K; k += 1024 * KW) {
    if (SRC == kFloat || k != first) ask(k);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (SRC != kFloat) v[j] = staged[row_place(min(k, K - 16) / 4 + j)];
      else look(v[j]);
    }
#pragma unroll
    for (int i = 0; i < RW; i++) {
      float c = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        constexpr float kDown = 0.00390625f;
        const uint32_t q = j < 2 ? w[i].x : w[i].y;
        const v2f a = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, kDown, 2) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, kDown, 0);
        const v2f b = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, kDown, 3) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, kDown, 1);
        c = fmaf(v[j].x, a[0], fmaf(v[j].y, a[1], fmaf(v[j].z, b[0], fmaf(v[j].w, b[1], c))));
      }
      c = s[i] == 255u ? __uint_as_float(0x7fc00000u) : ldexpf(c, (int)s[i] - 119);
      total[i] += k < K ? c : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < RW; i++) {
    const float t = wave_sum(SRC == kFloat ? total[i] + bad : total[i]);
    if (lane == 0) sums[wave][i] = t;
  }
  if constexpr (SRC != kFloat) {
    ss = wave_sum(ss + bad);
    if (lane == 0) sums[wave][RW] = ss;
  }
  __syncthreads();
  if (tid >= FW * kTile) return;
  const int f = tid / kTile, n = (int)blockIdx.x * FW * kTile + tid;
  const auto sum = [&](int wave, int count, int i) {
    float t = sums[wave][i];
    for (int k = 1; k < count; k++) t += sums[wave + k][i];
    return t;
  };
  const float row = SRC != kFloat ? sum(0, KW * FW, RW) : 0.f;                       // (of a merged row: 0 or NaN)
  const float inv = SRC == kNormed ? 1.0f / sqrtf(row / (float)K + R.eps) : 1.f;
  const float a = (sum(f * KW, KW, tid % kTile) + (SRC == kMerged ? row : 0.f)) * inv;
  if (n >= N) return;
  if constexpr (GATED) y[n] = gated(a, sum(f * KW, KW, tid % kTile + kTile) * inv);
  else y[n] = a;
}

template <int SRC, int RW, bool GATED>
static hipError_t launch_row_small(const uint8_t* W, const uint8_t* sw, int64_t N, int64_t K, int KW, int FW, float* y, const MxRow& R) {
  const int64_t rows = FW * (GATED ? RW / 2 : RW);
  const int lds = SRC != kFloat ? (int)(K / 4 + K / 64 + 1) * 16 : 0;
  const auto kernel = mx_row_small_kernel<SRC, RW, GATED>;
  if (const hipError_t e = allow_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess) return e;
  kernel<<<dim3((unsigned)((N + rows - 1) / rows)), dim3(64 * KW * FW), lds, ctx().stream>>>(W, sw, (int)N, (int)(K / kMxBlock), KW, FW, y, R);
  return hipGetLastError();
}

// Which kernel, by sizes (us so, and in the other forms; weights not in any cache; "gated" and "normed" as told, else plain):
//   up to 20 2^20 elements (behind a producer 9 2^20) or 1024 rows (of up to 32768 behind a producer), K from 512, from 896 where there are more
//     than 16384 rows (30000 x 640 5.6, 5.1 in mx_row_tiles_kernel; 20000 x 1024 4.8, 5.6): mx_row_small_kernel, a wavefront for every 1024 k
//     (896 x 4864 3.9, mx_rows_kernel 4.4; 3584 x 3584 4.1, 4.6; 1000 x 18944 5.2, 9.2; beyond, 8192 x 3584 6.0, 5.7. Normed 896 x 4864 4.3,
//     5.1; 9728 x 896 4.3, 4.5, gated 4.4, 4.8; 1000 x 18944 8.6, 12.0; beyond, 3584 x 3584 5.6, 5.1; 20000 x 512 5.0, 4.5). Four rows a
//     wavefront (1000 x 18944 5.2, two 6.2; 3584 x 3584 4.1, 4.4), two where that makes no more blocks than there are CUs (normed
//     896 x 4864 4.3, four 4.5); two sets of wavefronts a block share what is staged.
//   more than 4 tiles of 16 rows for each CU, K up to 4096: mx_row_tiles_kernel (152064 x 3584 51.6, row by row 55.2; 37888 x 3584 14.8, 16.0;
//     9728 x 896, 2.4 tiles: 4.2, 4.2; 16384 x 2048 6.4, 6.1); more than 2 from twelve units of 256 k on, where row by row is a block of
//     sixteen wavefronts a CU (12288 x 3584 7.6, 8.8, normed 8.6, 11.0; 8192 x 3584, 2 tiles: 6.6, 5.7);
//   K up to 1024: as many wavefronts share a row's K as it has units of 256, in several sets (9728 x 896 in two of four 4.2, in eight 4.4;
//     150000 x 64 in eight of one 4.8, in two of four 11.4);
//   up to twelve units of 256 k: eight; beyond: sixteen (3584 x 18944 9.8; eight 10.8; 4608 x 3584 4.8; 5.2), but eight where there are more blocks
//     than CUs, which hold one of sixteen (16384 x 8192 17.2, 19.5; 28672 x 8192 normed 30.4, 38.5; 32768 x 5120 gated 21.5, 30.1);
//   32 rows a block where there are more tiles of 16 than CUs (4608 x 3584 5.1, 16: 5.9; gated 6.6, 8.8; 3584 x 18944 12.9, 16: 9.8), and while
//     the scales of their rows leave room in LDS.
enum { kRowVector = 0, kRowWalk = 1, kRowTiles = 2 };
struct RowPlan {
  int form;                  // mx_row_small_kernel, mx_row_tiles_kernel, mx_rows_kernel
  int rows;                  // of the weight, that a wavefront has at a time
  int KW, waves;             // wavefronts that share a row, of a block
  int units;                 // kRowWalk: of 256 k, that a wavefront has
};
static RowPlan plan_row(int64_t N, int64_t K, int src, bool gated) {
  const int64_t nb = K / kMxBlock, units = (nb + 7) / 8, cus = cu_count();
  const int KW = units <= 1 ? 1 : units <= 2 ? 2 : units <= 4 ? 4 : 8;
  const int64_t rows = (gated ? 8 : 16) * (8 / KW);          // of a tile, gate rows if gated
  const int64_t all = gated ? 2 * N : N;                     // rows of the weight
  const int kw = (int)std::min<int64_t>(16, (K + 1023) / 1024);
  if (src == kFloat) {
    if ((all * K <= (int64_t)20 << 20 || all <= 4 * cus) && K >= 512 && (K >= 896 || all <= 64 * cus)) return RowPlan{kRowVector, 4, kw, kw, 0};
  } else {
    const int sets = kw <= 8 ? 2 : 1;
    if ((all * K <= (int64_t)9 << 20 || all <= 4 * cus) && K >= 512 && K <= 32768)
      return RowPlan{kRowVector, all <= 2 * sets * cus ? 2 : 4, kw, kw * sets, 0};
  }
  if (src != kMerged && units <= 16 && N % 16 == 0 && N > (units > 12 ? 2 : 4) * cus * rows && rows * nb % 16 == 0)
    return RowPlan{kRowWalk, 16, KW, 8, units <= KW ? 1 : 2};
  const bool two = all > 16 * cus && nb <= 1024;
  const int waves = units <= 12 || all > (two ? 32 : 16) * cus ? 8 : 16;
  return RowPlan{kRowTiles, two ? 32 : 16, units <= 8 ? KW : waves, waves, 0};
}

template <int SRC, bool GATED>
static hipError_t launch_row(const uint8_t* W, const uint8_t* sw, int64_t N, int64_t K, float* y, const MxRow& R) {
  const RowPlan P = plan_row(N, K, SRC, GATED);
  if (P.form == kRowVector) {
    if constexpr (SRC == kFloat) return launch_row_small<SRC, 4, false>(W, sw, N, K, P.KW, P.waves / P.KW, y, R);
    else return (P.rows == 2 ? launch_row_small<SRC, 2, GATED> : launch_row_small<SRC, 4, GATED>)(W, sw, N, K, P.KW, P.waves / P.KW, y, R);
  }
  if constexpr (SRC != kMerged)
    if (P.form == kRowWalk)
      return (P.units == 1 ? launch_row_tiles<SRC, 1, GATED, 1> : launch_row_tiles<SRC, 1, GATED, 2>)(W, sw, N, K, P.KW, 2, y, R);
  return (P.rows == 32 ? launch_rows<SRC, 2, GATED> : launch_rows<SRC, 1, GATED>)(nullptr, nullptr, W, sw, 1, N, K, P.KW, P.waves, y, nullptr, nullptr, R);
}

bool mx_few_rows_fit(int64_t N, int64_t K, bool gated) {
  // (a gated block has the scales of 64 rows in LDS beside 32 KB of sums)
  return !gated || 64 * (K / kMxBlock) <= 120 * 1024;
}
// 16 rows of the weight a block, 32 where there would be more blocks than CUs (77 x 896 x 4864 7.4 us, with 16 8.9)
int mx_few_rows_tiles(int64_t M, int64_t N, int64_t K) { return (N + 15) / 16 * ((M + 15) / 16) > cu_count() && K <= 32768 ? 2 : 1; }
// Up to a block on each CU it takes 2.9 us and 27 ns for each KB that a block reads, of both operands; up to two blocks twice that, beyond which
// tiles that share what they read are ahead (measured 17 to 256 rows by 896 x 896 to 4608 x 3584: 48 x 896 x 4864 5.6, estimated 6.0, in
// tiles 6.9; 112 x 1152 x 896 3.7, 3.9, 5.3; 48 x 3584 x 3584 9.7, 9.1, 9.1).
double mx_few_rows_us(int64_t M, int64_t N, int64_t K) {
  const int64_t nf = mx_few_rows_tiles(M, N, K), blocks = (N + 16 * nf - 1) / (16 * nf) * ((M + 15) / 16), cus = cu_count();
  if (blocks > 2 * cus) return M <= kMxFewRows ? 0 : 1e30;
  return 2.9 + (double)((blocks + cus - 1) / cus) * (double)(nf * K * 17 / 2 + std::min<int64_t>(M, 16) * K) / 1024 * 0.027;
}
hipError_t launch_mx_few_rows(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, int64_t M, int64_t N, int64_t K, float* C,
                              uint8_t* codes, uint8_t* scales) {
  const int64_t units = (K + 255) / 256;
  const int KW = units <= 1 ? 1 : units <= 2 ? 2 : units <= 4 ? 4 : 8;
  if (codes) return launch_rows<kCodes, 4, true>(A, sa, W, sw, M, N, K, KW, KW, C, codes, scales, MxRow{});
  return (mx_few_rows_tiles(M, N, K) == 2 ? launch_rows<kCodes, 2, false> : launch_rows<kCodes, 1, false>)(A, sa, W, sw, M, N, K, KW, KW, C, nullptr, nullptr,
                                                                                                  MxRow{});
}

}  // namespace tlhip

using namespace tlhip;

static const uint8_t* bytes(const void* p) { return static_cast<const uint8_t*>(p); }

extern "C" {

int tlhip_gemv_mxfp4(const void* a, const void* codes, const void* scales, void* y, int64_t N, int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemv_mxfp4";
  if (const int rc = check_mx_product(who, a, scales, codes, scales, y, 1, N, K, 4)) return rc;
  if (const int rc = check_mx_apart(who, y, {a, codes, scales})) return rc;
  const MxRow R{static_cast<const float*>(a), nullptr, nullptr, nullptr, 0.f, 0, 0, 0};
  const hipError_t e = launch_row<kFloat, false>(bytes(codes), bytes(scales), N, K, static_cast<float*>(y), R);
  if (e != hipSuccess) return hip_fail(e, who);
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMV_MXFP4);
}

int tlhip_gemv_mxfp4_attn(const void* parts, int64_t n_parts, int64_t heads, int64_t head_dim, const void* codes, const void* scales, void* y,
                          int64_t N, int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemv_mxfp4_attn";
  if (const int rc = check_mx_product(who, parts, scales, codes, scales, y, 1, N, K, 4)) return rc;
  if (const int rc = check_attn_merge(parts, n_parts, heads, head_dim, K, who)) return rc;
  if (const int rc = check_mx_apart(who, y, {parts, codes, scales})) return rc;
  const MxRow R{static_cast<const float*>(parts), nullptr, nullptr, nullptr, 0.f, (int)n_parts, (int)heads, (int)head_dim};
  const hipError_t e = launch_row<kMerged, false>(bytes(codes), bytes(scales), N, K, static_cast<float*>(y), R);
  if (e != hipSuccess) return hip_fail(e, who);
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMV_MXFP4);
}

static int normed(const char* who, const void* x, const void* delta, const void* norm_w, void* xout, const void* codes, const void* scales, void* y,
                  int64_t N, int64_t K, float eps, bool gate) {
  if (const int rc = check_mx_product(who, x, scales, codes, scales, y, 1, N, K, 4)) return rc;
  if (!norm_w) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (!aligned16(delta) || !aligned16(norm_w) || !aligned16(xout)) return fail(TLHIP_EINVAL, "%s: delta, norm_w and xout must be 16-byte aligned", who);
  if (xout && (xout == x || xout == delta)) return fail(TLHIP_EINVAL, "%s: xout must not alias x or delta", who);
  if (const int rc = check_mx_apart(who, y, {x, delta, norm_w, xout, codes, scales})) return rc;
  if (xout)
    if (const int rc = check_mx_apart(who, xout, {norm_w, codes, scales})) return rc;
  const MxRow R{static_cast<const float*>(x), static_cast<const float*>(delta), static_cast<const float*>(norm_w), static_cast<float*>(xout), eps,
                0, 0, 0};
  const hipError_t e = (gate ? launch_row<kNormed, true> : launch_row<kNormed, false>)(bytes(codes), bytes(scales), N, K, static_cast<float*>(y), R);
  if (e != hipSuccess) return hip_fail(e, who);
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMV_MXFP4);
}

int tlhip_gemv_mxfp4_rmsnorm(const void* x, const void* delta, const void* norm_w, void* xout, const void* codes, const void* scales, void* y,
                             int64_t N, int64_t K, float eps) {
  TLHIP_REQUIRE_READY();
  return normed("tlhip_gemv_mxfp4_rmsnorm", x, delta, norm_w, xout, codes, scales, y, N, K, eps, false);
}

int tlhip_gemv_mxfp4_rmsnorm_gateup(const void* x, const void* delta, const void* norm_w, void* xout, const void* codes, const void* scales, void* act,
                                    int64_t N2, int64_t K, float eps) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemv_mxfp4_rmsnorm_gateup";
  if (N2 % 2) return fail(TLHIP_EINVAL, "%s: need as many gate rows as up rows", who);
  return normed(who, x, delta, norm_w, xout, codes, scales, act, N2 / 2, K, eps, true);
}

int tlhip_plan_gemv_mxfp4(int64_t N, int64_t K, int producer, int gated, int plan[5]) {
  const char* who = "tlhip_plan_gemv_mxfp4";
  if (!plan || N <= 0 || !mx_row(K) || producer < 0 || producer > 2 || (gated && producer != 1)) return fail(TLHIP_EINVAL, "%s: bad arguments", who);
  if (N > (1 << 24) || K > kMxMaxK) return fail(TLHIP_EUNSUPPORTED, "%s: dimension too large", who);
  const RowPlan P = plan_row(N, K, producer == 0 ? kFloat : producer == 1 ? kNormed : kMerged, gated != 0);
  plan[0] = P.form;
  plan[1] = P.rows;
  plan[2] = P.KW;
  plan[3] = P.waves;
  plan[4] = P.units;
  return TLHIP_OK;
}

}  // extern "C"
