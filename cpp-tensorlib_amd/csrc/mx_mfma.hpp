// Products over MXFP4 weights (mx_formats.hpp) on the scaled matrix instructions: what gemm_mx.hip (MXFP8 rows) and gemv_mx.hip (few of
// them, or one f32 row) share.
//
// C[m][n] = sum over blocks b of 2^(sa + sw - 254) sum over 32 of a w: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows of
// 128 e2m1 elements by 16 rows of 128 e4m3 ones, each block of 32 with its own scale byte, into f32 sums. Lane l holds row l % 16 of both
// operands; with g = l / 16 its 16 bytes of e2m1 are k = 32 g .. 32 g + 31, its 32 bytes of e4m3 k = 16 g .. + 15 and 64 + 16 g
// .. + 15, and its scale bytes are those of block g. The weight is the first operand: lane l's four results are features 4 g .. 4 g + 3 of token
// l % 16, one 16-byte store.
//
// The instruction adds the products of eight neighbouring k to the precision of the largest of them: whatever of a product lies
// more than 13 binades below the sum of that one's exponents is cut off (measured: 2688 + 0.125 keeps the 0.125, 2688 + 0.0625
// does not; a random product over 18944 is 1.4e-5 off, f32 sums 3e-8). e4m3 spans 18 binades, so activations go in twice, the elements of
// at least 2 (bit 6 of the byte: exponent field 8 to 15) and the others apart. Of the first a product's last bit is 2^-2 x 2^-1 at
// least, the largest exponents add up to 8 + 2; of the others 2^-9 x 2^-1 and 0 + 2: nothing is cut off in either, and sums
// of eight and more are f32. Half the instruction's rate is what that costs.
//
// What lies past the end of a row is the row's last block again under the scale 2^-127 on both sides: 2^-254 times at most
// 32 x 448 x 6, which is 0 in f32.
#pragma once

#include <initializer_list>

#include "gemm_shared.hpp"
#include "gemv_shared.hpp"
#include "mx_formats.hpp"

namespace tlhip {

// Arguments of a product, as its entry point `who` checks them. K: what the weight's scales of 16 rows leave room for in LDS. align: of
// the result's address, 4 where it is stored number by number.
constexpr int64_t kMxMaxK = 65536;
inline int check_mx_product(const char* who, const void* a, const void* sa, const void* W, const void* sw, const void* out, int64_t M, int64_t N,
                            int64_t K, int align = 16) {
  if (!a || !sa || !W || !sw || !out) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (M <= 0 || N <= 0 || !mx_row(K)) return fail(TLHIP_EINVAL, "%s: need M, N > 0, K a positive multiple of 32", who);
  if (!aligned16(a) || !aligned16(W)) return fail(TLHIP_EINVAL, "%s: elements must be 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(out) % align) return fail(TLHIP_EINVAL, "%s: the result must be %d-byte aligned", who, align);
  if (M > (1 << 20) || N > (1 << 24) || K > kMxMaxK) return fail(TLHIP_EUNSUPPORTED, "%s: M up to 2^20, N up to 2^24, K up to 65536", who);
  if (M * N > (int64_t)1 << 37) return fail(TLHIP_EUNSUPPORTED, "%s: results of up to 2^37 numbers", who);
  return TLHIP_OK;
}

// out: written by some blocks while others read the rest
inline int check_mx_apart(const char* who, const void* out, std::initializer_list<const void*> operands) {
  for (const void* p : operands)
    if (p == out) return fail(TLHIP_EINVAL, "%s: the result must not be written over an operand", who);
  return TLHIP_OK;
}

// More than 64 KB of LDS a block (some of it static) has to be asked for
inline hipError_t allow_lds(const void* kernel, int lds) {
  return lds > 60 * 1024 ? hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) : hipSuccess;
}

// gemv_mx.hip: rows of MXFP8 by a weight, 16 of them a block; codes non-null: gated, [gate | up] rows of N each, into MXFP8 (up to
// kMxFewRows rows). mx_few_rows_us: what it takes without the gate, nothing where no other kernel reads the weight as fast.
constexpr int kMxFewRows = 16;
double mx_few_rows_us(int64_t M, int64_t N, int64_t K);
bool mx_few_rows_fit(int64_t N, int64_t K, bool gated);
int mx_few_rows_tiles(int64_t M, int64_t N, int64_t K);      // of 16 features, that a block has
hipError_t launch_mx_few_rows(const uint8_t* A, const uint8_t* sa, const uint8_t* W, const uint8_t* sw, int64_t M, int64_t N, int64_t K, float* C,
                              uint8_t* codes, uint8_t* scales);

#if defined(__HIPCC__)
__device__ __forceinline__ v4f mx_mma(const v8i w, const v8i a, const v4f c, int sw, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 4, 0, 0, sw, 0, sa);
}

// Keeps the instructions that formed c ahead of what follows. They read the registers of all 64 lanes, but the compiler holds them
// to be free to move: where only some lanes need a result it has put one under their branch, operands prepared there for
// those lanes only.
__device__ __forceinline__ void mx_done(v4f& c) { asm volatile("" : "+v"(c)); }

// The elements of at least 2 of a register of e4m3, and the others (zeros elsewhere, signs in both)
__device__ __forceinline__ void split_e4m3(const v8i a, v8i& large, v8i& small) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    // bytes 0xff where bit 6 is set: the permutation's selectors 8 to 11 spread the top bits of bytes 1, 3 (the second word's), 5 and 7
    const uint32_t w = (uint32_t)a[i], is = __builtin_amdgcn_perm(w << 1, w << 9, 0x0b090a08);
    large[i] = (int)(w & (is | 0x80808080u));
    small[i] = (int)(w & (~is | 0x80808080u));
  }
}
__device__ __forceinline__ v8i weight_operand(const frag16& w) { return v8i{(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0}; }
__device__ __forceinline__ v8i row_operand(const frag16& lo, const frag16& hi) {
  return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// What gemv_shared.hpp's gated() is, on the hardware's exponential and reciprocal (1 ulp each): e^-g = 2^t, t = -g log2 e in two terms, the
// lower one as the first two of its series; from t = 128 on 0. The reciprocal knows no subnormal numbers: it is of (1 + e^-g) / 4.
// As far from 64 bits as the exact operations are (4.7e-8 in the mean over gates of order one, 2.6e-7 at most; those 4.7e-8, 2.8e-7), in
// thirteen instructions instead of more than thirty: 1280 x 4160 gated x 96 15.0 us instead of 17.4, 2048 x 18944 x 3584 422 instead
// of 431 (with the results read back, 3.7 and 18 of them).
__device__ __forceinline__ float gated_fast(float g, float u) {
  const float t = g * -1.44269502f, r = fmaf(g, -1.92596299e-8f, fmaf(g, -1.44269502f, -t));
  float e = __builtin_amdgcn_exp2f(t);
  e = fabsf(t) < 128.f ? fmaf(e, r * 0.693147182f, e) : e;
  return g * 0.25f * __builtin_amdgcn_rcpf(fmaf(e, 0.25f, 0.25f)) * u;
}

// Gated activations of a token, features 4 g .. 4 g + 3 of two tiles of 16 (gates g0, g1, up values u0, u1): a block of 32, the lanes
// of one l % 16, as MXFP8
__device__ __forceinline__ void store_gated(const v4f& g0, const v4f& g1, const v4f& u0, const v4f& u1, int g, bool live, uint8_t* codes,
                                            uint8_t* scale) {
  float v[8];
  uint32_t big = 0;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    v[k] = gated_fast(g0[k], u0[k]);
    v[4 + k] = gated_fast(g1[k], u1[k]);
    big = max(big, max(magnitude(v[k]), magnitude(v[4 + k])));
  }
  const auto by16 = __builtin_amdgcn_permlane16_swap(big, big, false, false);      // with the lane 16 away, then 32
  big = max(by16[0], by16[1]);
  const auto by32 = __builtin_amdgcn_permlane32_swap(big, big, false, false);
  big = max(by32[0], by32[1]);
  const uint32_t s = mx_scale_of(big, kMx8Exp);
  const float up = mx_up(min(s, 252u));
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] = s == 255u ? 0.f : v[k] * up;
  if (live) {
    reinterpret_cast<uint32_t*>(codes)[g] = to_e4m3x4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint32_t*>(codes)[4 + g] = to_e4m3x4(v[4], v[5], v[6], v[7]);
    if (g == 0) *scale = (uint8_t)s;
  }
}

// Features n .. n + 3 of a token's row of N (whose address is a multiple of 16 bytes, or of 4 where N is no multiple of 4)
typedef float any4f __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void store_features(float* row, int n, int N, const v4f& v) {
  if (n >= N) return;
  if ((N & 3) == 0) *reinterpret_cast<v4f*>(row + n) = v;
  else if (n + 4 <= N) *reinterpret_cast<any4f*>(row + n) = v;
  else
    for (int k = 0; k < 4; k++)
      if (n + k < N) row[n + k] = v[k];
}
#endif

}  // namespace tlhip
