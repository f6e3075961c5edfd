// Products over MXFP4 weights (mx_formats.hpp): of one f32 row, and of MXFP8 rows, on the scaled matrix instructions.
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
#include "mx_formats.hpp"
#include "gemv_shared.hpp"

#include <algorithm>

namespace tlhip {

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
    const uint32_t w = (uint32_t)a[i], t = w & 0x40404040u;
    const uint32_t keep = (t << 1) + (0x80808080u - (t >> 6));        // bytes 0xff where bit 6 is set, else 0x80
    large[i] = (int)(w & keep);
    small[i] = (int)(w & (~keep | 0x80808080u));
  }
}
__device__ __forceinline__ v4f mx_mma_both(const v8i w, const v8i a, v4f c, int sw, int sa) {
  v8i large, small;
  split_e4m3(a, large, small);
  c = mx_mma(w, small, c, sw, sa);
  return mx_mma(w, large, c, sw, sa);
}

// One wavefront: 16 features (GU: 32 gate and the 32 up ones) by 16 tokens, operands straight from memory.
// What lies past the end of a row is the row's last block again under the scale 2^-127 on both sides: 2^-254 times at most 32 x 448 x 6,
// which is 0 in f32.
struct MxFrag { v8i v; int s; };
__device__ __forceinline__ MxFrag mx_weight(const uint8_t* W, const uint8_t* scales, int64_t row, int nb, int b) {
  const int at = min(b, nb - 1);
  const uint4 c = *reinterpret_cast<const uint4*>(W + (row * nb + at) * 16);
  return MxFrag{v8i{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0}, b < nb ? (int)scales[row * nb + at] : 0};
}
__device__ __forceinline__ MxFrag mx_act(const uint8_t* A, const uint8_t* scales, int64_t row, int nb, int b0, int g) {
  const int64_t K = (int64_t)nb * 32;
  const int c0 = min(2 * b0 + g, 2 * nb - 1), c1 = min(2 * b0 + 4 + g, 2 * nb - 1);        // 16-byte chunks of the row
  const uint4 lo = *reinterpret_cast<const uint4*>(A + row * K + 16 * c0), hi = *reinterpret_cast<const uint4*>(A + row * K + 16 * c1);
  return MxFrag{v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w},
                b0 + g < nb ? (int)scales[row * nb + b0 + g] : 0};
}

__global__ __launch_bounds__(64) void mx_gemm_simple_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ sa,
                                                            const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw,
                                                            float* __restrict__ C, int M, int N, int nb) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m = blockIdx.y * 16 + r;
  const int64_t wr = min(n0 + r, N - 1), ar = min(m, M - 1);
  v4f c = {0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < nb; b += 4) {
    const MxFrag w = mx_weight(W, sw, wr, nb, b + g), a = mx_act(A, sa, ar, nb, b, g);
    c = mx_mma_both(w.v, a.v, c, w.s, a.s);
  }
  mx_done(c);
  if (m >= M) return;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (n0 + 4 * g + i < N) C[(int64_t)m * N + n0 + 4 * g + i] = c[i];
}

// 32 features: two tiles of 16; token l % 16's block of 32 activations lies in the four lanes with that l % 16
__global__ __launch_bounds__(64) void mx_gated_simple_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ sa,
                                                             const uint8_t* __restrict__ W, const uint8_t* __restrict__ sw,
                                                             uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int M, int ff, int nb) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  const int f0 = blockIdx.x * 32, m = blockIdx.y * 16 + r;
  const int64_t ar = min(m, M - 1);
  v4f c[4];
#pragma unroll
  for (int t = 0; t < 4; t++) c[t] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < nb; b += 4) {
    const MxFrag a = mx_act(A, sa, ar, nb, b, g);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const MxFrag w = mx_weight(W, sw, f0 + 16 * (t & 1) + r + (t >> 1) * (int64_t)ff, nb, b + g);
      c[t] = mx_mma_both(w.v, a.v, c[t], w.s, a.s);
    }
  }
#pragma unroll
  for (int t = 0; t < 4; t++) mx_done(c[t]);
  float v[8];
  uint32_t big = 0;
#pragma unroll
  for (int t = 0; t < 8; t++) {
    v[t] = gated(c[t >> 2][t & 3], c[2 + (t >> 2)][t & 3]);
    big = max(big, magnitude(v[t]));
  }
  big = max(big, (uint32_t)__shfl_xor((int)big, 16, kWave));
  big = max(big, (uint32_t)__shfl_xor((int)big, 32, kWave));
  const uint32_t s = mx_scale_of(big, kMx8Exp);
  const float up = mx_up(min(s, 252u));
#pragma unroll
  for (int t = 0; t < 8; t++) v[t] = s == 255u ? 0.f : v[t] * up;
  if (m >= M) return;
#pragma unroll
  for (int t = 0; t < 2; t++)
    *reinterpret_cast<uint32_t*>(codes + (int64_t)m * ff + f0 + 16 * t + 4 * g) = to_e4m3x4(v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]);
  if (g == 0) scales[(int64_t)m * (ff / kMxBlock) + blockIdx.x] = (uint8_t)s;
}

// One wavefront a row of the weight
__global__ __launch_bounds__(256) void mx_gemv_simple_kernel(const float* __restrict__ a, const uint8_t* __restrict__ W,
                                                             const uint8_t* __restrict__ sw, float* __restrict__ y, int N, int nb) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  float sum = 0.f;
  for (int b = lane; b < nb; b += 64) {
    const uint4 c = *reinterpret_cast<const uint4*>(W + (n * nb + b) * 16);
    const uint32_t d[4] = {c.x, c.y, c.z, c.w};
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float* x = a + 32 * b + 8 * i;
      const v2f w0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 0), w1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 1);
      const v2f w2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 2), w3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 3);
      p = fmaf(w0[0], x[0], fmaf(w0[1], x[1], fmaf(w1[0], x[2], fmaf(w1[1], x[3], p))));
      p = fmaf(w2[0], x[4], fmaf(w2[1], x[5], fmaf(w3[0], x[6], fmaf(w3[1], x[7], p))));
    }
    sum = fmaf(p, mx_scale(sw[n * nb + b]), sum);
  }
  sum = wave_sum(sum);
  if (lane == 0) y[n] = sum;
}

static int check_product(const char* who, const void* a, const void* sa, const void* W, const void* sw, const void* out, int64_t M, int64_t N,
                         int64_t K) {
  if (!a || !sa || !W || !sw || !out) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (M <= 0 || N <= 0 || !mx_row(K)) return fail(TLHIP_EINVAL, "%s: need M, N > 0, K a positive multiple of 32", who);
  if (!aligned16(a) || !aligned16(W) || !aligned16(out)) return fail(TLHIP_EINVAL, "%s: elements and result must be 16-byte aligned", who);
  if (M > (1 << 20) || N > (1 << 24) || K > (1 << 20)) return fail(TLHIP_EUNSUPPORTED, "%s: M, K up to 2^20, N up to 2^24", who);
  return TLHIP_OK;
}

}  // namespace tlhip

using namespace tlhip;

extern "C" {

int tlhip_gemv_mxfp4(const void* a, const void* codes, const void* scales, void* y, int64_t N, int64_t K) {
  TLHIP_REQUIRE_READY();
  if (const int rc = check_product("tlhip_gemv_mxfp4", a, scales, codes, scales, y, 1, N, K)) return rc;
  mx_gemv_simple_kernel<<<dim3((unsigned)((N + 3) / 4)), dim3(256), 0, ctx().stream>>>(
      static_cast<const float*>(a), static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<float*>(y), (int)N,
      (int)(K / 32));
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMV_MXFP4);
}

int tlhip_gemm_mxfp4_nt_parts(const void* acodes, const void* ascales, const void* codes, const void* scales, void* parts, int64_t parts_bytes,
                              int64_t M, int64_t N, int64_t K, int* n_parts) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemm_mxfp4_nt_parts";
  if (const int rc = check_product(who, acodes, ascales, codes, scales, parts, M, N, K)) return rc;
  if (!n_parts) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (parts_bytes < M * N * 4) return fail(TLHIP_EINVAL, "%s: the parts need M * N * 4 bytes at least", who);
  mx_gemm_simple_kernel<<<dim3((unsigned)((N + 15) / 16), (unsigned)((M + 15) / 16)), dim3(64), 0, ctx().stream>>>(
      static_cast<const uint8_t*>(acodes), static_cast<const uint8_t*>(ascales), static_cast<const uint8_t*>(codes),
      static_cast<const uint8_t*>(scales), static_cast<float*>(parts), (int)M, (int)N, (int)(K / 32));
  *n_parts = 1;
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMM_MXFP4);
}

int tlhip_gemm_mxfp4_nt(const void* acodes, const void* ascales, const void* codes, const void* scales, void* C, int64_t M, int64_t N,
                        int64_t K) {
  TLHIP_REQUIRE_READY();
  if (const int rc = check_product("tlhip_gemm_mxfp4_nt", acodes, ascales, codes, scales, C, M, N, K)) return rc;
  mx_gemm_simple_kernel<<<dim3((unsigned)((N + 15) / 16), (unsigned)((M + 15) / 16)), dim3(64), 0, ctx().stream>>>(
      static_cast<const uint8_t*>(acodes), static_cast<const uint8_t*>(ascales), static_cast<const uint8_t*>(codes),
      static_cast<const uint8_t*>(scales), static_cast<float*>(C), (int)M, (int)N, (int)(K / 32));
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMM_MXFP4);
}

int tlhip_gemm_mxfp4_nt_swiglu(const void* acodes, const void* ascales, const void* codes, const void* scales, void* act_codes,
                               void* act_scales, int64_t M, int64_t ff, int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_gemm_mxfp4_nt_swiglu";
  if (const int rc = check_product(who, acodes, ascales, codes, scales, act_codes, M, ff, K)) return rc;
  if (!act_scales) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (!mx_row(ff)) return fail(TLHIP_EINVAL, "%s: ff must be a multiple of 32", who);
  mx_gated_simple_kernel<<<dim3((unsigned)(ff / 32), (unsigned)((M + 15) / 16)), dim3(64), 0, ctx().stream>>>(
      static_cast<const uint8_t*>(acodes), static_cast<const uint8_t*>(ascales), static_cast<const uint8_t*>(codes),
      static_cast<const uint8_t*>(scales), static_cast<uint8_t*>(act_codes), static_cast<uint8_t*>(act_scales), (int)M, (int)ff, (int)(K / 32));
  TLHIP_CHECK_LAUNCH(TLHIP_C_GEMM_MXFP4);
}

}  // extern "C"
