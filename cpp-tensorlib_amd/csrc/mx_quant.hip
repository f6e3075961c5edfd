// Rows into the microscaled formats and back: weights as a model file holds them to MXFP4, f32 activations to MXFP8, the
// RMS norm with the residual's addition whose result is MXFP8.
//
// A block of 32 has the scale 2^e, e the exponent of its largest magnitude less 2 (e2m1) or 8 (e4m3), and every element is the
// value over that, exact, rounded to nearest even. Nothing but the largest magnitude is shared, so a block's bytes depend on
// its own 32 values only. All of it is bound by memory: 18957 x 3584 bf16 rounded and read back as bf16 62 us, 5.5 TB/s where a
// copy reaches 5.35 (two or four times eight values a lane: 64, 65); 2048 x 18944 f32 to MXFP8 34 us.
#include "mx_formats.hpp"

#include <algorithm>

namespace tlhip {

// eight consecutive values, 16-byte aligned
template <int T> struct Eight;
template <> struct Eight<TLHIP_T_F32> {
  typedef float type;
  static __device__ __forceinline__ void load(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <> struct Eight<TLHIP_T_F16> {
  typedef uint16_t type;
  static __device__ __forceinline__ void load(const uint16_t* p, float (&v)[8]) {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    const half8 h = *reinterpret_cast<const half8*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)h[i];
  }
};
template <> struct Eight<TLHIP_T_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ void load(const uint16_t* p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = bf16_lo(d[i]); v[2 * i + 1] = bf16_hi(d[i]); }
  }
  static __device__ __forceinline__ void store(uint16_t* p, const float (&v)[8]) {
    uint4 w;
    w.x = f32_to_bf16_rne(v[0]) | (uint32_t)f32_to_bf16_rne(v[1]) << 16;
    w.y = f32_to_bf16_rne(v[2]) | (uint32_t)f32_to_bf16_rne(v[3]) << 16;
    w.z = f32_to_bf16_rne(v[4]) | (uint32_t)f32_to_bf16_rne(v[5]) << 16;
    w.w = f32_to_bf16_rne(v[6]) | (uint32_t)f32_to_bf16_rne(v[7]) << 16;
    *reinterpret_cast<uint4*>(p) = w;
  }
};

// Scale byte of the block whose 32 values four neighbouring lanes hold, eight each
__device__ __forceinline__ uint32_t quad_scale(const float (&v)[8], int largest) {
  uint32_t big = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) big = max(big, magnitude(v[i]));
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0xB1, 0xf, 0xf, true));   // quad_perm [1,0,3,2]
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x4E, 0xf, 0xf, true));   // quad_perm [2,3,0,1]
  return mx_scale_of(big, largest);
}
// The eight elements a lane writes; those of a block that reads as NaN are zeros.
__device__ __forceinline__ void scaled(float (&v)[8], uint32_t s) {
  const float up = mx_up(min(s, 252u));
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = s == 255u ? 0.f : v[i] * up;
}

// A lane takes eight values. (Eights past the end: the lanes of a block leave together, 32 values being four lanes'.)
template <int T, bool FP4>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const typename Eight<T>::type* __restrict__ src, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, int64_t eights) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= eights) return;
  float v[8];
  Eight<T>::load(src + 8 * i, v);
  const uint32_t s = quad_scale(v, FP4 ? kMx4Exp : kMx8Exp);
  scaled(v, s);
  if constexpr (FP4)
    reinterpret_cast<uint32_t*>(codes)[i] = to_e2m1x8(v);
  else
    reinterpret_cast<uint2*>(codes)[i] = make_uint2(to_e4m3x4(v[0], v[1], v[2], v[3]), to_e4m3x4(v[4], v[5], v[6], v[7]));
  if ((i & 3) == 0) scales[i >> 2] = (uint8_t)s;
}

template <int T, bool FP4>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            typename Eight<T>::type* __restrict__ dst, int64_t eights) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= eights) return;
  const float f = mx_scale(scales[i >> 2]);
  float v[8];
  if constexpr (FP4) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[i];
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const v2f c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  } else {
    const uint2 w = reinterpret_cast<const uint2*>(codes)[i];
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
    const v2f c = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  }
#pragma unroll
  for (int k = 0; k < 8; k++) v[k] *= f;
  Eight<T>::store(dst + 8 * i, v);
}

// Sum over the wavefront, in every lane
template <int CTRL>
__device__ __forceinline__ double dpp_read_f64(double v) {
  const long long b = __double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xf, 0xf, true), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  const auto halves = [](double d, auto swap) {
    const long long b = __double_as_longlong(d);
    const auto lo = swap((uint32_t)b), hi = swap((uint32_t)(b >> 32));
    return __longlong_as_double((long long)(((uint64_t)hi[0] << 32) | lo[0])) + __longlong_as_double((long long)(((uint64_t)hi[1] << 32) | lo[1]));
  };
  v = halves(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  v = halves(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  v += dpp_read_f64<0x128>(v);   // row_ror:8, 4, 2, 1
  v += dpp_read_f64<0x124>(v);
  v += dpp_read_f64<0x122>(v);
  v += dpp_read_f64<0x121>(v);
  return v;
}

// xout = x + (parts[0] + parts[1] + ...), h = xout / sqrt(mean(xout^2) + eps) * w, h as MXFP8: a block per row, a thread V times eight numbers,
// which stay in its registers. The statistic and h are formed in 64 bits and h is rounded to f32 once: an element next to the border
// between two codes then falls on the same side however the sum is split, so a row's bytes do not depend on the launch's shape.
// One row of 896 4.6 to 5.1 us from machine to machine (with the row in LDS and the sum through shuffles 0.7 more; an empty launch is 3.3), 301 of 3584 with three parts
// 7.1 (a copy's rate would be 4.2 beside the launch), 2048 of 8192 with two 58, 5.0 TB/s. Sixteen numbers a thread where eight would do: 301 of 3584
// with three parts 6.0 instead of 6.4 in a queue of launches, but 257 with two 4.8 instead of 4.5, 2048 of 8192 60 instead of 58.
template <int V>
__global__ __launch_bounds__(1024) void rmsnorm_mxfp8_kernel(const float* x, const float* __restrict__ parts, int S, const float* __restrict__ w,
                                                             float* xout, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int n,
                                                             double eps, double each) {
  __shared__ double red[16];
  const int64_t r = blockIdx.x, all = (int64_t)gridDim.x * n, row = r * n;
  const int tid = threadIdx.x, threads = blockDim.x;
  float v[V][8], g[V][8];
  double ss = 0;
#pragma unroll
  for (int k = 0; k < V; k++) {
    const int i = min(8 * (tid + k * threads), n - 8);          // (past the end: the last eight again, not counted, not stored)
    Eight<TLHIP_T_F32>::load(x + row + i, v[k]);
    Eight<TLHIP_T_F32>::load(w + i, g[k]);
    if (S > 0) {
      float t[8];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float4 d = sum_parts(S, [&](int s) { return *reinterpret_cast<const float4*>(parts + s * all + row + i + 4 * h); });
        t[4 * h] = d.x; t[4 * h + 1] = d.y; t[4 * h + 2] = d.z; t[4 * h + 3] = d.w;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) v[k][e] += t[e];
    }
  }
#pragma unroll
  for (int k = 0; k < V; k++) {
    const int i = 8 * (tid + k * threads);
    if (i < n) {
      if (xout) Eight<TLHIP_T_F32>::store(xout + row + i, v[k]);
#pragma unroll
      for (int e = 0; e < 8; e++) ss += (double)v[k][e] * v[k][e];
    }
  }
  ss = wave_sum_f64(ss);
  if (threads > 64) {
    if ((tid & 63) == 0) red[tid >> 6] = ss;
    __syncthreads();
    ss = 0;
    for (int k = 0; k < threads / 64; k++) ss += red[k];
  }
  const double inv = rsqrt(ss * each + eps);       // (each: 1 / n)
#pragma unroll
  for (int k = 0; k < V; k++) {
    const int i = 8 * (tid + k * threads);
#pragma unroll
    for (int e = 0; e < 8; e++) v[k][e] = (float)((double)v[k][e] * inv * (double)g[k][e]);
    const uint32_t s = quad_scale(v[k], kMx8Exp);
    scaled(v[k], s);
    if (i < n) {
      *reinterpret_cast<uint2*>(codes + row + i) = make_uint2(to_e4m3x4(v[k][0], v[k][1], v[k][2], v[k][3]), to_e4m3x4(v[k][4], v[k][5], v[k][6], v[k][7]));
      if ((tid & 3) == 0) scales[(row + i) / kMxBlock] = (uint8_t)s;
    }
  }
}
constexpr int64_t kNormMax = 32768;      // numbers of a row that 1024 threads hold, 32 each

template <int T, bool FP4>
static void launch_quantize(const void* src, void* codes, void* scales, int64_t eights) {
  // (a grid's x counts threads in 32 bits: at most 2^31 a launch)
  for (int64_t e0 = 0; e0 < eights; e0 += (int64_t)1 << 31) {
    const int64_t n = std::min<int64_t>(eights - e0, (int64_t)1 << 31);
    mx_quantize_kernel<T, FP4><<<dim3((unsigned)((n + 255) / 256)), dim3(256), 0, ctx().stream>>>(
        static_cast<const typename Eight<T>::type*>(src) + 8 * e0, static_cast<uint8_t*>(codes) + (FP4 ? 4 : 8) * e0,
        static_cast<uint8_t*>(scales) + e0 / 4, n);
  }
}

template <bool FP4>
static int dequantize(const char* who, const void* codes, const void* scales, void* dst, int dst_type, int64_t rows, int64_t K) {
  if (!codes || !scales || !dst) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (dst_type != TLHIP_T_F32 && dst_type != TLHIP_T_BF16) return fail(TLHIP_EUNSUPPORTED, "%s: element type %d", who, dst_type);
  if (rows <= 0 || !mx_row(K)) return fail(TLHIP_EINVAL, "%s: need rows > 0, K a positive multiple of 32", who);
  if (!aligned16(codes) || !aligned16(dst)) return fail(TLHIP_EINVAL, "%s: codes and dst must be 16-byte aligned", who);
  if (rows > ((int64_t)1 << 50) / K) return fail(TLHIP_EUNSUPPORTED, "%s: too many elements", who);
  if (dst == codes || dst == scales) return fail(TLHIP_EINVAL, "%s: dst must not be what it is read from", who);
  const int64_t eights = rows * K / 8;
  for (int64_t e0 = 0; e0 < eights; e0 += (int64_t)1 << 31) {
    const int64_t n = std::min<int64_t>(eights - e0, (int64_t)1 << 31);
    const dim3 grid((unsigned)((n + 255) / 256)), block(256);
    const uint8_t* c = static_cast<const uint8_t*>(codes) + (FP4 ? 4 : 8) * e0;
    const uint8_t* s = static_cast<const uint8_t*>(scales) + e0 / 4;
    if (dst_type == TLHIP_T_F32)
      mx_dequantize_kernel<TLHIP_T_F32, FP4><<<grid, block, 0, ctx().stream>>>(c, s, static_cast<float*>(dst) + 8 * e0, n);
    else
      mx_dequantize_kernel<TLHIP_T_BF16, FP4><<<grid, block, 0, ctx().stream>>>(c, s, static_cast<uint16_t*>(dst) + 8 * e0, n);
  }
  TLHIP_CHECK_LAUNCH(TLHIP_C_QUANTIZE_MX);
}

}  // namespace tlhip

using namespace tlhip;

extern "C" {

int tlhip_quantize_mxfp4(const void* src, int src_type, void* codes, void* scales, int64_t rows, int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_quantize_mxfp4";
  if (!src || !codes || !scales) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (src_type != TLHIP_T_F32 && src_type != TLHIP_T_F16 && src_type != TLHIP_T_BF16)
    return fail(TLHIP_EUNSUPPORTED, "%s: element type %d", who, src_type);
  if (rows <= 0 || !mx_row(K)) return fail(TLHIP_EINVAL, "%s: need rows > 0, K a positive multiple of 32", who);
  if (!aligned16(src) || !aligned16(codes)) return fail(TLHIP_EINVAL, "%s: src and codes must be 16-byte aligned", who);
  if (rows > ((int64_t)1 << 50) / K) return fail(TLHIP_EUNSUPPORTED, "%s: too many elements", who);
  if (src == codes || src == scales || codes == scales) return fail(TLHIP_EINVAL, "%s: src, codes and scales must not be the same", who);
  const int64_t eights = rows * K / 8;
  if (src_type == TLHIP_T_F32) launch_quantize<TLHIP_T_F32, true>(src, codes, scales, eights);
  else if (src_type == TLHIP_T_F16) launch_quantize<TLHIP_T_F16, true>(src, codes, scales, eights);
  else launch_quantize<TLHIP_T_BF16, true>(src, codes, scales, eights);
  TLHIP_CHECK_LAUNCH(TLHIP_C_QUANTIZE_MX);
}

int tlhip_quantize_mxfp8(const void* x, void* codes, void* scales, int64_t rows, int64_t K) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_quantize_mxfp8";
  if (!x || !codes || !scales) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (rows <= 0 || !mx_row(K)) return fail(TLHIP_EINVAL, "%s: need rows > 0, K a positive multiple of 32", who);
  if (!aligned16(x) || !aligned16(codes)) return fail(TLHIP_EINVAL, "%s: x and codes must be 16-byte aligned", who);
  if (rows > ((int64_t)1 << 50) / K) return fail(TLHIP_EUNSUPPORTED, "%s: too many elements", who);
  if (x == codes || x == scales || codes == scales) return fail(TLHIP_EINVAL, "%s: x, codes and scales must not be the same", who);
  launch_quantize<TLHIP_T_F32, false>(x, codes, scales, rows * K / 8);
  TLHIP_CHECK_LAUNCH(TLHIP_C_QUANTIZE_MX);
}

int tlhip_dequantize_mxfp4(const void* codes, const void* scales, void* dst, int dst_type, int64_t rows, int64_t K) {
  TLHIP_REQUIRE_READY();
  return dequantize<true>("tlhip_dequantize_mxfp4", codes, scales, dst, dst_type, rows, K);
}

int tlhip_dequantize_mxfp8(const void* codes, const void* scales, void* dst, int dst_type, int64_t rows, int64_t K) {
  TLHIP_REQUIRE_READY();
  return dequantize<false>("tlhip_dequantize_mxfp8", codes, scales, dst, dst_type, rows, K);
}

int tlhip_rmsnorm_res_mxfp8(const void* x, const void* parts, int64_t S, const void* w, void* xout, void* codes, void* scales, int64_t n,
                            float eps, int64_t rows) {
  TLHIP_REQUIRE_READY();
  const char* who = "tlhip_rmsnorm_res_mxfp8";
  if (!x || !w || !codes || !scales || (S > 0 && !parts)) return fail(TLHIP_EINVAL, "%s: null pointer", who);
  if (rows <= 0 || !mx_row(n)) return fail(TLHIP_EINVAL, "%s: need rows > 0, n a positive multiple of 32", who);
  if (S < 0 || S > 64 || n > kNormMax || rows > (1 << 20))
    return fail(TLHIP_EUNSUPPORTED, "%s: at most 64 parts, 2^20 rows of 32768", who);
  if (!aligned16(x) || !aligned16(parts) || !aligned16(w) || !aligned16(xout) || !aligned16(codes))
    return fail(TLHIP_EINVAL, "%s: x, parts, w, xout and codes must be 16-byte aligned", who);
  // a row's block writes while the blocks of other rows read: xout may be x, of which each block has its own row, and nothing else
  const void *read[] = {x, w, S > 0 ? parts : nullptr}, *written[] = {xout, codes, scales};
  for (int i = 0; i < 3; i++) {
    for (int j = i == 0 ? 1 : 0; j < 3; j++)
      if (written[i] && written[i] == read[j]) return fail(TLHIP_EINVAL, "%s: what is written must not be what is read, but xout x", who);
    for (int j = 0; j < i; j++)
      if (written[i] == written[j]) return fail(TLHIP_EINVAL, "%s: xout, codes and scales must not be the same", who);
  }
  const int64_t eights = n / 8, V = eights <= 1024 ? 1 : eights <= 2048 ? 2 : 4, threads = ((eights + V - 1) / V + 63) / 64 * 64;
  const auto kernel = V == 1 ? rmsnorm_mxfp8_kernel<1> : V == 2 ? rmsnorm_mxfp8_kernel<2> : rmsnorm_mxfp8_kernel<4>;
  kernel<<<dim3((unsigned)rows), dim3((unsigned)threads), 0, ctx().stream>>>(
      static_cast<const float*>(x), static_cast<const float*>(parts), (int)S, static_cast<const float*>(w), static_cast<float*>(xout),
      static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), (int)n, (double)eps, 1.0 / (double)n);
  TLHIP_CHECK_LAUNCH(TLHIP_C_RMSNORM_RES);
}

}  // extern "C"
