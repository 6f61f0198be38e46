// Residual addition, RMSNorm and per-token 8-bit codes in one pass over a row:
//   s     = x + residual                        (fp32; residual_out = s rounded to x's type)
//   y     = s * rsqrt(mean(s^2) + eps) * weight (fp32; the norm reads s before its rounding)
//   scale = max(max|y|, 1e-5) / top * clip      top = 127 (int8) or 448 (e4m3)
//   code  = clamp(rint(y / scale), -128, 127)   or  y / scale rounded to e4m3, saturating
// The row is loaded once and stays in registers as fp32 through both reductions (sum of squares,
// abs-max), so what moves is x, the residual in and out, one byte a value and four a row.
//
// Measured at 32760 x 5120 bf16 with residual: int8 180 us (6.51 TB/s on 7 bytes a value, 1.01 of the copy rate), e4m3 203 us;
// fp16 without residual int8 119 us (4.2 TB/s: the schedulers issue in 76 % of their cycles, the code conversions among it; codes by
// a reciprocal alone, off by one beside a border, took 110), e4m3 143 us.  Rows whose length or address allows no
// 128-bit access move one value an access: 20000 x 5121 with residual 439 us, four times the copy.  Worst case: a
// row of equal values in e4m3 is all largest values (32760 x 5120: 381 us).
//
// e4m3 codes are those of the exact quotient: its midpoints are 2^-4 of a value apart, so among millions of values
// some always lie within the fp32 roundings of one, and a code on the wrong side is a step of 6 %.  So every value is
// converted twice, with the reciprocal of the scale nudged up and down by 2^-20; the roundings on the way to a quotient (s and
// two products, the same for the largest value, scale, reciprocal, product: ten halves of 2^-23) are less.  A value with two
// codes (one in 2^15) is read again and decided in 64 bits, against the
// row's largest |s * weight|, of which 64 bits are kept too; the rsqrt cancels.  The largest is sought among all values
// within 2^-20 of the fp32 maximum, whose order three roundings each may have changed (2^-21.4).  In a row whose scale is the
// least one (max|y| <= 1e-5, or so near that 64 bits have to tell) the rsqrt does not cancel: it is computed again in 64
// bits, by each thread that needs it, and the nudges are 2^-18, for the sum of squares is off by up to 77 halves of 2^-23.
//
// A row whose sum of squares or whose y is not finite has no meaningful codes: its scale is NaN
// (whatever is computed from it shows it) and its codes are 0.  So it is for a row whose mean square and eps add up to less
// than the least normal number (squares below it have lost bits, or are 0), and for a scale without a normal reciprocal.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "quant_act.cuh"  // Chunk, row_reduce

namespace b200w4a4 {

enum : int { CODES_INT8 = 0, CODES_E4M3 = 1 };

struct RmsNormArgs {
  const void* x;         // [M, D], row pitch x_ld elements
  const void* residual;  // same type, row pitch r_ld, or null
  const void* weight;    // [D] of type w_dtype
  void* codes;           // [M, D] bytes
  float* scale;          // [M]
  void* residual_out;    // [M, D] of x's type, or null with residual
  long long x_ld, r_ld;
  float eps, clip;
  int w_dtype, format, M, D;
};

namespace detail {

__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ void store_f32(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }

// Eight values stored in x's type with one or two 128-bit stores.
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Eight weights; the weight vector is shared by every row, so it goes through the read-only cache.
template <typename W>
__device__ __forceinline__ void weight8(const W* p, float (&w)[8]) {
  if constexpr (sizeof(W) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    Chunk<W> c;
    c.raw = __ldg(reinterpret_cast<const uint4*>(p));
    c.values(w);
  }
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// the e4m3 value nearest to num / den (den > 0), a quotient near a midpoint; compared without dividing, so ties are seen
__device__ __forceinline__ float nearest_e4m3(double num, double den) {
  const double a = fabs(num);
  const float t = static_cast<float>(a / den);
  float low, next;  // the neighbours
  bool odd;
  if (t < 0.015625f) {  // steps of 2^-9
    const float step = floorf(t * 512.0f);
    low = step * 0.001953125f;
    next = (step + 1.0f) * 0.001953125f;
    odd = (static_cast<int>(step) & 1) != 0;
  } else {
    const uint32_t bits = __float_as_uint(t) & 0xfff00000u;
    low = __uint_as_float(bits);
    next = __uint_as_float(bits + 0x100000u);
    odd = (bits & 0x100000u) != 0;
  }
  const double mid = 0.5 * (static_cast<double>(low) + static_cast<double>(next)) * den;
  const bool up = a > mid || (a == mid && odd);  // ties to the even one
  return copysignf(up ? next : low, static_cast<float>(num));
}
__device__ __forceinline__ uint32_t code_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace detail

// TPR threads share a row and hold NCH * 8 of its values each.  VEC: eight consecutive values a
// chunk, moved with 128-bit accesses (D, pitches and addresses allow it).  Otherwise a chunk is
// eight values TPR apart and every access moves one value, coalesced across the threads.
template <typename T, int TPR, int NCH, bool VEC, bool E4M3>
__global__ void __launch_bounds__(256, NCH <= 5 ? 4 : 2) rms_norm_quant_kernel(const RmsNormArgs a) {
  constexpr int ROWS = 256 / TPR;
  __shared__ float red[2][8];
  __shared__ unsigned long long top64[8];  // a row's largest |s * weight| in 64 bits (e4m3)
  const int sub = threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const long long row = static_cast<long long>(blockIdx.x) * ROWS + sub;
  const bool row_ok = row < a.M;
  const T* xr = static_cast<const T*>(a.x) + (row_ok ? row : 0) * a.x_ld;
  const T* rr = static_cast<const T*>(a.residual);
  if (rr != nullptr) rr += (row_ok ? row : 0) * a.r_ld;
  T* ro = static_cast<T*>(a.residual_out) + row * a.D;
  // Cleared by the row's own first thread: the barriers of the row's reductions (for one warp a row, which reduces with
  // shuffles alone, the barrier of that warp) stand between this and the row's maxima.
  if constexpr (E4M3) {
    if (t == 0) top64[sub] = 0ull;
    if constexpr (TPR == 32) __syncwarp();
  }
  auto at = [&](int i, int e) { return VEC ? 8 * (t + i * TPR) + e : (8 * i + e) * TPR + t; };

  float v[NCH][8];
  float ss = 0.0f;
  if constexpr (VEC) {
    detail::Chunk<T> cx[NCH], cr[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (row_ok && at(i, 0) < a.D) cx[i].load(xr + at(i, 0));
    if (rr != nullptr) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        if (row_ok && at(i, 0) < a.D) cr[i].load(rr + at(i, 0));
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (row_ok && at(i, 0) < a.D) {
        cx[i].values(v[i]);
        if (rr != nullptr) {
          float r[8];
          cr[i].values(r);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] += r[e];
          detail::store8(ro + at(i, 0), v[i]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = row_ok && at(i, e) < a.D ? detail::load_f32(xr + at(i, e)) : 0.0f;
    if (rr != nullptr && row_ok) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float r[8];  // a chunk's loads come before its stores
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = at(i, e) < a.D ? detail::load_f32(rr + at(i, e)) : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[i][e] += r[e];
          if (at(i, e) < a.D) detail::store_f32(ro + at(i, e), v[i][e]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  ss = row_reduce<TPR, false>(ss, red[0], sub);
  const float mean = ss / static_cast<float>(a.D) + a.eps;
  const float rstd = rsqrtf(mean);

  float amax = 0.0f;
  auto normalise = [&](const auto* weight) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float w[8];
      if constexpr (VEC) {
        if (at(i, 0) >= a.D) continue;  // zeros
        detail::weight8(weight + at(i, 0), w);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = at(i, e) < a.D ? detail::load_f32(weight + at(i, e)) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = v[i][e] * rstd * w[e];
        amax = detail::max_nan(amax, fabsf(v[i][e]));
      }
    }
  };
  if (a.w_dtype == XDT_F16) normalise(static_cast<const __half*>(a.weight));
  else if (a.w_dtype == XDT_BF16) normalise(static_cast<const __nv_bfloat16*>(a.weight));
  else normalise(static_cast<const float*>(a.weight));
  // a NaN must survive the reduction too: it travels as +inf, which no finite row reaches
  if (!(amax < INFINITY)) amax = INFINITY;
  amax = row_reduce<TPR, true>(amax, red[1], sub);
  [[maybe_unused]] const bool least = amax < 1.0001e-5f;
  const float top = E4M3 ? 448.0f : 127.0f;
  const float s = __fmul_rn(__fdiv_rn(fmaxf(amax, 1e-5f), top), a.clip);
  constexpr float kLeast = 1.17549435e-38f, kMost = 8.5070592e37f;  // 2^-126, 2^126
  const bool good = ss < INFINITY && amax < INFINITY && (mean >= kLeast || amax == 0.0f) && s >= kLeast && s <= kMost;  // false for NaN
  [[maybe_unused]] float inv_up = 0.0f, inv_dn = 0.0f;
  if constexpr (E4M3) {
    const float inv = __fdiv_rn(1.0f, s), nudge = least ? 3.8146973e-06f : 9.5367432e-07f;  // 2^-18, 2^-20
    inv_up = inv * (1.0f + nudge);
    inv_dn = inv * (1.0f - nudge);
  }
  [[maybe_unused]] const detail::RowQuant rq = detail::row_quant_of<127>(s, a.clip);
  uint8_t* q = static_cast<uint8_t*>(a.codes) + (row_ok ? row : 0) * a.D;
  // e4m3: which of this thread's values may be the row's largest, and which lie near a midpoint
  constexpr int MW = E4M3 ? (NCH + 3) / 4 : 1;
  uint32_t largest[MW] = {}, near[MW] = {};
  [[maybe_unused]] const float near_top = amax * 0.99999905f;
  if (row_ok && t == 0) a.scale[row] = good ? s : __int_as_float(0x7fc00000);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    [[maybe_unused]] uint32_t c[8];  // int8 codes: low bytes
    [[maybe_unused]] uint32_t up[2];  // e4m3 codes, four a word
    if constexpr (E4M3) {
      uint32_t apart = 0, dn[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float* u = v[i] + 4 * h;
        up[h] = detail::code_e4m3x2(u[0] * inv_up, u[1] * inv_up) | detail::code_e4m3x2(u[2] * inv_up, u[3] * inv_up) << 16;
        dn[h] = detail::code_e4m3x2(u[0] * inv_dn, u[1] * inv_dn) | detail::code_e4m3x2(u[2] * inv_dn, u[3] * inv_dn) << 16;
        apart |= up[h] ^ dn[h];
      }
      if (apart != 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if ((up[e / 4] ^ dn[e / 4]) >> (8 * (e % 4)) & 0xff) near[i / 4] |= 1u << (8 * (i % 4) + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (fabsf(v[i][e]) >= near_top) largest[i / 4] |= 1u << (8 * (i % 4) + e);
    } else {
      detail::chunk_codes<127>(v[i], rq, c);
    }
    if constexpr (VEC) {
      if (at(i, 0) >= a.D) continue;
      uint2 o = make_uint2(0u, 0u);
      if (good) {
        if constexpr (E4M3) {
          o = make_uint2(up[0], up[1]);
        } else {
          o.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
          o.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
        }
      }
      if (row_ok) *reinterpret_cast<uint2*>(q + at(i, 0)) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (at(i, e) >= a.D) continue;
        uint32_t code = 0;
        if constexpr (E4M3) code = up[e / 4] >> (8 * (e % 4));
        else code = c[e];
        if (row_ok) q[at(i, e)] = static_cast<uint8_t>(good ? code : 0u);
      }
    }
  }
  if constexpr (E4M3) {
    auto sum64 = [&](int c) {  // one value of s, read again
      const double s64 = static_cast<double>(detail::load_f32(xr + c));
      return rr != nullptr ? s64 + static_cast<double>(detail::load_f32(rr + c)) : s64;
    };
    auto product64 = [&](int c) {  // s * weight
      const double s64 = sum64(c);
      if (a.w_dtype == XDT_F16) return s64 * static_cast<double>(detail::load_f32(static_cast<const __half*>(a.weight) + c));
      if (a.w_dtype == XDT_BF16) return s64 * static_cast<double>(detail::load_f32(static_cast<const __nv_bfloat16*>(a.weight) + c));
      return s64 * static_cast<double>(detail::load_f32(static_cast<const float*>(a.weight) + c));
    };
    const bool decide = row_ok && good && amax > 0.0f;  // in a row of zeros every value is the largest
    unsigned long long mine = 0;  // positive 64-bit floats order as integers
#pragma unroll
    for (int m = 0; m < MW; ++m)
      for (uint32_t left = decide ? largest[m] : 0u; left != 0; left &= left - 1) {
        const int k = 32 * m + __ffs(left) - 1, c = at(k >> 3, k & 7);
        if (c < a.D) mine = max(mine, static_cast<unsigned long long>(__double_as_longlong(fabs(product64(c)))));
      }
    if (mine != 0) atomicMax(&top64[sub], mine);
    __syncthreads();
    double den = __longlong_as_double(static_cast<long long>(top64[sub])) * static_cast<double>(a.clip);
    uint32_t any = 0;
#pragma unroll
    for (int m = 0; m < MW; ++m) any |= near[m];
    if (decide && least && any != 0) {  // |y| <= 1e-5 in the units of |s * weight|
      double ss64 = 0.0;
      for (int c = 0; c < a.D; ++c) ss64 = fma(sum64(c), sum64(c), ss64);
      den = fmax(den, 1e-5 * static_cast<double>(a.clip) * sqrt(ss64 / a.D + static_cast<double>(a.eps)));
    }
#pragma unroll
    for (int m = 0; m < MW; ++m)
      for (uint32_t left = decide ? near[m] : 0u; left != 0; left &= left - 1) {
        const int k = 32 * m + __ffs(left) - 1, c = at(k >> 3, k & 7);
        if (c >= a.D) continue;
        const double num = product64(c) * 448.0;
        if (fabs(num) < 448.0 * den)
          q[c] = static_cast<uint8_t>(detail::code_e4m3x2(detail::nearest_e4m3(num, den), 0.0f));
      }
  }
}

constexpr int kRmsNormMaxD = 16384;  // a row stays in the registers of 256 threads

template <typename T, bool VEC, bool E4M3>
inline cudaError_t launch_rms_norm_quant_as(const RmsNormArgs& a, cudaStream_t stream) {
#define B200W4A4_RMS_LAUNCH(TPR, NCH)                                                             \
  do {                                                                                             \
    constexpr int ROWS = 256 / (TPR);                                                              \
    const unsigned grid = static_cast<unsigned>((static_cast<long long>(a.M) + ROWS - 1) / ROWS);  \
    rms_norm_quant_kernel<T, TPR, NCH, VEC, E4M3><<<grid, 256, 0, stream>>>(a);                          \
  } while (0)
  const int chunks = (a.D + 7) / 8;
  // Threads a row by its length; four blocks of 256 threads an SM while 40 values a thread allow it (32760 x 5120 fp16
  // without residual: 119 us, 155 with 24 values and 256 threads a row).
  if (chunks <= 32) B200W4A4_RMS_LAUNCH(32, 1);
  else if (chunks <= 32 * 3) B200W4A4_RMS_LAUNCH(32, 3);
  else if (chunks <= 64 * 3) B200W4A4_RMS_LAUNCH(64, 3);
  else if (chunks <= 128 * 3) B200W4A4_RMS_LAUNCH(128, 3);
  else if (chunks <= 128 * 5) B200W4A4_RMS_LAUNCH(128, 5);
  else if (chunks <= 256 * 3) B200W4A4_RMS_LAUNCH(256, 3);
  else if (chunks <= 256 * 5) B200W4A4_RMS_LAUNCH(256, 5);
  else B200W4A4_RMS_LAUNCH(256, 8);
#undef B200W4A4_RMS_LAUNCH
  return cudaGetLastError();
}

template <typename T, bool VEC>
inline cudaError_t launch_rms_norm_quant(const RmsNormArgs& a, cudaStream_t stream) {
  return a.format == CODES_E4M3 ? launch_rms_norm_quant_as<T, VEC, true>(a, stream)
                                : launch_rms_norm_quant_as<T, VEC, false>(a, stream);
}

}  // namespace b200w4a4
