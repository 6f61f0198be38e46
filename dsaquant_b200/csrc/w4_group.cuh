// A few tokens times a 4-bit weight with group scales:
//   y[m,n] = act_scale[m] * sum_g scale[n,g] * sum_{k in g} x[m,k] * code[n,k] + bias[n]
// packed: row-major nibbles [N, K/2] (code 2b in the low, 2b+1 in the high nibble, two's complement),
// scale: fp16 [N, K/group].  x: fp16, bf16, or int8 with one fp32 scale a token.
//
// With so few tokens the weight is all that counts: it is read once, 16 rows and 128 codes of each
// a warp at a time, straight from its row-major form into the A fragments of mma.sync (the weight
// rows are the M of the tile, the tokens its N = 8).  tcgen05 would need 128 rows of widened codes in
// shared memory for the same 8 columns; here a code is widened in the register that feeds the product,
// and at one to sixteen tokens the tensor pipe is idle most of the time either way.
// The dot product's order of k is free as long as x follows it, so the words are used as they lie:
//   fp16 / bf16: nibbles (i, i+4) of a word become a pair by one mask, or'ed under the exponent of
//                1024 (fp16) or 128 (bf16), and an exact subtraction leaves the code;
//   int8:        word << 4 and word, masked with 0xF0F0F0F0, are bytes of 16 * code (the 16 goes
//                into the scale, exactly).
// Products of one group are summed by the tensor core in fp32 (int32 for int8), then enter the fp32
// total with the group's scale.  The warps of a CTA share its rows and split K; their totals are
// added in shared memory in a fixed order.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200w4a4 {

struct W4GroupArgs {
  const void* x;           // [M, K]
  const uint8_t* packed;   // [N, K/2]
  const __half* scale;     // [N, K/group]
  const float* act_scale;  // [M] (int8 x) or null
  const void* bias;        // [N] of the output type or null
  void* out;               // [M, N]
  int M, N, K, group;
  bool out_bf16;
};

namespace detail {

template <typename X>
struct W4Mma;

// D += A * B, A 16 x 16 (weights), B 16 x 8 (tokens)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight codes of a word as four pairs: p[i] = (code i, code i + 4).  u = code + 8 is a plain nibble.
__device__ __forceinline__ void widen(uint32_t word, uint32_t (&p)[4], __half) {
  const uint32_t u = word ^ 0x88888888u, v = u >> 8;
  const __half2 one = __half2half2(__ushort_as_half(0x6408));        // 1032
  const __half2 by = __half2half2(__ushort_as_half(0x2c00));         // 1/16
  const __half2 off = __half2half2(__ushort_as_half(0xd480));        // -72
  uint32_t w[4] = {(u & 0x000f000fu) | 0x64006400u, (u & 0x00f000f0u) | 0x64006400u,
                   (v & 0x000f000fu) | 0x64006400u, (v & 0x00f000f0u) | 0x64006400u};
  __half2* h = reinterpret_cast<__half2*>(w);
  h[0] = __hsub2(h[0], one);          // (1024 + u) - 1032
  h[1] = __hfma2(h[1], by, off);      // (1024 + 16 u) / 16 - 72
  h[2] = __hsub2(h[2], one);
  h[3] = __hfma2(h[3], by, off);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = w[i];
}
__device__ __forceinline__ void widen(uint32_t word, uint32_t (&p)[4], __nv_bfloat16) {
  const uint32_t u = word ^ 0x88888888u;
  const __nv_bfloat162 off = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));  // 136
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = ((u >> (4 * i)) & 0x000f000fu) | 0x43004300u;  // 128 + u
    __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&w), off);
    p[i] = *reinterpret_cast<uint32_t*>(&h);
  }
}

template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  } else if constexpr (WORDS == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));  // the next word's load finds the other half of the sector in L1
  }
}

}  // namespace detail

constexpr int kW4Warps = 8;

// GB: codes that are sure to share a scale (32, 64 or 128; a divisor of the group).  A superblock is
// 128 codes of a row; lane (g, t) holds the run of GB / 4 codes at t * GB / 4 of each of its 128 / GB
// parts, for rows g and g + 8 of each of the RT row tiles.  NT: tiles of 8 tokens.
template <typename X, int GB, int RT, int NT>
__global__ void __launch_bounds__(32 * kW4Warps) w4_group_kernel(const W4GroupArgs a) {
  constexpr bool S8 = sizeof(X) == 1;
  constexpr int PARTS = 128 / GB;
  constexpr int WORDS = GB / 32;  // words of a lane's run
  constexpr int U = RT == 1 ? 4 : 2;  // superblocks in flight
  __shared__ float total[kW4Warps][RT * 16][NT * 8 + 1];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * (RT * 16);
  const int tok0 = blockIdx.y * (NT * 8);
  const int nsb = (a.K + 127) >> 7;
  const int ngroups = a.K / a.group;
  const X* x = static_cast<const X*>(a.x);

  // rows behind the last one repeat it: nothing of theirs is stored
  const uint8_t* wp[2 * RT];
  const __half* sp[2 * RT];
#pragma unroll
  for (int r = 0; r < 2 * RT; ++r) {
    const long long row = min(row0 + g + 8 * r, a.N - 1);
    wp[r] = a.packed + row * (a.K >> 1) + t * (GB / 8);
    sp[r] = a.scale + row * ngroups;
  }

  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;

  for (int sb0 = warp; sb0 < nsb; sb0 += kW4Warps * U) {
    uint32_t w[U][2 * RT][PARTS][WORDS];
    float s[U][2 * RT][PARTS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k0 = (sb0 + u * kW4Warps) << 7;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const int k = k0 + p * GB;
        if (k < a.K) {
          const int grp = k / a.group;
#pragma unroll
          for (int r = 0; r < 2 * RT; ++r) {
            detail::load_words<WORDS>(wp[r] + (k >> 1), w[u][r][p]);
            s[u][r][p] = __half2float(__ldg(sp[r] + grp));
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k0 = (sb0 + u * kW4Warps) << 7;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const int k = k0 + p * GB;
        if (k >= a.K) continue;  // the same for the whole warp
        if constexpr (S8) {
          int part[RT][NT][4];
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) part[r][n][i] = 0;
#pragma unroll
          for (int j = 0; j < WORDS; ++j) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int tok = tok0 + 8 * n + g;
              uint2 v = make_uint2(0u, 0u);
              if (tok < a.M)
                v = __ldg(reinterpret_cast<const uint2*>(x + static_cast<long long>(tok) * a.K + k + t * (GB / 4) + 8 * j));
              const uint32_t b0 = __byte_perm(v.x, v.y, 0x6420), b1 = __byte_perm(v.x, v.y, 0x7531);
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const uint32_t w0 = w[u][2 * r][p][j], w1 = w[u][2 * r + 1][p][j];
                const uint32_t f[4] = {(w0 << 4) & 0xF0F0F0F0u, (w1 << 4) & 0xF0F0F0F0u, w0 & 0xF0F0F0F0u, w1 & 0xF0F0F0F0u};
                detail::mma_s8(part[r][n], f, b0, b1);
              }
            }
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float s0 = s[u][2 * r][p] * 0.0625f, s1 = s[u][2 * r + 1][p] * 0.0625f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[r][n][0] = fmaf(s0, static_cast<float>(part[r][n][0]), acc[r][n][0]);
              acc[r][n][1] = fmaf(s0, static_cast<float>(part[r][n][1]), acc[r][n][1]);
              acc[r][n][2] = fmaf(s1, static_cast<float>(part[r][n][2]), acc[r][n][2]);
              acc[r][n][3] = fmaf(s1, static_cast<float>(part[r][n][3]), acc[r][n][3]);
            }
          }
        } else {
          float part[RT][NT][4];
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) part[r][n][i] = 0.0f;
#pragma unroll
          for (int j = 0; j < WORDS; ++j) {
            uint32_t c[2 * RT][4];
#pragma unroll
            for (int r = 0; r < 2 * RT; ++r) detail::widen(w[u][r][p][j], c[r], X());
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int tok = tok0 + 8 * n + g;
              uint4 v = make_uint4(0u, 0u, 0u, 0u);
              if (tok < a.M)
                v = __ldg(reinterpret_cast<const uint4*>(x + static_cast<long long>(tok) * a.K + k + t * (GB / 4) + 8 * j));
              const uint32_t b[4] = {__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                     __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632)};
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const uint32_t f0[4] = {c[2 * r][0], c[2 * r + 1][0], c[2 * r][1], c[2 * r + 1][1]};
                const uint32_t f1[4] = {c[2 * r][2], c[2 * r + 1][2], c[2 * r][3], c[2 * r + 1][3]};
                detail::mma_f16(part[r][n], f0, b[0], b[1], X());
                detail::mma_f16(part[r][n], f1, b[2], b[3], X());
              }
            }
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float s0 = s[u][2 * r][p], s1 = s[u][2 * r + 1][p];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[r][n][0] = fmaf(s0, part[r][n][0], acc[r][n][0]);
              acc[r][n][1] = fmaf(s0, part[r][n][1], acc[r][n][1]);
              acc[r][n][2] = fmaf(s1, part[r][n][2], acc[r][n][2]);
              acc[r][n][3] = fmaf(s1, part[r][n][3], acc[r][n][3]);
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      total[warp][16 * r + g][8 * n + 2 * t] = acc[r][n][0];
      total[warp][16 * r + g][8 * n + 2 * t + 1] = acc[r][n][1];
      total[warp][16 * r + g + 8][8 * n + 2 * t] = acc[r][n][2];
      total[warp][16 * r + g + 8][8 * n + 2 * t + 1] = acc[r][n][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < RT * 16 * NT * 8; i += 32 * kW4Warps) {
    const int r = i % (RT * 16), n = i / (RT * 16);
    const int row = row0 + r, tok = tok0 + n;
    if (row >= a.N || tok >= a.M) continue;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kW4Warps; ++w) y += total[w][r][n];
    if (a.act_scale != nullptr) y *= a.act_scale[tok];
    const long long o = static_cast<long long>(tok) * a.N + row;
    if (a.out_bf16) {
      if (a.bias != nullptr) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[row]);
      static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(y);
    } else {
      if (a.bias != nullptr) y += __half2float(static_cast<const __half*>(a.bias)[row]);
      static_cast<__half*>(a.out)[o] = __float2half_rn(y);
    }
  }
}

template <typename X, int GB>
inline cudaError_t launch_w4_group(const W4GroupArgs& a, cudaStream_t stream) {
#define B200W4A4_W4G_LAUNCH(RT, NT)                                                             \
  w4_group_kernel<X, GB, RT, NT><<<dim3(static_cast<unsigned>((a.N + 16 * (RT)-1) / (16 * (RT))), \
                                        static_cast<unsigned>((a.M + 8 * (NT)-1) / (8 * (NT)))),  \
                                   32 * kW4Warps, 0, stream>>>(a)
  if (a.M <= 8) B200W4A4_W4G_LAUNCH(1, 1);
  else if (a.M <= 16) B200W4A4_W4G_LAUNCH(1, 2);
  else B200W4A4_W4G_LAUNCH(2, 4);
#undef B200W4A4_W4G_LAUNCH
  return cudaGetLastError();
}

// ---- quantiser (load time): scale = max(absmax, 1e-5) / 7 in fp16, code = clamp(rint(w / scale), -8, 7)
template <typename W>
__global__ void w4_group_scale_kernel(const W* __restrict__ w, __half* __restrict__ scale, long long groups, int group) {
  const long long i = static_cast<long long>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  if (i >= groups) return;
  float m = 0.0f;
  for (int k = threadIdx.x & 31; k < group; k += 32) m = fmaxf(m, fabsf(static_cast<float>(w[i * group + k])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) scale[i] = __float2half_rn(fminf(__fdiv_rn(fmaxf(m, 1e-5f), 7.0f), 65504.0f));
}
template <typename W>
__global__ void w4_group_pack_kernel(const W* __restrict__ w, const __half* __restrict__ scale, uint8_t* __restrict__ packed,
                                     long long bytes, int group) {
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= bytes) return;
  const float s = __half2float(scale[2 * i / group]);
  uint32_t b = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float t = fminf(fmaxf(__fdiv_rn(static_cast<float>(w[2 * i + e]), s), -8.0f), 7.0f);
    b |= (static_cast<uint32_t>(__float2int_rn(t)) & 15u) << (4 * e);
  }
  packed[i] = static_cast<uint8_t>(b);
}

template <typename W>
inline cudaError_t launch_w4_group_quantize(const W* w, uint8_t* packed, __half* scale, int N, int K, int group,
                                            cudaStream_t stream) {
  const long long groups = static_cast<long long>(N) * (K / group), bytes = static_cast<long long>(N) * (K / 2);
  w4_group_scale_kernel<W><<<static_cast<unsigned>((groups + 7) / 8), 256, 0, stream>>>(w, scale, groups, group);
  w4_group_pack_kernel<W><<<static_cast<unsigned>((bytes + 255) / 256), 256, 0, stream>>>(w, scale, packed, bytes, group);
  return cudaGetLastError();
}

}  // namespace b200w4a4
