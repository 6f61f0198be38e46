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
//   fp16 / bf16: nibbles (i, i+4) of a word become a pair by one mask and one exclusive or: the exponent of
//                1024 (fp16) or 128 (bf16) with the nibble, sign bit flipped, in the mantissa; an exact
//                subtraction leaves the code (it runs on the FMA pipe, the masks on the slower ALU);
//   int8:        word << 4 and word, masked with 0xF0F0F0F0, are bytes of 16 * code (the 16 goes
//                into the scale, exactly).
// Products of one group are summed by the tensor core in fp32 (int32 for int8), then enter the fp32
// total with the group's scale.  The warps of a CTA share its rows and split K; their totals are
// added in shared memory in a fixed order.
//
// Measured (device time, weights past L2): 1 x 5120 -> 15360 bf16, groups of 128: 18.1 us (2.2 TB/s of weight and scales;
// the copy rate would take 6.3); 8 x 13824 -> 5120 fp16, groups of 64: 19.6 us; 5 x 1536 -> 8960 int8, groups of 32: 8.1 us.  The
// ALU is 59 % busy with the masks while the SMs are, half of the stalls wait for memory, DRAM is 24 % busy, and a call this
// short spends some 3 us on its launch and its last wave (2.16 waves of blocks at the first shape).  Slower, each measured at the first shape against the form of its time:
// the same stream through a per-warp cp.async ring in shared memory (27 us) or a register ring (27), leaving the bias of the
// pairs in and taking it out through a product with ones (24), shifts as multiplications' high words (21).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "rms_norm.cuh"  // max_nan

namespace b200w4a4 {

struct W4GroupArgs {
  const void* x;           // [M, K]
  const uint8_t* packed;   // [N, K/2]
  const __half* scale;     // [N, K/group]
  const float* act_scale;  // [M] (int8 x) or null
  const void* bias;        // [N] of the output type, or null
  const float* bias32;     // [N] fp32, or null
  void* out;               // [M, N]
  int M, N, K, group;
  int group_runs;          // group / GB (set by the launcher), and the multiplier that divides by it:
  uint32_t group_mul;      // ceil(2^32 / group_runs), exact for the run numbers of K < 2^20
  bool out_bf16;
};

namespace detail {

// D = A * B + C, A 16 x 16 (weights), B 16 x 8 (tokens)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4], __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4], __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// Eight codes of a word as four pairs: p[i] = (code i, code i + 4).  A nibble n with its sign bit flipped is code + 8.
__device__ __forceinline__ void widen(uint32_t w, uint32_t (&p)[4], __half) {
  const __half2 one = __half2half2(__ushort_as_half(0x6408));  // 1032
  const __half2 by = __half2half2(__ushort_as_half(0x2c00));   // 1/16
  const __half2 off = __half2half2(__ushort_as_half(0xd480));  // -72
  const uint32_t v = w >> 8;
  p[0] = (w & 0x000f000fu) ^ 0x64086408u;  // 1024 + 8 + code
  p[1] = (w & 0x00f000f0u) ^ 0x64806480u;  // 1024 + 16 (8 + code)
  p[2] = (v & 0x000f000fu) ^ 0x64086408u;
  p[3] = (v & 0x00f000f0u) ^ 0x64806480u;
  __half2* h = reinterpret_cast<__half2*>(p);
  h[0] = __hsub2(h[0], one);
  h[1] = __hfma2(h[1], by, off);
  h[2] = __hsub2(h[2], one);
  h[3] = __hfma2(h[3], by, off);
}
__device__ __forceinline__ void widen(uint32_t w, uint32_t (&p)[4], __nv_bfloat16) {
  const __nv_bfloat162 off = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));  // 136
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = ((w >> (4 * i)) & 0x000f000fu) ^ 0x43084308u;  // 128 + 8 + code
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&p[i]);
    *h = __hsub2(*h, off);
  }
}

// A lane's run of 8 * WORDS codes; the weight is read once, so it does not go through L1 where whole sectors
// are read by one instruction.
template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 4) {
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  } else if constexpr (WORDS == 2) {
    asm("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));  // the next run's load finds the other half of the sector in L1
  }
}

}  // namespace detail

constexpr int kW4Warps = 8;
// At most so many warps an SM are asked for when K is split; up to eight tokens 24 are resident, so this is 2.2 waves of blocks:
// 1 x 5120 -> 15360 takes 18.9 us with 48 (K in four, 1.1 waves of longer blocks), 18.0 with 64 (in eight).
constexpr int kW4WarpsPerSm = 64;

// GB: codes that are sure to share a scale (32, 64 or 128; a divisor of the group).  A superblock is
// 128 codes of a row; lane (g, t) multiplies the run of GB / 4 codes at t * GB / 4 of each of its 128 / GB
// parts, for rows g and g + 8 of each of the RT row tiles.  NT: tiles of 8 tokens.
//
// `split` warps (a power of two) share a tile's K, superblocks in turn; a CTA holds kW4Warps / split tiles.
// A warp takes U superblocks at a time: all their words, scales and x are asked for before the first product,
// so a batch costs one memory latency.
template <typename X, int GB, int RT, int NT, int U>
__global__ void __launch_bounds__(32 * kW4Warps, NT == 4 ? 1 : 3) w4_group_kernel(const W4GroupArgs a, int split) {
  constexpr bool S8 = sizeof(X) == 1;
  constexpr int PARTS = 128 / GB;
  constexpr int WORDS = GB / 32;  // words of a lane's run
  constexpr int XR = PARTS * WORDS;  // runs of eight values of x a lane takes from a superblock
  using XVec = typename std::conditional<S8, uint2, uint4>::type;
  using Part = typename std::conditional<S8, int, float>::type;
  __shared__ float total[kW4Warps][RT * 16][NT * 8 + 1];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int tiles = kW4Warps / split;
  const int cta_row0 = blockIdx.x * tiles * (RT * 16);
  const int row0 = cta_row0 + warp / split * (RT * 16);
  const int tok0 = blockIdx.y * (NT * 8);
  const int toks = min(a.M - tok0, NT * 8);
  const int nsb = (a.K + 127) >> 7;
  const int ngroups = a.K / a.group;

  // rows behind the last one repeat it, and tokens likewise: nothing of theirs is stored
  const uint8_t* wp[2 * RT];
  const __half* sp[2 * RT];
#pragma unroll
  for (int r = 0; r < 2 * RT; ++r) {
    const long long row = min(row0 + g + 8 * r, a.N - 1);
    wp[r] = a.packed + row * (a.K >> 1) + t * (GB / 8);
    sp[r] = a.scale + row * ngroups;
  }
  const X* xp[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    xp[n] = static_cast<const X*>(a.x) + static_cast<long long>(tok0 + min(8 * n + g, toks - 1)) * a.K + t * (GB / 4);

  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;

  // one batch of UU superblocks; WHOLE: all of them exist and hold 128 codes
  auto batch = [&](int sb0, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    uint32_t w[U][2 * RT][PARTS][WORDS];
    __half s[U][2 * RT][PARTS];
    [[maybe_unused]] XVec xv[NT == 1 ? U : 1][NT == 1 ? XR : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int sb = sb0 + u * split;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        if (!WHOLE && (sb << 7) + p * GB >= a.K) continue;  // the same for the warp
        const uint32_t q = sb * PARTS + p;
        const uint32_t grp = a.group_runs == 1 ? q : __umulhi(q, a.group_mul);
#pragma unroll
        for (int r = 0; r < 2 * RT; ++r) {
          detail::load_words<WORDS>(wp[r] + sb * 64 + p * (GB / 2), w[u][r][p]);
          s[u][r][p] = __ldg(sp[r] + grp);
        }
        if constexpr (NT == 1) {
#pragma unroll
          for (int j = 0; j < WORDS; ++j)
            xv[u][p * WORDS + j] = __ldg(reinterpret_cast<const XVec*>(xp[0] + (sb << 7) + p * GB + 8 * j));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int sb = sb0 + u * split;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        if (!WHOLE && (sb << 7) + p * GB >= a.K) continue;
        Part part[RT][NT][4];
#pragma unroll
        for (int j = 0; j < WORDS; ++j) {
          constexpr Part zero[4] = {0, 0, 0, 0};
          uint32_t c[2 * RT][4];
#pragma unroll
          for (int r = 0; r < 2 * RT; ++r) {
            const uint32_t word = w[u][r][p][j];
            if constexpr (S8) {
              c[r][0] = (word << 4) & 0xF0F0F0F0u;
              c[r][1] = word & 0xF0F0F0F0u;
            } else {
              detail::widen(word, c[r], X());
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            XVec v;
            if constexpr (NT == 1) v = xv[u][p * WORDS + j];
            else v = __ldg(reinterpret_cast<const XVec*>(xp[n] + (sb << 7) + p * GB + 8 * j));
            if constexpr (S8) {
              const uint32_t b0 = __byte_perm(v.x, v.y, 0x6420), b1 = __byte_perm(v.x, v.y, 0x7531);
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const uint32_t f[4] = {c[2 * r][0], c[2 * r + 1][0], c[2 * r][1], c[2 * r + 1][1]};
                if (j == 0) detail::mma_s8(part[r][n], f, b0, b1, zero);
                else detail::mma_s8(part[r][n], f, b0, b1, part[r][n]);
              }
            } else {
              const uint32_t b[4] = {__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                     __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632)};
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const uint32_t f0[4] = {c[2 * r][0], c[2 * r + 1][0], c[2 * r][1], c[2 * r + 1][1]};
                const uint32_t f1[4] = {c[2 * r][2], c[2 * r + 1][2], c[2 * r][3], c[2 * r + 1][3]};
                if (j == 0) detail::mma_f16(part[r][n], f0, b[0], b[1], zero, X());
                else detail::mma_f16(part[r][n], f0, b[0], b[1], part[r][n], X());
                detail::mma_f16(part[r][n], f1, b[2], b[3], part[r][n], X());
              }
            }
          }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float by = S8 ? 0.0625f : 1.0f;  // int8 words hold 16 * code
          const float s0 = __half2float(s[u][2 * r][p]) * by, s1 = __half2float(s[u][2 * r + 1][p]) * by;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][n][i] = fmaf(i < 2 ? s0 : s1, static_cast<float>(part[r][n][i]), acc[r][n][i]);
        }
      }
    }
  };
  int sb = warp & (split - 1);
  for (; sb + (U - 1) * split < (a.K >> 7); sb += U * split) batch(sb, std::true_type());
  for (; sb < nsb; sb += U * split) batch(sb, std::false_type());

#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[warp][16 * r + g + (i >> 1) * 8][8 * n + 2 * t + (i & 1)] = acc[r][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < tiles * RT * 16 * toks; i += 32 * kW4Warps) {
    const int r = i % (tiles * RT * 16), n = i / (tiles * RT * 16);
    const int row = cta_row0 + r, tok = tok0 + n;
    if (row >= a.N) continue;
    const int tile = r / (RT * 16), in_tile = r % (RT * 16);
    float y = 0.0f;
    for (int v = 0; v < split; ++v) y += total[tile * split + v][in_tile][n];
    if (a.act_scale != nullptr) y *= a.act_scale[tok];
    const long long o = static_cast<long long>(tok) * a.N + row;
    if (a.bias32 != nullptr) y += a.bias32[row];
    if (a.out_bf16) {
      if (a.bias != nullptr) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[row]);
      static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(y);
    } else {
      if (a.bias != nullptr) y += __half2float(static_cast<const __half*>(a.bias)[row]);
      static_cast<__half*>(a.out)[o] = __float2half_rn(y);
    }
  }
}

template <typename X, int GB, int RT, int NT, int U>
inline cudaError_t launch_w4_group_tile(W4GroupArgs a, int sm_count, cudaStream_t stream) {
  const long long row_tiles = (static_cast<long long>(a.N) + 16 * RT - 1) / (16 * RT);
  const long long tok_tiles = (a.M + 8 * NT - 1) / (8 * NT);
  const int nsb = (a.K + 127) / 128;
  a.group_runs = a.group / GB;
  a.group_mul = static_cast<uint32_t>(((1ull << 32) + a.group_runs - 1) / a.group_runs);
  int split = 1;
  while (split < kW4Warps && 2 * split <= nsb && row_tiles * tok_tiles * split * 2 <= static_cast<long long>(sm_count) * kW4WarpsPerSm) split *= 2;
  const int per = kW4Warps / split;
  w4_group_kernel<X, GB, RT, NT, U><<<dim3(static_cast<unsigned>((row_tiles + per - 1) / per), static_cast<unsigned>(tok_tiles)),
                                      32 * kW4Warps, 0, stream>>>(a, split);
  return cudaGetLastError();
}

// Up to 16 tokens 16 rows a warp and two superblocks a batch; with 32 rows a warp one token takes 17.8 instead of 18.8 us at
// 15360 rows, but 10.0 instead of 9.0 at 5120 and 14 instead of 10 at 1000, where fewer warps are left.  From 17 tokens on
// 32 rows and 32 tokens a warp (64 tokens: 33 us; two blocks an SM instead of one 41).
template <typename X, int GB>
inline cudaError_t launch_w4_group(const W4GroupArgs& a, int sm_count, cudaStream_t stream) {
  if (a.M <= 8) return launch_w4_group_tile<X, GB, 1, 1, 2>(a, sm_count, stream);
  if (a.M <= 16) return launch_w4_group_tile<X, GB, 1, 2, 2>(a, sm_count, stream);
  return launch_w4_group_tile<X, GB, 2, 4, 2>(a, sm_count, stream);
}

// ---- quantiser (load time): scale = max(absmax, 1e-5) / 7 in fp16, code = clamp(rint(w / scale), -8, 7).  A group that holds a
// NaN or an infinity, or whose scale passes fp16's range, has scale NaN and codes 0, so that every product with it shows.
template <typename W>
__global__ void w4_group_scale_kernel(const W* __restrict__ w, __half* __restrict__ scale, long long groups, int group) {
  const long long i = static_cast<long long>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  if (i >= groups) return;
  float m = 0.0f;
  for (int k = threadIdx.x & 31; k < group; k += 32) m = detail::max_nan(m, fabsf(static_cast<float>(w[i * group + k])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = detail::max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) {
    const __half s = __float2half_rn(__fdiv_rn(detail::max_nan(m, 1e-5f), 7.0f));
    scale[i] = __half2float(s) < INFINITY ? s : __ushort_as_half(0x7fff);
  }
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
    const float t = isnan(s) ? 0.0f : fminf(fmaxf(__fdiv_rn(static_cast<float>(w[2 * i + e]), s), -8.0f), 7.0f);
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
