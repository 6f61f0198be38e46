// tcgen05 form of the windowed attention, for prompts (see window_attn.cuh for the mathematics).
//
// A CTA owns 256 queries of one head as two tiles of 128 rows, A and B, that share every key tile:
//   warps 0-3    softmax of tile A, one thread a row
//   warps 4-7    softmax of tile B
//   warp 8       owns TMEM; one lane issues every MMA
//   warp 9       TMA producer: Q once, then K and V tiles of 128 keys through one ring
// TMEM: scores S_A, S_B (128 x 128 fp32 each) and outputs O_A, O_B (128 x HD fp32).  A row's thread reads its
// 128 scores, and writes its weights P over them as 16-bit pairs: the A operand of the second product
// comes from TMEM, so the weights never touch shared memory, whose bandwidth the first product needs
// (both its operands are read from there).
//   S_X(n) = Q_X K(n)^T;   P_X(n) = exp2(S sc - m);   O_X += P_X(n) V(n)
// The issue order O_A(n), S_A(n+1), O_B(n), S_B(n+1) keeps the tensor pipe on one tile while the other's
// softmax runs.  S_X(n+1) overwrites P_X(n) behind the product that reads it: MMAs of one thread
// execute in order.  One commit after S_X(n+1) therefore also says that O_X(n) is complete, which is all the
// rescaling below needs.
//
// The running maximum m is moved only when a score exceeds it by more than 2^8 (then O and the row sum
// are rescaled): fp32 sums and 16-bit weights up to 256 lose nothing, and after the first tiles hardly
// any row moves, so the round trip of O through registers is rare.
//
// V rows of keys that no row of the CTA sees are overwritten with zeros in shared memory (tile A's threads,
// before they hand over P): 0 * garbage must not reach O.  Every wait is bounded.
#pragma once
#include <cuda.h>

#include "../../include/b200w4a4.h"
#include "device_state.cuh"
#include "gemm_w4a4.cuh"  // bounded waits, ring cursor, K-major descriptor
#include "ptx.cuh"
#include "window_attn.cuh"
#include <type_traits>

namespace b200w4a4 {

constexpr int DEV_TIMEOUT_ATTENTION = 106;
constexpr int kAttnTcMinQueries = 128;

template <int HD>
struct AttnTcCfg {
  static constexpr int BM = 128, BN = 128;         // rows of a tile, keys of a tile
  static constexpr int ATOM = 128 * 128;           // 128 rows of 64 values (one 128-byte swizzle row each)
  static constexpr int TILE = ATOM * (HD / 64);    // a Q, K or V tile
  static constexpr int S = HD == 128 ? 5 : 8;      // ring stages
  static constexpr int OFF_RING = 2 * TILE;
  static constexpr int OFF_BAR = OFF_RING + S * TILE;
  // full[S], free[S], q, s[2], p[2], then the abort flag and the TMEM address
  static constexpr int NUM_BARS = 2 * S + 5;
  static constexpr int SMEM = OFF_BAR + 8 * NUM_BARS + 16 + 1024;
  static constexpr int THREADS = 320;
  static constexpr int TMEM_COLS = 512;
  static constexpr int COL_O = 256;                // S at 0 and 128, O at 256 and 256 + HD
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct AttnTcParams {
  WindowAttnArgs a;
  int* status;
  unsigned* abort_word;
  unsigned launch_id;
};

namespace attn {

// B operand whose N runs along the 128-byte swizzle rows (V: dims contiguous, keys down the rows): 64-value
// column blocks `atom` bytes apart (leading offset), groups of eight keys 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t mn_major_sw128_desc(uint32_t smem_addr, uint32_t atom) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(atom >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// Instruction descriptor of kind::f16: D fp32 (bit 4), A and B fp16 (0) or bf16 (1) at bits 7 and 10, B's
// major at bit 16 (1: MN), N >> 3 at 17, M >> 4 at 24.
template <typename T>
__host__ __device__ constexpr uint32_t f16_idesc(int n, bool b_mn) {
  const uint32_t f = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

// Whether rows at positions [p0, p1] see anything of the 128 keys from j0 on.
__device__ __forceinline__ bool tile_active(int p0, int p1, int j0, int window, int sinks) {
  return j0 <= p1 && p1 >= 0 && (j0 + 127 > max(p0, 0) - window || j0 < sinks);
}

}  // namespace attn

template <typename T, int HD>
__global__ void __launch_bounds__(AttnTcCfg<HD>::THREADS, 1)
window_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const AttnTcParams prm) {
  using namespace attn;
  using C = AttnTcCfg<HD>;
  const WindowAttnArgs& a = prm.a;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - ptx::smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const uint32_t bar0 = base + C::OFF_BAR;
  auto bar_full = [&](uint32_t s) { return bar0 + 8u * s; };
  auto bar_free = [&](uint32_t s) { return bar0 + 8u * (C::S + s); };
  const uint32_t bar_q = bar0 + 8u * (2 * C::S);
  auto bar_s = [&](int x) { return bar0 + 8u * (2 * C::S + 1 + x); };
  auto bar_p = [&](int x) { return bar0 + 8u * (2 * C::S + 3 + x); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::OFF_BAR + 8 * C::NUM_BARS);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(gen + C::OFF_BAR + 8 * C::NUM_BARS + 8);
  const detail::WaitCtx wctx{abort_flag, prm.status, prm.abort_word, prm.launch_id};
  auto wait = [&](uint32_t bar, uint32_t parity) { return detail::wait_bar(bar, parity, wctx, DEV_TIMEOUT_ATTENTION); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::S; ++s) {
      ptx::mbar_init(bar_full(s), 1);
      ptx::mbar_init(bar_free(s), 1);
    }
    ptx::mbar_init(bar_q, 1);
    for (int x = 0; x < 2; ++x) {
      ptx::mbar_init(bar_s(x), 1);
      ptx::mbar_init(bar_p(x), 4);  // one arrival a warp
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 8) {
    ptx::tmem_alloc<1>(ptx::smem_u32(tmem_holder), C::TMEM_COLS);
    ptx::tmem_relinquish<1>();
  }
  if (warp == 9 && lane == 0) {
    ptx::prefetch_tensormap(&tm_q);
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_holder);

  // the longest runs (the last queries) first
  const int i0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * (2 * C::BM);
  const int hq = blockIdx.y, b = blockIdx.z;
  const int i1 = min(i0 + 2 * C::BM, a.Lq) - 1;
  const Span sp = span_of<C::BN>(a, b, i0, i1);
  auto tile_key = [&](int n) { return (n < sp.n_sink ? n : sp.w0 + n - sp.n_sink) * C::BN; };
  // positions of tile x's first and last query (last < first: no queries)
  auto first_pos = [&](int x) { return sp.p0 + x * C::BM; };
  auto last_pos = [&](int x) { return min(sp.p0 + x * C::BM + C::BM - 1, sp.p1); };
  auto active = [&](int x, int n) {
    return first_pos(x) <= sp.p1 && tile_active(first_pos(x), last_pos(x), tile_key(n), a.window, a.sinks);
  };

  if (warp == 9) {
    if (lane == 0 && sp.n > 0) {
      ptx::mbar_arrive_expect_tx(bar_q, 2 * C::TILE);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
          ptx::tma_load_4d(base + x * C::TILE + c * C::ATOM, &tm_q, bar_q, 64 * c, hq, i0 + x * C::BM, b);
      RingPos<C::S> pos;
      bool alive = true;
      const int hk = hq / a.G;
      for (int n = 0; n < sp.n && alive; ++n) {
        const int j0 = tile_key(n);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!wait(bar_free(pos.slot), pos.phase ^ 1)) {
            alive = false;
            break;
          }
          ptx::mbar_arrive_expect_tx(bar_full(pos.slot), C::TILE);
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
            ptx::tma_load_4d(base + C::OFF_RING + pos.slot * C::TILE + c * C::ATOM, kv ? &tm_v : &tm_k, bar_full(pos.slot),
                             64 * c, hk, j0, b);
          pos.advance();
        }
      }
      if (!alive) {  // loads in flight get a bounded time to land before the block ends
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  } else if (warp == 8) {
    if (lane == 0 && sp.n > 0) {
      constexpr uint32_t id_s = f16_idesc<T>(C::BN, false), id_o = f16_idesc<T>(HD, true);
      auto score = [&](int x, uint32_t k_tile) {
        const uint64_t dq = make_kmajor_sw128_desc(base + x * C::TILE), dk = make_kmajor_sw128_desc(k_tile);
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
          const uint64_t step = (j >> 2) * (C::ATOM >> 4) + (j & 3) * 2;
          ptx::mma_f16_ss(tmem + x * C::BN, dq + step, dk + step, id_s, j > 0);
        }
        ptx::mma_commit(bar_s(x));
      };
      auto output = [&](int x, uint32_t v_tile, bool accumulate) {
        const uint64_t dv = mn_major_sw128_desc(v_tile, C::ATOM);
#pragma unroll
        for (int j = 0; j < C::BN / 16; ++j)
          ptx::mma_f16_ts(tmem + C::COL_O + x * HD, tmem + x * C::BN + 8 * j, dv + j * (2048 >> 4), id_o, accumulate || j > 0);
      };
      auto tile_at = [&](uint32_t slot) { return base + C::OFF_RING + slot * C::TILE; };
      RingPos<C::S> pos;
      uint32_t p_phase[2] = {0, 0};
      bool started[2] = {false, false};
      bool alive = wait(bar_q, 0) && wait(bar_full(0), 0);
      if (alive) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (active(x, 0)) score(x, tile_at(0));
        ptx::mma_commit(bar_free(0));
        pos.advance();
      }
      for (int n = 0; n < sp.n && alive; ++n) {
        const uint32_t v_slot = pos.slot, v_phase = pos.phase;
        pos.advance();
        const uint32_t k_slot = pos.slot, k_phase = pos.phase;
        if (!wait(bar_full(v_slot), v_phase)) {
          alive = false;
          break;
        }
        bool have_k = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (active(x, n)) {
            if (!wait(bar_p(x), p_phase[x])) {
              alive = false;
              break;
            }
            p_phase[x] ^= 1;
            ptx::tc_fence_after_sync();
            output(x, tile_at(v_slot), started[x]);
            started[x] = true;
          }
          if (n + 1 < sp.n) {
            if (!have_k && !wait(bar_full(k_slot), k_phase)) {
              alive = false;
              break;
            }
            have_k = true;
            if (active(x, n + 1)) score(x, tile_at(k_slot));
          }
        }
        if (!alive) break;
        ptx::mma_commit(bar_free(v_slot));
        if (n + 1 < sp.n) {
          ptx::mma_commit(bar_free(k_slot));
          pos.advance();
        }
      }
      if (alive) {
        ptx::mma_commit(bar_s(0));  // the outputs are complete
        ptx::mma_commit(bar_s(1));
      } else {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  } else {
    const int x = warp >> 2;
    const int r = (warp & 3) * 32 + lane;           // row of the tile = TMEM lane
    const int qi = i0 + x * C::BM + r;
    const int p = first_pos(x) + r;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + x * C::BN, t_o = tmem + lanes + C::COL_O + x * HD;
    // the lanes of a warp give up together: the TMEM accesses below want all of them
    auto wait_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    const float sc = a.scale * kLog2e;
    const int pa = first_pos(x), pz = last_pos(x);
    float m = -INFINITY, l = 0.0f;
    uint32_t s_phase = 0;
    bool alive = true, started = false;
    for (int n = 0; n < sp.n && alive; ++n) {
      const int j0 = tile_key(n);
      if (!active(x, n)) continue;
      if (!wait_all(bar_s(x), s_phase)) {
        alive = false;
        break;
      }
      s_phase ^= 1;
      ptx::tc_fence_after_sync();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(t_s + 32 * c, s[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_wait_for(s[c]);
      const bool whole = j0 + C::BN - 1 <= pa && (j0 > pz - a.window || j0 + C::BN <= a.sinks);
      if (!whole) {
        // key j is seen when j <= p and (j > p - window or j < sinks)
        const int hi = p - j0, lo = p - a.window - j0, first = a.sinks - j0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int j = 32 * c + i;
            if (!(j <= hi && (j > lo || j < first))) s[c][i] = 0xff800000u;
          }
      }
      float top = -INFINITY;
      {
        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) t4[i & 3] = fmaxf(t4[i & 3], __uint_as_float(s[c][i]));
        top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * sc;
      }
      // move the maximum only when the weights would pass 2^8
      const bool move = top > m + 8.0f;
      if (__any_sync(0xffffffffu, move)) {
        const float next = move ? top : m;
        const float f = next == m ? 1.0f : exp2_fast(m - next);  // 0 for a row that starts here
        m = next;
        l *= f;
        if (started) {
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            ptx::tmem_ld_32x32(t_o + 32 * c, o);
            ptx::tmem_ld_wait_for(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st_32x32(t_o + 32 * c, o);
          }
        }
      }
      started = true;
      const float neg = m == -INFINITY ? 0.0f : -m;
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e0 = exp2_fast(fmaf(__uint_as_float(s[c][2 * i]), sc, neg));
          const float e1 = exp2_fast(fmaf(__uint_as_float(s[c][2 * i + 1]), sc, neg));
          sum[0] += e0;
          sum[1] += e1;
          w[i] = pack2(e0, e1, T());
        }
        ptx::tmem_st_32x16(t_s + 16 * c, w);
      }
      l += sum[0] + sum[1];
      ptx::tmem_st_wait();
      if (x == 0 || !active(0, n)) {
        const bool cover = j0 + C::BN - 1 <= sp.hi && (j0 >= sp.lo || j0 + C::BN <= a.sinks);
        if (!cover) {
          // V(n) follows K(n) in the ring
          const uint32_t at = 2 * n + 1, slot = at % C::S;
          if (!wait_all(bar_full(slot), (at / C::S) & 1)) {
            alive = false;
            break;
          }
          const int j = j0 + r;
          if (!(j <= sp.hi && (j >= sp.lo || j < a.sinks))) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                detail::sts128(base + C::OFF_RING + slot * C::TILE + c * C::ATOM + r * 128 + 16 * i, make_uint4(0, 0, 0, 0));
          }
          ptx::fence_proxy_async_smem();
        }
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_p(x));
    }
    if (alive && sp.n > 0) {
      alive = wait_all(bar_s(x), s_phase);
      ptx::tc_fence_after_sync();
    }
    if (alive) {
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
      const bool ok = qi < a.Lq;
      if (ok && a.lse != nullptr)
        a.lse[(static_cast<long long>(b) * a.Hq + hq) * a.Lq + qi] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
      T* out = static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.Lq + qi) * a.Hq + hq) * HD;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        if (started) {  // the same for the whole warp
          ptx::tmem_ld_32x32(t_o + 32 * c, o);
          ptx::tmem_ld_wait_for(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (ok) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              w[j] = pack2(__uint_as_float(o[8 * i + 2 * j]) * inv, __uint_as_float(o[8 * i + 2 * j + 1]) * inv, T());
            *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<1>(tmem, C::TMEM_COLS);
  }
}

// [batch, token, head, HD] as a 4-D map (HD, head, token, batch) with boxes of 64 values x 128 tokens.
inline int encode_attn_map(CUtensorMap* map, bool bf16, const void* base, int hd, int heads, int tokens, int batch,
                           long long p_head, long long p_tok, long long p_batch) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Encode enc = reinterpret_cast<Encode>(tensor_map_encoder());
  if (enc == nullptr) return B200W4A4_ECUDA;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens),
                              static_cast<cuuint64_t>(batch)};
  // the pitch of a dimension of one is never used
  const cuuint64_t strides[3] = {heads > 1 ? static_cast<cuuint64_t>(2 * p_head) : 256u,
                                 tokens > 1 ? static_cast<cuuint64_t>(2 * p_tok) : 256u,
                                 batch > 1 ? static_cast<cuuint64_t>(2 * p_batch) : 256u};
  const cuuint32_t box[4] = {64, 1, 128, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200W4A4_OK : B200W4A4_ECUDA;
}

template <typename T, int HD>
inline int launch_window_attn_tc(const WindowAttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  using C = AttnTcCfg<HD>;
  const bool bf16 = !std::is_same<T, __half>::value;
  CUtensorMap q, k, v;
  int rc = encode_attn_map(&q, bf16, a.q, HD, a.Hq, a.Lq, a.B, a.q_h, a.q_t, a.q_b);
  if (rc == B200W4A4_OK) rc = encode_attn_map(&k, bf16, a.k, HD, a.Hkv, a.Lk, a.B, a.k_h, a.k_t, a.k_b);
  if (rc == B200W4A4_OK) rc = encode_attn_map(&v, bf16, a.v, HD, a.Hkv, a.Lk, a.B, a.v_h, a.v_t, a.v_b);
  if (rc != B200W4A4_OK) return rc;
  if (cudaFuncSetAttribute(window_attn_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
    return B200W4A4_ECUDA;
  AttnTcParams prm{a, dev.status, dev.abort_word, new_launch_id()};
  const dim3 grid(static_cast<unsigned>((a.Lq + 2 * C::BM - 1) / (2 * C::BM)), static_cast<unsigned>(a.Hq),
                  static_cast<unsigned>(a.B));
  window_attn_tc_kernel<T, HD><<<grid, C::THREADS, C::SMEM, stream>>>(q, k, v, prm);
  return cudaGetLastError() == cudaSuccess ? B200W4A4_OK : B200W4A4_ECUDA;
}

}  // namespace b200w4a4
