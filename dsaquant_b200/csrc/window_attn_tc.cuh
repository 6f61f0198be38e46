// tcgen05 form of the windowed attention, for prompts (see window_attn.cuh for the mathematics).
//
// A CTA owns 256 queries of one head as two tiles of 128 rows, A and B, that share every key tile:
//   warps 0-7    softmax of tile A, two threads a row (32 keys of each key tile)
//   warps 8-15   softmax of tile B
//   warps 16, 17 one lane of each issues the MMAs of tile A, of tile B; warp 16 owns TMEM
//   warp 18      TMA producer: Q once, then K and V tiles of 64 keys through one ring (warp 19 idles)
// TMEM: two score buffers a tile (128 x 64 fp32 each) and the outputs O_A, O_B (128 x HD fp32).  A thread reads
// its 32 scores and writes its weights P over them as 16-bit pairs: the A operand of the second product comes from
// TMEM, so the weights never touch shared memory, whose bandwidth the first product needs.
//   S_X(n) = Q_X K(n)^T;   P_X(n) = exp2(S sc - m);   O_X += P_X(n) V(n)
// S_X(n + 1) is issued before P_X(n) is waited for, into the other buffer, so the softmax warps always find
// their next scores ready.  (128 keys a tile fill both buffers: a tile's softmax, 2200 cycles, and its products, 1250,
// then took turns, and the tensor pipe idled 40 % of the time however the softmax was spread over warps.)
// Four softmax warps on each scheduler hide one another's waits, TMEM accesses and barriers; with two, 64 keys cost 2000
// cycles a pair of tiles, of which the exponentials are 1024.
// An issuer's waits and commits take as long as its products (830 of 1800 cycles when one warp did both tiles); with
// two, one tile's products fill the pipe meanwhile.
// S_X(n + 2) overwrites P_X(n) behind the product that reads it: MMAs of one thread execute in order.
//
// A row's maximum is found in its first tile and again only when the weights of half a tile add up to over 2^9: until
// then fp32 sums and 16-bit weights lose nothing by a maximum that is a little old, a tile costs no pass for
// it, and O is hardly ever rescaled.
//
// V rows of keys that no row of the CTA sees are overwritten with zeros in shared memory (by each tile's threads,
// before they hand over P), and so are values that are not finite in the key tiles that some row of the CTA does not see
// entirely (the rows that see them get them at the very end): 0 * inf must not reach O.  Both tiles do so in the same key tiles,
// also where all rows of one of them see every key: its product would else meet such a value or a zero, by which tile came
// first.  Every wait is bounded.
//
// Measured, 12 heads of 128 x 32760 queries, window 4096, 64 first keys, bf16: 821 us in bursts of a few calls, 0.786 TFLOP at
// 957 TFLOP/s, 0.58 of the library product's burst rate (the mma.sync form: 2842 us); call after call for seconds 933 us.
// Tensor pipe and special-function unit are each 44 % busy: what is left is latency between the roles, instruction fetch
// (four roles share the caches) and a tenth in a block's start and end.  Clearing values of V that are not finite is in it
// (810 us without, when such a value made rows NaN that do not see it).
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
// From one full tile of queries on.  Measured against the mma.sync form: 32 x 128 queries on 4096 keys, 40 query and 8 key heads
// of 128: 494 and 1263 us; 8 x 128 of them: 166 and 376; 512 on 512: 21 and 38; 3 x 517, 8 heads of 64, window 300: 19.9 and 20.2.
// The rule does not ask how many blocks there are, and this form never splits the keys: where a call is a few blocks the
// other one would be faster (128 queries, 12 heads: 10.1 and 8.4 us on 128 keys, 55 and 28 on 4096; 8 heads on 32768 keys: 381 and 81).
constexpr int kAttnTcMinQueries = 128;

template <int HD>
struct AttnTcCfg {
  static constexpr int BM = 128, BN = 64;            // rows of a tile, keys of a tile
  static constexpr int Q_ATOM = BM * 128, K_ATOM = BN * 128;  // 64 values of each row (one 128-byte swizzle row each)
  static constexpr int Q_TILE = Q_ATOM * (HD / 64), K_TILE = K_ATOM * (HD / 64);
  static constexpr int S = HD == 128 ? 10 : 16;      // ring stages
  static constexpr int OFF_RING = 2 * Q_TILE;
  static constexpr int OFF_BAR = OFF_RING + S * K_TILE;
  // full[S], free[S], q, s[2][2], p[2][2], o[2][2], then the abort flag, the TMEM address and a float a row of both tiles
  static constexpr int NUM_BARS = 2 * S + 13;
  static constexpr int OFF_ROWS = OFF_BAR + 8 * NUM_BARS + 16;
  static constexpr int SMEM = OFF_ROWS + 2 * BM * 4 + 1024;
  static constexpr int SOFTMAX_WARPS = 16, WARP_MMA = 16, WARP_TMA = 18;
  static constexpr int THREADS = 640;
  static constexpr int TMEM_COLS = 512;
  static constexpr int COL_O = 256;                  // S_A at 0, 64; S_B at 128, 192; O at 256 and 256 + HD
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

// the low n bits, n clamped to 0..32
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The waiting part of a bounded wait, out of line: the roles' loops share the instruction caches.
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                         unsigned* abort_word, unsigned launch_id) {
  return b200w4a4::detail::wait_bar(bar, parity, b200w4a4::detail::WaitCtx{abort_flag, status, abort_word, launch_id},
                                    DEV_TIMEOUT_ATTENTION);
}

// Whether rows at positions [p0, p1] see anything of the 64 keys from j0 on.
__device__ __forceinline__ bool tile_active(int p0, int p1, int j0, int window, int sinks) {
  return j0 <= p1 && p1 >= 0 && (j0 + 63 > max(p0, 0) - window || j0 < sinks);
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
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  const uint32_t bar0 = base + C::OFF_BAR;
  auto bar_full = [&](uint32_t s) { return bar0 + 8u * s; };
  auto bar_free = [&](uint32_t s) { return bar0 + 8u * (C::S + s); };
  const uint32_t bar_q = bar0 + 8u * (2 * C::S);
  auto bar_s = [&](int x, uint32_t buf) { return bar0 + 8u * (2 * C::S + 1 + 2 * x + buf); };
  // one for each buffer: a warp may be through tile n + 1 before another of its tile is through n
  auto bar_p = [&](int x, uint32_t buf) { return bar0 + 8u * (2 * C::S + 5 + 2 * x + buf); };
  auto bar_o = [&](int x, uint32_t buf) { return bar0 + 8u * (2 * C::S + 9 + 2 * x + buf); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + C::OFF_BAR + 8 * C::NUM_BARS);
  // set before the first value is cleared; the CTA reads it behind its last barrier
  volatile int* cleared = reinterpret_cast<volatile int*>(gen + C::OFF_BAR + 8 * C::NUM_BARS + 4);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(gen + C::OFF_BAR + 8 * C::NUM_BARS + 8);
  auto wait = [&](uint32_t bar, uint32_t parity) {
    return ptx::mbar_probe(bar, parity) || wait_longer(bar, parity, abort_flag, prm.status, prm.abort_word, prm.launch_id);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::S; ++s) {
      ptx::mbar_init(bar_full(s), 1);
      ptx::mbar_init(bar_free(s), 2);  // both issuers
    }
    ptx::mbar_init(bar_q, 1);
    for (int x = 0; x < 2; ++x) {
      ptx::mbar_init(bar_s(x, 0), 1);
      ptx::mbar_init(bar_s(x, 1), 1);
      ptx::mbar_init(bar_p(x, 0), 8);  // one arrival a warp
      ptx::mbar_init(bar_p(x, 1), 8);
      ptx::mbar_init(bar_o(x, 0), 1);
      ptx::mbar_init(bar_o(x, 1), 1);
    }
    *abort_flag = 0;
    *cleared = 0;
    ptx::fence_mbar_init();
  }
  if (warp == C::WARP_MMA) {
    ptx::tmem_alloc<1>(ptx::smem_u32(tmem_holder), C::TMEM_COLS);
    ptx::tmem_relinquish<1>();
  }
  if (warp == C::WARP_TMA && lane == 0) {
    ptx::prefetch_tensormap(&tm_q);
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(tmem_holder), 0);

  // the longest runs (the last queries) first
  const int i0 = static_cast<int>(gridDim.x - 1 - blockIdx.x) * (2 * C::BM);
  const int hq = blockIdx.y, b = blockIdx.z;
  const int i1 = min(i0 + 2 * C::BM, a.Lq) - 1;
  const Span sp = span_of<C::BN>(a, b, i0, i1);
  auto tile_key = [&](int n) { return (n < sp.n_sink ? n : sp.w0 + n - sp.n_sink) * C::BN; };
  // positions of tile x's first and last query (last < first: no queries)
  auto first_pos = [&](int x) { return sp.p0 + x * C::BM; };
  auto last_pos = [&](int x) { return min(sp.p0 + x * C::BM + C::BM - 1, sp.p1); };
  // key tiles that some row of tile x sees: those of the sinks, and [from, to] of the window's (rows are
  // consecutive, so are these; one more look covers a first window tile that only holds sinks)
  auto last_tile = [&](int x) {
    return first_pos(x) <= sp.p1 && last_pos(x) >= 0 ? sp.n_sink + last_pos(x) / C::BN - sp.w0 : -1;
  };
  auto first_tile = [&](int x, int last) {
    int n = sp.n_sink;
    while (n <= last && !tile_active(first_pos(x), last_pos(x), tile_key(n), a.window, a.sinks)) ++n;
    return n;
  };
  // whether every row of the CTA sees all keys of the tile from j0 on
  auto cta_sees = [&](int j0) { return j0 + C::BN - 1 <= sp.p0 && (j0 > sp.p1 - a.window || j0 + C::BN <= a.sinks); };
  const int to_a = last_tile(0), to_b = last_tile(1), from_a = first_tile(0, to_a), from_b = first_tile(1, to_b);
  auto active = [&](int x, int n) {
    const int to = x == 0 ? to_a : to_b, from = x == 0 ? from_a : from_b;
    return n <= to && (n < sp.n_sink || n >= from);
  };

  if (warp == C::WARP_TMA) {
    if (lane == 0 && sp.n > 0) {
      ptx::mbar_arrive_expect_tx(bar_q, 2 * C::Q_TILE);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
          for (int half = 0; half < 2; ++half)  // a box is 64 rows
            ptx::tma_load_4d(base + x * C::Q_TILE + c * C::Q_ATOM + half * (C::Q_ATOM / 2), &tm_q, bar_q, 64 * c, hq,
                             i0 + x * C::BM + half * 64, b);
      RingPos<C::S> pos;
      const int hk = hq / a.G;
      auto load = [&](const CUtensorMap* map, int n) {
        if (!wait(bar_free(pos.slot), pos.phase ^ 1)) return false;
        ptx::mbar_arrive_expect_tx(bar_full(pos.slot), C::K_TILE);
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
          ptx::tma_load_4d(base + C::OFF_RING + pos.slot * C::K_TILE + c * C::K_ATOM, map, bar_full(pos.slot), 64 * c, hk,
                           tile_key(n), b);
        pos.advance();
        return true;
      };
      // in the order of use: K(0), then K(n + 1), V(n)
      bool alive = load(&tm_k, 0);
      for (int n = 0; n < sp.n && alive; ++n) alive = (n + 1 == sp.n || load(&tm_k, n + 1)) && load(&tm_v, n);
      if (!alive) {  // loads in flight get a bounded time to land before the block ends
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  } else if (warp == C::WARP_MMA || warp == C::WARP_MMA + 1) {
    if (sp.n > 0) {
      // the whole warp walks through the loop, one lane's products count
      const uint32_t one = ptx::elect_one();
      const int x = warp - C::WARP_MMA;
      constexpr uint32_t id_s = f16_idesc<T>(C::BN, false), id_o = f16_idesc<T>(HD, true);
      // The issuer's instructions are on the critical path: descriptors are split into words, of which only the low
      // ones (addresses) change, by constants that are known at compile time.
      const uint64_t dq = make_kmajor_sw128_desc(base + x * C::Q_TILE), dr = make_kmajor_sw128_desc(base + C::OFF_RING);
      const uint64_t dv = mn_major_sw128_desc(base + C::OFF_RING, C::K_ATOM);
      const uint32_t a_lo = static_cast<uint32_t>(dq), k_hi = static_cast<uint32_t>(dr >> 32);
      const uint32_t r_lo = static_cast<uint32_t>(dr), v_lo0 = static_cast<uint32_t>(dv), v_hi = static_cast<uint32_t>(dv >> 32);
      const uint32_t t_x = tmem + x * 128, t_o = tmem + C::COL_O + x * HD;
      uint32_t scored = 0, done = 0;  // score and output products issued so far
      auto wait_warp = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
      // The weights are waited for without suspending: the tensor pipe may have nothing else to do.
      auto wait_soon = [&](uint32_t bar, uint32_t parity) {
        for (int i = 0; i < 4096; ++i)
          if (__all_sync(0xffffffffu, ptx::mbar_probe(bar, parity))) return true;
        return wait_warp(bar, parity);
      };
      RingPos<C::S> pos;
      auto scores = [&](int n) {
        if (!wait_warp(bar_full(pos.slot), pos.phase)) return false;
        if (active(x, n)) {
          const uint32_t buf = scored++ & 1, t_s = t_x + buf * C::BN, b_lo = r_lo + pos.slot * (C::K_TILE >> 4);
          ptx::mma_f16_ss<false>(one, t_s, a_lo, k_hi, b_lo, k_hi, id_s);
#pragma unroll
          for (int j = 1; j < HD / 16; ++j)
            ptx::mma_f16_ss<true>(one, t_s, a_lo + (j >> 2) * (C::Q_ATOM >> 4) + (j & 3) * 2, k_hi,
                                  b_lo + (j >> 2) * (C::K_ATOM >> 4) + (j & 3) * 2, k_hi, id_s);
          ptx::mma_commit_if(one, bar_s(x, buf));
        }
        ptx::mma_commit_if(one, bar_free(pos.slot));
        pos.advance();
        return true;
      };
      auto output = [&](int n) {
        if (!wait_warp(bar_full(pos.slot), pos.phase)) return false;
        if (active(x, n)) {
          const uint32_t buf = done & 1, t_p = t_x + buf * C::BN, b_lo = v_lo0 + pos.slot * (C::K_TILE >> 4);
          if (!wait_soon(bar_p(x, buf), (done >> 1) & 1)) return false;
          ptx::tc_fence_after_sync();
#pragma unroll
          for (int j = 0; j < C::BN / 16; ++j)
            ptx::mma_f16_ts(one, t_o, t_p + (j >> 1) * 32 + (j & 1) * 8, b_lo + j * (2048 >> 4), v_hi, id_o,
                            j > 0 || done > 0 ? 1u : 0u);  // the weights of keys 32.. start at column 32
          ptx::mma_commit_if(one, bar_o(x, buf));
          ++done;
        }
        ptx::mma_commit_if(one, bar_free(pos.slot));
        pos.advance();
        return true;
      };
      bool alive = wait_warp(bar_q, 0) && scores(0);
      for (int n = 0; n < sp.n && alive; ++n) alive = (n + 1 == sp.n || scores(n + 1)) && output(n);
      if (!alive) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  } else if (warp < C::SOFTMAX_WARPS) {
    const int x = warp >> 3, h = (warp >> 2) & 1;   // tile, and half of its keys and of O's columns
    const int r = (warp & 3) * 32 + lane;           // row of the tile = TMEM lane
    const int qi = i0 + x * C::BM + r;
    const int p = min(first_pos(x) + r, sp.p1);     // rows behind the last query see what that one sees
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + C::COL_O + x * HD + h * (HD / 2);
    float* row_float = reinterpret_cast<float*>(gen + C::OFF_ROWS) + x * C::BM + r;
    // The two warps of the same rows meet at a barrier of their own.  A wait that runs out does not end their loops -
    // the other warp would wait at the next meeting - they go on to the end (every other wait gives up at
    // once) and store nothing.
    const int pair_id = 1 + x * 4 + (warp & 3);
    auto meet = [&]() { asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair_id) : "memory"); };
    auto meet_any = [&](bool mine) {
      uint32_t any;
      asm volatile(
          "{\n\t"
          ".reg .pred p, q;\n\t"
          "setp.ne.u32 p, %2, 0;\n\t"
          "barrier.cta.red.or.pred q, %1, 64, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t"
          "}\n" : "=r"(any) : "r"(pair_id), "r"(static_cast<uint32_t>(mine)) : "memory");
      return any != 0;
    };
    // what both threads of a row know, out of what each knows of its half
    auto exchange = [&](float v, auto join) {
      if (h == 0) *row_float = v;
      meet();
      if (h == 1) {
        v = join(*row_float, v);
        *row_float = v;
      }
      meet();
      return h == 0 ? *row_float : v;
    };
    const float sc = a.scale * kLog2e;
    const int pa = first_pos(x), pz = last_pos(x);
    float m = -INFINITY, l = 0.0f;  // the row's maximum, this half's sum
    uint32_t count = 0;             // tiles this row has been through
    bool alive = true;
    for (int n = 0; n < sp.n; ++n) {
      if (!active(x, n)) continue;
      const int j0 = tile_key(n);
      const uint32_t t_s = tmem + lanes + x * 128 + (count & 1) * C::BN + 32 * h;
      alive &= wait(bar_s(x, count & 1), (count >> 1) & 1);
      __syncwarp();
      ptx::tc_fence_after_sync();
      uint32_t s[32];
      ptx::tmem_ld_32x32(t_s, s);
      ptx::tmem_ld_wait_for(s);
      const bool whole = j0 + C::BN - 1 <= pa && (j0 > pz - a.window || j0 + C::BN <= a.sinks);
      // A loop of at most one turn: as a plain condition the whole body is predicated and issued for every tile.
#pragma unroll 1
      for (bool edge = !whole; edge; edge = false) {
        // key j is seen when j <= p and (j > p - window or j < sinks)
        const int j1 = j0 + 32 * h;
        const uint32_t seen = bits_below(p - j1 + 1) & (~bits_below(p - a.window - j1 + 1) | bits_below(a.sinks - j1));
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(seen >> i & 1)) s[i] = 0xff800000u;
      }
      // Weights against the maximum known so far.  A row that has none yet, or whose weights of this tile add up to
      // over 2^9 in one half (the only sign that the maximum moved far), makes its warps find the maximum and do
      // them again.  Only such a row's maximum moves, so what a row gets does not depend on the rows beside it.  One more
      // turn is always enough - a row that has found its maximum here has weights of at most 1, the others' sums stay as they
      // were - and the loop ends there whatever the scores are: sums that are not finite would ask for ever.
      float sum;
      bool mine = m == -INFINITY, find = __any_sync(0xffffffffu, mine);  // the same for both halves
#pragma unroll 1
      for (int turn = 0;; ++turn) {
        if (find) {
          float top = __uint_as_float(s[0]);  // a NaN score makes it NaN
#pragma unroll
          for (int i = 1; i < 32; ++i) top = detail::max_nan(top, __uint_as_float(s[i]));
          top = sc * exchange(top, [](float u, float v) { return detail::max_nan(u, v); });
          const bool move = mine && !(top <= m);
          const float f = move ? exp2_fast(m - top) : 1.0f;  // 0 for a row that starts here
          if (move) m = top;
          l *= f;
          if (count > 0 && __any_sync(0xffffffffu, move)) {
            // the product of the tile before has to be in O (the one before that is: these scores came behind it)
            alive &= wait(bar_o(x, (count - 1) & 1), ((count - 1) >> 1) & 1);
            __syncwarp();
            ptx::tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < HD / 64; ++c) {
              uint32_t o[32];
              ptx::tmem_ld_32x32(t_o + 32 * c, o);
              ptx::tmem_ld_wait_for(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              ptx::tmem_st_32x32(t_o + 32 * c, o);
            }
          }
        }
        // an infinite maximum leaves no weights: NaN, as inf - inf would
        const float neg = m == -INFINITY ? 0.0f : (m == INFINITY ? __int_as_float(0x7fc00000) : -m);
        const uint64_t sc2 = pair(sc, sc), neg2 = pair(neg, neg);
        uint64_t both = pair(0.0f, 0.0f);
        // Exponentials run LAG pairs ahead of their sums and conversions: a warp that asks for a result at once
        // waits out the special-function unit's latency at every pair.  (A quarter of them as a polynomial on the FMA pipe,
        // made safe for masked, infinite and NaN scores, took 890 us instead of 850 at 12 heads x 32760.)
        constexpr int LAG = 4;
        float e[32];
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16 + LAG; ++i) {
          if (i < 16) {
            const uint64_t y = fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sc2, neg2);
            float y0, y1;
            unpair(y, y0, y1);
            e[2 * i] = exp2_fast(y0);
            e[2 * i + 1] = exp2_fast(y1);
          }
          if (i >= LAG) {
            const int j = i - LAG;
            both = add2(both, pair(e[2 * j], e[2 * j + 1]));
            w[j] = pack2(e[2 * j], e[2 * j + 1], T());
          }
        }
        ptx::tmem_st_32x16(t_s, w);
        float sum1;
        unpair(both, sum, sum1);
        sum += sum1;
        if (turn > 0) break;
        const bool bad = !mine && !(sum <= 512.0f);  // a row that just moved has weights of at most 1
        find = meet_any(bad);
        if (!find) break;
        mine = exchange(bad ? 1.0f : 0.0f, [](float u, float v) { return fmaxf(u, v); }) != 0.0f;
        meet();
        ptx::tmem_st_wait();  // the weights are written again
      }
      l += sum;
#pragma unroll 1
      for (bool edge = !cta_sees(j0); edge; edge = false) {  // behind the weights: V(n) has had their time to arrive
        const uint32_t at = n + 1 < sp.n ? 2 * n + 2 : 2 * n + 1, slot = at % C::S;  // V(n) in the ring
        const bool here = wait(bar_full(slot), (at / C::S) & 1);
        alive &= here;
        if (here) {
          const int row = r & 63, j = j0 + row;
          const bool covered = j <= sp.hi && (j >= sp.lo || j < a.sinks);  // by some row
#pragma unroll
          for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint8_t* chunk = gen + C::OFF_RING + slot * C::K_TILE + c * C::K_ATOM + row * 128 + 16 * (i + 2 * (r >> 6) + 4 * h);
              if (!covered) {
                *reinterpret_cast<uint4*>(chunk) = make_uint4(0, 0, 0, 0);
              } else if (any_not_finite<T>(chunk)) {
                *cleared = 1;
                __threadfence_block();
                clear_not_finite<T>(chunk);
              }
            }
        }
        // Whoever wrote: what the other tile cleared may have been read here as finite already.
        ptx::fence_proxy_async_smem();
      }
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_p(x, count & 1));
      ++count;
    }
    if (count > 0) {
      alive &= wait(bar_o(x, (count - 1) & 1), ((count - 1) >> 1) & 1);
      __syncwarp();
      ptx::tc_fence_after_sync();
    }
    l = exchange(l, [](float u, float v) { return u + v; });
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    const bool ok = qi < a.Lq && alive;
    if (h == 0 && ok && a.lse != nullptr)
      a.lse[(static_cast<long long>(b) * a.Hq + hq) * a.Lq + qi] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    T* out = static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.Lq + qi) * a.Hq + hq) * HD + h * (HD / 2);
#pragma unroll 1
    for (int c = 0; c < HD / 64; ++c) {
      uint32_t o[32];
      if (count > 0) {  // the same for the whole warp
        ptx::tmem_ld_32x32(t_o + 32 * c, o);
        ptx::tmem_ld_wait_for(o);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0u;
      }
      if (ok) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[j] = pack2(__uint_as_float(o[8 * i + 2 * j]) * inv, __uint_as_float(o[8 * i + 2 * j + 1]) * inv, T());
          *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == C::WARP_MMA) {
    __syncwarp();
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<1>(tmem, C::TMEM_COLS);
  }
  if (*cleared != 0 && *abort_flag == 0 && warp < C::SOFTMAX_WARPS) {
    // each warp its rows and columns, a lane a column (or two) of one row after another
    const int x = warp >> 3, h = (warp >> 2) & 1;
    const T* v = static_cast<const T*>(a.v) + b * a.v_b + (hq / a.G) * a.v_h + h * (HD / 2) + lane;
#pragma unroll 1
    for (int r = 0; r < 32; ++r) {
      const int qi = i0 + x * C::BM + (warp & 3) * 32 + r, p = sp.p0 + qi - i0;
      if (qi > i1) break;
      float bad[HD / 64] = {};
      for (int n = 0; n < sp.n; ++n) {
        const int j0 = tile_key(n);
        if (cta_sees(j0)) continue;
#pragma unroll 4
        for (int j = j0; j < j0 + C::BN; ++j) {
          if (!(j <= p && (j > p - a.window || j < a.sinks))) continue;
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) {
            const float y = static_cast<float>(v[j * a.v_t + 32 * c]);
            if (!(fabsf(y) < INFINITY)) bad[c] += y;
          }
        }
      }
      T* out = static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.Lq + qi) * a.Hq + hq) * HD + h * (HD / 2) + lane;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c)
        if (bad[c] != 0.0f) out[32 * c] = static_cast<T>(static_cast<float>(out[32 * c]) + bad[c]);
    }
  }
}

// [batch, token, head, HD] as a 4-D map (HD, head, token, batch) with boxes of 64 values x 64 tokens.
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
  const cuuint32_t box[4] = {64, 1, 64, 1}, one[4] = {1, 1, 1, 1};
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
