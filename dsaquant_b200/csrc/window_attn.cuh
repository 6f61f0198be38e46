// Causal attention with a sliding window and a few first keys that stay visible (sinks).
// Query i of a sequence whose cache holds `len` keys sits at position p = len - Lq + i and sees key j when
//   j <= p  and  (j > p - window  or  j < sinks).
//   out = sum_j softmax_j(q . k_j * scale) v_j,   lse = log sum_j exp(q . k_j * scale)
// A query that sees nothing (p < 0) has out = 0 and lse = -inf.
//
// A tile is ROWS (query, head) rows of the heads that share one key head: row r is query r / G, head r % G,
// so a cached key tile serves the whole group, for prompts and single tokens alike.  The keys that any row
// of the tile sees are two runs of key tiles - [0, first) for the sinks and [w0, w1] for the window - and only
// those are visited; the mask is evaluated only in tiles that some row does not see entirely.
// Keys that no row of the tile sees are read as zeros, so whatever lies there (freed or unwritten cache
// lines, NaN among them) has no effect.  A key that some rows of the tile see and others do not enters the second
// product of all of them, of the others with weight 0 - and 0 * inf is NaN.  So in the key tiles that some row does not see
// entirely, values of V that are not finite are replaced by zeros in shared memory, and only if there were any, the rows that
// see them get them added at the end: their sum is then inf or NaN as by the formula, whatever the finite rest is.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200w4a4 {

struct WindowAttnArgs {
  const void *q, *k, *v;  // [B, Lq, Hq, HD], [B, Lk, Hkv, HD]
  void* out;              // [B, Lq, Hq, HD] contiguous
  float* lse;             // [B, Hq, Lq] or null
  const int* kv_lens;     // [B] or null: Lk
  long long q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;  // pitches in elements
  int B, Lq, Lk, Hq, Hkv, G;
  int window, sinks;
  float scale;
  int splits;       // key runs a row's tiles are split into; > 1: partial results go to the workspace
  float* part_o;    // [splits, B, Hq, Lq, HD]
  float* part_lse;  // [splits, B, Hq, Lq], in units of log2
};

namespace attn {

// What a tile of rows [r0, r1] of one sequence has to visit.
struct Span {
  int p0, p1;     // positions of its first and last query
  int lo, hi;     // keys [lo, hi] cover every row's window (hi < lo: nothing)
  int n_sink, w0, n;  // key tiles: [0, n_sink) and [w0, w0 + n - n_sink)
};

template <int BN>
__device__ __forceinline__ Span span_of(const WindowAttnArgs& a, int b, int i0, int i1) {
  Span s;
  int len = a.Lk;
  if (a.kv_lens != nullptr) len = min(max(a.kv_lens[b], 0), a.Lk);
  s.p0 = len - a.Lq + i0;
  s.p1 = len - a.Lq + i1;
  s.hi = s.p1;
  const int first = max(s.p0, 0);  // rows before position 0 see nothing
  s.lo = max(0, first - a.window + 1);
  if (s.hi < 0) {
    s.n_sink = s.w0 = s.n = 0;
    s.lo = 0;
    return s;
  }
  s.w0 = s.lo / BN;
  s.n_sink = min((min(a.sinks, s.lo) + BN - 1) / BN, s.w0);
  s.n = s.n_sink + s.hi / BN - s.w0 + 1;
  return s;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// 16 bytes global -> shared; zeros when !ok (nothing is read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Element offset of 16-byte chunk c of row r in a [rows][HD] tile: chunks of a row are permuted by
// the row's low bits, so the eight rows that one ldmatrix phase touches sit in different banks.
template <int HD>
__device__ __forceinline__ int swz(int r, int c) {
  return r * HD + ((c ^ (r & 7)) << 3);
}

// Bit 15 of each 16-bit half that is an infinity or a NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t w, __half) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ uint32_t not_finite(uint32_t w, __nv_bfloat16) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

template <typename T>
__device__ __forceinline__ bool any_not_finite(const void* p) {
  const uint4 v = *static_cast<const uint4*>(p);
  return (not_finite(v.x, T()) | not_finite(v.y, T()) | not_finite(v.z, T()) | not_finite(v.w, T())) != 0;
}

// Eight values in shared memory: those that are not finite become 0.  True if there were any.
template <typename T>
__device__ __forceinline__ bool clear_not_finite(void* p) {
  uint4 v = *static_cast<const uint4*>(p);
  const uint32_t x = not_finite(v.x, T()), y = not_finite(v.y, T()), z = not_finite(v.z, T()), w = not_finite(v.w, T());
  if ((x | y | z | w) == 0) return false;
  v.x &= ~((x >> 15) * 0xffffu);
  v.y &= ~((y >> 15) * 0xffffu);
  v.z &= ~((z >> 15) * 0xffffu);
  v.w &= ~((w >> 15) * 0xffffu);
  *static_cast<uint4*>(p) = v;
  return true;
}

// Adds the values that are not finite of V's keys [j0, j0 + KEYS) to a thread's two rows (columns 8 h + 2 t and the next) that see them.
template <typename T, int HD, int KEYS>
__device__ __forceinline__ void add_not_finite(float (&o)[HD / 8][4], const T* v, long long v_t, int j0, const int (&pos)[2],
                                               int window, int sinks) {
#pragma unroll 1
  for (int j = j0; j < j0 + KEYS; ++j) {
    bool sees[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) sees[i] = j <= pos[i] && (j > pos[i] - window || j < sinks);
    if (!sees[0] && !sees[1]) continue;
    const uint32_t* row = reinterpret_cast<const uint32_t*>(v + j * v_t);
#pragma unroll
    for (int h = 0; h < HD / 8; ++h) {
      const uint32_t w = __ldg(row + 4 * h), bad = not_finite(w, T());
      const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (sees[k >> 1] && (bad >> (16 * (k & 1) + 15) & 1) != 0) o[h][k] += static_cast<float>(x[k & 1]);
    }
  }
}

}  // namespace attn

// Short chunks (more rows than the single-token kernel takes, fewer than 128 queries), and prompts whose pitches no
// tensor map can express: mma.sync, four warps of 16 rows each, key tiles of 64 in two cp.async stages.
// Measured: 2 x 60 queries on 8000 keys, 8 heads of 128: 35 us; 8 x 127 on up to 8000 keys, 12 heads: 147; 32 x 127 on 16000
// keys, 40 query and 8 key heads: 4.85 ms, 0.27 PFLOP/s.  What bounds it is mma.sync: every warp reads each key tile again
// from shared memory, for 16 rows.
constexpr int kAttnRows = 64, kAttnBN = 64;

template <typename T, int HD>
__global__ void __launch_bounds__(128) window_attn_kernel(const WindowAttnArgs a) {
  using namespace attn;
  constexpr int BN = kAttnBN, KT = HD / 16;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  T* sk = reinterpret_cast<T*>(smem_raw);  // [2][BN][HD]
  T* sv = sk + 2 * BN * HD;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int hk = blockIdx.y;
  const int b = blockIdx.z / a.splits, split = blockIdx.z % a.splits;
  const long long rows = static_cast<long long>(a.Lq) * a.G;
  const long long r0 = static_cast<long long>(blockIdx.x) * kAttnRows;
  const long long r1 = min(r0 + kAttnRows, rows) - 1;
  const Span sp = span_of<BN>(a, b, static_cast<int>(r0 / a.G), static_cast<int>(r1 / a.G));
  const int per = (sp.n + a.splits - 1) / a.splits;
  const int first = min(split * per, sp.n), last = min(first + per, sp.n);

  // this thread's two rows
  int pos[2];
  long long q_off[2];
  bool row_ok[2];
  int qi[2], qh[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const long long r = r0 + 16 * warp + g + 8 * i;
    row_ok[i] = r < rows;
    qi[i] = static_cast<int>((row_ok[i] ? r : rows - 1) / a.G);
    qh[i] = hk * a.G + static_cast<int>((row_ok[i] ? r : rows - 1) % a.G);
    pos[i] = sp.p0 - static_cast<int>(r0 / a.G) + qi[i];
    q_off[i] = b * a.q_b + qi[i] * a.q_t + qh[i] * a.q_h;
  }
  uint32_t qf[KT][4];
  {
    const T* q = static_cast<const T*>(a.q);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qf[kt][i] = __ldg(reinterpret_cast<const uint32_t*>(q + q_off[i & 1] + 16 * kt + 2 * t + 8 * (i >> 1)));
  }

  const T* kb = static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h;
  const T* vb = static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h;
  auto tile_key = [&](int n) { return (n < sp.n_sink ? n : sp.w0 + n - sp.n_sink) * BN; };
  auto load = [&](int n, int stage) {
    const int j0 = tile_key(n);
    constexpr int CH = HD / 8;
#pragma unroll
    for (int i = 0; i < BN * CH / 128; ++i) {
      const int c = threadIdx.x + i * 128;
      const int r = c / CH, ch = c % CH;
      const int j = j0 + r;
      const bool ok = j <= sp.hi && (j >= sp.lo || j < a.sinks);
      cp16(smem_addr(sk + stage * BN * HD + swz<HD>(r, ch)), kb + (ok ? j * a.k_t + ch * 8 : 0), ok);
      cp16(smem_addr(sv + stage * BN * HD + swz<HD>(r, ch)), vb + (ok ? j * a.v_t + ch * 8 : 0), ok);
    }
  };

  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  const float sc = a.scale * kLog2e;

  // every row sees the whole tile when its last key is at or before the first position and its first
  // key is inside the last position's window
  auto sees_all = [&](int j0) { return j0 + BN - 1 <= sp.p0 && (j0 > sp.p1 - a.window || j0 + BN <= a.sinks); };
  bool cleared = false;  // of V, somewhere
  if (first < last) load(first, 0);
  cp_commit();
  for (int n = first; n < last; ++n) {
    const int stage = (n - first) & 1;
    const int j0 = tile_key(n);
    const bool whole = sees_all(j0);
    if (n + 1 < last) load(n + 1, stage ^ 1);
    cp_commit();
    cp_wait<1>();
    if (!whole && sp.p0 != sp.p1) {  // (rows of one position see the same keys)
#pragma unroll
      for (int i = 0; i < BN * (HD / 8) / 128; ++i) {  // the chunks that this thread copied
        const int c = threadIdx.x + i * 128;
        cleared |= clear_not_finite<T>(sv + stage * BN * HD + swz<HD>(c / (HD / 8), c % (HD / 8)));
      }
    }
    __syncthreads();
    const T* ks = sk + stage * BN * HD;
    const T* vs = sv + stage * BN * HD;
    float s[BN / 8][4];
#pragma unroll
    for (int i = 0; i < BN / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int nt = 0; nt < BN / 16; ++nt) {
        // matrices: keys 0-7 | k lo, keys 0-7 | k hi, keys 8-15 | k lo, keys 8-15 | k hi
        uint32_t f[4];
        ldsm4(f, smem_addr(ks + swz<HD>(16 * nt + (lane & 7) + ((lane >> 4) << 3), 2 * kt + ((lane >> 3) & 1))));
        mma(s[2 * nt], qf[kt], f[0], f[1], T());
        mma(s[2 * nt + 1], qf[kt], f[2], f[3], T());
      }
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < BN / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = j0 + 8 * i + 2 * t + (j & 1), p = pos[j >> 1];
          if (!(key <= p && (key > p - a.window || key < a.sinks))) s[i][j] = -INFINITY;
        }
    }
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int i = 0; i < BN / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx[j >> 1] = fmaxf(mx[j >> 1], s[i][j] * sc);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float base = mx[i] == -INFINITY ? 0.0f : mx[i];
      const float f = exp2_fast(m[i] - base);
      m[i] = mx[i];
      l[i] *= f;
#pragma unroll
      for (int h = 0; h < HD / 8; ++h) {
        o[h][2 * i] *= f;
        o[h][2 * i + 1] *= f;
      }
      mx[i] = base;
    }
#pragma unroll
    for (int i = 0; i < BN / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2_fast(fmaf(s[i][j], sc, -mx[j >> 1]));
        l[j >> 1] += s[i][j];
      }
#pragma unroll
    for (int kt = 0; kt < BN / 16; ++kt) {
      const uint32_t p[4] = {pack2(s[2 * kt][0], s[2 * kt][1], T()), pack2(s[2 * kt][2], s[2 * kt][3], T()),
                             pack2(s[2 * kt + 1][0], s[2 * kt + 1][1], T()), pack2(s[2 * kt + 1][2], s[2 * kt + 1][3], T())};
#pragma unroll
      for (int ht = 0; ht < HD / 16; ++ht) {
        // transposed: keys lo | dims 0-7, keys hi | dims 0-7, keys lo | dims 8-15, keys hi | dims 8-15
        uint32_t f[4];
        ldsm4t(f, smem_addr(vs + swz<HD>(16 * kt + (lane & 15), 2 * ht + (lane >> 4))));
        mma(o[2 * ht], p, f[0], f[1], T());
        mma(o[2 * ht + 1], p, f[2], f[3], T());
      }
    }
    __syncthreads();
  }

  if (__syncthreads_or(cleared))
    for (int n = first; n < last; ++n)
      if (!sees_all(tile_key(n))) add_not_finite<T, HD, BN>(o, vb + 2 * t, a.v_t, tile_key(n), pos, a.window, a.sinks);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (!row_ok[i]) continue;
    const float inv = l[i] > 0.0f ? 1.0f / l[i] : (l[i] == 0.0f ? 0.0f : l[i]);
    const float lse2 = l[i] == 0.0f ? -INFINITY : m[i] + log2f(l[i]);
    const long long head_row = (static_cast<long long>(b) * a.Hq + qh[i]) * a.Lq + qi[i];
    if (a.splits > 1) {
      const long long at = static_cast<long long>(split) * a.B * a.Hq * a.Lq + head_row;
      if (t == 0) a.part_lse[at] = lse2;
      float2* po = reinterpret_cast<float2*>(a.part_o + at * HD) + t;
#pragma unroll
      for (int h = 0; h < HD / 8; ++h) po[4 * h] = make_float2(o[h][2 * i] * inv, o[h][2 * i + 1] * inv);
    } else {
      if (t == 0 && a.lse != nullptr) a.lse[head_row] = lse2 * kLn2;
      T* out = static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.Lq + qi[i]) * a.Hq + qh[i]) * HD + 2 * t;
#pragma unroll
      for (int h = 0; h < HD / 8; ++h)
        *reinterpret_cast<uint32_t*>(out + 8 * h) = pack2(o[h][2 * i] * inv, o[h][2 * i + 1] * inv, T());
    }
  }
}

// Single tokens: at most 16 rows a tile.  What bounds it is reading the keys and values once, so a CTA's four warps
// each take 16 keys of every 64-key tile through a ring of their own (cp.async, kAttnDecodeStages deep, no barrier
// between the warps), keep their own maximum, sum and output, and meet at the end in shared memory.
// Measured, 16 sequences of 0 to 8192 keys, 40 query and 8 key heads of 128, window 4096: 44 us with the joining kernel
// for 206 MB (4.7 TB/s, 0.72 of the copy rate); the 64-row form above took 67.5.  96 KB of ring allow two blocks an SM, whose
// blocks of unequal length come in 2.2 waves.
constexpr int kAttnDecodeRows = 16, kAttnDecodeStages = 3;

template <typename T, int HD>
__global__ void __launch_bounds__(128) window_attn_decode_kernel(const WindowAttnArgs a) {
  using namespace attn;
  constexpr int BN = kAttnBN, WN = 16, KT = HD / 16, CH = HD / 8, D = kAttnDecodeStages;
  constexpr int TILE = WN * HD;  // values of a warp's K (or V) tile
  extern __shared__ __align__(128) uint8_t smem_raw[];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int hk = blockIdx.y;
  const int b = blockIdx.z / a.splits, split = blockIdx.z % a.splits;
  const int rows = a.Lq * a.G;
  const int r0 = blockIdx.x * kAttnDecodeRows;
  const int r1 = min(r0 + kAttnDecodeRows, rows) - 1;
  const Span sp = span_of<BN>(a, b, r0 / a.G, r1 / a.G);
  const int per = (sp.n + a.splits - 1) / a.splits;
  const int first = min(split * per, sp.n), last = min(first + per, sp.n);

  T* ring = reinterpret_cast<T*>(smem_raw) + warp * (D * 2 * TILE);
  const T* kb = static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h;
  const T* vb = static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h;
  auto tile_key = [&](int n) { return (n < sp.n_sink ? n : sp.w0 + n - sp.n_sink) * BN + warp * WN; };
  auto load = [&](int n, int stage) {
    const int j0 = tile_key(n);
    T* sk = ring + stage * (2 * TILE);
#pragma unroll
    for (int i = 0; i < WN * CH / 32; ++i) {
      const int r = lane / CH + i * (32 / CH), ch = lane % CH;
      const long long j = j0 + r;
      const bool ok = j <= sp.hi && (j >= sp.lo || j < a.sinks);
      cp16(smem_addr(sk + swz<HD>(r, ch)), kb + (ok ? j * a.k_t + ch * 8 : 0), ok);
      cp16(smem_addr(sk + TILE + swz<HD>(r, ch)), vb + (ok ? j * a.v_t + ch * 8 : 0), ok);
    }
  };
#pragma unroll
  for (int d = 0; d < D - 1; ++d) {
    if (first + d < last) load(first + d, d);
    cp_commit();
  }

  int pos[2];
  uint32_t qf[KT][4];
  {
    const T* q = static_cast<const T*>(a.q);
    long long off[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = min(r0 + g + 8 * i, rows - 1);  // rows behind the last one repeat it and are not stored
      pos[i] = sp.p0 - r0 / a.G + r / a.G;
      off[i] = b * a.q_b + (r / a.G) * a.q_t + (hk * a.G + r % a.G) * a.q_h;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qf[kt][i] = __ldg(reinterpret_cast<const uint32_t*>(q + off[i & 1] + 16 * kt + 2 * t + 8 * (i >> 1)));
  }

  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  const float sc = a.scale * kLog2e;

  auto sees_all = [&](int j0) { return j0 + WN - 1 <= sp.p0 && (j0 > sp.p1 - a.window || j0 + WN <= a.sinks); };
  bool cleared = false;  // of V, somewhere
  int stage = 0;
  for (int n = first; n < last; ++n) {
    const int j0 = tile_key(n);
    const bool whole = sees_all(j0);
    cp_wait<D - 2>();
    if (!whole && sp.p0 != sp.p1) {  // (rows of one position see the same keys)
#pragma unroll
      for (int i = 0; i < WN * CH / 32; ++i)  // the chunks that this lane copied
        cleared |= clear_not_finite<T>(ring + stage * (2 * TILE) + TILE + swz<HD>(lane / CH + i * (32 / CH), lane % CH));
    }
    __syncwarp();  // the warp's copies have landed, and it is done with the stage that is filled next
    if (n + D - 1 < last) load(n + D - 1, stage == 0 ? D - 1 : stage - 1);
    cp_commit();
    const T* ks = ring + stage * (2 * TILE);
    const T* vs = ks + TILE;
    stage = stage == D - 1 ? 0 : stage + 1;
    if (j0 > sp.p1) continue;  // this warp's share of the last tile is behind every row
    float s[2][4] = {};
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      uint32_t f[4];
      ldsm4(f, smem_addr(ks + swz<HD>((lane & 7) + ((lane >> 4) << 3), 2 * kt + ((lane >> 3) & 1))));
      mma(s[0], qf[kt], f[0], f[1], T());
      mma(s[1], qf[kt], f[2], f[3], T());
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = j0 + 8 * i + 2 * t + (j & 1), p = pos[j >> 1];
          if (!(key <= p && (key > p - a.window || key < a.sinks))) s[i][j] = -INFINITY;
        }
    }
    float mx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1])) * sc;
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
    }
    // the maximum moves only when a weight would pass 2^8: sums and outputs are fp32, weights 16 bits up to 256
    const bool move0 = mx[0] > m[0] + 8.0f, move1 = mx[1] > m[1] + 8.0f;
    if (__any_sync(0xffffffffu, move0 || move1)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float next = (i ? move1 : move0) ? mx[i] : m[i];
        const float f = next == m[i] ? 1.0f : exp2_fast(m[i] - next);
        m[i] = next;
        l[i] *= f;
#pragma unroll
        for (int h = 0; h < HD / 8; ++h) {
          o[h][2 * i] *= f;
          o[h][2 * i + 1] *= f;
        }
      }
    }
    const float neg[2] = {m[0] == -INFINITY ? 0.0f : -m[0], m[1] == -INFINITY ? 0.0f : -m[1]};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2_fast(fmaf(s[i][j], sc, neg[j >> 1]));
        l[j >> 1] += s[i][j];
      }
    const uint32_t p[4] = {pack2(s[0][0], s[0][1], T()), pack2(s[0][2], s[0][3], T()), pack2(s[1][0], s[1][1], T()),
                           pack2(s[1][2], s[1][3], T())};
#pragma unroll
    for (int ht = 0; ht < HD / 16; ++ht) {
      uint32_t f[4];
      ldsm4t(f, smem_addr(vs + swz<HD>(lane & 15, 2 * ht + (lane >> 4))));
      mma(o[2 * ht], p, f[0], f[1], T());
      mma(o[2 * ht + 1], p, f[2], f[3], T());
    }
  }

  if (__any_sync(0xffffffffu, cleared))
    for (int n = first; n < last; ++n)
      if (!sees_all(tile_key(n))) add_not_finite<T, HD, WN>(o, vb + 2 * t, a.v_t, tile_key(n), pos, a.window, a.sinks);

  // the four warps' results: [warp][row][HD] outputs, then maxima and sums
  constexpr int OP = HD + 8;  // row pitch: the rows of a store land in different banks
  float* po = reinterpret_cast<float*>(smem_raw);
  float* pm = po + 4 * kAttnDecodeRows * OP;
  float* pl = pm + 4 * kAttnDecodeRows;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = warp * kAttnDecodeRows + g + 8 * i;
#pragma unroll
    for (int h = 0; h < HD / 8; ++h)
      *reinterpret_cast<float2*>(po + r * OP + 8 * h + 2 * t) = make_float2(o[h][2 * i], o[h][2 * i + 1]);
    if (t == 0) {
      pm[r] = m[i];
      pl[r] = l[i];
    }
  }
  __syncthreads();
  constexpr int LANES = HD / 4;  // threads of a row, four values each
  for (int r = threadIdx.x / LANES; r <= r1 - r0; r += 128 / LANES) {
    const int c = threadIdx.x % LANES * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, pm[w * kAttnDecodeRows + r]);
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, acc[4] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_fast(pm[w * kAttnDecodeRows + r] - base);
      total = fmaf(pl[w * kAttnDecodeRows + r], f, total);
      const float4 v = *reinterpret_cast<const float4*>(po + (w * kAttnDecodeRows + r) * OP + c);
      acc[0] = fmaf(v.x, f, acc[0]);
      acc[1] = fmaf(v.y, f, acc[1]);
      acc[2] = fmaf(v.z, f, acc[2]);
      acc[3] = fmaf(v.w, f, acc[3]);
    }
    const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
    const float lse2 = total == 0.0f ? -INFINITY : base + log2f(total);
    const int qi = (r0 + r) / a.G, qh = hk * a.G + (r0 + r) % a.G;
    const long long head_row = (static_cast<long long>(b) * a.Hq + qh) * a.Lq + qi;
    if (a.splits > 1) {
      const long long at = static_cast<long long>(split) * a.B * a.Hq * a.Lq + head_row;
      if (c == 0) a.part_lse[at] = lse2;
      if (lse2 != -INFINITY)
        *reinterpret_cast<float4*>(a.part_o + at * HD + c) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      if (c == 0 && a.lse != nullptr) a.lse[head_row] = lse2 * kLn2;
      T* out = static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.Lq + qi) * a.Hq + qh) * HD + c;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2(acc[0] * inv, acc[1] * inv, T()), pack2(acc[2] * inv, acc[3] * inv, T()));
    }
  }
}

// Joins the partial results of the splits: one warp a (batch, head, query) row.
template <typename T, int HD>
__global__ void __launch_bounds__(128) window_attn_join_kernel(const WindowAttnArgs a) {
  using namespace attn;
  const long long rows = static_cast<long long>(a.B) * a.Hq * a.Lq;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, a.part_lse[s * rows + row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float base = m == -INFINITY ? 0.0f : m;
  float total = 0.0f;
  float acc[HD / 32] = {};
  for (int s0 = 0; s0 < a.splits; s0 += 4) {  // four runs' loads at a time
    float w[4], o[4][HD / 32];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = s0 + u < a.splits ? a.part_lse[(s0 + u) * rows + row] : -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)  // a run without keys: its partial output is not read
        o[u][i] = w[u] == -INFINITY ? 0.0f : a.part_o[((s0 + u) * rows + row) * HD + lane + 32 * i];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      w[u] = exp2_fast(w[u] - base);
      total += w[u];
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) acc[i] = fmaf(w[u], o[u][i], acc[i]);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int qi = static_cast<int>(row % a.Lq);
  const long long bh = row / a.Lq;
  const int h = static_cast<int>(bh % a.Hq), b = static_cast<int>(bh / a.Hq);
  if (lane == 0 && a.lse != nullptr) a.lse[row] = total == 0.0f ? -INFINITY : (base + log2f(total)) * kLn2;
  T* out = static_cast<T*>(a.out) + ((static_cast<long long>(b) * a.Lq + qi) * a.Hq + h) * HD + lane;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) out[32 * i] = static_cast<T>(acc[i] * inv);
}

// The form of a call without tensor-core tiles of queries: rows up to 32 take the single-token kernel (a second tile of
// 16 rows reads the keys again, from L2), more the one with 64-row tiles.
inline bool window_attn_decodes(long long rows) { return rows <= 2 * kAttnDecodeRows; }

// Runs the keys of a row tile are split into: enough for four CTAs an SM, none shorter than two key tiles, at most 64 (and at
// most 65535 / B, see attention_splits).  The single-token kernel's are also no longer than 1024 keys while that allows it, so
// that sequences of unequal lengths share the GPU evenly; its partial outputs, 32 rows a key head at most, are then a
// thirtieth of the keys and values.  In the 64-row form they would be an eighth for every tile of rows (1.3 GB for 32 x 127
// queries of 40 heads of 128 on 16000 keys, for 42 MB of output), so there the first rule alone counts.
inline int window_attn_splits(int B, int Lq, int Lk, int Hkv, int G, int window, int sinks, int sm_count) {
  const long long rows = static_cast<long long>(Lq) * G;
  const int per_tile = window_attn_decodes(rows) ? kAttnDecodeRows : kAttnRows;
  const long long tiles = (rows + per_tile - 1) / per_tile * Hkv * B;
  if (tiles <= 0) return 1;
  const long long reach = static_cast<long long>(window) + per_tile / G + 1;
  const long long keys = Lk < reach ? Lk : (Lk < reach + sinks ? Lk : reach + sinks);
  const long long key_tiles = (keys + kAttnBN - 1) / kAttnBN + 1;  // a window need not start at a tile's edge
  long long s = (4LL * sm_count + tiles - 1) / tiles;
  if (window_attn_decodes(rows) && s < (key_tiles + 15) / 16) s = (key_tiles + 15) / 16;
  if (s > key_tiles / 2) s = key_tiles / 2;
  if (s > 64) s = 64;
  return s < 1 ? 1 : static_cast<int>(s);
}

template <typename T, int HD>
inline cudaError_t launch_window_attn(const WindowAttnArgs& a, cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.Lq) * a.G;
  const bool decode = window_attn_decodes(rows);
  constexpr int ring = 4 * kAttnDecodeStages * 2 * 16 * HD * 2, meet = 4 * kAttnDecodeRows * (HD + 8 + 2) * 4;
  const int smem = decode ? (ring > meet ? ring : meet) : 4 * kAttnBN * HD * 2;
  const int per_tile = decode ? kAttnDecodeRows : kAttnRows;
  const auto kernel = decode ? window_attn_decode_kernel<T, HD> : window_attn_kernel<T, HD>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>((rows + per_tile - 1) / per_tile), static_cast<unsigned>(a.Hkv),
                  static_cast<unsigned>(a.B * a.splits));
  kernel<<<grid, 128, smem, stream>>>(a);
  if (a.splits > 1) {
    const long long total = static_cast<long long>(a.B) * a.Hq * a.Lq;
    window_attn_join_kernel<T, HD><<<static_cast<unsigned>((total + 3) / 4), 128, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace b200w4a4
