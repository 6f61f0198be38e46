// Rotary positions on q and k in one launch.  Pair i of a head (i < rotary_dim / 2) at position p:
//   u = a cos(p f_i) - b sin(p f_i),  v = a sin(p f_i) + b cos(p f_i)
// (a, b) are the values i and i + rotary_dim / 2 of the head ("half" layout) or 2i and 2i + 1
// (interleaved); values behind rotary_dim are copied.  cos and sin come from a table built in 64
// bits, one row a position, so a far position is as exact as a near one.
//
// HBM-bound: every value is read and written once.  A head is cut into units that one thread moves
// with 128-bit accesses, and a thread keeps its unit for all heads of its token that it visits, so
// the pairs' cos and sin are fetched once a thread and not once a head.  Blocks of 128 threads, two heads a thread at
// a time (one in fp32).  Measured at 32760 tokens: 40 + 40 heads of 128 in pairs 212 us (6.40 TB/s, 0.99 of the copy rate),
// 40 + 8 heads in halves 148 us (5.57), 12 + 2 heads with half of each rotated 70 us; with 256 threads 234, 162 and 94 us, with
// four heads at a time 213, 188 and 121 us.
//
// A token at a negative position is copied unchanged (in place: left alone): the padding behind the
// last sequence.  A position behind the table gives NaN in the rotated part.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "rms_norm.cuh"  // Chunk, store8, load_f32, store_f32

namespace b200w4a4 {

namespace detail {
template <typename T>
__device__ __forceinline__ void store_raw(T* p, const Chunk<T>& c) {
  *reinterpret_cast<uint4*>(p) = c.raw;
}
__device__ __forceinline__ void store_raw(float* p, const Chunk<float>& c) {
  reinterpret_cast<float4*>(p)[0] = c.lo;
  reinterpret_cast<float4*>(p)[1] = c.hi;
}
}  // namespace detail

struct RotaryArgs {
  const void* in[2];  // q, k: [T, heads, head_dim], token and head pitches in elements
  void* out[2];
  long long in_tok[2], in_head[2], out_tok[2], out_head[2];
  int heads[2];
  const float* cos_sin;   // [max_pos, rotary_dim / 2, 2]
  const void* positions;  // int32 or int64 [T]
  long long max_pos, T;
  int head_dim, rotary_dim;
  int units;           // units a head is cut into
  int rows_per_block;  // (token, head) rows a block holds at once; threads = units * rows_per_block
  int tokens_per_block;
  bool pos64;
  float sign;  // -1 rotates back
};

constexpr int kRotaryThreads = 128;
constexpr int kRotaryMaxHeadDim = 512;

template <typename T, bool INTERLEAVED, bool VEC>
__global__ void __launch_bounds__(512) rotary_kernel(const RotaryArgs a) {
  // pairs a unit holds: 16 values in two vectors (half), 8 in one (interleaved), or one pair
  constexpr int P = VEC ? (INTERLEAVED ? 4 : 8) : 1;
  constexpr int COPY = VEC ? 8 : 1;  // values of a unit behind the rotated part
  const int unit = threadIdx.x % a.units;
  const int row0 = threadIdx.x / a.units;
  const int heads = a.heads[0] + a.heads[1];
  const long long token = static_cast<long long>(blockIdx.x) * a.tokens_per_block + row0 / heads;
  if (token >= a.T || row0 / heads >= a.tokens_per_block) return;
  const long long pos = a.pos64 ? static_cast<const long long*>(a.positions)[token]
                                : static_cast<long long>(static_cast<const int*>(a.positions)[token]);
  const int rot_units = a.rotary_dim / (2 * P);
  const bool rotated = unit < rot_units;
  float c[P], s[P];
#pragma unroll
  for (int i = 0; i < P; ++i) c[i] = 1.0f, s[i] = 0.0f;
  if (rotated && pos >= 0) {
    if (pos < a.max_pos) {
      const float* row = a.cos_sin + pos * a.rotary_dim + 2 * P * unit;
      if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < P; i += 2) {
          const float4 cs = __ldg(reinterpret_cast<const float4*>(row + 2 * i));
          c[i] = cs.x;
          s[i] = cs.y * a.sign;
          c[i + 1] = cs.z;
          s[i + 1] = cs.w * a.sign;
        }
      } else {
        const float2 cs = __ldg(reinterpret_cast<const float2*>(row));
        c[0] = cs.x;
        s[0] = cs.y * a.sign;
      }
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
    }
  }
  const int half = a.rotary_dim / 2;
  // first value of the unit, and of its second vector
  const int at0 = rotated ? (INTERLEAVED ? 2 * P * unit : P * unit) : a.rotary_dim + COPY * (unit - rot_units);
  // a few heads at a time: their loads come before the stores, which may go to the same place
  constexpr int BATCH = sizeof(T) == 4 ? 1 : 2;
  for (int head0 = row0 % heads; head0 < heads; head0 += BATCH * a.rows_per_block) {
    const T* in[BATCH];
    T* out[BATCH];
#pragma unroll
    for (int m = 0; m < BATCH; ++m) {
      const int head = head0 + m * a.rows_per_block;
      const int which = head >= a.heads[0];
      const int h = which ? head - a.heads[0] : head;
      in[m] = static_cast<const T*>(a.in[which]) + token * a.in_tok[which] + h * a.in_head[which] + at0;
      out[m] = static_cast<T*>(a.out[which]) + token * a.out_tok[which] + h * a.out_head[which] + at0;
    }
    auto valid = [&](int m) { return head0 + m * a.rows_per_block < heads; };
    if constexpr (VEC) {
      detail::Chunk<T> x[BATCH], y[BATCH];
#pragma unroll
      for (int m = 0; m < BATCH; ++m)
        if (valid(m)) {
          x[m].load(in[m]);
          if (!INTERLEAVED && rotated) y[m].load(in[m] + half);
        }
#pragma unroll
      for (int m = 0; m < BATCH; ++m) {
        if (!valid(m)) continue;
        if (!rotated || pos < 0) {
          detail::store_raw(out[m], x[m]);  // bit for bit
          if (!INTERLEAVED && rotated) detail::store_raw(out[m] + half, y[m]);
          continue;
        }
        float p[8], q[8], u[8], w[8];
        x[m].values(p);
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[2 * i] = p[2 * i] * c[i] - p[2 * i + 1] * s[i];
            u[2 * i + 1] = p[2 * i] * s[i] + p[2 * i + 1] * c[i];
          }
          detail::store8(out[m], u);
        } else {
          y[m].values(q);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u[i] = p[i] * c[i] - q[i] * s[i];
            w[i] = p[i] * s[i] + q[i] * c[i];
          }
          detail::store8(out[m], u);
          detail::store8(out[m] + half, w);
        }
      }
    } else {
      const int second = INTERLEAVED ? 1 : half;
      T x[BATCH], y[BATCH];
#pragma unroll
      for (int m = 0; m < BATCH; ++m)
        if (valid(m)) {
          x[m] = in[m][0];
          y[m] = rotated ? in[m][second] : x[m];
        }
#pragma unroll
      for (int m = 0; m < BATCH; ++m) {
        if (!valid(m)) continue;
        if (!rotated || pos < 0) {
          out[m][0] = x[m];
          if (rotated) out[m][second] = y[m];
        } else {
          const float p = detail::load_f32(&x[m]), q = detail::load_f32(&y[m]);
          detail::store_f32(out[m], p * c[0] - q * s[0]);
          detail::store_f32(out[m] + second, p * s[0] + q * c[0]);
        }
      }
    }
  }
}

template <typename T>
inline cudaError_t launch_rotary(RotaryArgs a, bool interleaved, bool vec, cudaStream_t stream) {
  const int heads = a.heads[0] + a.heads[1];
  a.units = vec ? a.rotary_dim / (interleaved ? 8 : 16) + (a.head_dim - a.rotary_dim) / 8
                : a.rotary_dim / 2 + a.head_dim - a.rotary_dim;
  // Whole tokens while they fit in kRotaryThreads threads, else one token whose heads the block walks through in equal turns.
  const int most = a.units >= kRotaryThreads ? 1 : kRotaryThreads / a.units;
  a.tokens_per_block = most >= heads ? most / heads : 1;
  if (most >= heads) {
    a.rows_per_block = heads;
  } else {
    const int turns = (heads + most - 1) / most;
    a.rows_per_block = (heads + turns - 1) / turns;
  }
  const int threads = a.units * a.rows_per_block * a.tokens_per_block;
  const unsigned grid = static_cast<unsigned>((a.T + a.tokens_per_block - 1) / a.tokens_per_block);
  if (interleaved) {
    if (vec) rotary_kernel<T, true, true><<<grid, threads, 0, stream>>>(a);
    else rotary_kernel<T, true, false><<<grid, threads, 0, stream>>>(a);
  } else {
    if (vec) rotary_kernel<T, false, true><<<grid, threads, 0, stream>>>(a);
    else rotary_kernel<T, false, false><<<grid, threads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace b200w4a4
