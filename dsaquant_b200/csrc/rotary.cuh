// Rotary positions on q and k in one launch.  Pair i of a head (i < rotary_dim / 2) at position p:
//   u = a cos(p f_i) - b sin(p f_i),  v = a sin(p f_i) + b cos(p f_i)
// (a, b) are the values i and i + rotary_dim / 2 of the head ("half" layout) or 2i and 2i + 1
// (interleaved); values behind rotary_dim are copied.  cos and sin come from a table built in 64
// bits, one row a position, so a far position is as exact as a near one.
//
// HBM-bound: every value is read and written once.  A head is cut into units that one thread moves
// with 128-bit accesses, and a thread keeps its unit for all heads of its token that it visits, so
// the pairs' cos and sin are fetched once a thread and not once a head.
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
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 cs = __ldg(reinterpret_cast<const float2*>(row) + i);
        c[i] = cs.x;
        s[i] = cs.y * a.sign;
      }
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
    }
  }
  const int half = a.rotary_dim / 2;
  // first value of the unit, and of its second vector
  const int at0 = rotated ? (INTERLEAVED ? 2 * P * unit : P * unit) : a.rotary_dim + COPY * (unit - rot_units);
  for (int head = row0 % heads; head < heads; head += a.rows_per_block) {
    const int which = head >= a.heads[0];
    const int h = which ? head - a.heads[0] : head;
    const T* in = static_cast<const T*>(a.in[which]) + token * a.in_tok[which] + h * a.in_head[which] + at0;
    T* out = static_cast<T*>(a.out[which]) + token * a.out_tok[which] + h * a.out_head[which] + at0;
    if constexpr (VEC) {
      detail::Chunk<T> x, y;
      x.load(in);
      if (!INTERLEAVED && rotated) y.load(in + half);
      if (!rotated || pos < 0) {
        detail::store_raw(out, x);  // bit for bit
        if (!INTERLEAVED && rotated) detail::store_raw(out + half, y);
        continue;
      }
      float p[8], q[8], u[8], w[8];
      x.values(p);
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[2 * i] = p[2 * i] * c[i] - p[2 * i + 1] * s[i];
          u[2 * i + 1] = p[2 * i] * s[i] + p[2 * i + 1] * c[i];
        }
        detail::store8(out, u);
      } else {
        y.values(q);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          u[i] = p[i] * c[i] - q[i] * s[i];
          w[i] = p[i] * s[i] + q[i] * c[i];
        }
        detail::store8(out, u);
        detail::store8(out + half, w);
      }
    } else {
      const int second = INTERLEAVED ? 1 : half;
      const T x = in[0];
      const T y = rotated ? in[second] : x;
      if (!rotated || pos < 0) {
        out[0] = x;
        if (rotated) out[second] = y;
      } else {
        const float p = detail::load_f32(&x), q = detail::load_f32(&y);
        detail::store_f32(out, p * c[0] - q * s[0]);
        detail::store_f32(out + second, p * s[0] + q * c[0]);
      }
    }
  }
}

template <typename T>
inline cudaError_t launch_rotary(RotaryArgs a, bool interleaved, bool vec, cudaStream_t stream) {
  const int heads = a.heads[0] + a.heads[1];
  a.units = vec ? a.rotary_dim / (interleaved ? 8 : 16) + (a.head_dim - a.rotary_dim) / 8
                : a.rotary_dim / 2 + a.head_dim - a.rotary_dim;
  // Whole tokens while they fit in 256 threads, else one token whose heads the block walks through.
  const int rows = a.units >= 256 ? 1 : 256 / a.units;
  a.tokens_per_block = rows >= heads ? rows / heads : 1;
  a.rows_per_block = rows >= heads ? heads : rows;
  const int threads = a.units * (rows >= heads ? a.tokens_per_block * heads : rows);
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
