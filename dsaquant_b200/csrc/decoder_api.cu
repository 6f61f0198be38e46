// C-ABI entry points of the decoder-layer operators (declared in include/b200w4a4_decoder.h).
// Host side only: argument checks and kernel launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200w4a4_decoder.h"
#include "device_state.cuh"
#include "rms_norm.cuh"
#include "rotary.cuh"
#include "w4_group.cuh"
#include "window_attn.cuh"
#include "window_attn_tc.cuh"

namespace {

using namespace b200w4a4;

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool float_dtype(int d) { return d == B200W4A4_F16 || d == B200W4A4_BF16 || d == B200W4A4_F32; }
unsigned size_of(int d) { return d == B200W4A4_F32 ? 4u : 2u; }
int launched(cudaError_t e) { return e == cudaSuccess ? B200W4A4_OK : B200W4A4_ECUDA; }

int attention_splits(int B, int Lq, int Lk, int q_heads, int k_heads, int window, int sinks, int sm_count) {
  if (window > Lk) window = Lk;
  if (sinks > Lk) sinks = Lk;
  if (Lq >= kAttnTcMinQueries) return 1;
  int s = window_attn_splits(B, Lq, Lk, k_heads, q_heads / k_heads, window, sinks, sm_count);
  if (static_cast<long long>(B) * s > 65535) s = 65535 / B;
  return s < 1 ? 1 : s;
}

bool attention_shape_ok(int B, int Lq, int Lk, int q_heads, int k_heads, int head_dim) {
  return B >= 0 && B <= 65535 && Lq >= 0 && Lk >= 0 && q_heads >= 1 && k_heads >= 1 && q_heads <= 65535 &&
         q_heads % k_heads == 0 && q_heads / k_heads <= 64 && (head_dim == 64 || head_dim == 128) &&
         static_cast<long long>(Lq) * (q_heads / k_heads) <= 0x7fffffffLL - kAttnRows && Lk <= 0x7fffffff - 1024;
}

}  // namespace

extern "C" {

int b200w4a4_rms_norm_quant(const void* x, int x_dtype, long long x_ld, const void* residual,
                            long long residual_ld, const void* weight, int w_dtype, float eps,
                            void* codes, int code_format, float* scale, void* residual_out, int M,
                            int D, float clip, void* stream) {
  if (!float_dtype(x_dtype) || !float_dtype(w_dtype)) return B200W4A4_EINVAL;
  if (code_format != B200W4A4_CODES_INT8 && code_format != B200W4A4_CODES_E4M3) return B200W4A4_EINVAL;
  if ((residual == nullptr) != (residual_out == nullptr)) return B200W4A4_EINVAL;
  if (!(clip > 0.0f) || !(eps >= 0.0f)) return B200W4A4_EINVAL;
  if (M < 0 || D < 1 || D > kRmsNormMaxD) return B200W4A4_ESHAPE;
  if (M == 0) return B200W4A4_OK;
  if (x == nullptr || weight == nullptr || codes == nullptr || scale == nullptr) return B200W4A4_EINVAL;
  if (residual_out != nullptr && (residual_out == x || residual_out == residual)) return B200W4A4_EINVAL;
  if ((M > 1 && x_ld < D) || (residual != nullptr && M > 1 && residual_ld < D)) return B200W4A4_ESHAPE;
  const unsigned es = size_of(x_dtype);
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(residual_out, es) || !aligned(weight, size_of(w_dtype)) ||
      !aligned(scale, 4))
    return B200W4A4_EALIGN;
  const int rc = current_device(nullptr);
  if (rc != B200W4A4_OK) return rc;
  RmsNormArgs a;
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.codes = codes;
  a.scale = scale;
  a.residual_out = residual_out;
  a.x_ld = x_ld;
  a.r_ld = residual_ld;
  a.eps = eps;
  a.clip = clip;
  a.w_dtype = w_dtype;
  a.format = code_format;
  a.M = M;
  a.D = D;
  // 128-bit accesses where every row allows them
  const bool vec = D % 8 == 0 && (M == 1 || x_ld % 8 == 0) && (residual == nullptr || M == 1 || residual_ld % 8 == 0) &&
                   aligned(x, 16) && aligned(residual, 16) && aligned(residual_out, 16) && aligned(weight, 16) &&
                   aligned(codes, 8);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (x_dtype) {
    case B200W4A4_F16: return launched(vec ? launch_rms_norm_quant<__half, true>(a, s) : launch_rms_norm_quant<__half, false>(a, s));
    case B200W4A4_BF16:
      return launched(vec ? launch_rms_norm_quant<__nv_bfloat16, true>(a, s) : launch_rms_norm_quant<__nv_bfloat16, false>(a, s));
    default: return launched(vec ? launch_rms_norm_quant<float, true>(a, s) : launch_rms_norm_quant<float, false>(a, s));
  }
}

int b200w4a4_quantize_weight_grouped(const void* w, int w_dtype, void* packed, void* scale, int N,
                                     int K, int group, void* stream) {
  if (w == nullptr || packed == nullptr || scale == nullptr || !float_dtype(w_dtype)) return B200W4A4_EINVAL;
  if (N < 1 || K < 32 || group < 32 || group % 32 != 0 || K % group != 0 || K > (1 << 20)) return B200W4A4_ESHAPE;
  if (!aligned(w, size_of(w_dtype)) || !aligned(scale, 2)) return B200W4A4_EALIGN;
  const int rc = current_device(nullptr);
  if (rc != B200W4A4_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* p = static_cast<uint8_t*>(packed);
  __half* sc = static_cast<__half*>(scale);
  switch (w_dtype) {
    case B200W4A4_F16: return launched(launch_w4_group_quantize(static_cast<const __half*>(w), p, sc, N, K, group, s));
    case B200W4A4_BF16: return launched(launch_w4_group_quantize(static_cast<const __nv_bfloat16*>(w), p, sc, N, K, group, s));
    default: return launched(launch_w4_group_quantize(static_cast<const float*>(w), p, sc, N, K, group, s));
  }
}

int b200w4a4_linear_w4_group(const void* x, int x_dtype, const float* act_scale, const void* packed,
                             const void* scale, const void* bias, void* out, int out_dtype, int M,
                             int N, int K, int group, void* stream) {
  if (x_dtype != B200W4A4_F16 && x_dtype != B200W4A4_BF16 && x_dtype != B200W4A4_X_INT8) return B200W4A4_EINVAL;
  const bool bias_f32 = (out_dtype & B200W4A4_BIAS_F32) != 0;
  out_dtype &= ~B200W4A4_BIAS_F32;
  if (out_dtype != B200W4A4_F16 && out_dtype != B200W4A4_BF16) return B200W4A4_EINVAL;
  if (M < 0 || N < 1 || K < 32 || group < 32 || group % 32 != 0 || K % group != 0) return B200W4A4_ESHAPE;
  if (M > 65535 * 8 || K > (1 << 20) || N > 0x7fffffff - 511) return B200W4A4_ESHAPE;  // row numbers of the last block are 32 bits
  if (M == 0) return B200W4A4_OK;
  if (x == nullptr || packed == nullptr || scale == nullptr || out == nullptr) return B200W4A4_EINVAL;
  if ((x_dtype == B200W4A4_X_INT8) != (act_scale != nullptr)) return B200W4A4_EINVAL;
  if (!aligned(x, 16) || !aligned(packed, 16) || !aligned(scale, 2) || !aligned(out, 2) ||
      !aligned(bias, bias_f32 ? 4 : 2) || !aligned(act_scale, 4))
    return B200W4A4_EALIGN;
  DeviceInfo dev;
  const int rc = current_device(&dev);
  if (rc != B200W4A4_OK) return rc;
  W4GroupArgs a;
  a.x = x;
  a.packed = static_cast<const uint8_t*>(packed);
  a.scale = static_cast<const __half*>(scale);
  a.act_scale = act_scale;
  a.bias = bias_f32 ? nullptr : bias;
  a.bias32 = bias_f32 ? static_cast<const float*>(bias) : nullptr;
  a.out = out;
  a.M = M;
  a.N = N;
  a.K = K;
  a.group = group;
  a.out_bf16 = out_dtype == B200W4A4_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the widest run of codes that surely shares a scale
  const int gb = group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32;
#define B200W4A4_W4G_DISPATCH(X)                                       \
  launched(gb == 128  ? launch_w4_group<X, 128>(a, dev.sm_count, s)                  \
           : gb == 64 ? launch_w4_group<X, 64>(a, dev.sm_count, s)                   \
                      : launch_w4_group<X, 32>(a, dev.sm_count, s))
  if (x_dtype == B200W4A4_F16) return B200W4A4_W4G_DISPATCH(__half);
  if (x_dtype == B200W4A4_BF16) return B200W4A4_W4G_DISPATCH(__nv_bfloat16);
  return B200W4A4_W4G_DISPATCH(int8_t);
#undef B200W4A4_W4G_DISPATCH
}

int b200w4a4_rotary(const void* q, long long q_tok, long long q_head, void* q_out, long long qo_tok,
                    long long qo_head, int q_heads, const void* k, long long k_tok, long long k_head,
                    void* k_out, long long ko_tok, long long ko_head, int k_heads, int dtype,
                    const float* cos_sin, long long max_pos, const void* positions, int positions_int64,
                    long long T, int head_dim, int rotary_dim, int interleaved, int inverse, void* stream) {
  if (!float_dtype(dtype) || (positions_int64 != 0 && positions_int64 != 1) || (interleaved != 0 && interleaved != 1) ||
      (inverse != 0 && inverse != 1))
    return B200W4A4_EINVAL;
  if (T < 0 || T > 0x7fffffffLL || q_heads < 1 || k_heads < 0 || q_heads > 65536 || k_heads > 65536 || max_pos < 1)
    return B200W4A4_ESHAPE;
  if (head_dim < 2 || head_dim > kRotaryMaxHeadDim || rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return B200W4A4_ESHAPE;
  if (T == 0) return B200W4A4_OK;
  if (q == nullptr || q_out == nullptr || cos_sin == nullptr || positions == nullptr) return B200W4A4_EINVAL;
  if (k_heads > 0 && (k == nullptr || k_out == nullptr)) return B200W4A4_EINVAL;
  const unsigned es = size_of(dtype);
  if (!aligned(q, es) || !aligned(q_out, es) || !aligned(cos_sin, 8) || !aligned(positions, positions_int64 ? 8 : 4))
    return B200W4A4_EALIGN;
  if (k_heads > 0 && (!aligned(k, es) || !aligned(k_out, es))) return B200W4A4_EALIGN;
  const int rc = current_device(nullptr);
  if (rc != B200W4A4_OK) return rc;
  RotaryArgs a;
  a.in[0] = q; a.in_tok[0] = q_tok; a.in_head[0] = q_head;
  a.out[0] = q_out; a.out_tok[0] = qo_tok; a.out_head[0] = qo_head;
  a.heads[0] = q_heads;
  a.in[1] = k; a.in_tok[1] = k_tok; a.in_head[1] = k_head;
  a.out[1] = k_out; a.out_tok[1] = ko_tok; a.out_head[1] = ko_head;
  a.heads[1] = k_heads;
  a.cos_sin = cos_sin;
  a.positions = positions;
  a.max_pos = max_pos;
  a.T = T;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  a.pos64 = positions_int64 != 0;
  a.sign = inverse ? -1.0f : 1.0f;
  // 128-bit accesses: whole vectors in the rotated part (in each of its halves) and behind it
  bool vec = rotary_dim % (interleaved ? 8 : 16) == 0 && head_dim % 8 == 0 && aligned(cos_sin, 16);
  for (int i = 0; i < (k_heads > 0 ? 2 : 1); ++i)
    vec = vec && aligned(a.in[i], 16) && aligned(a.out[i], 16) && a.in_tok[i] % 8 == 0 && a.in_head[i] % 8 == 0 &&
          a.out_tok[i] % 8 == 0 && a.out_head[i] % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200W4A4_F16: return launched(launch_rotary<__half>(a, interleaved != 0, vec, s));
    case B200W4A4_BF16: return launched(launch_rotary<__nv_bfloat16>(a, interleaved != 0, vec, s));
    default: return launched(launch_rotary<float>(a, interleaved != 0, vec, s));
  }
}

size_t b200w4a4_window_attention_workspace_bytes(int B, int Lq, int Lk, int q_heads, int k_heads,
                                                 int head_dim, int window, int sinks) {
  if (!attention_shape_ok(B, Lq, Lk, q_heads, k_heads, head_dim) || window < 1 || sinks < 0 || B == 0 || Lq == 0) return 0;
  DeviceInfo dev;
  if (current_device(&dev) != B200W4A4_OK) return 0;
  const int splits = attention_splits(B, Lq, Lk, q_heads, k_heads, window, sinks, dev.sm_count);
  if (splits == 1) return 0;
  return static_cast<size_t>(splits) * B * q_heads * Lq * (head_dim + 1) * sizeof(float);
}

int b200w4a4_window_attention(const void* q, long long q_b, long long q_tok, long long q_head,
                              const void* k, long long k_b, long long k_tok, long long k_head,
                              const void* v, long long v_b, long long v_tok, long long v_head,
                              const int* kv_lens, void* out, float* lse, int dtype, int B, int Lq, int Lk,
                              int q_heads, int k_heads, int head_dim, int window, int sinks, float scale,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != B200W4A4_F16 && dtype != B200W4A4_BF16) return B200W4A4_EINVAL;
  if (!attention_shape_ok(B, Lq, Lk, q_heads, k_heads, head_dim)) return B200W4A4_ESHAPE;
  if (window < 1 || sinks < 0 || !(scale > 0.0f)) return B200W4A4_EINVAL;
  if (B == 0 || Lq == 0) return B200W4A4_OK;
  if (q == nullptr || out == nullptr || (Lk > 0 && (k == nullptr || v == nullptr))) return B200W4A4_EINVAL;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(lse, 4) ||
      !aligned(kv_lens, 4) || !aligned(workspace, 16))
    return B200W4A4_EALIGN;
  const long long pitches[9] = {q_b, q_tok, q_head, k_b, k_tok, k_head, v_b, v_tok, v_head};
  for (long long p : pitches)
    if (p % 8 != 0) return B200W4A4_EALIGN;
  DeviceInfo dev;
  const int rc = current_device(&dev);
  if (rc != B200W4A4_OK) return rc;
  WindowAttnArgs a;
  a.q = q; a.k = k; a.v = v;
  a.out = out;
  a.lse = lse;
  a.kv_lens = kv_lens;
  a.q_b = q_b; a.q_t = q_tok; a.q_h = q_head;
  a.k_b = k_b; a.k_t = k_tok; a.k_h = k_head;
  a.v_b = v_b; a.v_t = v_tok; a.v_h = v_head;
  a.B = B; a.Lq = Lq; a.Lk = Lk;
  a.Hq = q_heads; a.Hkv = k_heads; a.G = q_heads / k_heads;
  a.window = window > Lk ? (Lk > 0 ? Lk : 1) : window;
  a.sinks = sinks > Lk ? Lk : sinks;
  a.scale = scale;
  a.splits = attention_splits(B, Lq, Lk, q_heads, k_heads, window, sinks, dev.sm_count);
  a.part_o = a.part_lse = nullptr;
  if (a.splits > 1) {
    const size_t rows = static_cast<size_t>(a.splits) * B * q_heads * Lq;
    if (workspace == nullptr) return B200W4A4_EINVAL;
    if (workspace_bytes < rows * (head_dim + 1) * sizeof(float)) return B200W4A4_EWORKSPACE;
    a.part_o = static_cast<float*>(workspace);
    a.part_lse = a.part_o + rows * head_dim;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // tensor maps take no pitch of 0 (heads or sequences that share memory) and none of 2^40 bytes
  const int extents[9] = {B, Lq, q_heads, B, Lk, k_heads, B, Lk, k_heads};
  bool mapped = true;
  for (int i = 0; i < 9; ++i) mapped = mapped && (extents[i] <= 1 || (pitches[i] > 0 && pitches[i] < (1LL << 39)));
  if (a.Lq >= kAttnTcMinQueries && a.Lk > 0 && mapped) {
    if (dtype == B200W4A4_F16)
      return head_dim == 64 ? launch_window_attn_tc<__half, 64>(a, dev, s) : launch_window_attn_tc<__half, 128>(a, dev, s);
    return head_dim == 64 ? launch_window_attn_tc<__nv_bfloat16, 64>(a, dev, s) : launch_window_attn_tc<__nv_bfloat16, 128>(a, dev, s);
  }
  if (dtype == B200W4A4_F16)
    return launched(head_dim == 64 ? launch_window_attn<__half, 64>(a, s) : launch_window_attn<__half, 128>(a, s));
  return launched(head_dim == 64 ? launch_window_attn<__nv_bfloat16, 64>(a, s) : launch_window_attn<__nv_bfloat16, 128>(a, s));
}

}  // extern "C"
