// Gated delta rule: shared definitions of the one-token / token-loop kernel and the chunked kernels.
//
// Per sequence (slot) and value head a state S [dv][dk] in fp32, per token
//   k^ = k / sqrt(|k|^2 + 1e-6), q^ likewise (qk_norm; else as given)
//   g = -exp(A_log) softplus(a + dt_bias),  beta = sigmoid(b)
//   S <- e^g S + beta (v - e^g S k^) k^^T,   o = scale S q^
// Value heads h share the key head h / (v_heads / k_heads).
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace dfssm {

constexpr float kQkEps = 1e-6f;

struct GatedDeltaArgs {
  const void *q, *k, *v, *a, *b;  // 16-bit rows, one per token
  int ld_q, ld_k, ld_v, ld_a, ld_b, ld_o;
  const float *A_log, *dt_bias;  // [v_heads]
  float* state;                  // [n_slots][v_heads][dv][dk]
  int n_slots;
  const int* slots;  // [n_seq] or NULL: sequence i in slot i
  const int* cu;     // [n_seq + 1] token offsets, or NULL: one token per sequence
  int n_seq, tokens;
  void* o;
  int k_heads, v_heads, dv;
  float scale;
  int qk_norm;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// Log decay of one token; softplus(x) = x from 20 on, where e^-x is below half an fp32 ulp of x.  It ends at -256:
// e^-256 times any fp32 number is 0 in fp32, and sums of what is left tell the later tokens' decays apart, which a gate
// of -1e20 or -infinity (the largest values of a) would drown.  A NaN stays.
__device__ __forceinline__ float gd_log_decay(float a, float dt_bias, float A_log) {
  const float x = a + dt_bias;
  const float g = -expf(A_log) * (x > 20.f ? x : log1pf(expf(x)));
  return g < -256.f ? -256.f : g;
}
// k.q of unit vectors from that of the raw ones and the product of their factors.  A factor is 0 where a square overflowed: the
// vector counts as zero, although the raw product may be infinite.
__device__ __forceinline__ float unit_dot(float kq, float factors) { return factors == 0.f ? 0.f : kq * factors; }
__device__ __forceinline__ float gd_beta(float b) { return 1.0f / (1.0f + expf(-b)); }

// Tokens [first, first + count) of sequence i, clamped to the rows that exist whatever cu holds.
__device__ __forceinline__ void gd_range(const int* cu, int i, int tokens, int& first, int& count) {
  if (!cu) {
    first = i;
    count = 1;
    return;
  }
  const int b = min(max(cu[i], 0), tokens), e = min(max(cu[i + 1], 0), tokens);
  first = b;
  count = max(e - b, 0);
}

// The slot of sequence i, or -1 when the sequence takes no part: its slot is out of range, or an earlier
// sequence of the call has the same one (two writers of one state would race).  Every thread of the
// block calls it and gets the same answer; it ends with a block-wide barrier when there are slots.
__device__ __forceinline__ int gd_slot(const int* slots, int i, int n_slots, int tid, int nthreads) {
  if (!slots) return i < n_slots ? i : -1;
  const int s = slots[i];
  int twice = 0;
  for (int j = tid; j < i; j += nthreads) twice |= slots[j] == s;
  twice = __syncthreads_or(twice);
  return (s < 0 || s >= n_slots || twice) ? -1 : s;
}

}  // namespace dfssm
