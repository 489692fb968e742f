// Gated delta rule ops: the token-loop kernel (one token per sequence, short sequences) and the C ABI.
#include "gated_delta_chunk.cuh"

#include <cmath>

#include "op_host.h"

namespace dfssm {

// ------------------------------------------------------------------ token loop
//
// A warp owns R rows of one head's state; a lane holds DK/32 neighbouring columns of each, so a row is one
// coalesced access.  Both dot products come from the state before the token's update,
//   S k and S q,  u = beta (v - e^g S k),  o = scale (e^g S q + (k.q) u),  S <- e^g S + u k^T,
// so a token costs one reduction over the lanes for the 2R sums: a transposing butterfly, where each
// exchange halves the values a lane holds (2R + 5 - log2(2R) shuffles).
//
// Bound: HBM.  A one-token call reads and writes 8 dk dv bytes of state per head and computes 7 dk dv
// operations, far below the balance of the machine.
constexpr int kGdWarps = 4;
// Which prompts take the loop (gd_plan): sequences of up to kGdLoopMost tokens, looked for in calls of less than
// kGdMixed tokens per sequence.
constexpr int kGdLoopMost = 12, kGdMixed = 32;

// Sequences of more than `most` tokens are left to the chunked kernels.
template <typename T, int DK, int R>
__global__ void __launch_bounds__(kGdWarps * 32)
gated_delta_loop_kernel(const GatedDeltaArgs p, int row_blocks, int most) {
  constexpr int NV = DK / 32;  // columns per lane
  static_assert(R == 8, "the butterfly below is written for 16 sums");
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int blk = blockIdx.x;
  const int rb = blk % row_blocks, h = (blk / row_blocks) % p.v_heads, seq = blk / (row_blocks * p.v_heads);
  const int slot = gd_slot(p.slots, seq, p.n_slots, threadIdx.x, blockDim.x);
  if (slot < 0) return;
  int first, count;
  gd_range(p.cu, seq, p.tokens, first, count);
  const int row0 = (rb * kGdWarps + wid) * R;
  if (count == 0 || count > most || row0 >= p.dv) return;  // dv is a multiple of 16: a warp's 8 rows are all there or none
  const int hk = h / (p.v_heads / p.k_heads);
  float* S = p.state + (((size_t)slot * p.v_heads + h) * p.dv + row0) * DK + lane * NV;
  float s[R][NV];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if constexpr (NV == 4) {
      const float4 x = *reinterpret_cast<const float4*>(S + r * DK);
      s[r][0] = x.x, s[r][1] = x.y, s[r][2] = x.z, s[r][3] = x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(S + r * DK);
      s[r][0] = x.x, s[r][1] = x.y;
    }
  }
  const T* qp = static_cast<const T*>(p.q) + hk * DK + lane * NV;
  const T* kp = static_cast<const T*>(p.k) + hk * DK + lane * NV;
  const T* vp = static_cast<const T*>(p.v) + h * p.dv + row0;
  const T* ap = static_cast<const T*>(p.a) + h;
  const T* bp = static_cast<const T*>(p.b) + h;
  T* op = static_cast<T*>(p.o) + h * p.dv + row0;
  const float A_log = p.A_log[h], dt_bias = p.dt_bias[h];
  const int rsel = (lane >> 1) & 7;  // the row whose sum the butterfly leaves in this lane
  for (int t = first; t < first + count; ++t) {
    float q[NV], k[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q[j] = to_f(qp[(size_t)t * p.ld_q + j]);
      k[j] = to_f(kp[(size_t)t * p.ld_k + j]);
    }
    const float vr = to_f(vp[(size_t)t * p.ld_v + rsel]);
    const float eg = expf(gd_log_decay(to_f(ap[(size_t)t * p.ld_a]), dt_bias, A_log));
    const float beta = gd_beta(to_f(bp[(size_t)t * p.ld_b]));
    float qq = 0.f, kk = 0.f, kq = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      qq += q[j] * q[j];
      kk += k[j] * k[j];
      kq += k[j] * q[j];
    }
    kq = warp_sum(kq);
    if (p.qk_norm) {
      const float rq = 1.0f / sqrtf(warp_sum(qq) + kQkEps), rk = 1.0f / sqrtf(warp_sum(kk) + kQkEps);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        q[j] *= rq;
        k[j] *= rk;
      }
      kq = unit_dot(kq, rq * rk);
    }
    // sums[0..7] = S k of the rows, sums[8..15] = S q
    float sums[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        x += s[r][j] * k[j];
        y += s[r][j] * q[j];
      }
      sums[r] = x;
      sums[R + r] = y;
    }
#pragma unroll
    for (int n = 2 * R, off = 16; n > 1; n >>= 1, off >>= 1) {
      const bool up = (lane & off) != 0;
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const float send = up ? sums[i] : sums[i + n / 2];
        const float keep = up ? sums[i + n / 2] : sums[i];
        sums[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
      }
    }
    sums[0] += __shfl_xor_sync(0xffffffffu, sums[0], 1);
    // lanes 0..15 hold S k of row rsel, lanes 16..31 S q of it; the former know u
    const float uown = beta * (vr - eg * sums[0]);
    const float u = __shfl_sync(0xffffffffu, uown, lane & 15);
    if (lane >= 16 && (lane & 1) == 0) op[(size_t)t * p.ld_o + rsel] = from_f<T>(p.scale * (eg * sums[0] + kq * u));
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float ur = __shfl_sync(0xffffffffu, uown, 2 * r);
#pragma unroll
      for (int j = 0; j < NV; ++j) s[r][j] = fmaf(ur, k[j], eg * s[r][j]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if constexpr (NV == 4)
      *reinterpret_cast<float4*>(S + r * DK) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
    else
      *reinterpret_cast<float2*>(S + r * DK) = make_float2(s[r][0], s[r][1]);
  }
}

namespace {

int launch_loop(const GatedDeltaArgs& p, int dk, int dtype, int most, cudaStream_t s) {
  const int rows = kGdWarps * 8, row_blocks = (p.dv + rows - 1) / rows;
  const long long blocks = (long long)p.n_seq * p.v_heads * row_blocks;
  if (blocks > 0x7fffffffLL) return dfssm_fail(DFSSM_ERR_ARG, "%d sequences x %d heads are too many", p.n_seq, p.v_heads);
  const auto fn = dtype == DFSSM_F16 ? (dk == 128 ? gated_delta_loop_kernel<__half, 128, 8> : gated_delta_loop_kernel<__half, 64, 8>)
                                     : (dk == 128 ? gated_delta_loop_kernel<__nv_bfloat16, 128, 8>
                                                  : gated_delta_loop_kernel<__nv_bfloat16, 64, 8>);
  fn<<<(unsigned)blocks, kGdWarps * 32, 0, s>>>(p, row_blocks, most);
  DFSSM_CU(cudaGetLastError());
  return DFSSM_OK;
}

// What a prompt call launches, from its sizes alone.
struct GdPlan {
  bool loop, chunks;  // which kernels
  int most;           // sequences of up to so many tokens are the loop's,
  int least;          // of at least so many the chunked kernels'
  int walkers;        // no more sequences than this can be so long
};
GdPlan gd_plan(int tokens, int n_seq) {
  // The token loop for sequences of few tokens: it takes about 1.1 us a token of the longest one, the chunked kernels
  // 15 us and more whatever the length up to 64 (64 heads of 64 x 128, one sequence of 12 / 16 tokens: 14.5 / 18.5 us
  // against 15.1; 64 sequences of 8: 150 us for both launched as below, 241 by chunks).  The lengths are not known here:
  // where they average less than kGdMixed tokens, both run, each for its sequences (200 sequences of 1 token and 4 of
  // 500: 297 us, 818 by chunks alone; 255 of 1 and one of 700: 286, by the loop alone 1012; where one of them finds
  // nothing to do it costs 2 to 12%; 599 of 1 and one of 1700: 550, by the loop alone 2444; 600 of 1: 385, 366 by the loop alone).
  if (tokens <= kGdLoopMost) return {true, false, tokens, 0, 0};
  if (n_seq > 1 && tokens < (long long)kGdMixed * n_seq) {
    const int least = kGdLoopMost + 1;
    return {true, true, kGdLoopMost, least, tokens / least < n_seq ? tokens / least : n_seq};
  }
  return {false, true, 0, 1, n_seq};
}

// Bytes for the chunks' T, P and factors, the fp16 forms of bf16 rows, and the order of the sequences; kGdScratch where the
// loop takes the whole call and uses none.
constexpr size_t kGdScratch = 256;
size_t gd_workspace(int tokens, int n_seq, int k_heads, int v_heads, int dk, int dtype) {
  const GdPlan plan = gd_plan(tokens, n_seq);
  if (!plan.chunks) return kGdScratch;
  const size_t n = (size_t)gd_chunk_slots(tokens, n_seq, plan.least);
  return n * v_heads * kGdBlock + (dtype == DFSSM_BF16 ? n * k_heads * 2 * kGdC * dk * 2 : 0) + (size_t)plan.walkers * 16;
}

template <typename T, int DK, bool DEEP>
int launch_walk(const GatedDeltaArgs& p, const char* blocks, const __half* kq16, const int4* order, int slots_total,
                int walkers, int least, cudaStream_t s) {
  static SmemLimit limit;
  constexpr int bytes = gd_chunk_smem<DK, DEEP>();
  const auto fn = gated_delta_chunk_kernel<T, DK, DEEP>;
  DFSSM_CU(limit.raise(reinterpret_cast<const void*>(fn), bytes));
  const int parts = (p.dv + 16 * kGdGroups - 1) / (16 * kGdGroups);
  const long long grid = (long long)walkers * p.v_heads * parts;
  if (grid > 0x7fffffffLL) return dfssm_fail(DFSSM_ERR_ARG, "%d sequences x %d heads are too many", p.n_seq, p.v_heads);
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(128 * kGdGroups);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  DFSSM_CU(cudaLaunchKernelEx(&cfg, fn, p, blocks, kq16, order, parts, slots_total, least));
  return DFSSM_OK;
}

// Sequences of at least plan.least tokens by the chunked kernels (1: all that have any).
template <typename T, int DK>
int launch_chunked(const GatedDeltaArgs& p, char* workspace, const GdPlan& plan, cudaStream_t s) {
  static SmemLimit limit;
  constexpr int bytes = gd_prep_smem<DK>();
  const int least = plan.least, walkers = plan.walkers;
  const long long n = gd_chunk_slots(p.tokens, p.n_seq, least);
  const int rep = p.v_heads / p.k_heads;
  int dev = 0, sms = 0;
  DFSSM_CU(cudaGetDevice(&dev));
  DFSSM_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  // Heads of one key per prep block: the more, the less is computed twice, as long as there are blocks for every SM
  // (64 heads on one key, 64 prompts of 64 tokens, whole call: 253 us with 2, 242 with 4, 235 with 8, 235 with 16, before
  // the look at how far values lie apart, which adds 20).
  int per_group = rep < 8 ? rep : 8;
  while (per_group > 1 && n * p.k_heads * ((rep + per_group - 1) / per_group) < 4 * sms) per_group /= 2;
  const int groups = (rep + per_group - 1) / per_group;
  const long long grid = n * p.k_heads * groups;
  if (grid > 0x7fffffffLL) return dfssm_fail(DFSSM_ERR_ARG, "%d tokens x %d heads are too many", p.tokens, p.v_heads);
  __half* kq16 = std::is_same<T, __half>::value ? nullptr
                                               : reinterpret_cast<__half*>(workspace + (size_t)n * p.v_heads * kGdBlock);
  const bool at_once = (long long)walkers * p.v_heads * ((p.dv + 31) / 32) <= sms;  // every block of the walk has an SM
  // A list of the sequences, the long ones first (one that starts last runs alone), where there are fewer walkers than
  // sequences, or where not all start at once; many of them even out by themselves, and each block looks for itself.
  const bool ordered = walkers < p.n_seq || (!at_once && p.n_seq <= kGdOrdered);
  const size_t all = gd_workspace(p.tokens, p.n_seq, p.k_heads, p.v_heads, DK, std::is_same<T, __half>::value ? DFSSM_F16 : DFSSM_BF16);
  int4* order = ordered ? reinterpret_cast<int4*>(workspace + all - (size_t)walkers * 16) : nullptr;
  const auto fn = gated_delta_prep_kernel<T, DK>;
  DFSSM_CU(limit.raise(reinterpret_cast<const void*>(fn), bytes));
  fn<<<(unsigned)grid, kPrepThreads, bytes, s>>>(p, workspace, kq16, order, groups, per_group, least, walkers);
  DFSSM_CU(cudaGetLastError());
  return at_once ? launch_walk<T, DK, true>(p, workspace, kq16, order, (int)n, walkers, least, s)
                 : launch_walk<T, DK, false>(p, workspace, kq16, order, (int)n, walkers, least, s);
}

// What both entry points ask of their arguments.
int check_args(const GatedDeltaArgs& p, int dk, int dtype) {
  // arrays without rows have no address
  if ((p.tokens != 0 && (!p.q || !p.k || !p.v || !p.a || !p.b || !p.o)) || !p.A_log || !p.dt_bias || !p.state)
    return dfssm_fail(DFSSM_ERR_ARG, "NULL argument");
  if (dtype != DFSSM_F16 && dtype != DFSSM_BF16) return dfssm_fail(DFSSM_ERR_UNSUPPORTED, "dtype %d (16-bit types only)", dtype);
  if (dk != 64 && dk != 128) return dfssm_fail(DFSSM_ERR_UNSUPPORTED, "dk=%d (built for 64 and 128)", dk);
  if (p.dv < 16 || p.dv > 256 || p.dv % 16)
    return dfssm_fail(DFSSM_ERR_UNSUPPORTED, "dv=%d (multiples of 16 up to 256)", p.dv);
  if (p.k_heads < 1 || p.v_heads < 1 || p.v_heads % p.k_heads || p.v_heads > 65535)
    return dfssm_fail(DFSSM_ERR_ARG, "k_heads=%d v_heads=%d: v_heads must be a multiple of k_heads", p.k_heads, p.v_heads);
  if (p.n_seq < 0 || p.tokens < 0 || p.n_slots < 1) return dfssm_fail(DFSSM_ERR_ARG, "bad sizes");
  if (!p.slots && p.n_seq > p.n_slots) return dfssm_fail(DFSSM_ERR_ARG, "%d sequences in %d slots", p.n_seq, p.n_slots);
  if ((long long)p.ld_q < (long long)p.k_heads * dk || (long long)p.ld_k < (long long)p.k_heads * dk ||
      (long long)p.ld_v < (long long)p.v_heads * p.dv || (long long)p.ld_o < (long long)p.v_heads * p.dv ||
      p.ld_a < p.v_heads || p.ld_b < p.v_heads)
    return dfssm_fail(DFSSM_ERR_ARG, "a row stride is shorter than its row");
  if ((p.ld_q | p.ld_k | p.ld_v | p.ld_o) % 8)
    return dfssm_fail(DFSSM_ERR_ARG, "the row strides of q, k, v and o must be multiples of 8");
  if (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.o | (uintptr_t)p.state) & 15)
    return dfssm_fail(DFSSM_ERR_ARG, "q, k, v, o and state must be 16-byte aligned");
  if (!std::isfinite(p.scale)) return dfssm_fail(DFSSM_ERR_ARG, "scale is not finite");
  return DFSSM_OK;
}

}  // namespace
}  // namespace dfssm

using namespace dfssm;

extern "C" {

int dfssm_gated_delta_step(const void* q, int ld_q, const void* k, int ld_k, const void* v, int ld_v, const void* a,
                           int ld_a, const void* b, int ld_b, const float* A_log, const float* dt_bias, float* state,
                           int n_slots, const int32_t* slots, int batch, void* o, int ld_o, int k_heads, int v_heads,
                           int dk, int dv, float scale, int qk_norm, int dtype, void* stream) {
  const GatedDeltaArgs p{q,     k,       v,     a,     b,       ld_q,  ld_k,  ld_v, ld_a,    ld_b,    ld_o, A_log, dt_bias,
                         state, n_slots, slots, nullptr, batch, batch, o, k_heads, v_heads, dv, scale, qk_norm};
  if (const int rc = check_args(p, dk, dtype)) return rc;
  if (batch == 0) return DFSSM_OK;
  return launch_loop(p, dk, dtype, 1, static_cast<cudaStream_t>(stream));
}

size_t dfssm_gated_delta_workspace(int tokens, int n_seq, int k_heads, int v_heads, int dk, int dv, int dtype) {
  (void)dv;
  if (tokens < 1 || n_seq < 1 || k_heads < 1 || v_heads < 1 || dk < 1) return 0;
  return gd_workspace(tokens, n_seq, k_heads, v_heads, dk, dtype);
}

int dfssm_gated_delta_prefill(const void* q, int ld_q, const void* k, int ld_k, const void* v, int ld_v, const void* a,
                              int ld_a, const void* b, int ld_b, const float* A_log, const float* dt_bias,
                              float* state, int n_slots, const int32_t* slots, const int32_t* cu_seqlens, int n_seq,
                              int tokens, void* o, int ld_o, int k_heads, int v_heads, int dk, int dv, float scale,
                              int qk_norm, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const GatedDeltaArgs p{q,     k,       v,     a,     b,       ld_q,  ld_k,  ld_v, ld_a,    ld_b,    ld_o, A_log, dt_bias,
                         state, n_slots, slots, cu_seqlens, n_seq, tokens, o, k_heads, v_heads, dv, scale, qk_norm};
  if (!cu_seqlens) return dfssm_fail(DFSSM_ERR_ARG, "NULL argument");
  if (const int rc = check_args(p, dk, dtype)) return rc;
  const size_t need = dfssm_gated_delta_workspace(tokens, n_seq, k_heads, v_heads, dk, dv, dtype);
  if (need && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need))
    return dfssm_fail(DFSSM_ERR_ARG, "the workspace must be %zu bytes, 256-byte aligned", need);
  if (n_seq == 0 || tokens == 0) return DFSSM_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const GdPlan plan = gd_plan(tokens, n_seq);
  char* w = static_cast<char*>(workspace);
  if (plan.loop) {
    if (const int rc = launch_loop(p, dk, dtype, plan.most, s)) return rc;
  }
  if (!plan.chunks) return DFSSM_OK;
  if (dtype == DFSSM_F16) return dk == 128 ? launch_chunked<__half, 128>(p, w, plan, s) : launch_chunked<__half, 64>(p, w, plan, s);
  return dk == 128 ? launch_chunked<__nv_bfloat16, 128>(p, w, plan, s) : launch_chunked<__nv_bfloat16, 64>(p, w, plan, s);
}

}  // extern "C"
