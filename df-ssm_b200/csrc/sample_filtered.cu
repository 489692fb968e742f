// Filtered sampling: the next token of every row from its logits and a given uniform number.
//
// Per row, with T the row's temperature and tokens ordered by falling x, the lower index first among equals:
//   x = fp32(l / T), divided by rep_penalty for the tokens of the row's seen bitmap;  w = exp(x - max x)
//   top-k   the first k tokens;   top-p   a token stays while the weight before it is <= top_p of the sum
//   of the top-k tokens' weights;   min-p   w >= min_p (the first token always stays)
//   the draw: the first kept token in vocabulary order whose running weight passes u x the kept weight.
// T <= 0 takes the first token.  NaN and -inf logits are never taken; tokens at +inf share the row.
//
// Which token is drawn must not depend on how the sums were split, so weights are 64-bit integers: exp in
// double precision times 2^S with S = 62 - ceil(log2 V), rounded.  Their sums are exact in any order, and
// the rounding moves a boundary by about sqrt(V) 2^-S of the largest weight, some 1e-12, where fp32 sums
// would move it by 1e-7 and pick other tokens once in a thousand rows.
#include <cuda_bf16.h>

#include "common.cuh"
#include "op_host.h"

namespace dfssm {

constexpr int kSfThreads = 1024;
constexpr int kSfWarps = kSfThreads / 32;

typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  long long ld;
  int vocab;
  const float *temperature, *top_p, *min_p, *uniform;
  const int* top_k;
  const uint32_t* seen;
  float rep;
  int *next, *kept;
  float* prob;
  double unit;  // 2^S
};

__device__ __forceinline__ float sf_logit(const float* p) { return *p; }
__device__ __forceinline__ float sf_logit(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float sf_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Order-preserving key of x; 0 for NaN and -inf, which are never taken.
__device__ __forceinline__ uint32_t sf_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sf_unkey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename T>
struct Row {
  const T* l;
  const uint32_t* seen;
  float temp, rep;
  __device__ __forceinline__ uint32_t key(int i) const {
    float x = __fdiv_rn(sf_logit(l + i), temp);
    if (seen && ((seen[i >> 5] >> (i & 31)) & 1u)) x = __fdiv_rn(x, rep);
    return sf_key(x);
  }
};

// w of a key as a double in [0, 1]
__device__ __forceinline__ double sf_weight(uint32_t key, uint32_t top) {
  if (key == top) return 1.0;
  return key == 0u ? 0.0 : exp((double)sf_unkey(key) - (double)sf_unkey(top));
}
__device__ __forceinline__ u64 sf_fix(double w, double unit) { return (u64)__double2ll_rn(w * unit); }

__device__ __forceinline__ u64 sf_block_sum(u64 v, u64* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 s = 0;
  for (int j = 0; j < kSfWarps; ++j) s += red[j];
  return s;
}

// The last kept token of the order, as (key, how many of the tokens with that key stay).
struct Cut {
  uint32_t key;
  int ties;
};

// Finds the group of equal keys in which the budget (a count, or a weight) runs out, among the keys >= floor:
// four rounds over 8 bits of the key, each a histogram of the keys that share the digits found so far.
// by_weight: a token stays while the weight before it is <= budget; else `budget` tokens stay.
// Returns {floor_key, floor_ties} when the budget outlasts all of them.
template <typename T>
__device__ Cut sf_cut(const Row<T>& row, int V, uint32_t top, Cut fl, bool by_weight, u64 budget, double unit,
                      unsigned* cnt, unsigned* lo, unsigned* hi) {
  uint32_t prefix = 0;
  u64 used = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSfThreads) cnt[i] = lo[i] = hi[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kSfThreads) {
      const uint32_t k = row.key(i);
      if (k == 0u || k < fl.key || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
      const int d = (k >> shift) & 255;
      atomicAdd(cnt + d, 1u);
      if (by_weight) {
        const u64 w = sf_fix(sf_weight(k, top), unit);
        const unsigned wl = (unsigned)w, old = atomicAdd(lo + d, wl);
        const unsigned wh = (unsigned)(w >> 32) + (old + wl < old ? 1u : 0u);
        if (wh) atomicAdd(hi + d, wh);
      }
    }
    __syncthreads();
    int d = 255;  // every thread walks the digits from the top; all come to the same one
    for (; d >= 0; --d) {
      const u64 m = by_weight ? ((u64)hi[d] << 32) + lo[d] : cnt[d];
      if (cnt[d] && (by_weight ? used + m > budget : used + m >= budget)) break;
      used += m;
    }
    __syncthreads();
    if (d < 0) return fl;
    prefix = (prefix << 8) | (uint32_t)d;
    if (shift == 0) {
      const int n = prefix == fl.key ? fl.ties : (int)cnt[d];
      int stay;
      if (by_weight) {
        const u64 w = sf_fix(sf_weight(prefix, top), unit);
        stay = w == 0 ? n : (int)min((u64)n, (budget - used) / w + 1);
      } else {
        stay = (int)(budget - used);
      }
      __syncthreads();
      return Cut{prefix, min(stay, n)};
    }
  }
  return fl;
}

template <typename T>
__global__ void __launch_bounds__(kSfThreads) sample_filtered_kernel(const SampleArgs p) {
  __shared__ unsigned cnt[256], lo[256], hi[256];
  __shared__ u64 red[kSfWarps];
  __shared__ int ties_of[kSfWarps];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, V = p.vocab;
  Row<T> row;
  row.l = static_cast<const T*>(p.logits) + (long long)b * p.ld;
  row.seen = p.seen ? p.seen + (size_t)b * ((V + 31) / 32) : nullptr;
  row.rep = p.rep;
  const float temp = p.temperature ? p.temperature[b] : 1.0f;
  const bool greedy = !(temp > 0.f);
  row.temp = greedy ? 1.0f : temp;
  const int k = greedy ? 1 : (p.top_k ? p.top_k[b] : 0);
  const float top_p = p.top_p ? p.top_p[b] : 1.0f, min_p = p.min_p ? p.min_p[b] : 0.f;
  // the largest key
  uint32_t top = 0;
  for (int i = tid; i < V; i += kSfThreads) top = max(top, row.key(i));
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) cnt[wid] = top;
  __syncthreads();
  for (int j = 0; j < kSfWarps; ++j) top = max(top, cnt[j]);
  __syncthreads();
  if (top == 0u) {  // nothing to take in this row
    if (tid == 0) {
      p.next[b] = -1;
      if (p.kept) p.kept[b] = 0;
      if (p.prob) p.prob[b] = 0.f;
    }
    return;
  }
  Cut cut{1u, 0x7fffffff};
  if (k > 0 && k < V) cut = sf_cut(row, V, top, cut, false, (u64)k, p.unit, cnt, lo, hi);
  if (top_p < 1.f) {
    u64 m = 0;
    for (int i = tid; i < V; i += kSfThreads) {
      const uint32_t key = row.key(i);
      if (key > cut.key) m += sf_fix(sf_weight(key, top), p.unit);
    }
    m = sf_block_sum(m, red);
    if (cut.ties != 0x7fffffff) m += (u64)cut.ties * sf_fix(sf_weight(cut.key, top), p.unit);
    const u64 budget = (u64)(fmax((double)top_p, 0.0) * (double)m);
    cut = sf_cut(row, V, top, cut, true, budget, p.unit, cnt, lo, hi);
  }
  // the draw: every warp owns a run of the vocabulary
  const int run = (V + kSfThreads - 1) / kSfThreads * 32, i0 = min(V, wid * run), i1 = min(V, i0 + run);
  auto weight = [&](uint32_t key) -> double {  // negative: not kept by key and min_p
    if (key < cut.key || key == 0u) return -1.0;
    const double w = sf_weight(key, top);
    return (key == top || w >= (double)min_p) ? w : -1.0;
  };
  int ties = 0;
  for (int i = i0 + lane; i < i1; i += 32) ties += row.key(i) == cut.key;
  ties = warp_sum(ties);
  if (lane == 0) ties_of[wid] = ties;
  __syncthreads();
  int tie0 = 0;  // equal keys in the runs before this one
  for (int j = 0; j < wid; ++j) tie0 += ties_of[j];
  u64 mass = 0;
  int count = 0, tie = tie0;
  for (int i = i0; i < i1; i += 32) {
    const uint32_t key = i + lane < i1 ? row.key(i + lane) : 0u;
    const unsigned eq = __ballot_sync(0xffffffffu, key == cut.key);
    const double w = weight(key);
    const bool stay = w >= 0.0 && (key != cut.key || tie + __popc(eq & ((1u << lane) - 1)) < cut.ties);
    if (stay) mass += sf_fix(w, p.unit), ++count;
    tie += __popc(eq);
  }
  mass = warp_sum(mass);
  count = warp_sum(count);
  __syncthreads();
  if (lane == 0) red[wid] = mass, ties_of[wid] = count;
  __syncthreads();
  u64 total = 0, before = 0;
  int kept = 0;
  for (int j = 0; j < kSfWarps; ++j) {
    if (j < wid) before += red[j];
    total += red[j];
    kept += ties_of[j];
  }
  float u = p.uniform[b];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  const u64 target = min((u64)((double)u * (double)total), total - 1);  // total >= 2^S: the first token is kept
  if (target < before || target >= before + mass) return;
  tie = tie0;
  for (int i = i0; i < i1; i += 32) {
    const uint32_t key = i + lane < i1 ? row.key(i + lane) : 0u;
    const unsigned eq = __ballot_sync(0xffffffffu, key == cut.key);
    const double w = weight(key);
    const bool stay = w >= 0.0 && (key != cut.key || tie + __popc(eq & ((1u << lane) - 1)) < cut.ties);
    const u64 mine = stay ? sf_fix(w, p.unit) : 0;
    u64 upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        p.next[b] = i + lane;
        if (p.kept) p.kept[b] = kept;
        if (p.prob) p.prob[b] = (float)((double)mine / (double)total);
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    tie += __popc(eq);
  }
}

}  // namespace dfssm

using namespace dfssm;

extern "C" int dfssm_sample_filtered(const void* logits, int64_t ld, int dtype, int batch, int vocab,
                                     const float* temperature, const int32_t* top_k, const float* top_p,
                                     const float* min_p, const uint32_t* seen_bits, float rep_penalty,
                                     const float* uniform, int32_t* next, int32_t* kept_count, float* prob,
                                     void* stream) {
  if (batch != 0 && (!logits || !uniform || !next)) return dfssm_fail(DFSSM_ERR_ARG, "NULL argument");
  if (dtype != DFSSM_F16 && dtype != DFSSM_BF16 && dtype != DFSSM_F32) return dfssm_fail(DFSSM_ERR_UNSUPPORTED, "dtype %d", dtype);
  if (batch < 0 || vocab < 1 || ld < vocab) return dfssm_fail(DFSSM_ERR_ARG, "batch %d vocab %d ld %lld", batch, vocab, (long long)ld);
  if (vocab > (1 << 24)) return dfssm_fail(DFSSM_ERR_UNSUPPORTED, "vocab %d (up to 2^24)", vocab);
  if (seen_bits && !(rep_penalty > 0.f)) return dfssm_fail(DFSSM_ERR_ARG, "rep_penalty must be > 0");
  if (batch == 0) return DFSSM_OK;
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  const SampleArgs p{logits,    ld,  vocab,       temperature, top_p,      min_p, uniform,
                     top_k, seen_bits, rep_penalty, next,        kept_count, prob,  (double)(1ull << (62 - bits))};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == DFSSM_F32)
    sample_filtered_kernel<float><<<batch, kSfThreads, 0, s>>>(p);
  else if (dtype == DFSSM_F16)
    sample_filtered_kernel<__half><<<batch, kSfThreads, 0, s>>>(p);
  else
    sample_filtered_kernel<__nv_bfloat16><<<batch, kSfThreads, 0, s>>>(p);
  DFSSM_CU(cudaGetLastError());
  return DFSSM_OK;
}
