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
// double precision times 2^S with S = min(50, 62 - ceil(log2 V)), rounded.  Their sums are exact in any order,
// and the rounding moves a boundary by about sqrt(V) 2^-S of the largest weight, some 1e-12, where fp32 sums
// would move it by 1e-7 and pick other tokens once in a thousand rows.
//
// A cluster of 1 to 8 blocks of 1024 threads per row, each with a slice of the vocabulary and its x in shared memory
// where it fits (about 51,000 tokens; else every pass reads the logits again, from L2).  No pass sorts or selects
// over the whole row:
//   - with top-k, the k-th largest of the threads' own largest values bounds the k-th largest x from below;
//     the few tokens above it go to a list that the cluster's first block sorts, filters and draws from, and the
//     rest of the row is not looked at again;
//   - with top-p alone, a histogram of the weights (1024 bins of x, one pass) finds the bin that holds the
//     boundary, whose tokens are sorted for the cut {x, how many of the tokens equal to it stay}, and the draw is
//     one more pass that weighs what the cut keeps.
// Rows where the list would overflow (thousands of equal logits at the cut, top_k in the thousands) select the
// cut by four rounds over 8 bits of x's order-preserving key instead.
//
// Bound: instructions.  A weight is 25 of them, 10 in 64-bit floating point, and a row without top-k needs one
// for every token; with top-k the first pass over the logits (a division each) is most of it.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "op_host.h"

namespace dfssm {

constexpr int kSfThreads = 1024;
constexpr int kSfWarps = kSfThreads / 32;
constexpr int kSfList = 2048;  // tokens that are sorted
constexpr int kSfBins = 1024;  // one per thread
constexpr int kSfAll = 0x7fffffff;
constexpr int kSfBlocks = 8;   // of a row, at most

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
  int shift;      // S
  int slice;      // tokens per block of a row's cluster, a multiple of 128
  int in_shared;  // x of the slice in shared memory
  int ordered;    // > 0: the number of rows, which are taken by falling cost
};

__device__ __forceinline__ float sf_logit(const float* p) { return *p; }
__device__ __forceinline__ float sf_logit(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float sf_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Order-preserving key of x; 0 for -inf (and NaN), which is never taken.
__device__ __forceinline__ uint32_t sf_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sf_unkey(uint32_t k) {
  if (k == 0u) return -INFINITY;
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// A row's x.  from4 computes four of them from the logits: divided by T with the rounding of an IEEE division
// (two corrections bring q within an ulp of l / T and then, Markstein, to the rounded quotient, as long as
// nothing under- or overflows; -inf, NaN and large negative logits end as NaN on the way, which fmaxf turns
// into -inf; zero, tiny and large positive ones take the division itself).  -inf stands for every token
// that cannot be taken.
template <typename T>
struct Row {
  const T* l;
  const uint32_t* seen;
  float* xs;        // `shared`: the slice's x in shared memory, token i at xs[i - from]; else every pass computes them again
  int V;            // the row's tokens
  int from, to;     // the block's slice of them
  float temp, rtemp, rep;
  bool divide, mild, aligned, shared;  // aligned: four logits at a time
  bool lift;  // the row's largest x is +inf: tokens there count as 0, all others as -inf (in xs they already are)
  __device__ __forceinline__ float4 from4(float4 v, int i) const {
    float* e = reinterpret_cast<float*>(&v);
    if (divide) {
      bool odd = !mild;
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= e[j] > 0x1p100f || fabsf(e[j]) < 0x1p-79f;
      if (odd) {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = __fdiv_rn(e[j], temp);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float q = __fmul_rn(e[j], rtemp);
          q = __fmaf_rn(__fmaf_rn(-q, temp, e[j]), rtemp, q);
          e[j] = __fmaf_rn(__fmaf_rn(-q, temp, e[j]), rtemp, q);
        }
      }
    }
    if (seen) {
      const uint32_t bits = seen[i >> 5] >> (i & 31);  // i is a multiple of 4
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((bits >> j) & 1u) e[j] = __fdiv_rn(e[j], rep);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = fmaxf(e[j], -INFINITY);
    return v;
  }
  // logits i .. i + 3 (i a multiple of 4, i < V), -inf behind the row's end (a slice ends at a multiple of 4 or there)
  __device__ __forceinline__ float4 logits4(int i) const {
    float4 v;
    if (aligned && i + 4 <= V) {
      if constexpr (sizeof(T) == 4) {
        v = *reinterpret_cast<const float4*>(l + i);
      } else {
        const uint2 raw = *reinterpret_cast<const uint2*>(l + i);
        const T* e = reinterpret_cast<const T*>(&raw);
        v = make_float4(sf_logit(e), sf_logit(e + 1), sf_logit(e + 2), sf_logit(e + 3));
      }
    } else {
      v.x = sf_logit(l + i);
      v.y = i + 1 < V ? sf_logit(l + i + 1) : -INFINITY;
      v.z = i + 2 < V ? sf_logit(l + i + 2) : -INFINITY;
      v.w = i + 3 < V ? sf_logit(l + i + 3) : -INFINITY;
    }
    return v;
  }
  static __device__ __forceinline__ float lifted(float x) { return x == INFINITY ? 0.f : -INFINITY; }
  template <bool SHARED>
  __device__ __forceinline__ float4 x4(int i) const {
    if constexpr (SHARED) {
      return *reinterpret_cast<const float4*>(xs + (i - from));
    } else {
      float4 v = from4(logits4(i), i);
      if (lift) v = make_float4(lifted(v.x), lifted(v.y), lifted(v.z), lifted(v.w));
      return v;
    }
  }
  // f(std::true_type or std::false_type for x4's argument): a pass compiled for each
  template <typename F>
  __device__ __forceinline__ void pass(F f) const {
    if (shared) f(std::true_type());
    else f(std::false_type());
  }
  // f(x, index) for four tokens at a time
  template <typename F>
  __device__ __forceinline__ void each4(F f) const {
    pass([&](auto where) {
      for (int i = from + 4 * threadIdx.x; i < to; i += 4 * kSfThreads) {
        const float4 v = x4<decltype(where)::value>(i);
        const float x[4] = {v.x, v.y, v.z, v.w};
        f(x, i);
      }
    });
  }
  // f(x, index) for every token; behind the row's end x is -inf
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each4([&](const float(&x)[4], int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f(x[j], i + j);
    });
  }
};

// Weights: exp(x - m) by table and polynomial (Tang's scheme): x - m = n ln2 / 64 + r, |r| <= ln2 / 128,
// exp = 2^(n / 64) (1 + r + r^2/2 + r^3/6 + r^4/24), off by 4e-14; the table holds 2^(S + j / 64).  No branches:
// tokens beyond `far`, whose weight rounds to 0, are computed and dropped.  A row whose largest x is
// +inf comes lifted: its tokens there as 0 and the others as -inf.
struct Weigh {
  const double* table;
  double m;
  float top, far;  // the largest x, and the distance from it beyond which a weight rounds to 0
  __device__ __forceinline__ double scaled(float x) const {  // w 2^S
    const double magic = 6755399441055744.0;  // 1.5 2^52: the sum's low word is the rounded integer
    const double t = (double)x - m, z = fma(t, 92.33248261689366, magic);
    const int n = __double2loint(z);
    const double r = fma(z - magic, -0.010830424696249145, t);
    double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    p *= table[n & 63];
    const double w = __hiloint2double(__double2hiint(p) + (n & ~63) * (1 << 14), __double2loint(p));
    return top - x < far ? w : 0.0;
  }
  // v rounded to an integer, as the low bits of a double in [2^52, 2^53): sums of these patterns are sums of the
  // integers plus kBias each (modulo 2^64).
  static constexpr u64 kBias = 0x4330000000000000ull;
  static __device__ __forceinline__ u64 biased(double v) { return (u64)__double_as_longlong(v + 4503599627370496.0); }
  static __device__ __forceinline__ u64 fix(double v) { return biased(v) - kBias; }  // v < 2^51
  __device__ __forceinline__ u64 of(float x) const { return fix(scaled(x)); }
};

// Adds a weight to a bin's two words in shared memory (64-bit shared atomics are loops: 74 us instead of 60 for 148 rows
// of 50,280 with top-p).
__device__ __forceinline__ void add_weight(unsigned* lo, unsigned* hi, u64 w) {
  const unsigned wl = (unsigned)w, old = atomicAdd(lo, wl);
  const unsigned wh = (unsigned)(w >> 32) + (old + wl < old ? 1u : 0u);
  if (wh) atomicAdd(hi, wh);
}

// The last kept token of the order: its x, and how many of the tokens with that x stay (lowest indices first).
struct Cut {
  float x;
  int ties;
};

struct Shared {
  u64 red[kSfWarps];
  int ired[kSfWarps];
  float fred[kSfWarps];
  double table[64];
  u64 found;
  int count, pick, row;
  // written by the cluster's blocks in one another's copy, a slot for each; two sets, used in turn
  float bmax[2][kSfBlocks];
  u64 bmass[2][kSfBlocks];
  int bcount[2][kSfBlocks];
  // written by the first block in everybody's
  Cut cut;
  u64 budget, above;
  float scale;
  int state;
};

// The blocks of one row.
struct Group {
  int rank, blocks, turn;
  __device__ __forceinline__ void sync() const {
    if (blocks == 1) __syncthreads();
    else cooperative_groups::this_cluster().sync();
  }
  template <typename V>
  __device__ __forceinline__ V* at(V* p, int block) const {  // that block's copy of a shared variable
    return blocks == 1 ? p : cooperative_groups::this_cluster().map_shared_rank(p, block);
  }
  // Every block's value, the same in all its threads, to every block: read slots[turn][...] after the sync in it.
  template <typename V>
  __device__ __forceinline__ const V* share(V (&slots)[2][kSfBlocks], V v) {
    turn ^= 1;
    if (threadIdx.x < blocks) *at(&slots[turn][rank], threadIdx.x) = v;
    sync();
    return slots[turn];
  }
};

// Block-wide reductions and an exclusive scan, the same value in every thread.
template <typename V>
__device__ __forceinline__ V sf_sum(V v, V* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(red[threadIdx.x & 31]);
}
__device__ __forceinline__ float sf_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_max(red[threadIdx.x & 31]);
}
__device__ __forceinline__ u64 sf_scan(u64 v, u64* red, u64& total) {  // sum over the threads before this one
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  u64 upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  __syncthreads();
  if (lane == 31) red[wid] = upto;
  __syncthreads();
  u64 w = red[lane], wupto = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, wupto, o);
    if (lane >= o) wupto += x;
  }
  total = __shfl_sync(0xffffffffu, wupto, 31);
  return __shfl_sync(0xffffffffu, wupto - w, wid) + upto - v;
}

// From one value per warp in red[]: the sum over the warps before `wid`, and over all.
template <typename V>
__device__ __forceinline__ V sf_warps(const V* red, int wid, V& total) {
  const int lane = threadIdx.x & 31;
  const V own = red[lane];
  V upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  total = __shfl_sync(0xffffffffu, upto, 31);
  return __shfl_sync(0xffffffffu, upto - own, wid);
}

// Adds the tokens of a warp's tile that `take` accepts to the warp's pool (kSfPool floats, `have` < 32 in use) and runs
// use(x) for 32 of them as often as there are as many.
constexpr int kSfPool = 192;
template <typename F, typename G>
__device__ __forceinline__ void sf_pool(float* pool, int& have, const float4& v, F take, G use) {
  const int lane = threadIdx.x & 31;
  const float x[4] = {v.x, v.y, v.z, v.w};
  bool in[4], any = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) any |= in[j] = take(x[j]);
  if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned all = __ballot_sync(0xffffffffu, in[j]);
    if (in[j]) pool[have + __popc(all & ((1u << lane) - 1))] = x[j];
    have += __popc(all);
  }
  __syncwarp();
  while (have >= 32) {
    have -= 32;
    use(pool[have + lane]);
  }
  __syncwarp();
}

// Compare-exchange steps of a bitonic sort at distances 32 .. 1 among the 64 keys of a warp, for the merges of length
// k: lane l holds the keys base + l and base + l + 32.
__device__ __forceinline__ void sf_merge64(u64 (&e)[2], int base, int k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 32; j > 0; j >>= 1) {
    if (j >= k) continue;
    if (j == 32) {
      const u64 a = max(e[0], e[1]), b = min(e[0], e[1]);
      const bool falling = (base & k) == 0;
      e[0] = falling ? a : b, e[1] = falling ? b : a;
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u64 o = __shfl_xor_sync(0xffffffffu, e[h], j);
        const bool falling = ((base + lane + 32 * h) & k) == 0;
        e[h] = falling == ((lane & j) == 0) ? max(e[h], o) : min(e[h], o);
      }
    }
  }
}
// Descending sort of 64 keys by one warp.
__device__ __forceinline__ void sf_sort64(u64 (&e)[2], int base = 0) {
#pragma unroll 1
  for (int k = 2; k <= 64; k <<= 1) sf_merge64(e, base, k);
}
// Sum over the keys before each of two: e = 0 stands before e = 1 of every lane (positions l and l + 32).
__device__ __forceinline__ void sf_scan64(const u64 (&v)[2], u64 (&before)[2], u64& total) {
  const int lane = threadIdx.x & 31;
  u64 a = v[0], b = v[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  const u64 first = __shfl_sync(0xffffffffu, a, 31);
  before[0] = a - v[0];
  before[1] = first + b - v[1];
  total = first + __shfl_sync(0xffffffffu, b, 31);
}
// The places of a warp's two keys (or zeros) among list[0..n): how many there are larger.
__device__ __forceinline__ void sf_places(const u64* list, int n, const u64 (&key)[2], int (&place)[2]) {
  place[0] = place[1] = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) {
    const u64 o = list[j];
    place[0] += o > key[0];
    place[1] += o > key[1];
  }
}

// The draw among list[0..kept), kept <= 64, {key of x, complement of the index}, by one warp; exact: the weights of the
// lane's keys, l and l + 32.  The list is overwritten.
__device__ __forceinline__ void sf_draw64(const SampleArgs& p, int b, float u, u64* list, const double (&exact)[2], int kept) {
  const int lane = threadIdx.x & 31;
  u64 key[2], w[2], before[2], total;
  int place[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const u64 k = lane + 32 * e < kept ? list[lane + 32 * e] : 0ull;
    key[e] = (k << 32) | (k >> 32);
  }
  __syncwarp();
  list[lane] = key[0];
  list[lane + 32] = key[1];
  __syncwarp();
  sf_places(list, kept, key, place);  // in vocabulary order
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 32 * e < kept) list[place[e]] = Weigh::fix(exact[e]);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 2; ++e) w[e] = lane + 32 * e < kept ? list[lane + 32 * e] : 0ull;
  sf_scan64(w, before, total);
  const u64 target = min((u64)((double)u * (double)total), total - 1);
  int at = -1;  // the place that is drawn
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (target >= before[e] && target < before[e] + w[e]) at = lane + 32 * e;
  at = __reduce_max_sync(0xffffffffu, at);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (lane + 32 * e < kept && place[e] == at) {
      p.next[b] = (int)(0xffffffffu - (unsigned)(key[e] >> 32));
      if (p.kept) p.kept[b] = kept;
      if (p.prob) p.prob[b] = (float)(exact[e] / (double)total);
    }
  }
}

// Descending sort of list[0..n), n <= kSfList, all different.  Up to 256 by counting.  More go to kSfBins buckets by
// bin(key), which must not fall along the order, and are counted within theirs (2 us for some 1500 keys; a bitonic sort takes
// 15); where a bucket holds more than kSfCrowd, by a bitonic sort, padded with zeros to a power of two, by half as many
// threads as entries: distances below 64 in registers, the others through the list.  bins: kSfBins words.  Begins and
// ends with a block barrier.
constexpr int kSfCrowd = 64;
template <typename F>
__device__ __forceinline__ void sf_sort(u64* list, int n, unsigned* bins, u64* red, F bin) {
  int size = 64;
  while (size < n) size <<= 1;
  __syncthreads();
  if (size <= 256) {
    // few: every key's place is the number of larger ones, counted by several threads
    const int per = kSfThreads / size, i = threadIdx.x / per, part = threadIdx.x % per;
    const u64 key = i < n ? list[i] : 0ull;
    int place = 0;
    for (int j = part; j < n; j += per) place += list[j] > key;
    for (int o = per / 2; o > 0; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    __syncthreads();
    if (part == 0 && i < n) list[place] = key;
    __syncthreads();
    return;
  }
  {
    bins[threadIdx.x] = 0u;
    __syncthreads();
    u64 e[2], total;
    int b[2], at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = threadIdx.x + h * kSfThreads;
      if (i < n) {
        e[h] = list[i];
        b[h] = bin(e[h]);
        at[h] = atomicAdd(bins + b[h], 1u);
      }
    }
    __syncthreads();
    const unsigned here = bins[threadIdx.x], first = (unsigned)sf_scan((u64)here, red, total);
    const bool crowded = __syncthreads_or(here > kSfCrowd);
    if (!crowded) {
      bins[threadIdx.x] = first | here << 16;
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if ((int)threadIdx.x + h * kSfThreads < n) list[(bins[b[h]] & 0xffff) + at[h]] = e[h];
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if ((int)threadIdx.x + h * kSfThreads < n) {
          const unsigned from = bins[b[h]] & 0xffff, to = from + (bins[b[h]] >> 16);
          at[h] = from;
          for (unsigned j = from; j < to; ++j) at[h] += list[j] > e[h];
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if ((int)threadIdx.x + h * kSfThreads < n) list[at[h]] = e[h];
      __syncthreads();
      return;
    }
  }
  const int workers = size / 2;
  if (threadIdx.x < workers) {
    const int base = (threadIdx.x >> 5) * 64, i0 = base + (threadIdx.x & 31), i1 = i0 + 32;
    u64 e[2] = {i0 < n ? list[i0] : 0ull, i1 < n ? list[i1] : 0ull};
    auto meet = [&] { asm volatile("bar.sync 1, %0;" ::"r"(workers) : "memory"); };
    sf_sort64(e, base);
    for (int k = 128; k <= size; k <<= 1) {
      for (int j = k >> 1; j >= 64; j >>= 1) {
        meet();
        list[i0] = e[0];
        list[i1] = e[1];
        meet();
        const bool upper = (base & j) != 0, falling = (base & k) == 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u64 o = list[(h ? i1 : i0) ^ j];
          e[h] = falling != upper ? max(e[h], o) : min(e[h], o);
        }
      }
      sf_merge64(e, base, k);
    }
    meet();
    list[i0] = e[0];
    list[i1] = e[1];
  }
  __syncthreads();
}

// Appends the cluster's tokens that `take` accepts (none at -inf) to the first block's list, as {key of x,
// complement of the index}; returns how many there are, which may be more than were stored.
template <typename T, typename F>
__device__ int sf_gather(const Row<T>& row, Group& grp, u64* list, Shared& sh, F take) {
  if (grp.rank == 0 && threadIdx.x == 0) sh.count = 0;
  grp.sync();
  u64* const to = grp.at(list, 0);
  int* const count = grp.at(&sh.count, 0);
  const int lane = threadIdx.x & 31;
  row.pass([&](auto where) {
    for (int i0 = row.from + 4 * (threadIdx.x - lane); i0 < row.to; i0 += 4 * kSfThreads) {
      const int i = i0 + 4 * lane;
      const float4 v = i < row.to ? row.template x4<decltype(where)::value>(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      const float x[4] = {v.x, v.y, v.z, v.w};
      bool in[4], any = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) any |= in[j] = take(x[j]);
      if (!__any_sync(0xffffffffu, any)) continue;
      unsigned all[4];
      int found = 0, at = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) found += __popc(all[j] = __ballot_sync(0xffffffffu, in[j]));
      if (lane == 0) at = atomicAdd(count, found);
      at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int place = at + __popc(all[j] & ((1u << lane) - 1));
        if (in[j] && place < kSfList) to[place] = ((u64)sf_key(x[j]) << 32) | (0xffffffffu - (unsigned)(i + j));
        at += __popc(all[j]);
      }
    }
  });
  grp.sync();
  const int n = *count;
  grp.sync();  // everybody has read it: the list may be used again
  return n;
}

// The cut by four rounds over 8 bits of the key, for what does not fit the list.  by_weight: a token stays while
// the weight before it is <= budget; else `budget` tokens stay.  Looks at the tokens that `floor` keeps and
// returns it when the budget outlasts them.
template <typename T>
__device__ __noinline__ Cut sf_radix_cut(const Row<T>& row, Group& grp, const Weigh& weigh, Cut floor, bool by_weight,
                                         u64 budget, unsigned* cnt, unsigned* lo, unsigned* hi) {
  const uint32_t least = max(sf_key(floor.x), 1u);
  uint32_t prefix = 0;
  u64 used = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    grp.sync();
    for (int i = threadIdx.x; i < 256; i += kSfThreads) cnt[i] = lo[i] = hi[i] = 0u;
    __syncthreads();
    row.each([&](float x, int) {
      const uint32_t k = sf_key(x);
      if (k < least || (shift < 24 && (k >> (shift + 8)) != prefix)) return;
      const int d = (k >> shift) & 255;
      atomicAdd(cnt + d, 1u);
      if (by_weight) add_weight(lo + d, hi + d, weigh.of(x));
    });
    grp.sync();
    if (grp.blocks > 1) {  // every block adds up everybody's
      unsigned c = 0;
      u64 m = 0;
      if (threadIdx.x < 256) {
        for (int r = 0; r < grp.blocks; ++r) {
          c += grp.at(cnt, r)[threadIdx.x];
          m += ((u64)grp.at(hi, r)[threadIdx.x] << 32) + grp.at(lo, r)[threadIdx.x];
        }
      }
      grp.sync();
      if (threadIdx.x < 256) cnt[threadIdx.x] = c, lo[threadIdx.x] = (unsigned)m, hi[threadIdx.x] = (unsigned)(m >> 32);
      __syncthreads();
    }
    int d = 255;  // every thread walks the digits from the top; all come to the same one
    for (; d >= 0; --d) {
      const u64 m = by_weight ? ((u64)hi[d] << 32) + lo[d] : cnt[d];
      if (cnt[d] && (by_weight ? used + m > budget : used + m >= budget)) break;
      used += m;
    }
    const int here = d < 0 ? 0 : (int)cnt[d];
    grp.sync();
    if (d < 0) return floor;
    prefix = (prefix << 8) | (uint32_t)d;
    if (shift == 0) {
      const float x = sf_unkey(prefix);
      const int n = x == floor.x ? min(floor.ties, here) : here;
      if (!by_weight) return Cut{x, min(n, (int)(budget - used))};
      const u64 w = weigh.of(x);
      return Cut{x, w == 0 ? n : (int)min((u64)n, (budget - used) / w + 1)};
    }
  }
  return floor;
}

// The row of the place-th block when there are more rows than run at once: first those that weigh every token and
// select by weight (three times the time of the others), last the greedy ones; a long row that starts last runs alone
// (256 rows of 50,280 with settings of all kinds: 53 us, 64 in their own order; all with top-p alone: 112, 108).
constexpr int kSfOrdered = 4 * kSfThreads;
__device__ __forceinline__ int sf_row(const SampleArgs& p, int place, Shared& sh) {
  const int per = (p.ordered + kSfThreads - 1) / kSfThreads, r0 = threadIdx.x * per;
  u64 counts = 0, total;  // of the three kinds, 16 bits each
  unsigned kinds = 0;
  for (int j = 0; j < per && r0 + j < p.ordered; ++j) {
    const int r = r0 + j, k = p.top_k ? p.top_k[r] : 0;
    const bool greedy = k == 1 || (p.temperature && !(p.temperature[r] > 0.f));
    const bool heavy = (k <= 0 || k > kSfList) && p.top_p && p.top_p[r] < 1.f;
    const unsigned kind = greedy ? 2 : heavy ? 0 : 1;
    kinds |= kind << (2 * j);
    counts += 1ull << (16 * kind);
  }
  u64 before = sf_scan(counts, sh.red, total);
  before += (total << 16) + (total << 32);  // the kinds ahead of each
  for (int j = 0; j < per && r0 + j < p.ordered; ++j) {
    const unsigned kind = kinds >> (2 * j) & 3;
    if ((int)(before >> (16 * kind) & 0xffff) == place) sh.row = r0 + j;
    before += 1ull << (16 * kind);
  }
  __syncthreads();
  return sh.row;
}

template <typename T>
__global__ void __launch_bounds__(kSfThreads) sample_filtered_kernel(const SampleArgs p) {
  extern __shared__ __align__(16) char dyn[];
  __shared__ Shared sh;
  u64* list = reinterpret_cast<u64*>(dyn);  // [kSfList]; before it is filled, the histograms' words
  unsigned* cnt = reinterpret_cast<unsigned*>(dyn);
  unsigned *lo = cnt + 256, *hi = lo + kSfBins;
  unsigned* bins = reinterpret_cast<unsigned*>(list + kSfList);  // [2 kSfBins] of a sort
  float* pool = reinterpret_cast<float*>(dyn) + (threadIdx.x >> 5) * kSfPool;  // in the draw: one per warp, over both
  float* xs = reinterpret_cast<float*>(bins + 2 * kSfBins);
  static_assert(kSfWarps * kSfPool * 4 == kSfList * 8 + 2 * kSfBins * 4, "");
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, V = p.vocab;
  Group grp{0, 1, 0};
  if (gridDim.y > 1) {  // a cluster is the blocks of one row
    grp.blocks = gridDim.y;
    grp.rank = blockIdx.y;
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");  // this block runs: the wait is below
  }
  const int b = p.ordered ? sf_row(p, blockIdx.x, sh) : blockIdx.x;
  const bool chief = grp.rank == 0;
  Row<T> row;
  row.l = static_cast<const T*>(p.logits) + (long long)b * p.ld;
  row.seen = p.seen ? p.seen + (size_t)b * ((V + 31) / 32) : nullptr;
  row.xs = xs;
  row.shared = p.in_shared;
  row.V = V;
  row.from = min(V, grp.rank * p.slice);
  row.to = min(V, row.from + p.slice);
  row.lift = false;
  row.aligned = (reinterpret_cast<uintptr_t>(row.l) & (4 * sizeof(T) - 1)) == 0;
  const float temp = p.temperature ? p.temperature[b] : 1.0f;
  const bool greedy = !(temp > 0.f);
  row.temp = greedy ? 1.0f : temp;
  row.rep = p.rep;
  row.rtemp = __frcp_rn(row.temp);
  row.divide = row.temp != 1.f;
  row.mild = row.temp > 0x1p-20f && row.temp < 0x1p20f;
  const int k = greedy ? 1 : (p.top_k ? p.top_k[b] : 0);
  const float top_p = p.top_p ? p.top_p[b] : 1.0f, min_p = p.min_p ? p.min_p[b] : 0.f;
  float u = p.uniform[b];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;

  // ---- x of the slice, each thread's largest, the row's largest
  float mine2[2] = {-INFINITY, -INFINITY};  // of the thread's tokens, split in two
  constexpr int kAhead = 4;
  for (int i0 = row.from + 4 * tid; i0 < row.to; i0 += kAhead * 4 * kSfThreads) {
    float4 v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * 4 * kSfThreads;
      if (i < row.to) v[j] = row.logits4(i);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * 4 * kSfThreads;
      if (i < row.to) {
        const float4 x = row.from4(v[j], i);
        if (p.in_shared) *reinterpret_cast<float4*>(xs + (i - row.from)) = x;
        mine2[j & 1] = fmaxf(mine2[j & 1], fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));
      }
    }
  }
  const float mine = fmaxf(mine2[0], mine2[1]);
  if (tid < 64) sh.table[tid] = ldexp(exp2(tid / 64.0), p.shift);
  if (tid == 0) sh.pick = V;
  float top = sf_max(mine, sh.fred);
  if (grp.blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all run: their memory can be written
  {
    const float* all = grp.share(sh.bmax, top);
    for (int r = 0; r < grp.blocks; ++r) top = fmaxf(top, all[r]);
  }
  if (top == -INFINITY) {  // nothing to take in this row
    if (chief && tid == 0) {
      p.next[b] = -1;
      if (p.kept) p.kept[b] = 0;
      if (p.prob) p.prob[b] = 0.f;
    }
    grp.sync();
    return;
  }
  if (k == 1) {  // the first token of the order
    int* const pick = grp.at(&sh.pick, 0);
    if (mine == top) row.each([&](float x, int i) { if (x == top) atomicMin(pick, i); });
    grp.sync();
    if (chief && tid == 0) {
      p.next[b] = sh.pick;
      if (p.kept) p.kept[b] = 1;
      if (p.prob) p.prob[b] = 1.f;
    }
    return;
  }
  if (top == INFINITY) {
    row.lift = true;
    top = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) mine2[e] = Row<T>::lifted(mine2[e]);
    if (row.shared) {
      for (int i = row.from + tid; i < row.to; i += kSfThreads) xs[i - row.from] = Row<T>::lifted(xs[i - row.from]);
      __syncthreads();
    }
  }
  const Weigh weigh{sh.table, (double)top, top, (p.shift + 1) * 0.69314718f + 0.5f};
  const double unit = sh.table[0], least = (double)min_p * unit;
  Cut cut{-INFINITY, kSfAll};
  bool open_p = top_p < 1.f;  // top-p is still to be applied

  if (k > 0 && k < V) {
    // ---- top-k: a lower bound of the k-th largest x, the tokens from there on sorted
    float bound = -INFINITY;
    if (k <= 2 * kSfThreads) {
      // The c-th largest of the block's threads' largest (for larger c of both their halves), rounded down to a bin of a
      // histogram: at least c of the block's tokens are there or above.  With c = k / blocks in every block, the
      // least of the blocks' bounds bounds the row's k-th largest; where that is nothing (a block holds too few
      // tokens), with c = k, each one's does.
      auto reach = [&](int c) -> float {
        const bool halves = c > kSfThreads / 4;
        const float m0 = halves ? mine2[0] : fmaxf(mine2[0], mine2[1]), m1 = halves ? mine2[1] : -INFINITY;
        const float low = fminf(m0 > -INFINITY ? m0 : top, m1 > -INFINITY ? m1 : top);
        const float width = fmaxf(top + sf_max(-low, sh.fred), 1e-6f * fabsf(top) + 1e-30f), scale = (kSfBins - 1) / width;
        lo[tid] = 0u;
        __syncthreads();
        if (m0 > -INFINITY) atomicAdd(lo + min(kSfBins - 1, (int)((top - m0) * scale)), 1u);
        if (m1 > -INFINITY) atomicAdd(lo + min(kSfBins - 1, (int)((top - m1) * scale)), 1u);
        __syncthreads();
        u64 total;
        const int n = (int)lo[tid], before = (int)sf_scan((u64)n, sh.red, total);
        if (tid == 0) sh.scale = -INFINITY;
        __syncthreads();
        // a margin for the roundings of the bin's number
        if (before < c && before + n >= c) sh.scale = top - (tid + 1.01f) / scale - 1e-6f * fabsf(top);
        __syncthreads();
        return sh.scale;
      };
      bound = reach((k + grp.blocks - 1) / grp.blocks);
      if (grp.blocks > 1) {
        const float* bounds = grp.share(sh.bmax, bound);
        for (int r = 0; r < grp.blocks; ++r) bound = fminf(bound, bounds[r]);
        if (bound == -INFINITY) {
          bounds = grp.share(sh.bmax, reach(k));
          for (int r = 0; r < grp.blocks; ++r) bound = fmaxf(bound, bounds[r]);
        }
      }
    }
    int n = k > kSfList ? kSfList + 1
                        : sf_gather(row, grp, list, sh, [&](float x) { return x >= bound && x > -INFINITY; });
    if (n > kSfList && k <= kSfList) {
      // too many: halve the keys between by counting tokens, until at least k and no more than fit are left
      uint32_t low = sf_key(bound), high = sf_key(top);
      while (low < high) {
        const uint32_t mid = low + (high - low + 1) / 2;
        const float at = sf_unkey(mid);
        int c = 0;
        row.each([&](float x, int) { c += x >= at; });
        const int* all = grp.share(sh.bcount, sf_sum(c, sh.ired));
        c = 0;
        for (int r = 0; r < grp.blocks; ++r) c += all[r];
        if (c >= k) low = mid, n = c;
        else high = mid - 1;
        if (n <= kSfList) break;
      }
      bound = sf_unkey(low);
      if (n <= kSfList) n = sf_gather(row, grp, list, sh, [&](float x) { return x >= bound && x > -INFINITY; });
    }
    if (n <= kSfList) {
      // the first block orders them and draws
      if (chief) {
        const int n_k = min(n, k);
        if (n <= 64) {
          // one warp: order, weights, what stays; then the draw
          if (wid == 0) {
            u64 key[2], w[2], before[2], total;
            double exact[2];
            int place[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) key[e] = lane + 32 * e < n ? list[lane + 32 * e] : 0ull;
            sf_places(list, n, key, place);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (lane + 32 * e < n) list[place[e]] = key[e];
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              key[e] = lane + 32 * e < n_k ? list[lane + 32 * e] : 0ull;
              exact[e] = key[e] ? weigh.scaled(sf_unkey((uint32_t)(key[e] >> 32))) : 0.0;
              w[e] = Weigh::fix(exact[e]);
            }
            sf_scan64(w, before, total);
            const u64 budget = top_p < 1.f ? (u64)(fmax((double)top_p, 0.0) * (double)total) : ~0ull;
            int kept = 0;  // the first ones: every condition falls along the order
#pragma unroll
            for (int e = 0; e < 2; ++e)
              kept += __popc(__ballot_sync(0xffffffffu, key[e] && before[e] <= budget &&
                                                            (sf_unkey((uint32_t)(key[e] >> 32)) == top || exact[e] >= least)));
            sf_draw64(p, b, u, list, exact, kept);
          }
        } else {
          const float low = fmaxf(bound, -0x1.fffffep127f), per = kSfBins / fmaxf(top - low, 1e-30f);
          sf_sort(list, n, bins, sh.red, [&](u64 key) {
            return min(kSfBins - 1, (int)((top - sf_unkey((uint32_t)(key >> 32))) * per));
          });
          // weights in order: thread t has the tokens 2t and 2t + 1
          float x[2];
          u64 w[2], total;
          double exact[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 2 * tid + e;
            x[e] = i < n_k ? sf_unkey((uint32_t)(list[i] >> 32)) : -INFINITY;
            exact[e] = i < n_k ? weigh.scaled(x[e]) : 0.0;
            w[e] = Weigh::fix(exact[e]);
          }
          const u64 before = sf_scan(w[0] + w[1], sh.red, total);
          const u64 budget = top_p < 1.f ? (u64)(fmax((double)top_p, 0.0) * (double)total) : ~0ull;
          int stay = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            stay += 2 * tid + e < n_k && before + (e ? w[0] : 0) <= budget && (x[e] == top || exact[e] >= least);
          const int kept = sf_sum(stay, sh.ired);  // the first `kept` tokens: every condition falls along the order
          if (kept <= 64) {
            if (wid == 0) {
#pragma unroll
              for (int e = 0; e < 2; ++e)
                exact[e] = lane + 32 * e < kept ? weigh.scaled(sf_unkey((uint32_t)(list[lane + 32 * e] >> 32))) : 0.0;
              sf_draw64(p, b, u, list, exact, kept);
            }
            return;
          }
          // the kept tokens in vocabulary order: {complement of the index, key of x}
          u64 key[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) key[e] = list[2 * tid + e];
          __syncthreads();
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (2 * tid + e < kept) list[2 * tid + e] = (key[e] << 32) | (key[e] >> 32);
          const float per_token = (float)kSfBins / (float)V;
          sf_sort(list, kept, bins, sh.red, [&](u64 key) {
            return min(kSfBins - 1, (int)((float)(0xffffffffu - (unsigned)(key >> 32)) * per_token));
          });
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 2 * tid + e;
            exact[e] = i < kept ? weigh.scaled(sf_unkey((uint32_t)list[i])) : 0.0;
            w[e] = Weigh::fix(exact[e]);
          }
          u64 from = sf_scan(w[0] + w[1], sh.red, total);
          const u64 target = min((u64)((double)u * (double)total), total - 1);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (target >= from && target < from + w[e]) {
              p.next[b] = (int)(0xffffffffu - (unsigned)(list[2 * tid + e] >> 32));
              if (p.kept) p.kept[b] = kept;
              if (p.prob) p.prob[b] = (float)(exact[e] / (double)total);
            }
            from += w[e];
          }
        }
      }
      return;  // after the gather no block reaches into another's memory
    } else {
      cut = sf_radix_cut(row, grp, weigh, cut, false, (u64)k, cnt, lo, hi);
    }
  }

  if (open_p) {
    // ---- top-p over what top-k keeps (here: everything, or more tokens than the list holds)
    bool found = false;
    u64 budget = 0;
    if (cut.x == -INFINITY) {
      // Weights by x, in bins; even and odd warps have a copy each (fewer collide).  Tokens further below the top than
      // `range` weigh less than (1 - top_p) / V of it each, so together too little to hold the boundary: they are
      // only added up.  One thread per bin then adds up the copies and the blocks.
      const float range = fminf(weigh.far, logf(V / (1.f - fmaxf(top_p, 0.f))) + 0.01f), scale = kSfBins / range;
      unsigned *lo0 = cnt, *hi0 = cnt + 2 * kSfBins, *lo1 = lo0 + (wid & 1) * kSfBins, *hi1 = hi0 + (wid & 1) * kSfBins;
      lo0[tid] = lo0[kSfBins + tid] = hi0[tid] = hi0[kSfBins + tid] = 0u;
      __syncthreads();
      u64 rest = 0;
      row.each4([&](const float(&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float d = (top - x[j]) * scale;
          const u64 w = weigh.of(x[j]);
          if (d < (float)kSfBins) add_weight(lo1 + (int)d, hi1 + (int)d, w);
          else rest += w;
        }
      });
      rest = sf_sum(rest, sh.red);
      const u64* rests = grp.share(sh.bmass, rest);
      if (chief) {
        u64 w = 0, total;
#pragma unroll
        for (int r = 0; r < kSfBlocks; ++r) {
          if (r < grp.blocks) {
            const unsigned *l = grp.at(lo0, r), *h = grp.at(hi0, r);
            w += ((u64)h[tid] << 32) + l[tid] + ((u64)h[kSfBins + tid] << 32) + l[kSfBins + tid];
          }
        }
        const u64 before = sf_scan(w, sh.red, total);
        for (int r = 0; r < grp.blocks; ++r) total += rests[r];
        budget = (u64)(fmax((double)top_p, 0.0) * (double)total);
        if (tid < grp.blocks) *grp.at(&sh.budget, tid) = budget, *grp.at(&sh.state, tid) = -1;
        __syncthreads();
        if (before <= budget && before + w > budget) {
          for (int r = 0; r < grp.blocks; ++r) *grp.at(&sh.state, r) = tid;
          sh.above = before;
        }
      }
      grp.sync();
      budget = sh.budget;
      const float d0 = (float)sh.state, d1 = d0 + 1.f;
      int n = kSfList + 1;
      if (sh.state >= 0)
        n = sf_gather(row, grp, list, sh, [&](float x) {
          const float d = (top - x) * scale;
          return d >= d0 && d < d1;
        });
      if (n <= kSfList) {
        if (chief) {
          sf_sort(list, n, bins, sh.red, [&](u64 key) {
            const float d = (top - sf_unkey((uint32_t)(key >> 32))) * scale - d0;
            return min(kSfBins - 1, max(0, (int)(d * kSfBins)));
          });
          float x[2];
          u64 v[2], total;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 2 * tid + e;
            x[e] = i < n ? sf_unkey((uint32_t)(list[i] >> 32)) : -INFINITY;
            v[e] = i < n ? weigh.of(x[e]) : 0;
          }
          const u64 start = sh.above + sf_scan(v[0] + v[1], sh.red, total);
          int stay = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) stay += 2 * tid + e < n && start + (e ? v[0] : 0) <= budget;
          stay = sf_sum(stay, sh.ired);  // at least 1: the bin's first token has `above` <= budget before it
          const float last = sf_unkey((uint32_t)(list[stay - 1] >> 32));
          int equal = 0, ties = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool same = 2 * tid + e < n && x[e] == last;
            equal += same;
            ties += same && 2 * tid + e < stay;
          }
          equal = sf_sum(equal, sh.ired);
          ties = sf_sum(ties, sh.ired);
          if (tid < grp.blocks) *grp.at(&sh.cut, tid) = Cut{last, ties == equal ? kSfAll : ties};
        }
        grp.sync();
        cut = sh.cut;
        found = true;
      }
    } else {
      u64 m = 0;
      row.each4([&](const float(&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) m += x[j] > cut.x ? weigh.of(x[j]) : 0;
      });
      const u64* all = grp.share(sh.bmass, sf_sum(m, sh.red));
      m = (u64)cut.ties * weigh.of(cut.x);
      for (int r = 0; r < grp.blocks; ++r) m += all[r];
      budget = (u64)(fmax((double)top_p, 0.0) * (double)m);
    }
    if (!found) cut = sf_radix_cut(row, grp, weigh, cut, true, budget, cnt, lo, hi);
  }

  // ---- the draw: every warp owns a run of the slice, a lane four neighbouring tokens at a time
  const int run = (p.slice + kSfWarps * 128 - 1) / (kSfWarps * 128) * 128;
  const int i0 = min(row.to, row.from + wid * run), i1 = min(row.to, i0 + run);
  const bool count_ties = cut.ties != kSfAll;
  // tokens below this are not kept: the cut, and a bound of min_p's that leaves the comparison to the weights
  const float floor_p = min_p > 0.f ? fminf(top + logf(min_p) - 0.01f - 1e-5f * fabsf(top), top) : -INFINITY;
  const float floor_x = fmaxf(cut.x, floor_p);
  auto kept_by_x = [&](float x) { return x >= floor_x && x > -INFINITY; };
  auto weight = [&](float x) -> double {  // negative: not kept by x and min_p
    const double w = weigh.scaled(x);
    return kept_by_x(x) && (x == top || w >= least) ? w : -1.0;
  };
  u64 mass = 0;
  int count = 0, tie0 = 0;  // tie0: tokens equal to the cut before this warp's run
  row.pass([&](auto where) {
    if (!count_ties) {
      // the weights of the runs do not depend on the order within them
      auto add = [&](float x) {
        const double w = weight(x);
        mass += Weigh::fix(fmax(w, 0.0));
        count += w >= 0.0;
      };
      if (floor_x == -INFINITY) {
        for (int i = i0 + 4 * lane; i < i1; i += 128) {
          const float4 v = row.template x4<decltype(where)::value>(i);
          const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mass += Weigh::biased(weigh.scaled(x[j]));
            count += x[j] > -INFINITY;
          }
          mass -= 4 * Weigh::kBias;
        }
      } else {
        int have = 0;
        for (int i = i0; i < i1; i += 128) {
          const float4 v = i + 4 * lane < i1 ? row.template x4<decltype(where)::value>(i + 4 * lane) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          sf_pool(pool, have, v, kept_by_x, add);
        }
        __syncwarp();
        if (have) add(lane < have ? pool[lane] : -INFINITY);
      }
    } else {
      int ties = 0;
      for (int i = i0 + 4 * lane; i < i1; i += 128) {
        const float4 v = row.template x4<decltype(where)::value>(i);
        ties += (v.x == cut.x) + (v.y == cut.x) + (v.z == cut.x) + (v.w == cut.x);
      }
      ties = warp_sum(ties);
      __syncthreads();
      if (lane == 0) sh.ired[wid] = ties;
      __syncthreads();
      int all;
      tie0 = sf_warps(sh.ired, wid, all);
      const int* theirs = grp.share(sh.bcount, all);
      for (int r = 0; r < grp.rank; ++r) tie0 += theirs[r];
      int tie = tie0;
      for (int i = i0; i < i1; i += 128) {
        const float4 v = i + 4 * lane < i1 ? row.template x4<decltype(where)::value>(i + 4 * lane) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const float x[4] = {v.x, v.y, v.z, v.w};
        int before = tie;  // equal tokens before this lane's next one
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned eq = __ballot_sync(0xffffffffu, x[j] == cut.x);
          before += __popc(eq & ((1u << lane) - 1));
          tie += __popc(eq);
        }
        if (!kept_by_x(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])))) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double w = weight(x[j]);
          const bool same = x[j] == cut.x, stay = w >= 0.0 && !(same && before >= cut.ties);
          mass += Weigh::fix(stay ? w : 0.0);
          count += stay;
          before += same;
        }
      }
    }
  });
  mass = warp_sum(mass);
  count = warp_sum(count);
  __syncthreads();
  if (lane == 0) sh.red[wid] = mass, sh.ired[wid] = count;
  __syncthreads();
  u64 total, before = sf_warps(sh.red, wid, total);
  int kept;
  sf_warps(sh.ired, wid, kept);
  const u64 here = total;
  if (grp.blocks > 1) {
    const u64* masses = grp.share(sh.bmass, total);
    const int* counts = grp.share(sh.bcount, kept);  // the last use of another block's memory
    total = 0, kept = 0;
    u64 ahead = 0;
    for (int r = 0; r < grp.blocks; ++r) {
      if (r < grp.rank) ahead += masses[r];
      total += masses[r];
      kept += counts[r];
    }
    before += ahead;
    const u64 target = min((u64)((double)u * (double)total), total - 1);
    if (target < ahead || target >= ahead + here) return;
  }
  const u64 target = min((u64)((double)u * (double)total), total - 1);  // total >= 2^S: the first token is kept
  if (lane == 0 && target >= before && target < before + mass) {
    sh.pick = wid;
    sh.found = before;
    sh.count = tie0;
  }
  __syncthreads();
  // ... and the whole block walks the run that holds the target
  before = sh.found;
  int tie = sh.count;
  const int first = row.from + sh.pick * run, end = min(row.to, first + run);
  for (int i = first; i < end; i += 4 * kSfThreads) {
    const int at = i + 4 * tid;
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (at < end) row.pass([&](auto where) { v = row.template x4<decltype(where)::value>(at); });
    const float x[4] = {v.x, v.y, v.z, v.w};
    int rank = 0;
    if (count_ties) {
      u64 ties, own = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) own += x[j] == cut.x;
      rank = tie + (int)sf_scan(own, sh.red, ties);
      tie += (int)ties;
    }
    double w[4];
    u64 fixed[4], sum = 0, all;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = weight(x[j]);
      const bool same = count_ties && x[j] == cut.x;
      fixed[j] = w[j] >= 0.0 && !(same && rank >= cut.ties) ? Weigh::fix(w[j]) : 0;
      rank += same;
      sum += fixed[j];
    }
    u64 from = before + sf_scan(sum, sh.red, all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (target >= from && target < from + fixed[j]) {
        p.next[b] = at + j;
        if (p.kept) p.kept[b] = kept;
        if (p.prob) p.prob[b] = (float)(w[j] / (double)total);
      }
      from += fixed[j];
    }
    before += all;
    if (before > target) return;
  }
}

template <typename T>
int launch_sample(SampleArgs p, int batch, cudaStream_t s) {
  static SmemLimit limit;
  const auto fn = sample_filtered_kernel<T>;
  const int list = kSfWarps * kSfPool * 4, most = 232448 - 2048;  // 227 KB per block less the static part
  const int capacity = (most - list) / 512 * 128;
  DFSSM_CU(limit.raise(reinterpret_cast<const void*>(fn), list + capacity * 4));
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kSfThreads);
  cfg.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  // Blocks per row: the number that takes the fewest waves x (tokens per block + what a block costs apart from its
  // tokens), in tokens.  Measured at 50,280 logits: a pass over a block's tokens costs 0.2 to 0.6 cycles a token, the
  // rest of a block about 12,000 cycles; tokens that do not fit shared memory cost about half as much again.
  // rows_at_once: the clusters of that size that run together with a full block per SM (B200: 148, 74, 45, 33, ...).
  static std::atomic<int> rows_at_once[kSfBlocks + 1];
  int blocks = 1, at_once = 0;
  long long least = 0;
  for (int n = 1; n <= kSfBlocks && (n == 1 || p.vocab >= 4096 * n); ++n) {
    int rows = rows_at_once[n].load(std::memory_order_relaxed);
    if (rows == 0) {
      cfg.gridDim = dim3(1, n);
      cfg.dynamicSmemBytes = list + capacity * 4;
      cluster.val.clusterDim.y = n;
      cfg.numAttrs = 1;
      DFSSM_CU(cudaOccupancyMaxActiveClusters(&rows, fn, &cfg));
      if (rows < 1) rows = 1;
      rows_at_once[n].store(rows, std::memory_order_relaxed);
    }
    const long long slice = (p.vocab + n - 1) / n, waves = (batch + rows - 1) / rows;
    const long long cost = waves * ((slice <= capacity ? slice : slice + slice / 2) + 12000);
    if (n == 1 || cost < least) blocks = n, at_once = rows, least = cost;
    if (batch >= 2 * rows) break;  // more blocks per row only add waves
  }
  p.slice = ((p.vocab + blocks - 1) / blocks + 127) / 128 * 128;
  p.in_shared = p.slice <= capacity;
  p.ordered = p.top_p && batch > at_once && batch <= kSfOrdered ? batch : 0;
  const int bytes = list + (p.in_shared ? p.slice * 4 : 0);
  cfg.gridDim = dim3(batch, blocks);
  cfg.dynamicSmemBytes = bytes;
  cluster.val.clusterDim.y = blocks;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  DFSSM_CU(cudaLaunchKernelEx(&cfg, fn, p));
  return DFSSM_OK;
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
  SampleArgs p{logits,      ld,   vocab,      temperature, top_p,     min_p, uniform, top_k,
               seen_bits, rep_penalty, next, kept_count, prob,        62 - bits > 50 ? 50 : 62 - bits, 0, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == DFSSM_F32) return launch_sample<float>(p, batch, s);
  if (dtype == DFSSM_F16) return launch_sample<__half>(p, batch, s);
  return launch_sample<__nv_bfloat16>(p, batch, s);
}
