// Gated delta rule over prompts, chunked: matrix products on the tensor cores instead of a token loop.
//
// Inside a chunk of C = 64 tokens, with G_t the running sum of the log decays and S the state before it, the
// corrections u_t = v_t - e^g_t S_(t-1) k_t (before their beta) solve a triangular system, so that
//   T = (I + L)^-1,   L[t][w] = beta_w e^(G_t - G_w) k_t.k_w  for w < t
//   u   = T r,        r_t = v_t - e^G_t S k_t
//   o_t = scale e^G_t S q_t + sum_(w <= t) P[t][w] u_w,   P[t][w] = scale beta_w e^(G_t - G_w) q_t.k_w
//   S  <- e^G_C S + sum_w beta_w e^(G_C - G_w) u_w k_w^T
// (with beta in the columns, u has the size of v for every beta, down to 0).
// T and P do not depend on the state: gated_delta_prep_kernel computes them for every chunk and head at
// once.  gated_delta_chunk_kernel then walks a sequence's chunks with the state in registers.
//
// Precision.  The state is an fp32 result, so no product may lose more than fp32 sums do.  k and q are 16-bit
// inputs and exact as fp16 operands (bf16 rows are brought to fp16 by a power of two per row: bf16 has
// fewer mantissa bits, and what falls under fp16's smallest number is 2^-31 of the row's largest).  fp32
// operands are scaled by a power of two per row (T: for the whole matrix), so that the largest is below 2^14,
// and split in two fp16 numbers hi + lo, which keep 22 bits of what is above 2^-17 of that and 2^-39 of it
// below; a product of two such pairs takes three MMAs (hi hi, hi lo, lo hi).  The scales of S and P come
// from their largest elements; those of r and u from bounds known before the products end,
//   |r| <= max |v| + sqrt(dk) max |S| max |k|,   |u| <= max |r| max_t sum_w |T[t][w]|,
// and a chunk where what matters lies too far below these bounds is taken token by token instead (kGdRangeO).  So the errors are
// those of fp32 sums, relative to the largest that a row of the state has or, but for its decays, still has: an element far
// smaller than others of its row that are not forgotten is held in 39 bits below the row's largest in S k and S q.
// Sums run in fp32 accumulators, and the state's update in one of its own, added to the decayed state with one
// rounding.  Decays are differences of sums in double precision: in fp32 a sum of
// -100 already leaves e^(G_t - G_w) an error of 4e-6.
#pragma once
#include "gated_delta.cuh"

namespace dfssm {

constexpr int kGdC = 64;                // tokens per chunk
constexpr int kGdFrags = 20;            // 8 x 16 fragments of a lower triangular 64 x 64 matrix
constexpr int kGdTri = kGdFrags * 512;  // bytes of one such matrix as fp16 hi/lo pairs, in fragment order
// Factors of a chunk: per token -e^G / |k|, the update's beta e^(G_C - G) / |k| scaled to at most 1, scale e^G / |q|
// and the inverse scale of P's row; then e^G_C, the inverse scale of T, the largest absolute row sum of T, the
// update's scale, the largest norm of a key, and the largest weight a u could have in the update: the largest
// beta e^(G_C - G) / |k| times the largest norm of a key as it is staged.  Last, in the inputs' type, each token's own weight
// beta e^(G_C - G) |k| relative to that (to within 1/4: by powers of two), and the norm of its key as the products see it.
enum { kGdBk = 0, kGdC2 = 64, kGdOq = 128, kGdOp = 192, kGdLast = 256, kGdTdn, kGdTsum, kGdCdn, kGdKn, kGdWm, kGdWeights = 264,
       kGdNorms = kGdWeights + 32, kGdVecs = kGdNorms + 32 };
constexpr int kGdFactors = 1408;                   // bytes of them
constexpr int kGdBlock = 2 * kGdTri + kGdFactors;  // bytes per chunk and value head: T, P, factors
static_assert(kGdVecs * 4 <= kGdFactors && kGdBlock % 128 == 0, "");

// Chunks are numbered without a plan: sequence i's chunk c is cu[i] / 64 + i + c, or, where only sequences of `least` tokens and
// more have chunks and least > 1, cu[i] / 64 + cu[i] / least + c if that ends lower.  Either leaves at most one number
// per such sequence unused and gives no number twice: from one sequence's start to the next one's, the first part grows by the
// whole chunks between and the second by at least 1.
__host__ __device__ inline bool gd_by_rows(int tokens, int n_seq, int least) { return least > 1 && tokens / least + 1 < n_seq; }
__host__ __device__ inline long long gd_chunk_slots(int tokens, int n_seq, int least) {
  return (long long)tokens / kGdC + (gd_by_rows(tokens, n_seq, least) ? tokens / least + 1 : n_seq);
}
__device__ __forceinline__ int gd_chunk_base(int first, int i, bool by_rows, int least) {  // of sequence i, from row `first` on
  return first / kGdC + (by_rows ? first / least : i);
}

// Fragments of B = M^T (M lower triangular, rows t): n-tile j holds rows 8j..8j+7, k-step kk columns
// 16kk..16kk+15, kk <= j / 2.  Lane l: row 8j + l/4, columns 16kk + 2(l%4) + {0, 1} and + 8, as 16 bytes
// {hi, hi + 8, lo, lo + 8}.
__host__ __device__ constexpr int gd_frag(int j, int kk) { return ((j & 1) ? ((j + 1) / 2) * ((j + 1) / 2) : (j / 2) * (j / 2 + 1)) + kk; }
static_assert(gd_frag(0, 0) == 0 && gd_frag(1, 0) == 1 && gd_frag(2, 0) == 2 && gd_frag(3, 0) == 4 && gd_frag(4, 0) == 6 &&
                  gd_frag(5, 0) == 9 && gd_frag(6, 0) == 12 && gd_frag(7, 3) == kGdFrags - 1, "");

__device__ __forceinline__ unsigned h2_bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
// Two fp32 operations in one instruction (sm_100 packed fp32).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 dup(float x) { return make_float2(x, x); }
// Two fp32 values as fp16 pairs hi + lo (22 bits).
__device__ __forceinline__ void split2(float2 x, unsigned& hi, unsigned& lo) {
  const __half2 h = __float22half2_rn(x);
  const float2 d = fma2(__half22float2(h), dup(-1.f), x);
  hi = h2_bits(h);
  lo = h2_bits(__float22half2_rn(d));
}
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) { split2(make_float2(x, y), hi, lo); }
// The power of two that brings a row whose largest magnitude is m into [2^13, 2^14), and its inverse.
__device__ __forceinline__ void row_scale(float m, float& up, float& down) {
  const int e = (int)(__float_as_uint(m) >> 23);  // m >= 0
  const int s = min(max(267 - e, 1), 253);
  up = __uint_as_float((unsigned)s << 23);
  down = __uint_as_float((unsigned)(254 - s) << 23);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// m16n8k16 fp16 MMA that the compiler may schedule among the others
__device__ __forceinline__ void mma_acc(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Ordered among themselves and with the barriers (volatile), free to move among ordinary loads.
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void stsm4t(uint32_t addr, const unsigned (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]) : "memory");
}
// 16-byte asynchronous copy; `valid` false fills with zeros and reads nothing
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// The walk is launched while the last blocks of the prep kernel still run (programmatic dependent launch): prep_done
// returns when all of them have ended and what they wrote can be read.
__device__ __forceinline__ void let_walk_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void prep_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte unit u of row t in a K or Q tile [64][DK] of fp16: rows of 8 or 16 units, the units
// of a row permuted by its low three bits, so that eight rows' units of one column fall into different banks.
template <int DK>
__device__ __forceinline__ uint32_t kq_off(int t, int u) {
  return (uint32_t)(t * DK * 2 + ((u ^ (t & 7)) << 4));
}

// ------------------------------------------------------------------ T, P and the factors of every chunk
//
// One block per chunk, key head and group of the value heads that share it: k.k^T and q.k^T are taken once
// (mma.sync, kept in registers) and serve every head of the group, whose gates differ.  The decay between
// tokens of different 16-token blocks is a product of two factors that meet at the block boundary before t,
// each at most 1, so only the diagonal blocks take an exponential per element.  T is inverted blockwise: the
// 16 x 16 diagonal blocks by forward substitution in fp32, then the corners -T22 (L21 T11) of 32 and of 64 with
// TF32 MMAs on split operands.

constexpr int kPrepThreads = 128;
constexpr int kLS = 68;  // row stride of the fp32 matrices in shared memory

template <int DK>
__host__ __device__ constexpr int gd_prep_tiles() {  // K and Q; once they are multiplied, T [64][kLS]
  return 2 * kGdC * DK * 2 > kGdC * kLS * 4 ? 2 * kGdC * DK * 2 : kGdC * kLS * 4;
}
template <int DK>
__host__ __device__ constexpr int gd_prep_smem() { return gd_prep_tiles<DK>() + kGdC * kLS * 4 + 64 * 8 + 64 * 4 * 11 + 64; }

// Three TF32 MMAs for a product of fp32 values: a, b split here.  hi is cut off after 11 bits and lo, exact, rounded to
// 11 (finite values: adding half of its last place may carry into the exponent, as it should), 2^-23 of the value.
// By integer instructions: cvt.rna.tf32 runs at a fraction of their rate (64 prompts of 64 tokens, 64 heads:
// 235 us, 246 with it, before the look at how far values lie apart).
__device__ __forceinline__ void tf32_split2(float v, unsigned& hi, unsigned& lo) {
  hi = __float_as_uint(v) & 0xffffe000u;
  lo = (__float_as_uint(v - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}
__device__ __forceinline__ void mma_tf32_acc(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The corner of the 2N x 2N block of T at (o, o): Y = -T22 (L21 T11), taken transposed, M^T = T11^T L21^T and
// Y^T = -M^T T22^T, so that M^T passes from accumulators to left operands in registers (an operand's k-th
// and k+4-th columns are the accumulator's columns 2k and 2k+1; the right operand follows).  A warp takes 16
// rows mt of the transposed matrices and, of Y^T, half the columns.
template <int N>
__device__ __forceinline__ void corner(const float* L, float* X, int o, int half, int mt, int lane) {
  constexpr int NTI = N / 8;
  const int g = lane >> 2, c = lane & 3;
  const float* L21 = L + (o + N) * kLS + o;
  const float* T11 = X + o * kLS + o + 16 * mt;
  const float* T22 = X + (o + N) * kLS + o + N;
  float m[NTI][4] = {};
#pragma unroll
  for (int k = 0; k < N; k += 8) {
    if (k + 8 > 16 * mt) {  // T11^T is upper triangular
      unsigned ah[4], al[4];
      const float* x = T11 + (k + 2 * c) * kLS + g;
      tf32_split2(x[0], ah[0], al[0]);
      tf32_split2(x[8], ah[1], al[1]);
      tf32_split2(x[kLS], ah[2], al[2]);
      tf32_split2(x[kLS + 8], ah[3], al[3]);
#pragma unroll
      for (int j = 0; j < NTI; ++j) {
        const float2 l = *reinterpret_cast<const float2*>(L21 + (8 * j + g) * kLS + k + 2 * c);
        unsigned bh0, bl0, bh1, bl1;
        tf32_split2(l.x, bh0, bl0);
        tf32_split2(l.y, bh1, bl1);
        mma_tf32_acc(m[j], al, bh0, bh1);
        mma_tf32_acc(m[j], ah, bl0, bl1);
        mma_tf32_acc(m[j], ah, bh0, bh1);
      }
    }
  }
  float y[NTI / 2][4] = {};
#pragma unroll
  for (int i = 0; i < NTI; ++i) {  // columns 8 i.. of M^T
    unsigned ah[4], al[4];
    tf32_split2(m[i][0], ah[0], al[0]);
    tf32_split2(m[i][2], ah[1], al[1]);
    tf32_split2(m[i][1], ah[2], al[2]);
    tf32_split2(m[i][3], ah[3], al[3]);
#pragma unroll
    for (int j = 0; j < NTI / 2; ++j) {
      const float2 t = *reinterpret_cast<const float2*>(T22 + (8 * (half * (NTI / 2) + j) + g) * kLS + 8 * i + 2 * c);
      unsigned bh0, bl0, bh1, bl1;
      tf32_split2(t.x, bh0, bl0);
      tf32_split2(t.y, bh1, bl1);
      mma_tf32_acc(y[j], al, bh0, bh1);
      mma_tf32_acc(y[j], ah, bl0, bl1);
      mma_tf32_acc(y[j], ah, bh0, bh1);
    }
  }
#pragma unroll
  for (int j = 0; j < NTI / 2; ++j) {
    float* out = X + (o + N + 8 * (half * (NTI / 2) + j) + 2 * c) * kLS + o + 16 * mt + g;
    out[0] = -y[j][0];
    out[kLS] = -y[j][1];
    out[8] = -y[j][2];
    out[kLS + 8] = -y[j][3];
  }
}

// e^(G_t - G_w) rk_w beta_w of rows t, t + 8 and columns w, w + 1 of one diagonal block: the product of the
// tables' factors where the block's decay stays within e^kMild, so that neither factor overflows, else an
// exponential each.  Above the diagonal the values mean nothing (they may be infinite).
constexpr float kMild = 40.f;
__device__ __forceinline__ void diag_decay(float (&d)[4], bool mild, int t, int w, const double* G, const float* fk,
                                           const float* rowd, const float* cold) {
  if (mild) {
    const float a = rowd[t], b = rowd[t + 8];
    const float2 f = *reinterpret_cast<const float2*>(cold + w);
    d[0] = a * f.x, d[1] = a * f.y, d[2] = b * f.x, d[3] = b * f.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = fk[w + (i & 1)] * expf((float)(G[t + (i & 2) * 4] - G[w + (i & 1)]));
  }
}

// the n-tile of fragment i, three bits each
constexpr unsigned long long frag_rows() {
  unsigned long long v = 0;
  for (int j = 7; j >= 0; --j)
    for (int kk = j / 2; kk >= 0; --kk) v |= (unsigned long long)j << (3 * gd_frag(j, kk));
  return v;
}
constexpr unsigned long long kFragRow = frag_rows();

// For the chunk kernel, the sequences of `least` tokens and more as {first token, tokens, slot, number}, and entries without
// tokens up to `walkers`: by falling length and with their slots looked up (-1: takes no part) where there are no more than
// kGdOrdered of them in as many sequences, else the slot is kGdUnknown and each block of the walk looks; more than kGdOrdered come
// as they are.  One block does it: a scan over all lengths, and comparisons among the long ones alone, in shared memory (m: 2 kGdOrdered
// + 4 words).
constexpr int kGdOrdered = 512, kGdUnknown = -2;
__device__ __forceinline__ void gd_order(const GatedDeltaArgs& p, int4* walks, int walkers, int least, int* m, int tid) {
  int *const number = m, *const length = m + kGdOrdered, *const found = m + 2 * kGdOrdered;
  const int lane = tid & 31, wid = tid >> 5;
  auto put = [&](int place, int i) {
    int first, count;
    gd_range(p.cu, i, p.tokens, first, count);
    int slot = p.slots ? p.slots[i] : i;
    if (p.n_seq > kGdOrdered) {
      slot = kGdUnknown;
    } else if (p.slots) {
      bool mine = slot >= 0 && slot < p.n_slots;
      for (int j = 0; j < i; ++j) mine = mine && p.slots[j] != slot;
      if (!mine) slot = -1;
    }
    if (place < walkers) walks[place] = make_int4(first, count, slot, i);
  };
  int total = 0;
  for (int i0 = 0; i0 < p.n_seq; i0 += kPrepThreads) {
    int first, count = 0;
    if (i0 + tid < p.n_seq) gd_range(p.cu, i0 + tid, p.tokens, first, count);
    const bool in = count >= least;
    const unsigned all = __ballot_sync(0xffffffffu, in);
    if (lane == 0) found[wid] = __popc(all);
    __syncthreads();
    int place = total + __popc(all & ((1u << lane) - 1));
#pragma unroll
    for (int w = 0; w < kPrepThreads / 32; ++w) {
      if (w < wid) place += found[w];
      total += found[w];
    }
    if (in) {
      if (place < kGdOrdered) number[place] = i0 + tid, length[place] = count;
      else put(place, i0 + tid);
    }
    __syncthreads();
  }
  for (int e = tid; e < min(total, kGdOrdered); e += kPrepThreads) {
    int place = e;
    if (total <= kGdOrdered) {
      place = 0;
      for (int j = 0; j < total; ++j) place += length[j] > length[e] || (length[j] == length[e] && j < e);
    }
    put(place, number[e]);
  }
  for (int e = total + tid; e < walkers; e += kPrepThreads) walks[e] = make_int4(0, 0, -1, 0);
  __syncthreads();
}

// kq16: for bf16 inputs, the fp16 tiles K and Q [chunk][k_heads][2][64][DK] that the chunk kernel reads.  walks: NULL, or
// [walkers] entries to write (gd_order).
// Sequences of fewer than `least` tokens are not these kernels'.
template <typename T, int DK>
__global__ void __launch_bounds__(kPrepThreads, 4)
gated_delta_prep_kernel(const GatedDeltaArgs p, char* __restrict__ blocks, __half* __restrict__ kq16,
                        int4* __restrict__ walks, int groups, int per_group, int least, int walkers) {
  constexpr bool BF = !std::is_same<T, __half>::value;
  constexpr int UPR = DK / 8;  // 16-byte units per row
  extern __shared__ __align__(128) char smem[];
  __half* Ks = reinterpret_cast<__half*>(smem);
  __half* Qs = Ks + kGdC * DK;
  float* X = reinterpret_cast<float*>(smem);  // T, once K and Q have been multiplied
  float* L = reinterpret_cast<float*>(smem + gd_prep_tiles<DK>());  // [64][kLS]
  double* G = reinterpret_cast<double*>(L + kGdC * kLS);            // running log decay
  float* rk = reinterpret_cast<float*>(G + 64);                     // row factors of K and Q as staged
  float* rq = rk + 64;
  float* fk = rq + 64;      // rk beta
  float* rowf = fk + 64;    // e^(G_t - boundary before t's block)
  float* colf = rowf + 64;  // [3][64]: e^(boundary before block 1, 2, 3 - G_w) rk_w beta_w
  float* rowd = colf + 192;  // e^(G_t - last of t's block), where that is at most e^kMild
  float* cold = rowd + 64;   // e^(last of w's block - G_w) rk_w beta_w
  float* kst = cold + 64;    // norms of K's rows as staged
  float* knm = kst + 64;     // and as the products see them
  float* red = knm + 64;     // [4] max T, [4] row sums, [2] norms of keys, [2] max of the update's factors, [2] norms as staged
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, c = lane & 3;
  let_walk_start();
  const int rep = p.v_heads / p.k_heads;
  const int grp = blockIdx.x % groups, hk = (blockIdx.x / groups) % p.k_heads, num = blockIdx.x / (groups * p.k_heads);
  if (walks && blockIdx.x == 0) gd_order(p, walks, walkers, least, reinterpret_cast<int*>(smem), tid);
  // the sequence of chunk `num`: the last one whose first chunk is not behind it
  const bool by_rows = gd_by_rows(p.tokens, p.n_seq, least);
  int lo = 0, hi = p.n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (gd_chunk_base(min(max(p.cu[mid], 0), p.tokens), mid, by_rows, least) <= num) lo = mid;
    else hi = mid - 1;
  }
  int first, count;
  gd_range(p.cu, lo, p.tokens, first, count);
  const int cn = num - gd_chunk_base(first, lo, by_rows, least);
  if (cn < 0 || cn * kGdC >= count || count < least) return;
  first += cn * kGdC;
  count = min(count - cn * kGdC, kGdC);
  // K and Q rows as they are, then a thread per row (64 of K, 64 of Q) for its norm and, for bf16, its fp16 form
  const uint32_t ks = smem_u32(Ks), qs = smem_u32(Qs);
  for (int i = tid; i < kGdC * UPR; i += kPrepThreads) {
    const int t = i / UPR, u = i % UPR;
    const bool ok = t < count;
    const size_t r = (size_t)first + (ok ? t : 0);
    cp16(ks + kq_off<DK>(t, u), static_cast<const T*>(p.k) + r * p.ld_k + hk * DK + u * 8, ok);
    cp16(qs + kq_off<DK>(t, u), static_cast<const T*>(p.q) + r * p.ld_q + hk * DK + u * 8, ok);
  }
  cp_commit();
  cp_wait<0>();
  __syncthreads();
  {
    const int t = tid & 63;
    char* rowp = smem + (tid < 64 ? 0 : kGdC * DK * 2);
    float ss = 0.f, s1 = 0.f, mx = 0.f, staged;
#pragma unroll 4
    for (int u = 0; u < UPR; ++u) {
      const uint4 raw = *reinterpret_cast<const uint4*>(rowp + kq_off<DK>(t, u));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float x = to_f(e[j]), y = to_f(e[j + 1]);
        ss = fmaf(x, x, ss);
        s1 = fmaf(y, y, s1);
        if constexpr (BF) mx = fmaxf(mx, fmaxf(fabsf(x), fabsf(y)));
      }
    }
    ss += s1;
    float factor = p.qk_norm ? 1.0f / sqrtf(ss + kQkEps) : 1.0f;
    staged = sqrtf(ss);                       // the norm of the row in shared memory
    float kn = p.qk_norm ? 1.0f : staged;     // a bound of those that the products see
    const float seen = p.qk_norm ? fminf(staged * factor, 1.0f) : staged;
    if constexpr (BF) {
      float up, down;
      row_scale(mx, up, down);
      factor *= down;
      // within what the largest element allows: the sum of squares may have over- or underflowed
      staged = fminf(fmaxf(staged * up, mx * up), (DK == 128 ? 11.3137085f : 8.f) * (mx * up));
#pragma unroll 4
      for (int u = 0; u < UPR; ++u) {
        uint4* at = reinterpret_cast<uint4*>(rowp + kq_off<DK>(t, u));
        const uint4 raw = *at;
        const T* e = reinterpret_cast<const T*>(&raw);
        unsigned w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = h2_bits(__floats2half2_rn(to_f(e[2 * j]) * up, to_f(e[2 * j + 1]) * up));
        *at = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (tid < 64) {
      rk[t] = staged > 0.f ? factor : 0.f;  // a key of zeros adds nothing: its 1 / |k| is not to set the update's scale
      kst[t] = staged;
      knm[t] = seen;
      kn = warp_max(kn);
      staged = warp_max(staged);
      if (lane == 0) red[8 + wid] = kn, red[12 + wid] = staged;
    } else {
      rq[t] = factor;
    }
  }
  __syncthreads();
  if (BF && grp == 0) {
    __half* dst = kq16 + ((size_t)num * p.k_heads + hk) * 2 * kGdC * DK;
    for (int i = tid; i < 2 * kGdC * UPR; i += kPrepThreads) {
      const int t = i / UPR, u = i % UPR;  // rows 64.. are Q's: its tile follows K's here too
      *reinterpret_cast<uint4*>(dst + (size_t)i * 8) = *reinterpret_cast<const uint4*>(smem + (t >> 6) * kGdC * DK * 2 + kq_off<DK>(t & 63, u));
    }
  }
  // Q K^T rows 16 wid.. and K K^T rows 16 (3 - wid)..: ten 16 x 8 tiles for every warp
  const int mk = 3 - wid;
  float qk[8][4], kk_[8][4];
  {
    auto gram = [&](uint32_t a_tile, int mt, float (&acc)[8][4]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DK / 16; ++kk) {
        unsigned a[4];
        ldsm4(a, a_tile + kq_off<DK>(16 * mt + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
        for (int jp = 0; jp < 4; ++jp) {
          if (jp <= mt) {
            unsigned b[4];
            ldsm4(b, ks + kq_off<DK>(16 * jp + ((lane >> 4) << 3) + (lane & 7), 2 * kk + ((lane >> 3) & 1)));
            mma_acc(acc[2 * jp], a, b[0], b[1]);
            mma_acc(acc[2 * jp + 1], a, b[2], b[3]);
          }
        }
      }
    };
    gram(qs, wid, qk);
    gram(ks, mk, kk_);
  }
  __syncthreads();
  for (int i = tid; i < 512 / 4; i += kPrepThreads) {  // the two blocks of T above the diagonal that are read below
    const int o = 32 * (i >> 6), r = (i & 63) >> 2, w = (i & 3) * 4;
    *reinterpret_cast<float4*>(X + (o + r) * kLS + o + 16 + w) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int h1 = min(hk * rep + (grp + 1) * per_group, (hk + 1) * rep);
  for (int h = hk * rep + grp * per_group; h < h1; ++h) {
    // gates: one thread per token, the running sum in double precision
    if (tid < 64) {
      double gl = 0.0;
      float bt = 0.f;
      if (tid < count) {
        gl = gd_log_decay(to_f(static_cast<const T*>(p.a)[(size_t)(first + tid) * p.ld_a + h]), p.dt_bias[h], p.A_log[h]);
        bt = gd_beta(to_f(static_cast<const T*>(p.b)[(size_t)(first + tid) * p.ld_b + h]));
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, gl, o);
        if (lane >= o) gl += x;
      }
      G[tid] = gl;
      fk[tid] = rk[tid] * bt;
    }
    __syncthreads();
    if (tid >= 32 && tid < 64) G[tid] += G[31];
    __syncthreads();
    char* blk = blocks + ((size_t)num * p.v_heads + h) * kGdBlock;
    float* vec = reinterpret_cast<float*>(blk + 2 * kGdTri);
    {
      const int t = tid & 63;
      const double Gt = G[t], Ge = G[t | 15];  // of the token, and of the last in its block of 16
      if (tid < 64) {  // factors of the chunk kernel
        const float eg = expf((float)Gt), c2 = expf((float)(G[63] - Gt)) * fk[t];
        vec[kGdBk + t] = -eg * rk[t];
        vec[kGdOq + t] = p.scale * eg * rq[t];
        if (t == 0) vec[kGdLast] = expf((float)G[63]), vec[kGdKn] = fmaxf(red[8], red[9]);
        const float m = warp_max(fabsf(c2));
        if (lane == 0) red[10 + wid] = m;
        colf[128 + t] = c2;  // kept here until both warps' largest is known; e^(boundary 3 - G) follows
        rowd[t] = expf(fminf((float)(Gt - Ge), kMild));
      } else {  // factors of this one
        if (t >= 16) rowf[t] = expf((float)(Gt - G[(t & ~15) - 1]));
        if (t < 16) colf[t] = expf((float)(G[15] - Gt)) * fk[t];
        if (t < 32) colf[64 + t] = expf((float)(G[31] - Gt)) * fk[t];
        cold[t] = expf((float)(Ge - Gt)) * fk[t];
      }
      __syncthreads();
      if (tid < 64) {
        float up, down;
        const float c2max = fmaxf(red[10], red[11]);
        row_scale(c2max, up, down);
        vec[kGdC2 + t] = colf[128 + t] * (up * 0x1p-14f);
        const float kmax = fmaxf(red[12], red[13]);
        float kup, kdown;
        row_scale(kmax, kup, kdown);
        reinterpret_cast<T*>(vec + kGdWeights)[t] = from_f<T>((colf[128 + t] * (up * 0x1p-14f)) * (kst[t] * (kup * 0x1p-14f)));
        reinterpret_cast<T*>(vec + kGdNorms)[t] = from_f<T>(knm[t]);
        if (t == 0) vec[kGdCdn] = down * 0x1p14f, vec[kGdWm] = c2max * kmax;
        if (t < 48) colf[128 + t] = expf((float)(G[47] - Gt)) * fk[t];
      }
    }
    __syncthreads();
    // P: rows ta, tb of Q K^T
    {
      const int ta = 16 * wid + g, tb = ta + 8;
      const float ra = p.scale * rq[ta], rb = p.scale * rq[tb];
      float x[8][4], ma = 0.f, mb = 0.f;
      if (wid > 0) {
        const float fa = ra * rowf[ta], fb = rb * rowf[tb];
        const float* cf = colf + 64 * (wid - 1) + 2 * c;
#pragma unroll
        for (int j = 0; j < 6; ++j) {
          if (j < 2 * wid) {
            const float2 f = *reinterpret_cast<const float2*>(cf + 8 * j);
            x[j][0] = qk[j][0] * fa * f.x;
            x[j][1] = qk[j][1] * fa * f.y;
            x[j][2] = qk[j][2] * fb * f.x;
            x[j][3] = qk[j][3] * fb * f.y;
            ma = fmaxf(ma, fmaxf(fabsf(x[j][0]), fabsf(x[j][1])));
            mb = fmaxf(mb, fmaxf(fabsf(x[j][2]), fabsf(x[j][3])));
          }
        }
      }
      const bool mild = G[16 * wid] - G[16 * wid + 15] <= (double)kMild;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j == 2 * wid || j == 2 * wid + 1) {
          float d[4];
          diag_decay(d, mild, ta, 8 * j + 2 * c, G, fk, rowd, cold);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int w = 8 * j + 2 * c + i;
            x[j][i] = w <= ta ? qk[j][i] * ra * d[i] : 0.f;
            x[j][2 + i] = w <= tb ? qk[j][2 + i] * rb * d[2 + i] : 0.f;
            ma = fmaxf(ma, fabsf(x[j][i]));
            mb = fmaxf(mb, fabsf(x[j][2 + i]));
          }
        }
      }
      float ua, da, ub, db;
      row_scale(quad_max(ma), ua, da);
      row_scale(quad_max(mb), ub, db);
      if (c == 0) {
        vec[kGdOp + ta] = da;
        vec[kGdOp + tb] = db;
      }
      uint4* P = reinterpret_cast<uint4*>(blk + kGdTri);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        if (kk <= wid) {
          unsigned ha0, la0, ha1, la1, hb0, lb0, hb1, lb1;
          split2(x[2 * kk][0] * ua, x[2 * kk][1] * ua, ha0, la0);
          split2(x[2 * kk + 1][0] * ua, x[2 * kk + 1][1] * ua, ha1, la1);
          split2(x[2 * kk][2] * ub, x[2 * kk][3] * ub, hb0, lb0);
          split2(x[2 * kk + 1][2] * ub, x[2 * kk + 1][3] * ub, hb1, lb1);
          P[gd_frag(2 * wid, kk) * 32 + lane] = make_uint4(ha0, ha1, la0, la1);
          P[gd_frag(2 * wid + 1, kk) * 32 + lane] = make_uint4(hb0, hb1, lb0, lb1);
        }
      }
    }
    // L: rows of K K^T
    {
      const int ta = 16 * mk + g, tb = ta + 8;
      const float ra = rk[ta], rb = rk[tb];
      if (mk > 0) {
        const float fa = ra * rowf[ta], fb = rb * rowf[tb];
        const float* cf = colf + 64 * (mk - 1) + 2 * c;
#pragma unroll
        for (int j = 0; j < 6; ++j) {
          if (j < 2 * mk) {
            const float2 f = *reinterpret_cast<const float2*>(cf + 8 * j);
            *reinterpret_cast<float2*>(L + ta * kLS + 8 * j + 2 * c) = make_float2(kk_[j][0] * fa * f.x, kk_[j][1] * fa * f.y);
            *reinterpret_cast<float2*>(L + tb * kLS + 8 * j + 2 * c) = make_float2(kk_[j][2] * fb * f.x, kk_[j][3] * fb * f.y);
          }
        }
      }
      const bool mild = G[16 * mk] - G[16 * mk + 15] <= (double)kMild;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j == 2 * mk || j == 2 * mk + 1) {
          const int w = 8 * j + 2 * c;  // only what is left of the diagonal is read
          float d[4];
          diag_decay(d, mild, ta, w, G, fk, rowd, cold);
          *reinterpret_cast<float2*>(L + ta * kLS + w) = make_float2(kk_[j][0] * ra * d[0], kk_[j][1] * ra * d[1]);
          *reinterpret_cast<float2*>(L + tb * kLS + w) = make_float2(kk_[j][2] * rb * d[2], kk_[j][3] * rb * d[3]);
        }
      }
      __syncwarp();
      // the diagonal block of these rows: a lane per column of its inverse
      if (lane < 16) {
        const float* Lb = L + 16 * mk * kLS + 16 * mk;
        float* Xb = X + 16 * mk * kLS + 16 * mk + lane;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float l[16];
#pragma unroll
          for (int m = 0; m < i; m += 4) *reinterpret_cast<float4*>(l + m) = *reinterpret_cast<const float4*>(Lb + i * kLS + m);
          float s0 = i == lane ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
          for (int m = 0; m < i; ++m) {
            if (m & 1) s1 = fmaf(-l[m], y[m], s1);
            else s0 = fmaf(-l[m], y[m], s0);
          }
          y[i] = s0 + s1;
          Xb[i * kLS] = y[i];
        }
      }
    }
    __syncthreads();
    corner<16>(L, X, 32 * (wid >> 1), wid & 1, 0, lane);  // of the two 32 x 32 blocks
    __syncthreads();
    corner<32>(L, X, 0, wid >> 1, wid & 1, lane);
    __syncthreads();
    {  // the scale of T and its largest row sum
      const int t = tid >> 1, half = tid & 1;
      float m = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 32; w += 4) {
        if (32 * half + w <= t) {
          const float4 x = *reinterpret_cast<const float4*>(X + t * kLS + 32 * half + w);
          m = fmaxf(m, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
          sum += (fabsf(x.x) + fabsf(x.y)) + (fabsf(x.z) + fabsf(x.w));
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      m = warp_max_nonneg(m);
      sum = warp_max_nonneg(sum);
      if (lane == 0) red[wid] = m, red[4 + wid] = sum;
    }
    __syncthreads();
    float t_up, t_down;
    row_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), t_up, t_down);
    if (tid == 0) {
      vec[kGdTdn] = t_down;
      vec[kGdTsum] = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
    }
#pragma unroll
    for (int f = 0; f < kGdFrags / 4; ++f) {  // fragment 4 f + wid
      const int id = 4 * f + wid;
      const int j = (int)(kFragRow >> (3 * id)) & 7, kk = id - gd_frag(j, 0);
      const float* x = X + (8 * j + g) * kLS + 16 * kk + 2 * c;
      unsigned h0, l0, h1, l1;
      split2(mul2(*reinterpret_cast<const float2*>(x), dup(t_up)), h0, l0);
      split2(mul2(*reinterpret_cast<const float2*>(x + 8), dup(t_up)), h1, l1);
      reinterpret_cast<uint4*>(blk)[id * 32 + lane] = make_uint4(h0, h1, l0, l1);
    }
    // the next head's gates touch nothing that is still read: G and the factors were last used before
    // the barriers above
  }
}

// ------------------------------------------------------------------ the walk over a sequence's chunks
//
// A block owns 32 rows of one head's state, two groups of 16, and has eight warps.  Each group has two chain warps, which
// hold S^T as MMA accumulators, half of the dk columns each, and compute what the next chunk waits for: S k, r, u,
// the new S; and two output warps, which take the operands that the chain warps have split anyway (S and u as
// fp16 pairs, through shared memory), compute S q + u P^T and the rows of o, half of the tokens each, and fetch the next
// chunk (cp.async).  All products are taken transposed, with S, r and u as left operands: the accumulator layout of
// one product is the left operand's layout of the next.
//   S k, S q : [16 x dk] [dk x 64]     u = r T^T, u P^T : [16 x 64] [64 x 64]     u k : [16 x 64] [64 x dk]
// Between its two warps a chain passes, per chunk: half of each one's partial S k (A keeps tokens 0-31, B 32-63), A's r (B's
// u needs it), and both halves of the weighed u.  The splits of one product's operands are written among the MMAs of
// its earlier steps, so that a warp keeps its tensor core busy.
//
// K is double buffered, and Q, V, T, P and the factors are replaced as soon as they have been read, so that two blocks
// fit on an SM.  DEEP, for grids that give every block an SM of its own, has two of all of them and fetches a chunk ahead.
//
// Bound: per chunk and group, at dk = 128, 504 MMAs of 8 cycles (mma.sync runs 1024 multiply-adds per cycle and SM) and
// about 160 KB through shared memory, in a chain of dependent steps.  Alone on its SM a block takes 2.2 us a chunk
// (512 chunks of 32 heads, 128 blocks, in 1.12 ms; tensor cores 51% busy; one chain warp per group: 2.35 us where two took
// 2.1); two blocks on an SM take 4.1 us for a chunk each (tensor cores 51%, shared memory 69% busy).

constexpr int kGdGroups = 2;  // of 16 rows per block

// Where a chunk's values lie far apart, its pairs are not enough: what is 2^-38 of the row's bound or less is lost in r and
// u, and it may be all that matters, where a gate has forgotten the large values (of the chunk, or of the state before it)
// or where they come later.  Such a chunk is taken token by token in fp32 by the group's chain warps (gd_by_token).
// With U the bound of |u|, a row is safe where
//   - at every token, what the row holds (the largest of the state's elements and of beta |v| |k| so far, each decayed
//     since) is 2^-22 U times the largest weight, beta |k| decayed alike, that a token has in o, which is the scale of P's
//     row, or more: o is then off by some 2^-17 of what it could be; and
//   - at the end, the largest beta e^(G_C - G) |v| is 2^-17 U times the largest weight or more, or the largest of e^G_C S 2^-14:
//     what 64 tokens add to the row is off by some 2^-35 U times that weight.
// The output warps find the least |v| and the largest weighed one; the decays between are looked at only where some |v| is
// below 2^-22 U (else what is held cannot be either) and e^G_C S is too, which chance does to one chunk in 1000 or fewer.
// Looking costs 4 to 8% of a call (64 prompts of 64 tokens, 64 heads: 255 us, 235 without; 32768 tokens: 1.44 ms, 1.38), looking at
// the decays 2 us, a chunk token by token 25 us, 2 to 4 otherwise.
constexpr float kGdRangeO = 0x1p-22f, kGdRangeV = 0x1p-17f, kGdRangeS = 0x1p-14f;
constexpr int kGdOfV = 80, kGdByToken = 144;  // places among a group's scales

template <int DK>
__host__ __device__ constexpr int gd_exchange() { return DK / 16 * 1024 + 4096 + 4096 + 2048 + 640; }
template <int DK, bool DEEP>
__host__ __device__ constexpr int gd_chunk_smem() {
  return (DEEP ? 4 : 3) * kGdC * DK * 2 + (DEEP ? 2 : 1) * (kGdC * 32 * kGdGroups + kGdBlock) + kGdGroups * gd_exchange<DK>();
}

// Byte offset of 16-byte unit u of token t in the V tile [64][32]: two rows per 128 bytes, the units of four
// neighbouring pairs of rows permuted.
__device__ __forceinline__ uint32_t v_off(int t, int u) { return (uint32_t)(t * 64 + ((u ^ ((t >> 1) & 3)) << 4)); }
// Named barriers: 0 the block, 1 the output warps, 2 + 5 group + {0: the chain's two warps, 1: A's r is split, 2: S is
// split, 3: u is split, 4: S and u have been taken}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// x[i] += rows of (ah + al)[kk - K0] times the 64 x 64 triangular matrix in fragment order, for n-tiles J0 + i and the
// k-steps K0 .. K1 - 1 that they have
template <int J0, int K0, int K1, int NA>
__device__ __forceinline__ void tri_product(float (&x)[4][4], const unsigned (&ah)[NA][4], const unsigned (&al)[NA][4],
                                            const uint4* F) {
#pragma unroll
  for (int kk = K0; kk < K1; ++kk) {
    uint4 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (kk <= (J0 + i) / 2) b[i] = F[gd_frag(J0 + i, kk) * 32];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (kk <= (J0 + i) / 2) mma_acc(x[i], ah[kk - K0], b[i].z, b[i].w);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (kk <= (J0 + i) / 2) mma_acc(x[i], al[kk - K0], b[i].x, b[i].y);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (kk <= (J0 + i) / 2) mma_acc(x[i], ah[kk - K0], b[i].x, b[i].y);
  }
}
// One k-step's left operand from two neighbouring accumulator tiles, rows scaled by f0 (rows g) and f1 (g + 8).
__device__ __forceinline__ void split_tile(const float (&x)[4], const float (&y)[4], float f0, float f1, unsigned (&ah)[4],
                                           unsigned (&al)[4]) {
  split2(mul2(make_float2(x[0], x[1]), dup(f0)), ah[0], al[0]);
  split2(mul2(make_float2(x[2], x[3]), dup(f1)), ah[1], al[1]);
  split2(mul2(make_float2(y[0], y[1]), dup(f0)), ah[2], al[2]);
  split2(mul2(make_float2(y[2], y[3]), dup(f1)), ah[3], al[3]);
}
__device__ __forceinline__ void put_frag(uint4* to, const unsigned (&h)[4], const unsigned (&l)[4]) {
  to[0] = make_uint4(h[0], h[1], h[2], h[3]);
  to[32] = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void get_frag(const uint4* from, unsigned (&h)[4], unsigned (&l)[4]) {
  const uint4 a = from[0], b = from[32];
  h[0] = a.x, h[1] = a.y, h[2] = a.z, h[3] = a.w;
  l[0] = b.x, l[1] = b.y, l[2] = b.z, l[3] = b.w;
}
template <typename T>
struct PairOf;
template <>
struct PairOf<__half> {
  using type = __half2;
  static __device__ __forceinline__ float2 floats(__half2 x) { return __half22float2(x); }
};
template <>
struct PairOf<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ float2 floats(__nv_bfloat162 x) { return __bfloat1622float2(x); }
};
template <typename T>
__device__ __forceinline__ typename PairOf<T>::type as_pair(unsigned u) { return *reinterpret_cast<typename PairOf<T>::type*>(&u); }
template <typename P>
__device__ __forceinline__ unsigned pair_bits(P x) { return *reinterpret_cast<unsigned*>(&x); }

// Whether one of a group's rows comes to a token where it holds something, but less than w0 (rows g; w1: rows g + 8) times the
// largest weight.  m0, m1: the largest of the rows' state; v: the chunk's tile; norms: of its keys.
template <typename T>
__device__ __forceinline__ bool gd_forgets(const GatedDeltaArgs& p, const char* v, const T* norms, int group, int first, int n, int h, float m0,
                                           float m1, float w0, float w1) {
  const int lane = threadIdx.x & 31, g = lane >> 2;
  float weight = 0.f;
  bool bad = false;
#pragma unroll 1
  for (int t0 = 0; t0 < n; t0 += 32) {
    const size_t at = (size_t)first + min(t0 + lane, n - 1);  // the gates of 32 tokens, one per lane
    float keep = expf(gd_log_decay(to_f(static_cast<const T*>(p.a)[at * p.ld_a + h]), p.dt_bias[h], p.A_log[h]));
    float beta = gd_beta(to_f(static_cast<const T*>(p.b)[at * p.ld_b + h]));
    beta *= to_f(norms[t0 + lane]);
    if (t0 + lane >= n) keep = 1.f, beta = 0.f;
#pragma unroll 4
    for (int i = 0; i < 32; ++i) {
      const float e = __shfl_sync(0xffffffffu, keep, i), b = __shfl_sync(0xffffffffu, beta, i);
      const float x = fabsf(to_f(reinterpret_cast<const T*>(v + v_off(t0 + i, 2 * group))[g]));  // 0 behind the last token
      const float y = fabsf(to_f(reinterpret_cast<const T*>(v + v_off(t0 + i, 2 * group + 1))[g]));
      m0 = fmaxf(e * m0, b * x), m1 = fmaxf(e * m1, b * y), weight = fmaxf(e * weight, b);
      bad |= (m0 < w0 * weight && m0 != 0.f) || (m1 < w1 * weight && m1 != 0.f);
    }
  }
  return __any_sync(0xffffffffu, bad);
}

// The n tokens of a chunk one after the other, from the call's own arrays, for chunks whose values lie too far apart for
// pairs; first the gates, norms and k.q of all of them, a lane each (25 us a chunk; 85 with these in the tokens' turns).  s: the
// state as the chain warps hold it, s[j] the rows `row` and row + 8, columns half * DK / 2 + 8 j + 2 (lane % 4) +
// {0, 1}; the rows' sums pass between the two warps through ex (112 float4).
template <typename T, int DK>
__device__ __noinline__ void gd_by_token(const GatedDeltaArgs& p, float (&s)[DK / 16][4], int first, int n, int h, int hk, int row,
                                         int half, int bar, float4* ex) {
  constexpr int NH = DK / 16;
  using T2 = typename PairOf<T>::type;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  float4* const gates = ex + 32;                            // per token: e^g, beta and the factors of k and q
  float* const kqs = reinterpret_cast<float*>(ex + 96);     // and k.q
  if (const int t = 32 * half + lane; t < n) {  // a lane per token
    const size_t at = (size_t)first + t;
    const uint4* kp = reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + at * p.ld_k + hk * DK);
    const uint4* qp = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + at * p.ld_q + hk * DK);
    float kk[2] = {}, qq[2] = {}, kq[2] = {};
#pragma unroll 4
    for (int u = 0; u < DK / 8; ++u) {
      const uint4 x = kp[u], y = qp[u];
      const T *e = reinterpret_cast<const T*>(&x), *f = reinterpret_cast<const T*>(&y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float k = to_f(e[j]), q = to_f(f[j]);
        kk[j & 1] = fmaf(k, k, kk[j & 1]), qq[j & 1] = fmaf(q, q, qq[j & 1]), kq[j & 1] = fmaf(k, q, kq[j & 1]);
      }
    }
    const float rk = p.qk_norm ? 1.0f / sqrtf(kk[0] + kk[1] + kQkEps) : 1.0f, rq = p.qk_norm ? 1.0f / sqrtf(qq[0] + qq[1] + kQkEps) : 1.0f;
    gates[t] = make_float4(expf(gd_log_decay(to_f(static_cast<const T*>(p.a)[at * p.ld_a + h]), p.dt_bias[h], p.A_log[h])),
                           gd_beta(to_f(static_cast<const T*>(p.b)[at * p.ld_b + h])), rk, rq);
    kqs[t] = unit_dot(kq[0] + kq[1], rk * rq);
  }
  bar_sync(bar, 64);
  auto quad_sum = [](float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
  };
  const T* kp = static_cast<const T*>(p.k) + (size_t)first * p.ld_k + hk * DK + half * (DK / 2) + 2 * c;
  const T* qp = static_cast<const T*>(p.q) + (size_t)first * p.ld_q + hk * DK + half * (DK / 2) + 2 * c;
  const T* vp = static_cast<const T*>(p.v) + (size_t)first * p.ld_v + h * p.dv + row;
  T* op = static_cast<T*>(p.o) + (size_t)first * p.ld_o + h * p.dv + row;
#pragma unroll 1
  for (int t = 0; t < n; ++t, kp += p.ld_k, qp += p.ld_q, vp += p.ld_v, op += p.ld_o) {
    const float v0 = to_f(vp[0]), v1 = to_f(vp[8]);
    const float4 gate = gates[t];
    const float eg = gate.x, beta = gate.y, kq = kqs[t];
    float k[NH][2], q[NH][2];
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      const T2 x = *reinterpret_cast<const T2*>(kp + 8 * j), y = *reinterpret_cast<const T2*>(qp + 8 * j);
      k[j][0] = to_f(x.x) * gate.z, k[j][1] = to_f(x.y) * gate.z, q[j][0] = to_f(y.x) * gate.w, q[j][1] = to_f(y.y) * gate.w;
    }
    float4 sums = make_float4(0.f, 0.f, 0.f, 0.f);  // S k of the two rows, S q
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      sums.x = fmaf(s[j][0], k[j][0], fmaf(s[j][1], k[j][1], sums.x));
      sums.y = fmaf(s[j][2], k[j][0], fmaf(s[j][3], k[j][1], sums.y));
      sums.z = fmaf(s[j][0], q[j][0], fmaf(s[j][1], q[j][1], sums.z));
      sums.w = fmaf(s[j][2], q[j][0], fmaf(s[j][3], q[j][1], sums.w));
    }
    sums = make_float4(quad_sum(sums.x), quad_sum(sums.y), quad_sum(sums.z), quad_sum(sums.w));
    float4* const mail = ex + 16 * (t & 1);  // two, in turn: the other warp has read the one before the last
    if (c == 0) mail[8 * half + g] = sums;
    bar_sync(bar, 64);
    const float4 other = mail[8 * (1 - half) + g];
    const float u0 = beta * (v0 - eg * (sums.x + other.x)), u1 = beta * (v1 - eg * (sums.y + other.y));
    if (half == 0 && c == 0) {
      op[0] = from_f<T>(p.scale * fmaf(kq, u0, eg * (sums.z + other.z)));
      op[8] = from_f<T>(p.scale * fmaf(kq, u1, eg * (sums.w + other.w)));
    }
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      s[j][0] = fmaf(u0, k[j][0], eg * s[j][0]);
      s[j][1] = fmaf(u0, k[j][1], eg * s[j][1]);
      s[j][2] = fmaf(u1, k[j][0], eg * s[j][2]);
      s[j][3] = fmaf(u1, k[j][1], eg * s[j][3]);
    }
  }
}

// kq16: the fp16 tiles of K and Q for bf16 inputs; for fp16 inputs the tiles are rows of k and q themselves.
template <typename T, int DK, bool DEEP>
__global__ void __launch_bounds__(128 * kGdGroups, DEEP ? 1 : 2)
gated_delta_chunk_kernel(const __grid_constant__ GatedDeltaArgs p, const char* __restrict__ blocks, const __half* __restrict__ kq16,
                         const int4* __restrict__ walks, int parts, int slots_total, int least) {
  constexpr bool BF = !std::is_same<T, __half>::value;
  constexpr int NT = 128 * kGdGroups, NL = NT / 2, UPR = DK / 8;
  constexpr int NH = DK / 16, KH = DK / 32;  // n-tiles and k-steps of a chain warp's half of dk
  constexpr int TILE = kGdC * DK * 2;
  constexpr int V_AT = (DEEP ? 4 : 3) * TILE, B_AT = V_AT + kGdC * 32 * kGdGroups;  // K, K, Q (DEEP: twice), V, {T, P, factors}
  constexpr int STAGE = kGdC * 32 * kGdGroups + kGdBlock;                            // V and the rest (DEEP: two of them)
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, c = lane & 3;
  const int part = blockIdx.x % parts, h = (blockIdx.x / parts) % p.v_heads, nth = blockIdx.x / (parts * p.v_heads);
  int first, count, slot, seq;
  if (walks) {
    prep_done();
    const int4 w = walks[nth];
    first = w.x, count = w.y, slot = w.z, seq = w.w;
    if (slot == kGdUnknown) slot = gd_slot(p.slots, seq, p.n_slots, tid, NT);
  } else {
    seq = nth;
    gd_range(p.cu, seq, p.tokens, first, count);
    slot = gd_slot(p.slots, seq, p.n_slots, tid, NT);
  }
  if (slot < 0 || count < least) {
    prep_done();  // no block ends before the kernel ahead has
    return;
  }
  const int base = gd_chunk_base(first, seq, gd_by_rows(p.tokens, p.n_seq, least), least);
  const int chunks = min((count + kGdC - 1) / kGdC, slots_total - base);
  const int hk = h / (p.v_heads / p.k_heads);
  // Warps 0-3 are the chains', 4-7 the output warps'; w and w + 4 share a scheduler, a chain's B warp (more of u) with an
  // output warp of the first half (less of u P^T).
  const bool chain = wid < 2 * kGdGroups;
  const int group = (wid >> 1) % kGdGroups, half = chain ? wid & 1 : 1 - (wid & 1);
  const int dv0 = part * 16 * kGdGroups, row0 = dv0 + 16 * group;
  const bool active = row0 < p.dv;  // dv is a multiple of 16: a group's rows are all there or none
  char* ex = smem + V_AT + (DEEP ? 2 : 1) * STAGE + group * gd_exchange<DK>();
  uint4* s_ex = reinterpret_cast<uint4*>(ex) + lane;     // S: [dk / 16][hi, lo][32]
  uint4* u_ex = s_ex + DK / 16 * 64;                     // u: [4][hi, lo][32]
  uint4* d_ex = u_ex + 4 * 64;                           // weighed u, the same; before it, partial S k [A, B][4][32]
  uint4* r_ex = d_ex + 4 * 64;                           // A's r: [2][hi, lo][32]
  // [16] each: scale of S (A, B), max of S (A, B), scale of u; of v [2][8][4]: the largest, the least and the largest weighed
  // magnitudes of rows g and g + 8, as pairs, over either half of the tokens; whether the chunk goes token by token
  float* sc = reinterpret_cast<float*>(r_ex - lane + 2 * 64);
  const int bar = 2 + 5 * group;
  // lane parts of the ldmatrix addresses
  const int bt = ((lane >> 4) << 3) + (lane & 7), bu = (lane >> 3) & 1;  // B from [token][dk] rows, two n-tiles
  const int tt = (((lane >> 3) & 1) << 3) + (lane & 7), tu = lane >> 4;  // the same, transposed

  if (!chain) {
    // ---------------------------------------------------------------- output warp, tokens 32 half ..
    // A lane copies one 16-byte column of every RP-th row (K, Q), so that a copy costs a pointer step; rows past
    // the sequence's end are zeros.
    const int lt = tid - NT / 2;
    constexpr int RP = NL / UPR;  // rows per pass, a multiple of 8
    const uint32_t sm0 = smem_u32(smem);
    const int kt = lt / UPR, ku = lt % UPR;
    const uint32_t off = kq_off<DK>(kt, ku);
    auto load_tile = [&](int ch, uint32_t dst, const void* rows, int ld, int which) {  // K (0) or Q (1) of chunk ch
      const int n = count - ch * kGdC;
      const __half* src;
      size_t step;
      if constexpr (BF) {
        src = kq16 + ((((size_t)(base + ch) * p.k_heads + hk) * 2 + which) * kGdC + kt) * DK + ku * 8;
        step = RP * DK;
      } else {
        src = static_cast<const __half*>(rows) + ((size_t)first + (size_t)ch * kGdC + kt) * ld + hk * DK + ku * 8;
        step = (size_t)RP * ld;
      }
      if (BF || n >= kGdC) {
#pragma unroll
        for (int i = 0; i < kGdC / RP; ++i, src += step) cp16(dst + i * (RP * DK * 2) + off, src, true);
      } else {
        for (int i = 0; i < kGdC / RP; ++i, src += step) {
          const bool ok = kt + i * RP < n;
          cp16(dst + i * (RP * DK * 2) + off, ok ? src : static_cast<const __half*>(rows), ok);
        }
      }
    };
    auto load_k = [&](int ch) { load_tile(ch, sm0 + (ch & 1) * TILE, p.k, p.ld_k, 0); };
    auto load_q = [&](int ch) { load_tile(ch, sm0 + (2 + (DEEP ? ch & 1 : 0)) * TILE, p.q, p.ld_q, 1); };
    const int vu = lt & 3, vt = lt >> 2;  // 32 rows of V per pass
    const bool v_there = dv0 + vu * 8 < p.dv;
    auto load_vb = [&](int ch) {  // V, T, P and the factors of chunk ch
      const int n = count - ch * kGdC, stage = DEEP ? (ch & 1) * STAGE : 0;
      const T* src = static_cast<const T*>(p.v) + ((size_t)first + (size_t)ch * kGdC + vt) * p.ld_v + h * p.dv + dv0 + vu * 8;
#pragma unroll
      for (int i = 0; i < 2; ++i, src += (size_t)32 * p.ld_v) {
        const bool ok = v_there && vt + 32 * i < n;
        cp16(sm0 + V_AT + stage + v_off(vt + 32 * i, vu), ok ? src : static_cast<const T*>(p.v), ok);
      }
      const char* blk = blocks + ((size_t)(base + ch) * p.v_heads + h) * kGdBlock + lt * 16;
      const uint32_t dst = sm0 + B_AT + stage + lt * 16;
#pragma unroll
      for (int i = 0; i < kGdBlock / 16 / NL; ++i) cp16(dst + i * NL * 16, blk + i * NL * 16, true);
      constexpr int REST = kGdBlock / 16 % NL;
      if (lt < REST) cp16(dst + kGdBlock / 16 / NL * NL * 16, blk + kGdBlock / 16 / NL * NL * 16, true);
    };
    // |v| of each row over this half of chunk ch, for the chain's bound of r and for what it asks of the chunk
    auto sizes_of_v = [&](int ch) {
      const char* stage = smem + (DEEP ? (ch & 1) * STAGE : 0);
      const T* weights = reinterpret_cast<const T*>(stage + B_AT + 2 * kGdTri + 4 * kGdWeights) + 32 * half + 2 * c;
      const int n = count - ch * kGdC - 32 * half - 2 * c;
      using P = PairOf<T>;
      typename P::type most[2], least[2], weighed[2];  // of rows g, g + 8
      most[0] = most[1] = weighed[0] = weighed[1] = as_pair<T>(0u);
      least[0] = least[1] = as_pair<T>(0x7fff7fffu);  // no number: the others stay
#pragma unroll
      for (int jp = 0; jp < 2; ++jp) {
        unsigned v[4];  // {t, rows 0-7}, {t + 8, ..}, {t, rows 8-15}, {t + 8, ..}
        ldsm4t(v, smem_u32(stage) + V_AT + v_off(32 * half + 16 * jp + tt, 2 * group + tu));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = 16 * jp + 8 * i;
          const typename P::type f = *reinterpret_cast<const typename P::type*>(weights + t);
          const unsigned behind = (t < n ? 0u : 0x7fffu) | (t + 1 < n ? 0u : 0x7fff0000u);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const typename P::type x = __habs2(as_pair<T>(v[2 * r + i]));
            most[r] = __hmax2(most[r], x);
            least[r] = __hmin2(least[r], as_pair<T>(pair_bits(x) | behind));
            weighed[r] = __hmax2(weighed[r], __habs2(__hmul2(x, f)));
          }
        }
      }
      auto across = [&](typename P::type (&x)[2], auto op) {  // rows g and g + 8 of a pair, over the quad
        unsigned w = pair_bits(op(as_pair<T>(__byte_perm(pair_bits(x[0]), pair_bits(x[1]), 0x5410)),
                                  as_pair<T>(__byte_perm(pair_bits(x[0]), pair_bits(x[1]), 0x7632))));
        w = pair_bits(op(as_pair<T>(w), as_pair<T>(__shfl_xor_sync(0xffffffffu, w, 1))));
        return pair_bits(op(as_pair<T>(w), as_pair<T>(__shfl_xor_sync(0xffffffffu, w, 2))));
      };
      auto larger = [](typename P::type x, typename P::type y) { return __hmax2(x, y); };
      auto smaller = [](typename P::type x, typename P::type y) { return __hmin2(x, y); };
      const uint4 all = make_uint4(across(most, larger), across(least, smaller), across(weighed, larger), 0u);
      if (c == 0) reinterpret_cast<uint4*>(sc + kGdOfV)[8 * half + g] = all;
    };
    if (BF) prep_done();
    load_k(0);
    load_q(0);
    if (!DEEP) cp_commit();
    if (!BF) prep_done();
    load_vb(0);
    cp_commit();
    if constexpr (DEEP) {
      cp_wait<0>();
      bar_sync(1, NL);
      sizes_of_v(0);
      bar_arrive(0, NT);  // the chunk is there
    }
    for (int ch = 0; ch < chunks; ++ch) {
      const bool more = ch + 1 < chunks;
      const char* st = smem + (DEEP ? (ch & 1) * STAGE : 0);
      const uint32_t v_s = smem_u32(st) + V_AT, q_s = sm0 + (2 + (DEEP ? ch & 1 : 0)) * TILE;
      const float* vec = reinterpret_cast<const float*>(st + B_AT + 2 * kGdTri);
      if constexpr (DEEP) {
        bar_sync(bar + 2, 128);  // S is split
        bar_sync(1, NL);         // every chain is past the last chunk, and so are the output warps: the other stage is free
        if (more) load_k(ch + 1), load_q(ch + 1), load_vb(ch + 1);
        cp_commit();
      } else {
        cp_wait<1>();
        bar_sync(0, NT);  // K and Q are there, and nobody reads the other K any more
        if (more) load_k(ch + 1);
        cp_commit();
        cp_wait<1>();
        bar_sync(1, NL);  // V, T, P and the factors are there
        sizes_of_v(ch);
        bar_sync(0, NT);  // they are for the chains too, which have split S
      }
      float o[4][4] = {}, o2[4][4] = {};  // the two halves of dk have scales of their own
#pragma unroll
      for (int kk = 0; kk < DK / 16; ++kk) {
        unsigned ah[4], al[4], b[2][4];
        get_frag(s_ex + kk * 64, ah, al);
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) ldsm4(b[jp], q_s + kq_off<DK>(32 * half + 16 * jp + bt, 2 * kk + bu));
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_acc(kk < KH ? o[j] : o2[j], al, b[j / 2][2 * (j & 1)], b[j / 2][2 * (j & 1) + 1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_acc(kk < KH ? o[j] : o2[j], ah, b[j / 2][2 * (j & 1)], b[j / 2][2 * (j & 1) + 1]);
      }
      {
        const float a0 = sc[g], a1 = sc[g + 8], b0 = sc[16 + g], b1 = sc[24 + g];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 oq = *reinterpret_cast<const float2*>(vec + kGdOq + 32 * half + 8 * j + 2 * c);
          o[j][0] = oq.x * fmaf(o[j][0], a0, o2[j][0] * b0);
          o[j][1] = oq.y * fmaf(o[j][1], a0, o2[j][1] * b0);
          o[j][2] = oq.x * fmaf(o[j][2], a1, o2[j][2] * b1);
          o[j][3] = oq.y * fmaf(o[j][3], a1, o2[j][3] * b1);
        }
      }
      if constexpr (!DEEP) {
        bar_sync(1, NL);  // Q is free
        if (more) load_q(ch + 1);
        cp_commit();
      }
      bar_sync(bar + 3, 128);  // u is split
      unsigned ah[4][4], al[4][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        if (kk < 2 || half) get_frag(u_ex + kk * 64, ah[kk], al[kk]);
      const float du0 = sc[64 + g], du1 = sc[72 + g];
      const bool by_token = sc[kGdByToken] != 0.f;  // the chain warps write these rows of o
      if (more) bar_arrive(bar + 4, 128);
      if (DEEP && more) {
        cp_wait<0>();
        bar_sync(1, NL);
        sizes_of_v(ch + 1);
        bar_arrive(0, NT);  // the next chunk is there
      }
      const uint4* Pf = reinterpret_cast<const uint4*>(st + B_AT + kGdTri) + lane;
      float x[4][4] = {};
      if (half == 0) tri_product<0, 0, 2>(x, ah, al, Pf);
      else tri_product<4, 0, 4>(x, ah, al, Pf);
#pragma unroll
      for (int jp = 0; jp < 2; ++jp) {
        unsigned out[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = 2 * jp + i;
          const float2 op = *reinterpret_cast<const float2*>(vec + kGdOp + 32 * half + 8 * j + 2 * c);
          T r[4];
          r[0] = from_f<T>(fmaf(x[j][0], op.x * du0, o[j][0]));
          r[1] = from_f<T>(fmaf(x[j][1], op.y * du0, o[j][1]));
          r[2] = from_f<T>(fmaf(x[j][2], op.x * du1, o[j][2]));
          r[3] = from_f<T>(fmaf(x[j][3], op.y * du1, o[j][3]));
          out[i] = (unsigned)__builtin_bit_cast(unsigned short, r[0]) | (unsigned)__builtin_bit_cast(unsigned short, r[1]) << 16;
          out[2 + i] = (unsigned)__builtin_bit_cast(unsigned short, r[2]) | (unsigned)__builtin_bit_cast(unsigned short, r[3]) << 16;
        }
        // into the group's own columns of V, which its chain warps have read
        stsm4t(v_s + v_off(32 * half + 16 * jp + tt, 2 * group + tu), out);
      }
      __syncwarp();
      if (active && !by_token) {  // 16 rows of 32 bytes per store
        T* og = static_cast<T*>(p.o) + ((size_t)first + (size_t)ch * kGdC) * p.ld_o + h * p.dv + row0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = 32 * half + 16 * i + (lane >> 1);
          if (t < count - ch * kGdC)
            *reinterpret_cast<uint4*>(og + (size_t)t * p.ld_o + (lane & 1) * 8) =
                *reinterpret_cast<const uint4*>(st + V_AT + v_off(t, 2 * group + (lane & 1)));
        }
      }
      if constexpr (!DEEP) {
        bar_sync(1, NL);  // V, T, P and the factors are free: the chains left them before their u was split
        if (more) load_vb(ch + 1);
        cp_commit();
      }
    }
    cp_wait<0>();
    return;
  }

  // ------------------------------------------------------------------ chain warp, dk columns half * DK / 2 ..
  float* Sg = p.state + (((size_t)slot * p.v_heads + h) * p.dv + row0 + g) * DK + half * (DK / 2) + 2 * c;
  float s[NH][4], m0 = 0.f, m1 = 0.f;  // the state and its rows' largest magnitudes
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    float2 x = make_float2(0.f, 0.f), y = x;
    if (active) {
      x = *reinterpret_cast<const float2*>(Sg + 8 * j);
      y = *reinterpret_cast<const float2*>(Sg + 8 * DK + 8 * j);
    }
    s[j][0] = x.x, s[j][1] = x.y, s[j][2] = y.x, s[j][3] = y.y;
    m0 = fmaxf(m0, fmaxf(fabsf(x.x), fabsf(x.y)));
    m1 = fmaxf(m1, fmaxf(fabsf(y.x), fabsf(y.y)));
  }
  for (int ch = 0; ch < chunks; ++ch) {
    const uint32_t k_s = smem_u32(smem) + (ch & 1) * TILE;
    const char* st = smem + (DEEP ? (ch & 1) * STAGE : 0);
    const uint32_t v_s = smem_u32(st) + V_AT;
    const float* vec = reinterpret_cast<const float*>(st + B_AT + 2 * kGdTri);
    m0 = quad_max(m0);
    m1 = quad_max(m1);
    float up0, dn0, up1, dn1;
    row_scale(m0, up0, dn0);
    row_scale(m1, up1, dn1);
    if (ch) bar_sync(bar + 4, 128);  // the last chunk's S and u have been taken
    if (c == 0) {
      sc[16 * half + g] = dn0, sc[16 * half + 8 + g] = dn1;
      sc[32 + 16 * half + g] = m0, sc[40 + 16 * half + g] = m1;
    }
    unsigned sh[2][4], sl[2][4];
    split_tile(s[0], s[1], up0, up1, sh[0], sl[0]);
    bar_sync(0, NT);  // K and Q are there (DEEP: the whole chunk)
    // n-tiles 0-3 are this warp's tokens, 4-7 the other's
    float ks[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) ks[j][0] = ks[j][1] = ks[j][2] = ks[j][3] = 0.f;
    // this half's part of S k, the next step's split between the MMAs of this one
#pragma unroll
    for (int kk = 0; kk < KH; ++kk) {
      unsigned b[4][4];
#pragma unroll
      for (int jp = 0; jp < 4; ++jp)
        ldsm4(b[jp], k_s + (jp < 2 ? 0 : (1 - 2 * half) * 64 * DK) + kq_off<DK>(16 * (jp & 1) + 32 * half + bt, 2 * (half * KH + kk) + bu));
      const int now = kk & 1;
      put_frag(s_ex + (half * KH + kk) * 64, sh[now], sl[now]);
      if (DEEP && kk == KH - 1) bar_arrive(bar + 2, 128);  // S is split
      if (kk + 1 < KH) split_tile(s[2 * kk + 2], s[2 * kk + 3], up0, up1, sh[now ^ 1], sl[now ^ 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) mma_acc(ks[j], sl[now], b[j / 2][2 * (j & 1)], b[j / 2][2 * (j & 1) + 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) mma_acc(ks[j], sh[now], b[j / 2][2 * (j & 1)], b[j / 2][2 * (j & 1) + 1]);
    }
    // the other warp's tokens to it, in the place where it will put its weighed u
    float (&mine)[4][4] = *reinterpret_cast<float(*)[4][4]>(&ks[0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = mul2(make_float2(ks[4 + j][0], ks[4 + j][1]), dup(dn0)), b = mul2(make_float2(ks[4 + j][2], ks[4 + j][3]), dup(dn1));
      *reinterpret_cast<float4*>(d_ex + ((1 - half) * 4 + j) * 32) = make_float4(a.x, a.y, b.x, b.y);
    }
    if constexpr (DEEP) bar_sync(bar, 64);
    else bar_sync(0, NT);  // also: V, T, P and the factors are there; S is split
    // bounds of r and u, and the scales from them (measured: slower before or among the MMAs above)
    float ur0, dr0, ur1, dr1, uu0, du0, uu1, du1;
    const float root = (DK == 128 ? 11.3137085f : 8.f) * vec[kGdKn];
    const float s0 = fmaxf(sc[32 + g], sc[48 + g]), s1 = fmaxf(sc[40 + g], sc[56 + g]);
    const uint4 va = reinterpret_cast<const uint4*>(sc + kGdOfV)[g], vb = reinterpret_cast<const uint4*>(sc + kGdOfV)[8 + g];
    const float2 most = PairOf<T>::floats(__hmax2(as_pair<T>(va.x), as_pair<T>(vb.x)));
    const float r0 = fmaf(root, s0, most.x), r1 = fmaf(root, s1, most.y);
    const float u0 = r0 * vec[kGdTsum], u1 = r1 * vec[kGdTsum];
    row_scale(r0, ur0, dr0);
    row_scale(r1, ur1, dr1);
    row_scale(u0, uu0, du0);
    row_scale(u1, uu1, du1);
    const float tdn = vec[kGdTdn], el = vec[kGdLast], cdn = vec[kGdCdn];
    {  // both warps come to the same answers: they look at the same numbers
      const float2 least = PairOf<T>::floats(__hmin2(as_pair<T>(va.y), as_pair<T>(vb.y)));
      const float2 weighed = PairOf<T>::floats(__hmax2(as_pair<T>(va.z), as_pair<T>(vb.z)));
      const float k0 = el * s0, k1 = el * s1, w0 = u0 * kGdRangeO, w1 = u1 * kGdRangeO, kn = fmaxf(vec[kGdKn], 1.f), wm = vec[kGdWm] * kGdRangeS;
      const bool weak = (weighed.x < u0 * kGdRangeV && k0 < u0 * wm) || (weighed.y < u1 * kGdRangeV && k1 < u1 * wm);
      const bool low = (least.x < w0 && k0 < w0 * kn) || (least.y < w1 && k1 < w1 * kn);
      bool far = __any_sync(0xffffffffu, weak);
      if (!far && __any_sync(0xffffffffu, low))
        far = gd_forgets<T>(p, st + V_AT, reinterpret_cast<const T*>(vec + kGdNorms), group, first + ch * kGdC, min(count - ch * kGdC, kGdC), h, s0, s1, w0, w1);
      if (far && active) {
        if (half == 0 && lane == 0) sc[kGdByToken] = 1.f;
        bar_arrive(bar + 3, 128);  // the output warps need not wait: they leave this chunk's o alone
        float copy[NH][4];         // the state itself stays in registers
#pragma unroll
        for (int j = 0; j < NH; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) copy[j][i] = s[j][i];
        gd_by_token<T, DK>(p, copy, first + ch * kGdC, min(count - ch * kGdC, kGdC), h, hk, row0 + g, half, bar,
                           reinterpret_cast<float4*>(d_ex - lane));
        m0 = m1 = 0.f;
#pragma unroll
        for (int j = 0; j < NH; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] = copy[j][i];
          m0 = fmaxf(m0, fmaxf(fabsf(s[j][0]), fabsf(s[j][1])));
          m1 = fmaxf(m1, fmaxf(fabsf(s[j][2]), fabsf(s[j][3])));
        }
        continue;
      }
    }
    // r = v - e^G (S k) of this warp's tokens, split as the left operand of u = r T^T
    unsigned ah[4][4], al[4][4];
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {
      unsigned v[4];  // 16 tokens x 16 rows: {t, rows 0-7}, {t + 8, ..}, {t, rows 8-15}, {t + 8, ..}
      ldsm4t(v, v_s + v_off(32 * half + 16 * jp + tt, 2 * group + tu));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = 2 * jp + i;
        const float2 bk = *reinterpret_cast<const float2*>(vec + kGdBk + 32 * half + 8 * j + 2 * c);
        const float4 o = *reinterpret_cast<const float4*>(d_ex + (half * 4 + j) * 32);
        const T* x = reinterpret_cast<const T*>(&v[i]);
        const T* y = reinterpret_cast<const T*>(&v[2 + i]);
        const float2 a = fma2(bk, fma2(make_float2(mine[j][0], mine[j][1]), dup(dn0), make_float2(o.x, o.y)),
                              make_float2(to_f(x[0]), to_f(x[1])));
        const float2 b = fma2(bk, fma2(make_float2(mine[j][2], mine[j][3]), dup(dn1), make_float2(o.z, o.w)),
                              make_float2(to_f(y[0]), to_f(y[1])));
        mine[j][0] = a.x, mine[j][1] = a.y, mine[j][2] = b.x, mine[j][3] = b.y;
      }
      split_tile(mine[2 * jp], mine[2 * jp + 1], ur0, ur1, ah[2 + jp], al[2 + jp]);
    }
    const uint4* Tf = reinterpret_cast<const uint4*>(st + B_AT) + lane;
    float x[4][4] = {};  // u of this warp's tokens, scaled as r and T are
    {
      unsigned (&oh)[2][4] = *reinterpret_cast<unsigned(*)[2][4]>(&ah[2]), (&ol)[2][4] = *reinterpret_cast<unsigned(*)[2][4]>(&al[2]);
      if (half == 0) {
        put_frag(r_ex, oh[0], ol[0]);
        put_frag(r_ex + 64, oh[1], ol[1]);
        bar_arrive(bar + 1, 64);
        tri_product<0, 0, 2>(x, oh, ol, Tf);
      } else {
        tri_product<4, 2, 4>(x, oh, ol, Tf);
        bar_sync(bar + 1, 64);
        get_frag(r_ex, ah[0], al[0]);
        get_frag(r_ex + 64, ah[1], al[1]);
        tri_product<4, 0, 2>(x, ah, al, Tf);
      }
    }
    // beta e^(G_C - G) u, the left operand of the state's update, and u for the output warps
    const float fu0 = dr0 * uu0 * tdn, fu1 = dr1 * uu1 * tdn;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      float y[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 c2 = *reinterpret_cast<const float2*>(vec + kGdC2 + 32 * half + 16 * kk + 8 * i + 2 * c);
        const float2 a = mul2(make_float2(x[2 * kk + i][0], x[2 * kk + i][1]), c2);
        const float2 b = mul2(make_float2(x[2 * kk + i][2], x[2 * kk + i][3]), c2);
        y[i][0] = a.x, y[i][1] = a.y, y[i][2] = b.x, y[i][3] = b.y;
      }
      unsigned dh[4], dl[4];
      split_tile(y[0], y[1], fu0, fu1, dh, dl);
      put_frag(d_ex + (2 * half + kk) * 64, dh, dl);
    }
    bar_sync(bar, 64);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) get_frag(d_ex + kk * 64, ah[kk], al[kk]);
    // S <- e^G_C S + u k, and u for the output warps between the first MMAs
    const float ds0 = du0 * cdn, ds1 = du1 * cdn;
    m0 = m1 = 0.f;
#pragma unroll
    for (int jp = 0; jp < NH / 4; ++jp) {
      float z[4][4] = {};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        unsigned b[4], d[4];
        ldsm4t(b, k_s + kq_off<DK>(16 * kk + tt, half * NH + 4 * jp + tu));
        ldsm4t(d, k_s + kq_off<DK>(16 * kk + tt, half * NH + 4 * jp + 2 + tu));
        if (jp == 0 && kk < 2) {
          unsigned uh[4], ul[4];
          split_tile(x[2 * kk], x[2 * kk + 1], fu0, fu1, uh, ul);
          put_frag(u_ex + (2 * half + kk) * 64, uh, ul);
          if (kk == 1) {
            if (half == 0 && c == 0) sc[64 + g] = du0, sc[72 + g] = du1, sc[kGdByToken] = 0.f;
            bar_arrive(bar + 3, 128);  // u is split; this warp reads V, T and the factors no more
          }
        }
        mma_acc(z[0], al[kk], b[0], b[1]);
        mma_acc(z[1], al[kk], b[2], b[3]);
        mma_acc(z[2], al[kk], d[0], d[1]);
        mma_acc(z[3], al[kk], d[2], d[3]);
        mma_acc(z[0], ah[kk], b[0], b[1]);
        mma_acc(z[1], ah[kk], b[2], b[3]);
        mma_acc(z[2], ah[kk], d[0], d[1]);
        mma_acc(z[3], ah[kk], d[2], d[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float(&w)[4] = s[4 * jp + i];
        const float2 a = fma2(dup(el), make_float2(w[0], w[1]), mul2(make_float2(z[i][0], z[i][1]), dup(ds0)));
        const float2 b = fma2(dup(el), make_float2(w[2], w[3]), mul2(make_float2(z[i][2], z[i][3]), dup(ds1)));
        w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
        m0 = fmaxf(m0, fmaxf(fabsf(a.x), fabsf(a.y)));
        m1 = fmaxf(m1, fmaxf(fabsf(b.x), fabsf(b.y)));
      }
    }
  }
  if (!active) return;
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    *reinterpret_cast<float2*>(Sg + 8 * j) = make_float2(s[j][0], s[j][1]);
    *reinterpret_cast<float2*>(Sg + 8 * DK + 8 * j) = make_float2(s[j][2], s[j][3]);
  }
}

}  // namespace dfssm
