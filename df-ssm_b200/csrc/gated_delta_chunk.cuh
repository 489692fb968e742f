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
// operands (S, r, u, T, P) are scaled by a power of two per row, so that the row's largest is in [2^13, 2^14),
// and split in two fp16 numbers hi + lo, which keep 22 bits of what is above 2^-17 of the row's largest and
// 2^-39 of that below; a product of two such pairs takes three MMAs (hi hi, hi lo, lo hi).  Sums run in fp32 accumulators, and the state's update in one of its own, added to the
// decayed state with one rounding.  Decays are differences of sums in double precision: in fp32 a sum of
// -100 already leaves e^(G_t - G_w) an error of 4e-6.
#pragma once
#include "gated_delta.cuh"

namespace dfssm {

constexpr int kGdC = 64;                // tokens per chunk
constexpr int kGdFrags = 20;            // 8 x 16 fragments of a lower triangular 64 x 64 matrix
constexpr int kGdTri = kGdFrags * 512;  // bytes of one such matrix as fp16 hi/lo pairs, in fragment order
// per-token factors of a chunk, 64 floats each, then e^G_C
enum { kGdBk = 0, kGdC2 = 64, kGdOq = 128, kGdOp = 192, kGdTs = 256, kGdLast = 320, kGdVecs = 324 };
constexpr int kGdBlock = 2 * kGdTri + 1408;  // bytes per chunk and value head: T, P, factors
static_assert(kGdVecs * 4 <= 1408 && kGdBlock % 128 == 0, "");

// Chunks are numbered without a plan: sequence i's chunk c is cu[i] / 64 + i + c.  That leaves at most one
// number per sequence unused and gives no number twice.
__host__ __device__ inline long long gd_chunk_slots(int tokens, int n_seq) { return (long long)tokens / kGdC + n_seq; }
__device__ __forceinline__ int gd_chunk_base(const int* cu, int i, int tokens) {
  return min(max(cu[i], 0), tokens) / kGdC + i;
}

// Fragments of B = M^T (M lower triangular, rows t): n-tile j holds rows 8j..8j+7, k-step kk columns
// 16kk..16kk+15, kk <= j / 2.  Lane l: row 8j + l/4, columns 16kk + 2(l%4) + {0, 1} and + 8, as 16 bytes
// {hi, hi + 8, lo, lo + 8}.
__host__ __device__ constexpr int gd_frag(int j, int kk) { return ((j & 1) ? ((j + 1) / 2) * ((j + 1) / 2) : (j / 2) * (j / 2 + 1)) + kk; }
static_assert(gd_frag(0, 0) == 0 && gd_frag(1, 0) == 1 && gd_frag(2, 0) == 2 && gd_frag(3, 0) == 4 && gd_frag(4, 0) == 6 &&
                  gd_frag(5, 0) == 9 && gd_frag(6, 0) == 12 && gd_frag(7, 3) == kGdFrags - 1, "");

__device__ __forceinline__ unsigned h2_bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
// two fp32 values as fp16 pairs hi + lo (22 bits)
__device__ __forceinline__ void split2(float x, float y, unsigned& hi, unsigned& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2_bits(h);
  lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}
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
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
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
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte unit u of row t in a K or Q tile [64][DK] of fp16: rows of 8 or 16 units, the units
// of a row permuted by its low three bits, so that eight rows' units of one column fall into different banks.
template <int DK>
__device__ __forceinline__ uint32_t kq_off(int t, int u) {
  return (uint32_t)(t * DK * 2 + ((u ^ (t & 7)) << 4));
}

// ------------------------------------------------------------------ T, P and the factors of every chunk

constexpr int kPrepThreads = 128;
constexpr int kLS = 68;  // row stride of the fp32 matrices in shared memory

template <int DK>
__host__ __device__ constexpr int gd_prep_smem() { return 2 * kGdC * DK * 2 + 2 * kGdC * kLS * 4 + 1024 * 5 + 64 * 8; }

// One block per chunk number and value head.  kq16: for bf16 inputs, the fp16 tiles K and Q
// [chunk][k_heads][2][64][DK] that the chunk kernel reads.
template <typename T, int DK>
__global__ void __launch_bounds__(kPrepThreads)
gated_delta_prep_kernel(const GatedDeltaArgs p, char* __restrict__ blocks, __half* __restrict__ kq16) {
  constexpr bool BF = !std::is_same<T, __half>::value;
  constexpr int UPR = DK / 8;  // 16-byte units per row
  extern __shared__ __align__(128) char smem[];
  __half* Ks = reinterpret_cast<__half*>(smem);
  __half* Qs = Ks + kGdC * DK;
  float* L = reinterpret_cast<float*>(Qs + kGdC * DK);  // [64][kLS]
  float* X = L + kGdC * kLS;                            // [64][kLS]: T
  float* rk = X + kGdC * kLS;                           // row factors of K and Q as staged
  float* rq = rk + 64;
  float* beta = rq + 64;
  double* G = reinterpret_cast<double*>(beta + 64);  // running log decay
  float* tmax = reinterpret_cast<float*>(G + 64);    // [2][64]
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.x % p.v_heads, num = blockIdx.x / p.v_heads;
  // the sequence of chunk `num`: the last one whose first chunk is not behind it
  int lo = 0, hi = p.n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (gd_chunk_base(p.cu, mid, p.tokens) <= num) lo = mid;
    else hi = mid - 1;
  }
  int first, count;
  gd_range(p.cu, lo, p.tokens, first, count);
  const int cn = num - gd_chunk_base(p.cu, lo, p.tokens);
  if (cn < 0 || cn * kGdC >= count) return;
  first += cn * kGdC;
  count = min(count - cn * kGdC, kGdC);
  const int rep = p.v_heads / p.k_heads, hk = h / rep;
  // K and Q rows: DK / 8 lanes per row, one 16-byte unit each; the row's factor is 1 / |row| (qk_norm) times,
  // for bf16, the power of two that undoes the staging's
  {
    constexpr int RPI = kPrepThreads / UPR;  // rows per pass
    const int u = tid % UPR, r0 = tid / UPR;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const T* src = static_cast<const T*>(which ? p.q : p.k) + hk * DK + u * 8;
      const int ld = which ? p.ld_q : p.ld_k;
      uint4 raw[kGdC / RPI];
#pragma unroll
      for (int i = 0; i < kGdC / RPI; ++i) {
        const int t = r0 + i * RPI;
        raw[i] = t < count ? *reinterpret_cast<const uint4*>(src + (size_t)(first + t) * ld) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kGdC / RPI; ++i) {
        const int t = r0 + i * RPI;
        const T* e = reinterpret_cast<const T*>(&raw[i]);
        float f[8], ss = 0.f, mx = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[j] = to_f(e[j]);
          ss += f[j] * f[j];
          mx = fmaxf(mx, fabsf(f[j]));
        }
#pragma unroll
        for (int o = UPR / 2; o > 0; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if constexpr (BF) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
        float factor = p.qk_norm ? 1.0f / sqrtf(ss + kQkEps) : 1.0f;
        if constexpr (BF) {
          float up, down;
          row_scale(mx, up, down);
          factor *= down;
          uint4 out;
          unsigned* ow = reinterpret_cast<unsigned*>(&out);
#pragma unroll
          for (int j = 0; j < 4; ++j) ow[j] = h2_bits(__floats2half2_rn(f[2 * j] * up, f[2 * j + 1] * up));
          raw[i] = out;
          if (h % rep == 0)
            *reinterpret_cast<uint4*>(kq16 + ((((size_t)num * p.k_heads + hk) * 2 + which) * kGdC + t) * DK + u * 8) = out;
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<char*>(which ? Qs : Ks) + kq_off<DK>(t, u)) = raw[i];
        if (u == 0) (which ? rq : rk)[t] = factor;
      }
    }
  }
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
    beta[tid] = bt;
  }
  __syncthreads();
  if (tid >= 32 && tid < 64) G[tid] += G[31];
  __syncthreads();
  const double Glast = G[63];
  char* blk = blocks + ((size_t)num * p.v_heads + h) * kGdBlock;
  float* vec = reinterpret_cast<float*>(blk + 2 * kGdTri);
  // Q K^T rows 16 wid.. and K K^T rows 16 (3 - wid)..: ten 16 x 8 tiles for every warp
  const uint32_t ks = smem_u32(Ks), qs = smem_u32(Qs);
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
          mma_f16(acc[2 * jp], a[0], a[1], a[2], a[3], b[0], b[1]);
          mma_f16(acc[2 * jp + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
        }
      }
    }
  };
  {
    float acc[8][4];
    gram(qs, wid, acc);
    const int ta = 16 * wid + g, tb = ta + 8;
    const double Ga = G[ta], Gb = G[tb];
    const float fa = p.scale * rq[ta], fb = p.scale * rq[tb];
    float ma = 0.f, mb = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j <= 2 * wid + 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int w = 8 * j + 2 * c + i;
          const float ea = expf((float)(Ga - G[w])), eb = expf((float)(Gb - G[w]));
          const float fw = rk[w] * beta[w];
          acc[j][i] = w <= ta ? acc[j][i] * fa * fw * ea : 0.f;
          acc[j][2 + i] = w <= tb ? acc[j][2 + i] * fb * fw * eb : 0.f;
          ma = fmaxf(ma, fabsf(acc[j][i]));
          mb = fmaxf(mb, fabsf(acc[j][2 + i]));
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
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk <= wid) {
        unsigned ha0, la0, ha1, la1, hb0, lb0, hb1, lb1;
        split2(acc[2 * kk][0] * ua, acc[2 * kk][1] * ua, ha0, la0);
        split2(acc[2 * kk + 1][0] * ua, acc[2 * kk + 1][1] * ua, ha1, la1);
        split2(acc[2 * kk][2] * ub, acc[2 * kk][3] * ub, hb0, lb0);
        split2(acc[2 * kk + 1][2] * ub, acc[2 * kk + 1][3] * ub, hb1, lb1);
        uint4* P = reinterpret_cast<uint4*>(blk + kGdTri);
        P[gd_frag(2 * wid, kk) * 32 + lane] = make_uint4(ha0, ha1, la0, la1);
        P[gd_frag(2 * wid + 1, kk) * 32 + lane] = make_uint4(hb0, hb1, lb0, lb1);
      }
    }
  }
  {
    float acc[8][4];
    const int mt = 3 - wid;
    gram(ks, mt, acc);
    const int ta = 16 * mt + g, tb = ta + 8;
    const double Ga = G[ta], Gb = G[tb];
    const float fa = rk[ta], fb = rk[tb];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int w = 8 * j + 2 * c + i;
        const bool va = j <= 2 * mt + 1 && w < ta, vb = j <= 2 * mt + 1 && w < tb;
        const float fw = rk[w] * beta[w];
        L[ta * kLS + w] = va ? acc[j][i] * fa * fw * expf((float)(Ga - G[w])) : 0.f;
        L[tb * kLS + w] = vb ? acc[j][2 + i] * fb * fw * expf((float)(Gb - G[w])) : 0.f;
      }
    }
  }
  // per-token factors
  if (tid < 64) {
    const double Gt = G[tid];
    const float eg = expf((float)Gt);
    vec[kGdBk + tid] = -eg * rk[tid];
    vec[kGdC2 + tid] = expf((float)(Glast - Gt)) * rk[tid] * beta[tid];
    vec[kGdOq + tid] = p.scale * eg * rq[tid];
    if (tid == 0) vec[kGdLast] = expf((float)Glast);
  }
  __syncthreads();
  // T = (I + L)^-1: the 16 x 16 diagonal blocks by forward substitution, a lane per column ...
  for (int i = tid; i < kGdC * kLS; i += kPrepThreads) X[i] = 0.f;
  __syncthreads();
  if (lane < 16) {
    const float* Lb = L + 16 * wid * kLS + 16 * wid;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == lane ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) s = fmaf(-Lb[i * kLS + m], x[m], s);
      x[i] = s;
      X[(16 * wid + i) * kLS + 16 * wid + lane] = s;
    }
  }
  __syncthreads();
  // ... then pairs of blocks joined, 16 to 32 and 32 to 64: the corner is -T22 (L21 T11)
  float* M = reinterpret_cast<float*>(smem);  // K and Q are not read again: [2][16][20], then [32][36]
  {
    const int pair = tid >> 6, r = (tid & 63) >> 2, c0 = (tid & 3) * 4, o = 32 * pair;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 16; ++m) {
      const float l = L[(o + 16 + r) * kLS + o + m];
      const float4 x = *reinterpret_cast<const float4*>(X + (o + m) * kLS + o + c0);
      s[0] = fmaf(l, x.x, s[0]), s[1] = fmaf(l, x.y, s[1]), s[2] = fmaf(l, x.z, s[2]), s[3] = fmaf(l, x.w, s[3]);
    }
    *reinterpret_cast<float4*>(M + (pair * 16 + r) * 20 + c0) = make_float4(s[0], s[1], s[2], s[3]);
    __syncthreads();
    float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 16; ++m) {
      const float l = X[(o + 16 + r) * kLS + o + 16 + m];
      const float4 x = *reinterpret_cast<const float4*>(M + (pair * 16 + m) * 20 + c0);
      y[0] = fmaf(-l, x.x, y[0]), y[1] = fmaf(-l, x.y, y[1]), y[2] = fmaf(-l, x.z, y[2]), y[3] = fmaf(-l, x.w, y[3]);
    }
    *reinterpret_cast<float4*>(X + (o + 16 + r) * kLS + o + c0) = make_float4(y[0], y[1], y[2], y[3]);
  }
  __syncthreads();
  {
    const int r = (tid >> 3) * 2, c0 = (tid & 7) * 4;  // 16 x 8 threads of 2 x 4 outputs
    float s[2][4] = {};
#pragma unroll 8
    for (int m = 0; m < 32; ++m) {
      const float4 x = *reinterpret_cast<const float4*>(X + m * kLS + c0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float l = L[(32 + r + i) * kLS + m];
        s[i][0] = fmaf(l, x.x, s[i][0]), s[i][1] = fmaf(l, x.y, s[i][1]);
        s[i][2] = fmaf(l, x.z, s[i][2]), s[i][3] = fmaf(l, x.w, s[i][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(M + (r + i) * 36 + c0) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    __syncthreads();
    float y[2][4] = {};
#pragma unroll 8
    for (int m = 0; m < 32; ++m) {
      const float4 x = *reinterpret_cast<const float4*>(M + m * 36 + c0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float l = X[(32 + r + i) * kLS + 32 + m];
        y[i][0] = fmaf(-l, x.x, y[i][0]), y[i][1] = fmaf(-l, x.y, y[i][1]);
        y[i][2] = fmaf(-l, x.z, y[i][2]), y[i][3] = fmaf(-l, x.w, y[i][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(X + (32 + r + i) * kLS + c0) = make_float4(y[i][0], y[i][1], y[i][2], y[i][3]);
  }
  __syncthreads();
  {  // the rows' scales
    const int t = tid >> 1, half = tid & 1;
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < 32; w += 4) {
      const float4 x = *reinterpret_cast<const float4*>(X + t * kLS + 32 * half + w);
      m = fmaxf(m, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    float up, down;
    row_scale(m, up, down);
    if (half == 0) {
      tmax[t] = up;
      vec[kGdTs + t] = down;
    }
  }
  __syncthreads();
#pragma unroll
  for (int f = 0; f < kGdFrags / 4; ++f) {  // fragment 4 f + wid
    const int id = 4 * f + wid;
    int j = 0;
#pragma unroll
    for (int x = 1; x < 8; ++x) j += id >= gd_frag(x, 0);
    const int kk = id - gd_frag(j, 0), t = 8 * j + g;
    const float up = tmax[t];
    const float* x = X + t * kLS + 16 * kk + 2 * c;
    unsigned h0, l0, h1, l1;
    split2(x[0] * up, x[1] * up, h0, l0);
    split2(x[8] * up, x[9] * up, h1, l1);
    reinterpret_cast<uint4*>(blk)[id * 32 + lane] = make_uint4(h0, h1, l0, l1);
  }
}

// ------------------------------------------------------------------ the walk over a sequence's chunks
//
// A warp owns 16 rows of one head's state, S^T as MMA accumulators (64 registers per thread at dk = 128).  All
// products are taken transposed, with the state, r and u as left operands: the accumulator layout of one
// product is the left operand's layout of the next, so nothing but k, q, v, T and P passes through shared
// memory, and warps meet only where its buffers change hands.
//   S k, S q : [16 x dk] [dk x 64]     u = r T^T, u P^T : [16 x 64] [64 x 64]     u k : [16 x 64] [64 x dk]
// K is double buffered; Q, V, T, P and the factors of the next chunk arrive (cp.async) while the products that
// do not read them run.

template <int DK, int W>
__host__ __device__ constexpr int gd_chunk_smem() {
  return 3 * kGdC * DK * 2 + kGdC * 32 * W + kGdBlock;
}

// Byte offset of 16-byte unit u of token t in the V tile [64][16 W].
template <int W>
__device__ __forceinline__ uint32_t v_off(int t, int u) {
  const int f = W >= 4 ? (t & 7) : (W == 2 ? ((t >> 1) & 3) : ((t >> 2) & 1));
  return (uint32_t)(t * 32 * W + ((u ^ f) << 4));
}

// ldb: element strides of the K / Q tiles' rows.  For fp16 inputs kq16 is NULL and the tiles are rows of k and q.
template <typename T, int DK, int W>
__global__ void __launch_bounds__(32 * W, 8 / W)
gated_delta_chunk_kernel(const GatedDeltaArgs p, const char* __restrict__ blocks, const __half* __restrict__ kq16,
                         int parts, int slots_total) {
  constexpr bool BF = !std::is_same<T, __half>::value;
  constexpr int NT = 32 * W, NK = DK / 8, UPR = DK / 8;
  extern __shared__ __align__(128) char smem[];
  char* vt = smem + 3 * kGdC * DK * 2;
  char* tp = vt + kGdC * 32 * W;
  const float* vec = reinterpret_cast<const float*>(tp + 2 * kGdTri);
  const uint32_t k_s = smem_u32(smem), q_s = k_s + 2 * kGdC * DK * 2, v_s = smem_u32(vt), tp_s = smem_u32(tp);
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, c = lane & 3;
  const int part = blockIdx.x % parts, h = (blockIdx.x / parts) % p.v_heads, seq = blockIdx.x / (parts * p.v_heads);
  const int slot = gd_slot(p.slots, seq, p.n_slots, tid, NT);
  if (slot < 0) return;
  int first, count;
  gd_range(p.cu, seq, p.tokens, first, count);
  if (count == 0) return;
  const int base = gd_chunk_base(p.cu, seq, p.tokens);
  const int chunks = min((count + kGdC - 1) / kGdC, slots_total - base);
  const int hk = h / (p.v_heads / p.k_heads);
  const int dv0 = part * 16 * W, row0 = dv0 + 16 * wid;
  const bool active = row0 < p.dv;  // dv is a multiple of 16: a warp's rows are all there or none

  auto load_kq = [&](int ch) {  // K and Q of chunk ch
    const int n = count - ch * kGdC;
    const uint32_t kd = k_s + (ch & 1) * kGdC * DK * 2;
    const size_t row = (size_t)first + (size_t)ch * kGdC;
    for (int i = tid; i < kGdC * UPR; i += NT) {
      const int t = i / UPR, u = i % UPR;
      if constexpr (BF) {
        const __half* src = kq16 + (((size_t)(base + ch) * p.k_heads + hk) * 2 * kGdC + t) * DK + u * 8;
        cp16(kd + kq_off<DK>(t, u), src, true);
        cp16(q_s + kq_off<DK>(t, u), src + kGdC * DK, true);
      } else {
        const bool ok = t < n;
        const size_t r = ok ? row + t : row;
        cp16(kd + kq_off<DK>(t, u), static_cast<const __half*>(p.k) + r * p.ld_k + hk * DK + u * 8, ok);
        cp16(q_s + kq_off<DK>(t, u), static_cast<const __half*>(p.q) + r * p.ld_q + hk * DK + u * 8, ok);
      }
    }
    cp_commit();
  };
  auto load_vtp = [&](int ch) {  // V, T, P and the factors of chunk ch
    const int n = count - ch * kGdC;
    const size_t row = (size_t)first + (size_t)ch * kGdC;
    const int units = min(16 * W, p.dv - dv0) / 8;
    for (int i = tid; i < kGdC * 2 * W; i += NT) {
      const int t = i / (2 * W), u = i % (2 * W);
      const bool ok = t < n && u < units;
      cp16(v_s + v_off<W>(t, u), static_cast<const T*>(p.v) + (ok ? (row + t) * p.ld_v + h * p.dv + dv0 + u * 8 : 0), ok);
    }
    const char* blk = blocks + ((size_t)(base + ch) * p.v_heads + h) * kGdBlock;
    for (int i = tid; i < kGdBlock / 16; i += NT) cp16(tp_s + i * 16, blk + i * 16, true);
    cp_commit();
  };

  load_kq(0);
  load_vtp(0);
  float* Sg = p.state + (((size_t)slot * p.v_heads + h) * p.dv + row0 + g) * DK + 2 * c;
  float s[NK][4];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    float2 x = make_float2(0.f, 0.f), y = x;
    if (active) {
      x = *reinterpret_cast<const float2*>(Sg + 8 * j);
      y = *reinterpret_cast<const float2*>(Sg + 8 * DK + 8 * j);
    }
    s[j][0] = x.x, s[j][1] = x.y, s[j][2] = y.x, s[j][3] = y.y;
  }
  // lane parts of the ldmatrix addresses
  const int bt = ((lane >> 4) << 3) + (lane & 7), bu = (lane >> 3) & 1;   // B from [token][dk] rows, two n-tiles
  const int tt = (((lane >> 3) & 1) << 3) + (lane & 7), tu = lane >> 4;   // the same, transposed

  for (int ch = 0; ch < chunks; ++ch) {
    const uint32_t kd = k_s + (ch & 1) * kGdC * DK * 2;
    cp_wait<1>();
    __syncthreads();  // K and Q are there
    float ks[8][4], qs[8][4], up0, dn0, up1, dn1;
    {
      float m0 = 0.f, m1 = 0.f;
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        m0 = fmaxf(m0, fmaxf(fabsf(s[j][0]), fabsf(s[j][1])));
        m1 = fmaxf(m1, fmaxf(fabsf(s[j][2]), fabsf(s[j][3])));
      }
      row_scale(quad_max(m0), up0, dn0);
      row_scale(quad_max(m1), up1, dn1);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ks[j][0] = ks[j][1] = ks[j][2] = ks[j][3] = 0.f;
      qs[j][0] = qs[j][1] = qs[j][2] = qs[j][3] = 0.f;
    }
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
      unsigned ah[4], al[4];
      split2(s[2 * kk][0] * up0, s[2 * kk][1] * up0, ah[0], al[0]);
      split2(s[2 * kk][2] * up1, s[2 * kk][3] * up1, ah[1], al[1]);
      split2(s[2 * kk + 1][0] * up0, s[2 * kk + 1][1] * up0, ah[2], al[2]);
      split2(s[2 * kk + 1][2] * up1, s[2 * kk + 1][3] * up1, ah[3], al[3]);
#pragma unroll
      for (int jp = 0; jp < 4; ++jp) {
        unsigned b[4], q[4];
        ldsm4(b, kd + kq_off<DK>(16 * jp + bt, 2 * kk + bu));
        ldsm4(q, q_s + kq_off<DK>(16 * jp + bt, 2 * kk + bu));
        mma_f16(ks[2 * jp], ah[0], ah[1], ah[2], ah[3], b[0], b[1]);
        mma_f16(ks[2 * jp + 1], ah[0], ah[1], ah[2], ah[3], b[2], b[3]);
        mma_f16(qs[2 * jp], ah[0], ah[1], ah[2], ah[3], q[0], q[1]);
        mma_f16(qs[2 * jp + 1], ah[0], ah[1], ah[2], ah[3], q[2], q[3]);
        mma_f16(ks[2 * jp], al[0], al[1], al[2], al[3], b[0], b[1]);
        mma_f16(ks[2 * jp + 1], al[0], al[1], al[2], al[3], b[2], b[3]);
        mma_f16(qs[2 * jp], al[0], al[1], al[2], al[3], q[0], q[1]);
        mma_f16(qs[2 * jp + 1], al[0], al[1], al[2], al[3], q[2], q[3]);
      }
    }
    cp_wait<0>();
    __syncthreads();  // V, T and P are there; Q and the other K buffer are free
    if (ch + 1 < chunks) load_kq(ch + 1);
    else cp_commit();
    // r = v - e^G (S k), in ks
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int jp = 0; jp < 4; ++jp) {
      unsigned v[4];  // tokens 16 jp.. x 16 rows: {t, rows 0-7}, {t + 8, ..}, {t, rows 8-15}, {t + 8, ..}
      ldsm4t(v, v_s + v_off<W>(16 * jp + tt, 2 * wid + tu));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = 2 * jp + i, t = 8 * j + 2 * c;
        const float2 bk = *reinterpret_cast<const float2*>(vec + kGdBk + t);
        const T* x = reinterpret_cast<const T*>(&v[i]);
        const T* y = reinterpret_cast<const T*>(&v[2 + i]);
        ks[j][0] = fmaf(bk.x * dn0, ks[j][0], to_f(x[0]));
        ks[j][1] = fmaf(bk.y * dn0, ks[j][1], to_f(x[1]));
        ks[j][2] = fmaf(bk.x * dn1, ks[j][2], to_f(y[0]));
        ks[j][3] = fmaf(bk.y * dn1, ks[j][3], to_f(y[1]));
        m0 = fmaxf(m0, fmaxf(fabsf(ks[j][0]), fabsf(ks[j][1])));
        m1 = fmaxf(m1, fmaxf(fabsf(ks[j][2]), fabsf(ks[j][3])));
        // S q, complete: o = qs + P u
        const float2 oq = *reinterpret_cast<const float2*>(vec + kGdOq + t);
        qs[j][0] *= oq.x * dn0;
        qs[j][1] *= oq.y * dn0;
        qs[j][2] *= oq.x * dn1;
        qs[j][3] *= oq.y * dn1;
      }
    }
    row_scale(quad_max(m0), up0, dn0);
    row_scale(quad_max(m1), up1, dn1);
    unsigned ah[4][4], al[4][4];
    auto split_rows = [&](const float (&x)[8][4]) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        split2(x[2 * kk][0] * up0, x[2 * kk][1] * up0, ah[kk][0], al[kk][0]);
        split2(x[2 * kk][2] * up1, x[2 * kk][3] * up1, ah[kk][1], al[kk][1]);
        split2(x[2 * kk + 1][0] * up0, x[2 * kk + 1][1] * up0, ah[kk][2], al[kk][2]);
        split2(x[2 * kk + 1][2] * up1, x[2 * kk + 1][3] * up1, ah[kk][3], al[kk][3]);
      }
    };
    split_rows(ks);
    // u = r T^T, in ks
    const uint4* Tf = reinterpret_cast<const uint4*>(tp) + lane;
    m0 = m1 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk <= j / 2; ++kk) {
        const uint4 b = Tf[gd_frag(j, kk) * 32];
        mma_f16(x, ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], b.z, b.w);
        mma_f16(x, al[kk][0], al[kk][1], al[kk][2], al[kk][3], b.x, b.y);
        mma_f16(x, ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], b.x, b.y);
      }
      const float2 ts = *reinterpret_cast<const float2*>(vec + kGdTs + 8 * j + 2 * c);
      ks[j][0] = x[0] * (ts.x * dn0);
      ks[j][1] = x[1] * (ts.y * dn0);
      ks[j][2] = x[2] * (ts.x * dn1);
      ks[j][3] = x[3] * (ts.y * dn1);
      m0 = fmaxf(m0, fmaxf(fabsf(ks[j][0]), fabsf(ks[j][1])));
      m1 = fmaxf(m1, fmaxf(fabsf(ks[j][2]), fabsf(ks[j][3])));
    }
    row_scale(quad_max(m0), up0, dn0);
    row_scale(quad_max(m1), up1, dn1);
    split_rows(ks);
    // o = S q + u P^T
    const uint4* Pf = Tf + kGdFrags * 32;
#pragma unroll
    for (int jp = 0; jp < 4; ++jp) {
      unsigned out[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = 2 * jp + i;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk <= jp; ++kk) {
          const uint4 b = Pf[gd_frag(j, kk) * 32];
          mma_f16(x, ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], b.z, b.w);
          mma_f16(x, al[kk][0], al[kk][1], al[kk][2], al[kk][3], b.x, b.y);
          mma_f16(x, ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], b.x, b.y);
        }
        const float2 op = *reinterpret_cast<const float2*>(vec + kGdOp + 8 * j + 2 * c);
        T r[4];
        r[0] = from_f<T>(fmaf(x[0], op.x * dn0, qs[j][0]));
        r[1] = from_f<T>(fmaf(x[1], op.y * dn0, qs[j][1]));
        r[2] = from_f<T>(fmaf(x[2], op.x * dn1, qs[j][2]));
        r[3] = from_f<T>(fmaf(x[3], op.y * dn1, qs[j][3]));
        out[i] = *reinterpret_cast<unsigned*>(r);
        out[2 + i] = *reinterpret_cast<unsigned*>(r + 2);
      }
      stsm4t(v_s + v_off<W>(16 * jp + tt, 2 * wid + tu), out);  // into this warp's columns of V, read above
    }
    // beta e^(G_C - G) u for the state's update
    m0 = m1 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 c2 = *reinterpret_cast<const float2*>(vec + kGdC2 + 8 * j + 2 * c);
      ks[j][0] *= c2.x;
      ks[j][1] *= c2.y;
      ks[j][2] *= c2.x;
      ks[j][3] *= c2.y;
      m0 = fmaxf(m0, fmaxf(fabsf(ks[j][0]), fabsf(ks[j][1])));
      m1 = fmaxf(m1, fmaxf(fabsf(ks[j][2]), fabsf(ks[j][3])));
    }
    row_scale(quad_max(m0), up0, dn0);
    row_scale(quad_max(m1), up1, dn1);
    split_rows(ks);
    const float el = vec[kGdLast];
    __syncwarp();
    if (active) {  // 16 rows of 32 bytes per store
      T* og = static_cast<T*>(p.o) + ((size_t)first + (size_t)ch * kGdC) * p.ld_o + h * p.dv + row0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 16 * i + (lane >> 1);
        if (t < count - ch * kGdC)
          *reinterpret_cast<uint4*>(og + (size_t)t * p.ld_o + (lane & 1) * 8) =
              *reinterpret_cast<const uint4*>(vt + v_off<W>(t, 2 * wid + (lane & 1)));
      }
    }
    __syncthreads();  // V, T and P are free
    if (ch + 1 < chunks) load_vtp(ch + 1);
    else cp_commit();
    // S <- e^G_C S + u k
#pragma unroll
    for (int jp = 0; jp < NK / 4; ++jp) {
      float x[4][4] = {};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        unsigned b[4], d[4];
        ldsm4t(b, kd + kq_off<DK>(16 * kk + tt, 4 * jp + tu));
        ldsm4t(d, kd + kq_off<DK>(16 * kk + tt, 4 * jp + 2 + tu));
        mma_f16(x[0], al[kk][0], al[kk][1], al[kk][2], al[kk][3], b[0], b[1]);
        mma_f16(x[1], al[kk][0], al[kk][1], al[kk][2], al[kk][3], b[2], b[3]);
        mma_f16(x[2], al[kk][0], al[kk][1], al[kk][2], al[kk][3], d[0], d[1]);
        mma_f16(x[3], al[kk][0], al[kk][1], al[kk][2], al[kk][3], d[2], d[3]);
        mma_f16(x[0], ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], b[0], b[1]);
        mma_f16(x[1], ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], b[2], b[3]);
        mma_f16(x[2], ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], d[0], d[1]);
        mma_f16(x[3], ah[kk][0], ah[kk][1], ah[kk][2], ah[kk][3], d[2], d[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float(&z)[4] = s[4 * jp + i];
        z[0] = fmaf(el, z[0], x[i][0] * dn0);
        z[1] = fmaf(el, z[1], x[i][1] * dn0);
        z[2] = fmaf(el, z[2], x[i][2] * dn1);
        z[3] = fmaf(el, z[3], x[i][3] * dn1);
      }
    }
  }
  cp_wait<0>();
  if (!active) return;
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    *reinterpret_cast<float2*>(Sg + 8 * j) = make_float2(s[j][0], s[j][1]);
    *reinterpret_cast<float2*>(Sg + 8 * DK + 8 * j) = make_float2(s[j][2], s[j][3]);
  }
}

}  // namespace dfssm
