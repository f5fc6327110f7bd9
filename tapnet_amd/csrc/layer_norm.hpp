// Layer normalisation over the last axis, forward and backward (engine-free: any channel count, optional parameters).
//
//   y = (x - mean) rstd gamma + beta,   rstd = 1 / sqrt(var + eps), var = mean((x - mean)^2)
//   g = dy gamma,  u = (x - mean) rstd:   dx = rstd (g - mean(g) - u mean(g u)),  dgamma = sum_rows dy u,  dbeta = sum_rows dy
//
// One pass over memory: a row stays in the registers of LPR lanes (NCH chunks of EPT elements each) between its statistics and
// its output, so x is read once and y written once.  Statistics are two sums in f32 over those registers (mean first, then the
// squares of the centred values: no cancellation).  Bound: HBM, 2 x (forward) and 3 x (backward) the tensor's bytes.  49152 x 256 bf16:
// forward 10.3 us = 4.9 TB/s (21 us before the next rows were fetched under this step's sums), backward 15.9 us = 4.7 TB/s and 3.9 us for
// the shares of the parameters' gradients; 12288 x 512 f32: 10.0 + 14.6 + 3.4 us.  Rows stay in registers up to 2048 channels in aligned
// bf16 and 1024 otherwise; longer ones are read three times (layer_norm_long_kernel, layer_norm_bwd_long_kernel: twice, column sums in memory).
#pragma once
#include "common.hpp"

namespace tapir {

constexpr int LN_THREADS = 256;
constexpr int LN_MAX_CHANNELS = 1 << 30;   // columns are counted in 32 bits, a stride of threads past the last one included
constexpr int LN_REDUCE_COLS = 16;   // columns per workgroup of the partial sums' reduction

// columns of a row of partial sums: every row starts at a multiple of 16 bytes
__host__ __device__ __forceinline__ long ln_part_stride(int C) { return ((long)C + 3) & ~3L; }

struct LnArgs {
  const void* x; long ldx;        // [rows, C], row stride in elements
  const float* gamma;             // [C] or null (ones)
  const float* beta;              // [C] or null (zeros)
  void* y;                        // [rows, C] dense
  float *mean, *rstd;             // [rows] or null
  long rows; int C; float eps;
};

struct LnBwdArgs {
  const void* x; long ldx;
  const void* dy; long lddy;
  const float* gamma;
  const float *mean, *rstd;
  void* dx;                       // [rows, C] dense, or null
  float* part;                    // [grid][2][ln_part_stride(C)] partial sums of dgamma, dbeta (null: neither is wanted)
  long rows; int C;
};

// EPT consecutive elements at p as floats (EPT * sizeof(T) = 16 bytes, or one element)
template <typename T, int EPT> struct LnVec;
template <> struct LnVec<float, 4> {
  typedef tapir_f32x4 Raw;
  static __device__ __forceinline__ Raw get(const float* p) { return ldg_f4(p); }
  static __device__ __forceinline__ void split(const Raw& r, float (&v)[4]) { v[0] = r[0]; v[1] = r[1]; v[2] = r[2]; v[3] = r[3]; }
  static __device__ __forceinline__ void st(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <> struct LnVec<bf16_t, 8> {
  typedef uint4 Raw;
  static __device__ __forceinline__ Raw get(const bf16_t* p) { return ldg16(p); }
  static __device__ __forceinline__ void split(const Raw& r, float (&v)[8]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void st(bf16_t* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                              pack_bf16x2(v[6], v[7]));
  }
};
template <typename T> struct LnVec<T, 1> {
  typedef float Raw;
  static __device__ __forceinline__ Raw get(const T* p) { return Elem<T>::ld(p); }
  static __device__ __forceinline__ void split(Raw r, float (&v)[1]) { v[0] = r; }
  static __device__ __forceinline__ void st(T* p, const float (&v)[1]) { Elem<T>::st(p, v[0]); }
};

// sum over the LPR consecutive lanes that share a row; every lane receives it
template <int LPR> __device__ __forceinline__ float ln_sum(float v) {
  if (LPR == 64) return wave_sum(v);
#ifdef TAPIR_HIPEMU
#pragma unroll
  for (int m = LPR / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
#else
  v += dpp_f32<0xB1, 0xf>(0.f, v);                    // quad_perm [1,0,3,2]
  v += dpp_f32<0x4E, 0xf>(0.f, v);                    // quad_perm [2,3,0,1]
  if (LPR >= 8) v += dpp_f32<0x141, 0xf>(0.f, v);     // row_half_mirror
  if (LPR >= 16) v += dpp_f32<0x140, 0xf>(0.f, v);    // row_mirror
  if (LPR >= 32) v += __shfl_xor(v, 16);
#endif
  return v;
}

// sum over the workgroup, every thread receives it (used by the long-row forms only)
__device__ __forceinline__ float ln_block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < LN_THREADS / 64; ++w) s += red[w];
  return s;
}

// a lane's parameters: EPT consecutive columns from `col`, or the value of a missing parameter
template <int EPT> __device__ __forceinline__ void ln_param(const float* p, int col, int C, float missing, float (&v)[EPT]) {
  if (EPT >= 4 && p && col < C && ((uintptr_t)p & 15) == 0) {
#pragma unroll
    for (int e = 0; e < EPT; e += 4) {
      const tapir_f32x4 r = ldg_f4(p + col + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[EPT >= 4 ? e + i : 0] = r[i];
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < EPT; ++e) v[e] = p && col < C ? p[col + e] : missing;
}

// LPR lanes a row, LN_THREADS / LPR rows a workgroup and step; the next step's rows are on their way while this one's are worked on.
// C <= LPR * NCH * EPT.
template <typename T, int EPT, int LPR, int NCH>
__global__ __launch_bounds__(LN_THREADS) void layer_norm_kernel(LnArgs a) {
  constexpr int RPB = LN_THREADS / LPR;
  const int sub = threadIdx.x & (LPR - 1);
  typename LnVec<T, EPT>::Raw next[NCH];
  auto fetch = [&](long row0) {
    const long row = row0 + threadIdx.x / LPR;
    const T* xp = (const T*)a.x + (row < a.rows ? row : 0) * a.ldx;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * LPR + sub) * EPT;
      if (col < a.C) next[c] = LnVec<T, EPT>::get(xp + col);
    }
  };
  const long first = (long)blockIdx.x * RPB, step = (long)gridDim.x * RPB;
  if (first < a.rows) fetch(first);
  float gm[NCH][EPT], bt[NCH][EPT];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    ln_param(a.gamma, (c * LPR + sub) * EPT, a.C, 1.f, gm[c]);
    ln_param(a.beta, (c * LPR + sub) * EPT, a.C, 0.f, bt[c]);
  }
  const float inv = 1.f / (float)a.C;
  for (long row0 = first; row0 < a.rows; row0 += step) {
    const long row = row0 + threadIdx.x / LPR;
    float x[NCH][EPT];
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[c][e] = 0.f;
      if ((c * LPR + sub) * EPT < a.C) {
        LnVec<T, EPT>::split(next[c], x[c]);
#pragma unroll
        for (int e = 0; e < EPT; ++e) s += x[c][e];
      }
    }
    if (row0 + step < a.rows) fetch(row0 + step);
    const float mean = ln_sum<LPR>(s) * inv;
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if ((c * LPR + sub) * EPT < a.C) {
#pragma unroll
        for (int e = 0; e < EPT; ++e) { x[c][e] -= mean; ss = fmaf(x[c][e], x[c][e], ss); }
      }
    const float rstd = 1.f / sqrtf(ln_sum<LPR>(ss) * inv + a.eps);
    if (row >= a.rows) continue;
    T* yp = (T*)a.y + row * a.C;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * LPR + sub) * EPT;
      if (col < a.C) {
        float o[EPT];
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] = fmaf(x[c][e] * rstd, gm[c][e], bt[c][e]);
        LnVec<T, EPT>::st(yp + col, o);
      }
    }
    if (sub == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
  }
}

// Rows too long for registers: a workgroup a row, the row read three times (the second and third time out of L2).
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void layer_norm_long_kernel(LnArgs a) {
  __shared__ float red[LN_THREADS / 64];
  const float inv = 1.f / (float)a.C;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* xp = (const T*)a.x + row * a.ldx;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += LN_THREADS) s += Elem<T>::ld(xp + c);
    const float mean = ln_block_sum(s, red) * inv;
    float ss = 0.f;
    for (int c = threadIdx.x; c < a.C; c += LN_THREADS) { const float d = Elem<T>::ld(xp + c) - mean; ss = fmaf(d, d, ss); }
    const float rstd = 1.f / sqrtf(ln_block_sum(ss, red) * inv + a.eps);
    T* yp = (T*)a.y + row * a.C;
    for (int c = threadIdx.x; c < a.C; c += LN_THREADS)
      Elem<T>::st(yp + c, fmaf((Elem<T>::ld(xp + c) - mean) * rstd, a.gamma ? a.gamma[c] : 1.f, a.beta ? a.beta[c] : 0.f));
    if (threadIdx.x == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
  }
}

// dx, and this workgroup's share of dgamma / dbeta: a lane keeps the sums of its own columns over all rows it sees; the
// LN_THREADS / LPR lanes that own the same columns are added through LDS in a fixed order (no atomics: repeatable bits).
template <typename T, int EPT, int LPR, int NCH>
__global__ __launch_bounds__(LN_THREADS) void layer_norm_bwd_kernel(LnBwdArgs a) {
  constexpr int RPB = LN_THREADS / LPR;
  __shared__ float red[LN_THREADS * EPT];
  const int sub = threadIdx.x & (LPR - 1);
  float gm[NCH][EPT], dg[NCH][EPT], db[NCH][EPT];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * LPR + sub) * EPT;
#pragma unroll
    for (int e = 0; e < EPT; ++e) { dg[c][e] = 0.f; db[c][e] = 0.f; }
    ln_param(a.gamma, col, a.C, 1.f, gm[c]);
  }
  const float inv = 1.f / (float)a.C;
  typename LnVec<T, EPT>::Raw nx[NCH], ny[NCH];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](long row0) {
    const long row = row0 + threadIdx.x / LPR, r = row < a.rows ? row : 0;
    nmean = a.mean[r];
    nrstd = a.rstd[r];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * LPR + sub) * EPT;
      if (col < a.C) {
        nx[c] = LnVec<T, EPT>::get((const T*)a.x + r * a.ldx + col);
        ny[c] = LnVec<T, EPT>::get((const T*)a.dy + r * a.lddy + col);
      }
    }
  };
  const long first = (long)blockIdx.x * RPB, step = (long)gridDim.x * RPB;
  if (first < a.rows) fetch(first);
  for (long row0 = first; row0 < a.rows; row0 += step) {
    const long row = row0 + threadIdx.x / LPR;
    const bool live = row < a.rows;
    const float mean = nmean, rstd = nrstd;
    float u[NCH][EPT], g[NCH][EPT];
    float sg = 0.f, su = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (live && (c * LPR + sub) * EPT < a.C) {
        LnVec<T, EPT>::split(nx[c], u[c]);
        LnVec<T, EPT>::split(ny[c], g[c]);
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
          u[c][e] = (u[c][e] - mean) * rstd;
          dg[c][e] = fmaf(g[c][e], u[c][e], dg[c][e]);
          db[c][e] += g[c][e];
          g[c][e] *= gm[c][e];
          sg += g[c][e];
          su = fmaf(g[c][e], u[c][e], su);
        }
      }
    }
    if (row0 + step < a.rows) fetch(row0 + step);
    sg = ln_sum<LPR>(sg) * inv;
    su = ln_sum<LPR>(su) * inv;
    if (!live || !a.dx) continue;
    T* op = (T*)a.dx + row * a.C;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * LPR + sub) * EPT;
      if (col < a.C) {
        float o[EPT];
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] = rstd * (g[c][e] - sg - u[c][e] * su);
        LnVec<T, EPT>::st(op + col, o);
      }
    }
  }
  if (!a.part) return;
  const long ps = ln_part_stride(a.C);
  float* part = a.part + (long)blockIdx.x * 2 * ps;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EPT; ++e) red[threadIdx.x * EPT + e] = which ? db[c][e] : dg[c][e];
      __syncthreads();
      for (int k = threadIdx.x; k < LPR * EPT; k += LN_THREADS) {
        const int col = c * LPR * EPT + k;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < RPB; ++q) s += red[q * LPR * EPT + k];
        if (col < a.C) part[which * ps + col] = s;
      }
    }
  }
}

// Long rows: a workgroup a row and step; the sums of the columns live in the workgroup's own slice of `part`.
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void layer_norm_bwd_long_kernel(LnBwdArgs a) {
  __shared__ float red[LN_THREADS / 64];
  const float inv = 1.f / (float)a.C;
  const long ps = ln_part_stride(a.C);
  float* part = a.part ? a.part + (long)blockIdx.x * 2 * ps : nullptr;
  if (part)
    for (int c = threadIdx.x; c < a.C; c += LN_THREADS) { part[c] = 0.f; part[ps + c] = 0.f; }
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* xp = (const T*)a.x + row * a.ldx;
    const T* yp = (const T*)a.dy + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, su = 0.f;
    for (int c = threadIdx.x; c < a.C; c += LN_THREADS) {
      const float dy = Elem<T>::ld(yp + c), u = (Elem<T>::ld(xp + c) - mean) * rstd, g = a.gamma ? dy * a.gamma[c] : dy;
      sg += g;
      su = fmaf(g, u, su);
      if (part) { part[c] = fmaf(dy, u, part[c]); part[ps + c] += dy; }   // (a column belongs to one thread)
    }
    sg = ln_block_sum(sg, red) * inv;
    su = ln_block_sum(su, red) * inv;
    if (!a.dx) continue;
    T* op = (T*)a.dx + row * a.C;
    for (int c = threadIdx.x; c < a.C; c += LN_THREADS) {
      const float dy = Elem<T>::ld(yp + c), u = (Elem<T>::ld(xp + c) - mean) * rstd, g = a.gamma ? dy * a.gamma[c] : dy;
      Elem<T>::st(op + c, rstd * (g - sg - u * su));
    }
  }
}

// dgamma / dbeta = the sum of the workgroups' shares: LN_REDUCE_COLS columns a workgroup, four of them a thread, 64 rows of threads
// striding the shares (512 shares: eight loads a thread, in flight together).  Columns up to the padded stride are read and dropped.
__global__ __launch_bounds__(LN_THREADS) inline void layer_norm_reduce_kernel(const float* part, int shares, int C, float* dgamma,
                                                                              float* dbeta) {
  constexpr int CQ = LN_REDUCE_COLS / 4, RW = LN_THREADS / CQ;
  __shared__ __attribute__((aligned(16))) float red[LN_THREADS * 4];
  float* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  const int k = threadIdx.x % CQ, r = threadIdx.x / CQ;
  const long ps = ln_part_stride(C), col = (long)blockIdx.x * LN_REDUCE_COLS + 4 * k;
  tapir_f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (col < ps) {
#pragma unroll 8
    for (int p = r; p < shares; p += RW) s += ldg_f4(part + ((long)p * 2 + blockIdx.y) * ps + col);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[r * LN_REDUCE_COLS + 4 * k + i] = s[i];
  __syncthreads();
  // 256 threads: 16 a column, then one
  const int q = threadIdx.x / LN_REDUCE_COLS, j = threadIdx.x % LN_REDUCE_COLS;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < RW / (LN_THREADS / LN_REDUCE_COLS); ++i) v += red[(q * (RW / (LN_THREADS / LN_REDUCE_COLS)) + i) * LN_REDUCE_COLS + j];
  __syncthreads();
  red[threadIdx.x] = v;
  __syncthreads();
  const long c = (long)blockIdx.x * LN_REDUCE_COLS + threadIdx.x;
  if (threadIdx.x < LN_REDUCE_COLS && c < C) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < LN_THREADS / LN_REDUCE_COLS; ++i) t += red[i * LN_REDUCE_COLS + threadIdx.x];
    out[c] = t;
  }
}

}  // namespace tapir
