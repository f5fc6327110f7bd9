// Rotary positions of several axes: the channels of a head are split into one section per axis (time, height, width, ...), and
// pair i of a section of width w is turned by the angle  p base^(-2 i / w),  p the token's position on that axis (any real
// number: frame index, pixel coordinate of a point between cells):
//   (a, b) -> (a cos - b sin, a sin + b cos);   the gradient is the same map with -sin.
// The two channels of a pair are neighbours (interleaved) or i and i + w / 2 of the section (halves).  Channels behind the last
// section pass through.  Angles: turns = p * (base^(-2i/w) / 2 pi) in 64 bits (a product in 32 bits is off by 6e-3 at the
// hundred-thousandth frame), reduced there to an eighth of a turn, sine and cosine of the rest in 32 bits.
#pragma once
#include "common.hpp"

namespace tapir {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_PAIRS = 128;   // head dim <= 256
constexpr int ROT_MAX_AXES = 4;

struct RotaryArgs {
  const void* x; long sb, sn, sh;      // [B, N, H, D] strides in elements, last axis dense
  const float* pos; long pb;           // [B or 1, N, axes] dense, clip stride (0: shared)
  void* y;                             // [B, N, H, D] dense
  long B, N; int H, D, axes, pairs;    // pairs: rotated pairs of a head
  float sign;                          // +1 forward, -1 gradient
  double turns[ROT_MAX_PAIRS];         // base^(-2i/w) / 2 pi of every pair
  unsigned char axis[ROT_MAX_PAIRS], lo[ROT_MAX_PAIRS], hi[ROT_MAX_PAIRS];   // its axis and its two channels (< 256)
};

// cos and sin of 2 pi r.  r in turns: reduced to a quarter turn and scaled in 64 bits, rounded once (half a step of t), then Taylor's
// polynomials on |t| <= pi/4 (first dropped terms, absolute: t^10/10! < 2.5e-8, t^11/11! < 2e-9).  Off by less than 1.7 * 2^-24; with the
// turn rounded to 32 bits before the reduction it was 2.3 * 2^-24.
__device__ __forceinline__ void rot_sincos(double turns, float* sn, float* cs) {
  const double w = turns - rint(turns), k = rint(4.0 * w);
  const float t = (float)((w - 0.25 * k) * 6.283185307179586476925286766559);   // w - k/4 is exact
  const float t2 = t * t;
  float s = 2.7557319e-6f;
  s = fmaf(s, t2, -1.9841270e-4f); s = fmaf(s, t2, 8.3333333e-3f); s = fmaf(s, t2, -1.6666667e-1f);
  s = fmaf(s * t2, t, t);
  float c = 2.4801587e-5f;
  c = fmaf(c, t2, -1.3888889e-3f); c = fmaf(c, t2, 4.1666667e-2f); c = fmaf(c, t2, -0.5f);
  c = fmaf(c, t2, 1.f);
  const int q = (int)k & 3;
  const float a = (q & 1) ? c : s, b = (q & 1) ? s : c;
  *sn = (q & 2) ? -a : a;
  *cs = (q == 1 || q == 2) ? -b : b;
}

// Orders a wave's own LDS traffic (in order in hardware) for the compiler, whatever the accesses' types.
__device__ __forceinline__ void rot_wave_fence() {
  wave_sync();
#ifndef TAPIR_HIPEMU
  asm volatile("" ::: "memory");
#endif
}

template <typename T> struct RotVec;   // 16 bytes as floats and back
template <> struct RotVec<float> {
  static __device__ __forceinline__ void split(const uint4& r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 join(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct RotVec<bf16_t> {
  static __device__ __forceinline__ void split(const uint4& r, float (&v)[8]) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ uint4 join(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};

// One thread a (token, pair), for rows that are not whole 16-byte pieces: the angle is worked out once and serves all heads.  The
// channels behind the sections are copied by the threads past the last pair.
template <typename T>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotaryArgs a) {
  const int per = a.pairs + (a.D - 2 * a.pairs);   // threads a token
  const long total = a.B * a.N * per;
  for (long t = (long)blockIdx.x * ROT_THREADS + threadIdx.x; t < total; t += (long)gridDim.x * ROT_THREADS) {
    const long token = t / per;
    const int p = (int)(t - token * per);
    const long b = token / a.N, n = token - b * a.N;
    const T* x = (const T*)a.x + b * a.sb + n * a.sn;
    T* y = (T*)a.y + token * a.H * a.D;
    if (p < a.pairs) {
      const float at = a.pos[b * a.pb + n * a.axes + a.axis[p]];
      float sn, cs;
      rot_sincos((double)at * a.turns[p], &sn, &cs);
      sn *= a.sign;
      const int lo = a.lo[p], hi = a.hi[p];
      for (int h = 0; h < a.H; ++h) {
        const float u = Elem<T>::ld(x + h * a.sh + lo), v = Elem<T>::ld(x + h * a.sh + hi);
        Elem<T>::st(y + (long)h * a.D + lo, fmaf(u, cs, -v * sn));
        Elem<T>::st(y + (long)h * a.D + hi, fmaf(u, sn, v * cs));
      }
    } else {
      const int c = a.pairs + p;
      for (int h = 0; h < a.H; ++h) y[(long)h * a.D + c] = x[h * a.sh + c];
    }
  }
}

// The same, 16 bytes a lane: D / EPC lanes hold a row, a wave R = 64 / (D / EPC) tokens.  A lane works out the cosines and sines of
// its channels once and takes `heads` heads with them, ROT_HEADS at a time: their loads are in flight together, each row goes
// through LDS once (the other channel of a pair lies anywhere in it) and is stored in whole lanes.  Bound: HBM, the tensor read and
// written once: 2 x 49152 x 4 x 64 bf16 22.9 us = 4.4 TB/s (35 us with two bytes a lane).
constexpr int ROT_HEADS = 4;

struct RotaryRowArgs {
  const void* x; long sb, sn, sh;
  const float* pos; long pb;
  void* y;
  long B, N; int H, D, axes, heads;    // heads: of a workgroup (blockIdx.y takes the next ones)
  float sign;
  double turns[2 * ROT_MAX_PAIRS];     // of every channel
  unsigned char axis[2 * ROT_MAX_PAIRS], other[2 * ROT_MAX_PAIRS];   // its axis and the pair's other channel (itself: not turned)
};

template <typename T>
__global__ __launch_bounds__(ROT_THREADS) void rotary_rows_kernel(RotaryRowArgs a) {
  constexpr int EPC = 16 / (int)sizeof(T);
  __shared__ double turns[2 * ROT_MAX_PAIRS];
  __shared__ unsigned char axis[2 * ROT_MAX_PAIRS], other[2 * ROT_MAX_PAIRS];
  __shared__ __attribute__((aligned(16))) T rows[ROT_THREADS / 64][ROT_HEADS][64 * EPC];
  if ((int)threadIdx.x < a.D) {
    turns[threadIdx.x] = a.turns[threadIdx.x];
    axis[threadIdx.x] = a.axis[threadIdx.x];
    other[threadIdx.x] = a.other[threadIdx.x];
  }
  __syncthreads();
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int per = a.D / EPC, R = 64 / per, r = l / per, c0 = (l - r * per) * EPC;
  const long tokens = a.B * a.N, step = (long)gridDim.x * (ROT_THREADS / 64) * R;
  const double per_clip = 1.0 / (double)a.N;
  const int h0 = blockIdx.y * a.heads, h1 = h0 + a.heads < a.H ? h0 + a.heads : a.H;
  for (long first = ((long)blockIdx.x * (ROT_THREADS / 64) + w) * R; first < tokens; first += step) {
    const long token = first + r;
    const bool live = r < R && token < tokens;
    const long t = live ? token : 0;
    const long b = (long)(((double)t + 0.5) * per_clip), n = t - b * a.N;   // (exact: the half outweighs the rounding, t < 2^50)
    const T* const x = (const T*)a.x + b * a.sb + n * a.sn + c0;
    T* const y = (T*)a.y + t * a.H * a.D + c0;
    uint4 raw[ROT_HEADS];
#pragma unroll
    for (int u = 0; u < ROT_HEADS; ++u)
      if (live && h0 + u < h1) raw[u] = ldg16(x + (h0 + u) * a.sh);
    float cs[EPC], sn[EPC];
    int at[EPC];
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
      const int c = live ? c0 + e : 0;
      rot_sincos((double)a.pos[b * a.pb + n * a.axes + axis[c]] * turns[c], &sn[e], &cs[e]);
      const int o = other[c];
      sn[e] = o > c ? -a.sign * sn[e] : a.sign * sn[e];
      at[e] = o == c ? -1 : (r * per * EPC) + o;
    }
    for (int h = h0; h < h1; h += ROT_HEADS) {
#pragma unroll
      for (int u = 0; u < ROT_HEADS; ++u) {
        if (h > h0 && live && h + u < h1) raw[u] = ldg16(x + (h + u) * a.sh);
      }
      rot_wave_fence();
#pragma unroll
      for (int u = 0; u < ROT_HEADS; ++u)
        if (live && h + u < h1) *reinterpret_cast<uint4*>(&rows[w][u][l * EPC]) = raw[u];
      rot_wave_fence();
#pragma unroll
      for (int u = 0; u < ROT_HEADS; ++u) {
        if (!live || h + u >= h1) continue;
        float v[EPC];
        RotVec<T>::split(raw[u], v);
#pragma unroll
        for (int e = 0; e < EPC; ++e)
          if (at[e] >= 0) v[e] = fmaf(v[e], cs[e], Elem<T>::ld(&rows[w][u][at[e]]) * sn[e]);
        *reinterpret_cast<uint4*>(y + (long)(h + u) * a.D) = RotVec<T>::join(v);
      }
    }
  }
}

}  // namespace tapir
