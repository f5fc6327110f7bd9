// Rotary positions of several axes: the channels of a head are split into one section per axis (time, height, width, ...), and
// pair i of a section of width w is turned by the angle  p base^(-2 i / w),  p the token's position on that axis (any real
// number: frame index, pixel coordinate of a point between cells):
//   (a, b) -> (a cos - b sin, a sin + b cos);   the gradient is the same map with -sin.
// The two channels of a pair are neighbours (interleaved) or i and i + w / 2 of the section (halves).  Channels behind the last
// section pass through.  Angles: turns = p * (base^(-2i/w) / 2 pi) in 64 bits (a product in 32 bits is off by 6e-3 at the
// hundred-thousandth frame), reduced there to [-1/2, 1/2], sine and cosine of the rest in 32 bits.
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

// cos and sin of 2 pi r.  r in turns: reduced to a quarter turn, then Taylor's polynomials on |t| <= pi/4 (first dropped
// terms: t^10/10! < 2.5e-8 relative to cos, t^11/11! < 2e-9).
__device__ __forceinline__ void rot_sincos(double turns, float* sn, float* cs) {
  const double w = turns - rint(turns);
  const float r = (float)w;
  const float k = rintf(4.f * r);
  const float t = (r - 0.25f * k) * 6.28318530717958647692f;   // r - k/4 is exact
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

// One thread a (token, pair): the angle is worked out once and serves all heads.  The channels behind the sections are copied by
// the threads past the last pair.
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

}  // namespace tapir
