// Angles of rotary positions (headnorm.hip, paged.hip; rotary.hip takes the sines and keeps its
// own places): pair p of a token at position n turns by n f_p, positions with one entry per axis
// of a grid.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// sine and cosine of t turns
__device__ __forceinline__ void sincos_turns(double t, float& s, float& c) {
  const double q = rint(4.0 * t);
  const float x = (float)(t - 0.25 * q) * 6.28318530717958647692f;
  const float z = x * x;
  float ps = 2.75573192e-6f;                       // 1/9!
  ps = __builtin_fmaf(ps, z, -1.98412698e-4f);     // 1/7!
  ps = __builtin_fmaf(ps, z, 8.33333333e-3f);      // 1/5!
  ps = __builtin_fmaf(ps, z, -1.66666667e-1f);     // 1/3!
  ps = __builtin_fmaf(ps * z, x, x);
  float pc = 2.48015873e-5f;                       // 1/8!
  pc = __builtin_fmaf(pc, z, -1.38888889e-3f);     // 1/6!
  pc = __builtin_fmaf(pc, z, 4.16666667e-2f);      // 1/4!
  pc = __builtin_fmaf(pc, z, -0.5f);
  pc = __builtin_fmaf(pc, z, 1.0f);
  const int k = (int)(q - 4.0 * floor(0.25 * q));  // quarter turns mod 4
  const float a = (k & 1) ? pc : ps, b = (k & 1) ? ps : pc;
  s = (k & 2) ? -a : a;
  c = (k == 1 || k == 2) ? -b : b;
}

// the same in float64 (series to 1/15! and 1/16!: 5e-17 off on [-pi/4, pi/4])
__device__ __forceinline__ void sincos_turns(double t, double& s, double& c) {
  const double q = rint(4.0 * t);
  const double x = (t - 0.25 * q) * 6.28318530717958647692, z = x * x;
  double ps = -1.0 / 1307674368000.0;
  ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);
  ps = __builtin_fma(ps, z, -1.0 / 39916800.0);
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  ps = __builtin_fma(ps * z, x, x);
  double pc = 1.0 / 20922789888000.0;
  pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);
  pc = __builtin_fma(pc, z, 1.0 / 479001600.0);
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  pc = __builtin_fma(pc, z, -0.5);
  pc = __builtin_fma(pc, z, 1.0);
  const int k = (int)(q - 4.0 * floor(0.25 * q));
  const double a = (k & 1) ? pc : ps, b = (k & 1) ? ps : pc;
  s = (k & 2) ? -a : a;
  c = (k == 1 || k == 2) ? -b : b;
}

constexpr int kMaxAxes = 4;

struct Angles {
  const double* freqs;               // [pairs] radians per position
  const void* pos;                   // int32 / int64
  int64_t pb, ps, pa;                // strides of batch, token, axis
  int pos64, axes, axis_end[kMaxAxes];  // pairs below axis_end[a] (and not of an earlier axis) turn with axis a
  double amp;
  double sign;                       // -1: backwards
  // position of token n of sequence b as pair p takes it
  __device__ __forceinline__ double place(int b, int n, int p) const {
    int axis = 0;
    for (int x = 0; x + 1 < axes; ++x) axis += p >= axis_end[x];
    const int64_t i = (int64_t)b * pb + (int64_t)n * ps + (int64_t)axis * pa;
    return pos64 ? (double)((const int64_t*)pos)[i] : (double)((const int32_t*)pos)[i];
  }
  // sine and cosine, times amp, of pair p at that position (float or double)
  template <class F>
  __device__ __forceinline__ void turned(double at, int p, F& s, F& c) const {
    const double t = at * (freqs[p] * 0.15915494309189533577);  // turns
    sincos_turns(sign * (t - rint(t)), s, c);
    s *= (F)amp;
    c *= (F)amp;
  }
  __device__ __forceinline__ void at(int b, int n, int p, float& s, float& c) const { turned(place(b, n, p), p, s, c); }
};
