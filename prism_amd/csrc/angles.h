// Angles of rotary positions (rotary.hip, headnorm.hip, paged.hip): pair p of a
// token at position n turns by n f_p, positions with one entry per axis of a grid.
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

constexpr int kMaxAxes = 4;

struct Angles {
  const double* freqs;               // [pairs] radians per position
  const void* pos;                   // int32 / int64
  int64_t pb, ps, pa;                // strides of batch, token, axis
  int pos64, axes, axis_end[kMaxAxes];  // pairs below axis_end[a] (and not of an earlier axis) turn with axis a
  float amp;
  double sign;                       // -1: backwards
  // sine and cosine, times amp, of pair p of token n of sequence b
  __device__ __forceinline__ void at(int b, int n, int p, float& s, float& c) const {
    int axis = 0;
    for (int x = 0; x + 1 < axes; ++x) axis += p >= axis_end[x];
    const int64_t i = (int64_t)b * pb + (int64_t)n * ps + (int64_t)axis * pa;
    const double at = pos64 ? (double)((const int64_t*)pos)[i] : (double)((const int32_t*)pos)[i];
    const double t = at * (freqs[p] * 0.15915494309189533577);  // turns
    sincos_turns(sign * (t - rint(t)), s, c);
    s *= amp;
    c *= amp;
  }
};
