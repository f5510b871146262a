// Rotary positions on queries and keys (gfx950): pair (a, b) of pair index p
// at position n becomes
//   m (a cos t - b sin t,  a sin t + b cos t),   t = n f_p   (backward: -t)
// with pairs (2p, 2p + 1) (interleaved) or (p, p + R/2) of the first R
// channels of a head; the others are copied.  What the model applies to q and
// k before the attention (wan_video_dit.py:699-705), there with one position
// per axis of the video grid and the pairs split over the axes.
//
// Angles: n f / 2 pi is formed in float64 and reduced to a quarter turn there
// (three roundings of half a step: 1.1e-11 turns at n = 200,000, where float32 would
// lose 0.01 rad, and 1.1e-7 at 2^31), then sine and cosine by their Taylor series on
// [-pi/4, pi/4] in float32: four terms past the first each, 2e-9 and 3e-8 off.  No table
// is kept, so any position and any frequencies work.
//
// Bound: HBM (each element read and written once).  A thread owns one 16-byte
// piece of the head (two, half a rotation apart, where the pairs are), computes
// its angles once and walks the heads of q and k with them, four heads in
// flight.  The heads are cut over blockIdx.y until the launch fills the chip.
// Measured: 75,600 tokens of 40 + 40 heads of 128, bf16, three axes 583-606 us (5.1-5.3
// TB/s); 8 tokens 4.8 us.
#include <type_traits>

#include "common.h"
#include "elements.h"

namespace {

constexpr int kThreads = 256, kMaxHeadDim = 256, kMaxAxes = 4;

struct RotaryArgs {
  const void* x[2];                  // q, k: [B, H, S, D], channels adjacent
  void* o[2];
  int64_t xb[2], xh[2], xs[2], ob[2], oh[2], os[2];  // strides in elements
  int H[2];
  int64_t first, tokens;             // of this launch, of B * S
  int S, R, rot_units, units, tpb;   // units of a head: rot_units rotating, then copied; tokens per workgroup
  int heads_per;                     // heads (of q, then k) per blockIdx.y
  const double* freqs;               // [R/2] radians per position
  const void* pos;                   // int32 / int64
  int64_t pb, ps, pa;                // strides of batch, token, axis
  int pos64, axes, axis_end[kMaxAxes];  // pairs below axis_end[a] (and not of an earlier axis) turn with axis a
  float amp;
  double sign;
};

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

// VEC channels per unit (VEC = 1: one pair, or one copied channel, per unit)
template <class E, int VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int NP = VEC == 1 ? 1 : INTER ? VEC / 2 : VEC;  // pairs of a rotating unit
  constexpr int HEADS = 4;
  const int slot = (int)threadIdx.x / a.units, u = (int)threadIdx.x - slot * a.units;
  const int64_t token = a.first + (int64_t)blockIdx.x * a.tpb + slot;
  if (slot >= a.tpb || token >= a.tokens) return;
  const int b = (int)(token / a.S), n = (int)(token - (int64_t)b * a.S);
  const bool rot = u < a.rot_units;
  // first channel of the unit, and of its second piece (half layout; the pair's
  // other channel with VEC = 1)
  const int p0 = u * NP;
  const int c0 = !rot ? a.R + (u - a.rot_units) * VEC : INTER ? 2 * p0 : p0;
  const int c1 = !rot ? c0 : INTER ? 2 * p0 + 1 : p0 + a.R / 2;
  float cs[NP], sn[NP];
  if (rot) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int axis = 0;
      for (int x = 0; x + 1 < a.axes; ++x) axis += p0 + i >= a.axis_end[x];
      const int64_t at = (int64_t)b * a.pb + (int64_t)n * a.ps + (int64_t)axis * a.pa;
      const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
      const double t = pos * (a.freqs[p0 + i] * 0.15915494309189533577);  // turns
      sincos_turns(a.sign * (t - rint(t)), sn[i], cs[i]);
      sn[i] *= a.amp;
      cs[i] *= a.amp;
    }
  }
  typedef Pack<E, VEC> P;
  constexpr bool TWO = VEC == 1 || !INTER;  // two pieces per rotating unit
  auto head = [&](int h, int64_t& src, int64_t& dst, int& t) {
    t = h >= a.H[0];
    const int hh = t ? h - a.H[0] : h;
    src = (int64_t)b * a.xb[t] + (int64_t)hh * a.xh[t] + (int64_t)n * a.xs[t];
    dst = (int64_t)b * a.ob[t] + (int64_t)hh * a.oh[t] + (int64_t)n * a.os[t];
  };
  auto some = [&](int h, auto count) {
    constexpr int C = decltype(count)::value;
    P v0[C], v1[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      int64_t src, dst;
      int t;
      head(h + i, src, dst, t);
      v0[i] = P::load(a.x[t], src + c0);
      if constexpr (TWO) v1[i] = P::load(a.x[t], src + c1);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      int64_t src, dst;
      int t;
      head(h + i, src, dst, t);
      P o0 = v0[i], o1 = v0[i];
      if constexpr (TWO) o1 = v1[i];
      if (rot) {
        if constexpr (TWO) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const float x = v0[i].get(k), y = v1[i].get(k);
            o0.set(k, __builtin_fmaf(x, cs[k], -(y * sn[k])));
            o1.set(k, __builtin_fmaf(x, sn[k], y * cs[k]));
          }
        } else {
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            const float x = v0[i].get(2 * k), y = v0[i].get(2 * k + 1);
            o0.set(2 * k, __builtin_fmaf(x, cs[k], -(y * sn[k])));
            o0.set(2 * k + 1, __builtin_fmaf(x, sn[k], y * cs[k]));
          }
        }
      }
      o0.store(a.o[t], dst + c0);
      if constexpr (TWO)
        if (rot) o1.store(a.o[t], dst + c1);
    }
  };
  const int all = a.H[0] + a.H[1];
  int h = (int)blockIdx.y * a.heads_per;
  const int end = h + a.heads_per < all ? h + a.heads_per : all;
  for (; h + HEADS <= end; h += HEADS) some(h, std::integral_constant<int, HEADS>{});
  for (; h < end; ++h) some(h, std::integral_constant<int, 1>{});
}

template <class E, int VEC>
void launch_rotary(RotaryArgs a, int D, bool inter, hipStream_t stream) {
  const int np = VEC == 1 ? 1 : inter ? VEC / 2 : VEC;
  a.rot_units = a.R / 2 / np;
  a.units = a.rot_units + (D - a.R) / VEC;
  a.tpb = kThreads / a.units;
  const int64_t gx = (a.tokens + a.tpb - 1) / a.tpb;
  // heads per workgroup: all of them where the tokens alone give eight
  // workgroups a CU (2,048), else as few as that takes
  const int all = a.H[0] + a.H[1];
  const int64_t slices = gx >= 2048 ? 1 : (2048 + gx - 1) / gx;
  a.heads_per = slices >= all ? 1 : (int)((all + slices - 1) / slices);
  const unsigned grid_y = (unsigned)((all + a.heads_per - 1) / a.heads_per);
  const int64_t most = PRISM_MAX_THREADS / 2 / kThreads;  // workgroups at a time
  for (int64_t at = 0; at < gx; at += most) {
    const dim3 part((unsigned)(gx - at < most ? gx - at : most), grid_y);
    a.first = at * a.tpb;
    if (inter) rotary_kernel<E, VEC, true><<<part, kThreads, 0, stream>>>(a);
    else rotary_kernel<E, VEC, false><<<part, kThreads, 0, stream>>>(a);
  }
}

template <class E>
void launch_rotary_vec(const RotaryArgs& a, int D, bool inter, hipStream_t stream) {
  constexpr int ES = (int)sizeof(typename E::type);
  // the widest piece that every unit, stride and pointer is a multiple of
  auto fits = [&](int vec) {
    if (D % vec || (inter ? a.R % vec : (a.R / 2) % vec)) return false;
    for (int t = 0; t < 2; ++t) {
      if (!a.H[t]) continue;
      if ((uintptr_t)a.x[t] % (vec * ES) || (uintptr_t)a.o[t] % (vec * ES)) return false;
      for (int64_t s : {a.xb[t], a.xh[t], a.xs[t], a.ob[t], a.oh[t], a.os[t]})
        if (s % vec) return false;
    }
    return true;
  };
  if (fits(16 / ES)) launch_rotary<E, 16 / ES>(a, D, inter, stream);
  else if (fits(8 / ES)) launch_rotary<E, 8 / ES>(a, D, inter, stream);
  else launch_rotary<E, 1>(a, D, inter, stream);
}

}  // namespace

extern "C" int prism_rotary(const void* q, const void* k, int dtype, int B, int64_t S, int Hq, int Hk, int D, int R,
                            const int64_t* strides, const double* freqs, const void* pos, int pos64,
                            const int64_t* pos_strides, int axes, const int32_t* axis_end, int interleaved,
                            float amplitude, int inverse, void* out_q, void* out_k, hipStream_t stream) {
  PRISM_REQUIRE(dtype >= PRISM_F32 && dtype <= PRISM_F16, "prism_rotary: dtype code %d unknown", dtype);
  PRISM_REQUIRE(B >= 0 && S >= 0 && S < (1ll << 31) && Hq >= 0 && Hk >= 0 && Hq + (int64_t)Hk < (1 << 16),
                "prism_rotary: sizes out of range");
  PRISM_REQUIRE(D >= 2 && D <= kMaxHeadDim, "prism_rotary: head dim %d must be 2 to %d", D, kMaxHeadDim);
  PRISM_REQUIRE(R >= 2 && R <= D && R % 2 == 0, "prism_rotary: rotary dim %d must be even, 2 to the head dim", R);
  PRISM_REQUIRE(axes >= 1 && axes <= kMaxAxes, "prism_rotary: 1 to %d axes", kMaxAxes);
  if (B == 0 || S == 0 || Hq + Hk == 0) return PRISM_OK;
  PRISM_REQUIRE((!Hq || (q && out_q)) && (!Hk || (k && out_k)) && strides && freqs && pos && pos_strides && axis_end,
                "prism_rotary: null pointer");
  PRISM_REQUIRE(axis_end[axes - 1] == R / 2, "prism_rotary: the axes must share out all %d pairs", R / 2);
  PRISM_REQUIRE((int64_t)B * S < (1ll << 31), "prism_rotary: too many tokens");
  RotaryArgs a{};
  a.x[0] = q; a.x[1] = k; a.o[0] = out_q; a.o[1] = out_k;
  for (int t = 0; t < 2; ++t) {
    const int64_t* s = strides + 6 * t;
    a.xb[t] = s[0]; a.xh[t] = s[1]; a.xs[t] = s[2]; a.ob[t] = s[3]; a.oh[t] = s[4]; a.os[t] = s[5];
  }
  a.H[0] = Hq; a.H[1] = Hk;
  a.tokens = (int64_t)B * S; a.S = (int)S; a.R = R;
  a.freqs = freqs; a.pos = pos; a.pos64 = pos64;
  a.pb = pos_strides[0]; a.ps = pos_strides[1]; a.pa = pos_strides[2];
  a.axes = axes;
  for (int x = 0; x < axes; ++x) a.axis_end[x] = axis_end[x];
  a.amp = amplitude; a.sign = inverse ? -1.0 : 1.0;
  if (dtype == PRISM_F32) launch_rotary_vec<ElemF32>(a, D, interleaved != 0, stream);
  else if (dtype == PRISM_BF16) launch_rotary_vec<ElemBf16>(a, D, interleaved != 0, stream);
  else launch_rotary_vec<ElemF16>(a, D, interleaved != 0, stream);
  PRISM_LAUNCH_CHECK("prism_rotary");
  return PRISM_OK;
}
