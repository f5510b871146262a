// Root-mean-square norm of every query and key head, and its rotary positions, in
// one pass (gfx950):
//
//   inv = (mean(x^2) + eps)^-1/2,  y = m R(t) (x inv w)
//
// over the D channels of a head, R(t) turning the pairs of its first R channels as
// rotary.hip does (interleaved, or half a rotation apart).  Backward:
//
//   g = m R(-t) dy,  dx = inv (g w - x inv mean(g w x inv)),  dw = sum g x inv
//
// summed over tokens and heads.  Sums are fp32; y and dx are rounded once.
//
// Bound: HBM (each element read and written once, x and dy read in the backward).
// A head lies across lanes of one wave, 16 bytes a lane (bf16, D = 128: 16 lanes, so a
// wave holds four tokens' heads): its sum takes shuffles and no LDS, the other half
// of a rotation comes from the lane that holds it, and a lane keeps the angles of
// its token while it walks the heads, four in flight.  The backward's workgroups
// walk the tokens (kParts of them at most), keep dw of their lanes' channels in
// registers and leave one partial row each, which a second kernel adds in order: no
// atomics, the same bits every time.  Heads that are not whole pieces (odd sizes,
// unaligned rows) take one wave a row and single elements.
//
// Measured (bf16): 75,600 tokens, 40 + 40 heads of 128: 622 us, 3.03 GB, 4.9 TB/s (a copy
// of them runs at 4.8); loading the first heads before the angles: 678 us.  16 tokens, 32 +
// 8 heads: 6.5 us, the launch and its one trip to memory.  9,998 tokens, 16 + 4 heads of 64,
// 32 channels turning: forward 18.7 us (2.7 TB/s), backward 24.0 (3.2 TB/s) and 4.6 for the
// weights: the forward's 1,252 workgroups are 1.2 rounds (four a CU, 104 registers), the backward's
// 939 one; the vector unit issues 55% of the time (float64 angles, formed by every slice of heads
// anew; conversions), the rest waits for their first loads.
#include <type_traits>

#include "angles.h"
#include "common.h"
#include "elements.h"

namespace {

constexpr int kThreads = 256, kMaxHeadDim = 256, kParts = PRISM_HEAD_PARTS;

struct HeadArgs {
  const void* x[2];                  // q, k: [B, H, S, D], channels adjacent
  const void* g[2];                  // backward: gradients of y
  void* o[2];                        // y, backward: dx
  int64_t xb[2], xh[2], xs[2], gb[2], gh[2], gs[2], ob[2], oh[2], os[2];  // strides in elements
  const void* w[2];                  // [D] or null (ones)
  int w32;                           // weights are fp32 (else of x's type)
  int H[2];
  int64_t first, tokens;             // of this launch, of B * S
  int S, D, R, lanes, tpb;           // lanes of a head (a power of two), tokens per workgroup
  int heads_per;                     // heads (of q, then k) per blockIdx.y
  float eps;
  Angles at;
  float* partial;                    // backward: [2][parts][D]
  int parts;
};

template <class E>
__device__ __forceinline__ float weight_at(const HeadArgs& a, int t, int c) {
  if (!a.w[t]) return 1.0f;
  return a.w32 ? ((const float*)a.w[t])[c] : E::to_float(((const typename E::type*)a.w[t])[c]);
}

// The sines and cosines of a workgroup's tokens, [token][pair] in LDS, by all its threads:
// half a rotation apart two lanes need the same ones, and where a part of the head turns
// the other lanes have none (9,998 tokens of 16 + 4 heads of 64, 32 channels turning:
// forward 22.7 us with every lane's own, 18.7 with these, the sums below and fewer slices;
// backward 38.2 and 24.0)
template <int VEC>
__device__ __forceinline__ void put_angles(const HeadArgs& a, int64_t first, float2* table) {
  const int pairs = a.R >> 1;
  for (int x = (int)threadIdx.x; x < a.tpb * pairs; x += kThreads) {
    const int slot = x / pairs, p = x - slot * pairs;
    const int64_t token = first + slot < a.tokens ? first + slot : a.tokens - 1;
    const int b = (int)(token / a.S);
    a.at.at(b, (int)(token - (int64_t)b * a.S), p, table[x].x, table[x].y);
  }
}

// a lane's channels [c0, c0 + VEC) of a head: cosines and signed sines, and the lane
// that holds the pairs' other channels
template <int VEC, bool INTER>
struct LaneTurn {
  float cs[INTER ? VEC / 2 : VEC], sn[INTER ? VEC / 2 : VEC];
  int other;   // (half a rotation apart)
  bool turns;  // the lane's channels turn (a rotation ends between lanes)
  __device__ __forceinline__ void init(const HeadArgs& a, const float2* table, int slot, int u) {
    const int c0 = u * VEC, half = a.R / 2;
    const bool rot = c0 < a.R, upper = !INTER && c0 >= half;
    turns = rot;
    other = (int)threadIdx.x & 63;
    if (!INTER && rot) other += upper ? -(half / VEC) : half / VEC;
    const float2* mine = table + slot * half + (INTER ? c0 / 2 : upper ? c0 - half : c0);
#pragma unroll
    for (int i = 0; i < (INTER ? VEC / 2 : VEC); ++i) {
      cs[i] = 1.0f;
      sn[i] = 0.0f;
      if (rot) {
        sn[i] = INTER || upper ? mine[i].x : -mine[i].x;
        cs[i] = mine[i].y;
      }
    }
  }
  // v turned; p: the other channels' values (half a rotation apart)
  __device__ __forceinline__ void turn(float* v, const float* p) const {
    if constexpr (INTER) {
      if (!turns) return;  // (0 times an infinity beside it would make a channel NaN)
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float x = v[2 * i], y = v[2 * i + 1];
        v[2 * i] = __builtin_fmaf(x, cs[i], -(y * sn[i]));
        v[2 * i + 1] = __builtin_fmaf(x, sn[i], y * cs[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __builtin_fmaf(v[i], cs[i], p[i] * sn[i]);
    }
  }
};

// the piece that lane `lane` holds
template <class P>
__device__ __forceinline__ P from_lane(const P& v, int lane) {
  P r;
  if constexpr (sizeof(P) == 16) {
    r.w = make_uint4(__shfl(v.w.x, lane, 64), __shfl(v.w.y, lane, 64), __shfl(v.w.z, lane, 64), __shfl(v.w.w, lane, 64));
  } else {
    r.w = make_uint2(__shfl(v.w.x, lane, 64), __shfl(v.w.y, lane, 64));
  }
  return r;
}
// the sums of C values over the lanes of a head, in every one of them.  The values go
// through each step together (a step alone waits for the one before), by data-parallel
// moves inside a row of 16 lanes (after two steps a quad's lanes agree, so mirrors do)
template <int C>
__device__ __forceinline__ void head_sums(float* v, int lanes) {
  auto add = [&](auto ctrl) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      v[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v[i]), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if (lanes > 1) add(std::integral_constant<int, 0xb1>{});   // quad_perm [1, 0, 3, 2]
  if (lanes > 2) add(std::integral_constant<int, 0x4e>{});   // quad_perm [2, 3, 0, 1]
  if (lanes > 4) add(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if (lanes > 8) add(std::integral_constant<int, 0x140>{});  // row_mirror
  if (lanes > 16) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  }
  if (lanes > 32) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = xor32_add(v[i]);
  }
}

__device__ __forceinline__ float head_sum(float v) {
  head_sums<1>(&v, 64);
  return v;
}

// the heads [h, end) of tensor t that a slice of a.heads_per heads of q, then k, holds
__device__ __forceinline__ void slice_of(const HeadArgs& a, int t, int& h, int& end) {
  const int s0 = (int)blockIdx.y * a.heads_per - (t ? a.H[0] : 0), s1 = s0 + a.heads_per;
  h = s0 > 0 ? s0 : 0;
  end = s1 < a.H[t] ? s1 : a.H[t];
}

template <class E, int VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void head_norm_kernel(HeadArgs a) {
  typedef Pack<E, VEC> P;
  constexpr int HEADS = 4;
  const int u = (int)threadIdx.x & (a.lanes - 1), slot = (int)threadIdx.x / a.lanes;
  int64_t token = a.first + (int64_t)blockIdx.x * a.tpb + slot;
  const bool live = u * VEC < a.D && token < a.tokens;
  token = token < a.tokens ? token : a.tokens - 1;  // (every lane takes part in the shuffles)
  const int b = (int)(token / a.S), n = (int)(token - (int64_t)b * a.S), c0 = u * VEC;
  __shared__ float2 table[kThreads / 2 * VEC];  // (tokens x pairs: at most lanes x VEC / 2 pairs)
  put_angles<VEC>(a, a.first + (int64_t)blockIdx.x * a.tpb, table);
  __syncthreads();
  LaneTurn<VEC, INTER> turn;
  turn.init(a, table, slot, u);
  const float per = 1.0f / (float)a.D;
#pragma unroll 1
  for (int t = 0; t < 2; ++t) {
    int h, end;
    slice_of(a, t, h, end);
    if (h >= end) continue;
    float w[VEC], wp[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = wp[i] = c0 < a.D ? weight_at<E>(a, t, c0 + i) : 0.0f;
    if constexpr (!INTER)
#pragma unroll
      for (int i = 0; i < VEC; ++i) wp[i] = __shfl(w[i], turn.other, 64);
    const int64_t src = (int64_t)b * a.xb[t] + (int64_t)n * a.xs[t] + c0;
    const int64_t dst = (int64_t)b * a.ob[t] + (int64_t)n * a.os[t] + c0;
    auto some = [&](auto count) {
      constexpr int C = decltype(count)::value;
      P v[C];
#pragma unroll
      for (int i = 0; i < C; ++i) {
#pragma unroll
        for (int x = 0; x < VEC; ++x) v[i].set(x, 0.0f);
        if (live) v[i] = P::load(a.x[t], src + (int64_t)(h + i) * a.xh[t]);
      }
      float inv[C];
#pragma unroll
      for (int i = 0; i < C; ++i) {
        inv[i] = 0.0f;
#pragma unroll
        for (int x = 0; x < VEC; ++x) inv[i] = __builtin_fmaf(v[i].get(x), v[i].get(x), inv[i]);
      }
      head_sums<C>(inv, a.lanes);
#pragma unroll
      for (int i = 0; i < C; ++i) inv[i] = 1.0f / sqrtf(__builtin_fmaf(inv[i], per, a.eps));
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float f[VEC], p[VEC];
        if constexpr (!INTER) {
          const P o = from_lane(v[i], turn.other);
#pragma unroll
          for (int x = 0; x < VEC; ++x) p[x] = o.get(x) * inv[i] * wp[x];
        }
#pragma unroll
        for (int x = 0; x < VEC; ++x) f[x] = v[i].get(x) * inv[i] * w[x];
        turn.turn(f, p);
        P o;
#pragma unroll
        for (int x = 0; x < VEC; ++x) o.set(x, f[x]);
        if (live) o.store(a.o[t], dst + (int64_t)(h + i) * a.oh[t]);
      }
    };
    for (; h + HEADS <= end; h += HEADS) some(std::integral_constant<int, HEADS>{});
    for (; h + 2 <= end; h += 2) some(std::integral_constant<int, 2>{});
    if (h < end) some(std::integral_constant<int, 1>{});
  }
}

template <class E, int VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void head_norm_bwd_kernel(HeadArgs a) {
  typedef Pack<E, VEC> P;
  constexpr int HEADS = 2;
  __shared__ float red[kThreads * VEC];
  float2* const table = reinterpret_cast<float2*>(red);  // (until the sums at the end)
  const int u = (int)threadIdx.x & (a.lanes - 1), slot = (int)threadIdx.x / a.lanes, c0 = u * VEC;
  const float per = 1.0f / (float)a.D;
  const int64_t blocks = (a.tokens + a.tpb - 1) / a.tpb;
#pragma unroll 1
  for (int t = 0; t < 2; ++t) {
    int h0, end;
    slice_of(a, t, h0, end);
    float w[VEC], dw[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      w[i] = h0 < end && c0 < a.D ? weight_at<E>(a, t, c0 + i) : 0.0f;
      dw[i] = 0.0f;
    }
    for (int64_t block = blockIdx.x; h0 < end && block < blocks; block += gridDim.x) {
      int64_t token = block * a.tpb + slot;
      const bool live = c0 < a.D && token < a.tokens;
      token = token < a.tokens ? token : a.tokens - 1;
      const int b = (int)(token / a.S), n = (int)(token - (int64_t)b * a.S);
      __syncthreads();  // (nobody reads the last tokens' angles any more)
      put_angles<VEC>(a, block * a.tpb, table);
      __syncthreads();
      LaneTurn<VEC, INTER> turn;
      turn.init(a, table, slot, u);
      const int64_t src = (int64_t)b * a.xb[t] + (int64_t)n * a.xs[t] + c0;
      const int64_t grad = (int64_t)b * a.gb[t] + (int64_t)n * a.gs[t] + c0;
      const int64_t dst = (int64_t)b * a.ob[t] + (int64_t)n * a.os[t] + c0;
      int h = h0;
      auto some = [&](auto count) {
        constexpr int C = decltype(count)::value;
        P v[C], g[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            v[i].set(x, 0.0f);
            g[i].set(x, 0.0f);
          }
          if (live) {
            v[i] = P::load(a.x[t], src + (int64_t)(h + i) * a.xh[t]);
            g[i] = P::load(a.g[t], grad + (int64_t)(h + i) * a.gh[t]);
          }
        }
        float f[C][VEC], sums[2 * C];  // gradients turned back; sums of x^2 and of g w x
#pragma unroll
        for (int i = 0; i < C; ++i) {
          float p[VEC];
          if constexpr (!INTER) {
            const P o = from_lane(g[i], turn.other);
#pragma unroll
            for (int x = 0; x < VEC; ++x) p[x] = o.get(x);
          }
          sums[2 * i] = sums[2 * i + 1] = 0.0f;
#pragma unroll
          for (int x = 0; x < VEC; ++x) f[i][x] = g[i].get(x);
          turn.turn(f[i], p);  // (angles of the other sign)
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            const float y = v[i].get(x);
            sums[2 * i] = __builtin_fmaf(y, y, sums[2 * i]);
            sums[2 * i + 1] = __builtin_fmaf(f[i][x] * w[x], y, sums[2 * i + 1]);
          }
        }
        head_sums<2 * C>(sums, a.lanes);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float inv = 1.0f / sqrtf(__builtin_fmaf(sums[2 * i], per, a.eps)), mean = sums[2 * i + 1] * inv * per;
          P o;
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            const float xh = v[i].get(x) * inv;
            if (live) dw[x] = __builtin_fmaf(f[i][x], xh, dw[x]);
            o.set(x, inv * __builtin_fmaf(-xh, mean, f[i][x] * w[x]));
          }
          if (live) o.store(a.o[t], dst + (int64_t)(h + i) * a.oh[t]);
        }
      };
      for (; h + HEADS <= end; h += HEADS) some(std::integral_constant<int, HEADS>{});
      for (; h < end; ++h) some(std::integral_constant<int, 1>{});
    }
    if (!a.partial) continue;
    // the workgroup's partial row: its tokens' lanes in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VEC; ++i) red[(slot * a.lanes + u) * VEC + i] = dw[i];
    __syncthreads();
    const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    for (int c = (int)threadIdx.x; c < a.D; c += kThreads) {
      float s = 0.0f;
      for (int x = 0; x < a.tpb; ++x) s += red[x * a.lanes * VEC + c];
      a.partial[((int64_t)t * a.parts + part) * a.D + c] = s;
    }
  }
}

// any head: one wave a row, channels lane + 64 j
template <class E, bool BWD>
__global__ __launch_bounds__(kThreads) void head_norm_any_kernel(HeadArgs a, int inter) {
  constexpr int NC = kMaxHeadDim / 64;
  typedef typename E::type T;
  __shared__ float red[4][kMaxHeadDim];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const float per = 1.0f / (float)a.D;
  float w[NC], dw[NC];
#pragma unroll 1
  for (int t = 0; t < 2; ++t) {
    int h0, end;
    slice_of(a, t, h0, end);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      dw[j] = 0.0f;
      w[j] = h0 < end && lane + 64 * j < a.D ? weight_at<E>(a, t, lane + 64 * j) : 0.0f;
    }
    const int64_t step = BWD ? (int64_t)gridDim.x * 4 : a.tokens;
    for (int64_t token = a.first + (int64_t)blockIdx.x * 4 + wave; h0 < end && token < a.tokens; token += step) {
      const int b = (int)(token / a.S), n = (int)(token - (int64_t)b * a.S);
      float cs[NC], sn[NC];
      int other[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = lane + 64 * j, half = a.R / 2;
        const bool rot = c < a.R, upper = inter ? c & 1 : c >= half;
        cs[j] = 1.0f;
        sn[j] = 0.0f;
        other[j] = c;
        if (rot) {
          a.at.at(b, n, inter ? c >> 1 : upper ? c - half : c, sn[j], cs[j]);
          if (!upper) sn[j] = -sn[j];
          other[j] = inter ? c ^ 1 : upper ? c - half : c + half;
        }
      }
#pragma unroll 1
      for (int h = h0; h < end; ++h) {
        const T* x = (const T*)a.x[t] + (int64_t)b * a.xb[t] + (int64_t)h * a.xh[t] + (int64_t)n * a.xs[t];
        T* o = (T*)a.o[t] + (int64_t)b * a.ob[t] + (int64_t)h * a.oh[t] + (int64_t)n * a.os[t];
        float v[NC], g[NC], ss = 0.0f, sg = 0.0f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const int c = lane + 64 * j;
          v[j] = c < a.D ? E::to_float(x[c]) : 0.0f;
          ss = __builtin_fmaf(v[j], v[j], ss);
        }
        if constexpr (BWD) {
          const T* dy = (const T*)a.g[t] + (int64_t)b * a.gb[t] + (int64_t)h * a.gh[t] + (int64_t)n * a.gs[t];
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const int c = lane + 64 * j;
            g[j] = c < a.D ? __builtin_fmaf(E::to_float(dy[c]), cs[j], E::to_float(dy[other[j]]) * sn[j]) : 0.0f;
            sg = __builtin_fmaf(g[j] * w[j], v[j], sg);
          }
        }
        const float inv = 1.0f / sqrtf(__builtin_fmaf(head_sum(ss), per, a.eps));
        const float mean = BWD ? head_sum(sg) * inv * per : 0.0f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const int c = lane + 64 * j;
          if (c >= a.D) continue;
          const float xh = v[j] * inv;
          if constexpr (BWD) {
            dw[j] = __builtin_fmaf(g[j], xh, dw[j]);
            o[c] = E::from_float(inv * __builtin_fmaf(-xh, mean, g[j] * w[j]));
          } else {
            const float p = E::to_float(x[other[j]]) * inv * weight_at<E>(a, t, other[j]);
            o[c] = E::from_float(__builtin_fmaf(xh * w[j], cs[j], p * sn[j]));
          }
        }
      }
    }
    if (!BWD || !a.partial) continue;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NC; ++j) red[wave][lane + 64 * j] = dw[j];
    __syncthreads();
    const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int c = (int)threadIdx.x;
    if (c < a.D) a.partial[((int64_t)t * a.parts + part) * a.D + c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
  }
}

// dw of q (blockIdx.y = 0) and k: the partial rows' columns, 16 at a time, each by 16
// threads that take every 16th row, in order
template <class E>
__global__ __launch_bounds__(256) void head_norm_dw_kernel(const float* partial, int parts, int D, int w32, void* dwq, void* dwk) {
  __shared__ float red[16][17];
  const int c = (int)blockIdx.x * 16 + ((int)threadIdx.x & 15), y = (int)threadIdx.x >> 4, t = (int)blockIdx.y;
  void* const out = t ? dwk : dwq;
  if (!out) return;
  const float* p = partial + (int64_t)t * parts * D;
  float s = 0.0f;
  if (c < D)
#pragma unroll 8
    for (int x = y; x < parts; x += 16) s += p[(int64_t)x * D + c];
  red[y][threadIdx.x & 15] = s;
  __syncthreads();
  if (y || c >= D) return;
  for (int x = 1; x < 16; ++x) s += red[x][threadIdx.x & 15];
  if (w32) ((float*)out)[c] = s;
  else ((typename E::type*)out)[c] = E::from_float(s);
}

// How a launch is cut: `vec` elements a lane (0: one wave a row), tokens per
// workgroup, and heads per slice (blockIdx.y): as many slices as make 1,536 workgroups,
// six a CU, the backward 1,024, each leaving a partial row.  (A CU holds four of the backward
// and of the forward half a rotation apart in bfloat16, six in float16, seven
// interleaved, eight in halves of a piece; the numbers were measured for the clip and the
// training step above alone.)
struct HeadCut {
  int vec, lanes, tpb, heads_per;
  int64_t gx, gy;
};
HeadCut head_cut(int vec, int64_t tokens, int heads, int D, bool bwd) {
  HeadCut c{};
  c.vec = vec;
  c.lanes = 64;
  if (vec)
    for (c.lanes = 1; c.lanes * vec < D;) c.lanes *= 2;
  c.tpb = kThreads / c.lanes;
  c.gx = (tokens + c.tpb - 1) / c.tpb;
  const int64_t want = bwd ? kParts : 1536, slices = c.gx >= want ? 1 : want / c.gx;
  c.heads_per = slices >= heads ? 1 : (int)((heads + slices - 1) / slices);
  c.gy = (heads + c.heads_per - 1) / c.heads_per;
  if (bwd && c.gx * c.gy > kParts) c.gx = kParts / c.gy > 1 ? kParts / c.gy : 1;
  return c;
}

// the widest piece that the head, its rotation, every stride and pointer are multiples of
int piece_of(const HeadArgs& a, int es, bool inter, bool bwd) {
  for (int vec : {16 / es, 8 / es}) {
    if (a.D % vec || a.D > 64 * vec || (inter ? a.R % vec : (a.R / 2) % vec)) continue;
    bool ok = true;
    for (int t = 0; t < 2; ++t) {
      if (!a.H[t]) continue;
      ok = ok && (uintptr_t)a.x[t] % (vec * es) == 0 && (uintptr_t)a.o[t] % (vec * es) == 0 &&
           (!bwd || (uintptr_t)a.g[t] % (vec * es) == 0);
      for (int64_t s : {a.xb[t], a.xh[t], a.xs[t], a.ob[t], a.oh[t], a.os[t], bwd ? a.gb[t] : 0, bwd ? a.gh[t] : 0, bwd ? a.gs[t] : 0})
        ok = ok && s % vec == 0;
    }
    if (ok) return vec;
  }
  return 0;
}

template <class E>
void launch_fwd(HeadArgs a, bool inter, hipStream_t stream) {
  constexpr int ES = (int)sizeof(typename E::type);
  const HeadCut c = head_cut(piece_of(a, ES, inter, false), a.tokens, a.H[0] + a.H[1], a.D, false);
  a.lanes = c.lanes;
  a.tpb = c.tpb;
  a.heads_per = c.heads_per;
  const int64_t most = PRISM_MAX_THREADS / 2 / kThreads;  // workgroups at a time
  for (int64_t at = 0; at < c.gx; at += most) {
    const dim3 grid((unsigned)(c.gx - at < most ? c.gx - at : most), (unsigned)c.gy);
    a.first = at * c.tpb;
    if (c.vec == 16 / ES) {
      if (inter) head_norm_kernel<E, 16 / ES, true><<<grid, kThreads, 0, stream>>>(a);
      else head_norm_kernel<E, 16 / ES, false><<<grid, kThreads, 0, stream>>>(a);
    } else if (c.vec) {
      if (inter) head_norm_kernel<E, 8 / ES, true><<<grid, kThreads, 0, stream>>>(a);
      else head_norm_kernel<E, 8 / ES, false><<<grid, kThreads, 0, stream>>>(a);
    } else {
      head_norm_any_kernel<E, false><<<grid, kThreads, 0, stream>>>(a, inter);
    }
  }
}

template <class E>
void launch_bwd(HeadArgs a, bool inter, void* dwq, void* dwk, hipStream_t stream) {
  constexpr int ES = (int)sizeof(typename E::type);
  const HeadCut c = head_cut(piece_of(a, ES, inter, true), a.tokens, a.H[0] + a.H[1], a.D, true);
  a.lanes = c.lanes;
  a.tpb = c.tpb;
  a.heads_per = c.heads_per;
  a.parts = (int)(c.gx * c.gy);
  const dim3 grid((unsigned)c.gx, (unsigned)c.gy);
  if (c.vec == 16 / ES) {
    if (inter) head_norm_bwd_kernel<E, 16 / ES, true><<<grid, kThreads, 0, stream>>>(a);
    else head_norm_bwd_kernel<E, 16 / ES, false><<<grid, kThreads, 0, stream>>>(a);
  } else if (c.vec) {
    if (inter) head_norm_bwd_kernel<E, 8 / ES, true><<<grid, kThreads, 0, stream>>>(a);
    else head_norm_bwd_kernel<E, 8 / ES, false><<<grid, kThreads, 0, stream>>>(a);
  } else {
    head_norm_any_kernel<E, true><<<grid, kThreads, 0, stream>>>(a, inter);
  }
  if (a.partial)
    head_norm_dw_kernel<E><<<dim3((unsigned)((a.D + 15) / 16), 2), 256, 0, stream>>>(a.partial, a.parts, a.D, a.w32, dwq, dwk);
}

int check_heads(const char* name, int dtype, int wdtype, int B, int64_t S, int Hq, int Hk, int D, int R, int axes, float eps) {
  PRISM_REQUIRE(dtype >= PRISM_F32 && dtype <= PRISM_F16, "%s: dtype code %d unknown", name, dtype);
  PRISM_REQUIRE(wdtype == dtype || wdtype == PRISM_F32, "%s: weights must have the inputs' type or fp32", name);
  PRISM_REQUIRE(B >= 0 && S >= 0 && S < (1ll << 31) && Hq >= 0 && Hk >= 0 && Hq + (int64_t)Hk <= kParts,
                "%s: sizes out of range (at most %d heads)", name, kParts);
  PRISM_REQUIRE((int64_t)B * S < (1ll << 31), "%s: too many tokens", name);
  PRISM_REQUIRE(D >= 2 && D <= kMaxHeadDim, "%s: head dim %d must be 2 to %d", name, D, kMaxHeadDim);
  PRISM_REQUIRE(R >= 2 && R <= D && R % 2 == 0, "%s: rotary dim %d must be even, 2 to the head dim", name, R);
  PRISM_REQUIRE(axes >= 1 && axes <= kMaxAxes, "%s: 1 to %d axes", name, kMaxAxes);
  PRISM_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", name);
  return PRISM_OK;
}

HeadArgs head_args(const void* wq, const void* wk, int wdtype, int B, int64_t S, int Hq, int Hk, int D, int R, float eps,
                   const double* freqs, const void* pos, int pos64, const int64_t* pos_strides, int axes,
                   const int32_t* axis_end, float amplitude, bool bwd) {
  HeadArgs a{};
  a.w[0] = wq; a.w[1] = wk;
  a.w32 = wdtype == PRISM_F32;
  a.H[0] = Hq; a.H[1] = Hk;
  a.tokens = (int64_t)B * S; a.S = (int)S; a.D = D; a.R = R; a.eps = eps;
  a.at.freqs = freqs; a.at.pos = pos; a.at.pos64 = pos64;
  a.at.pb = pos_strides[0]; a.at.ps = pos_strides[1]; a.at.pa = pos_strides[2];
  a.at.axes = axes;
  for (int x = 0; x < axes; ++x) a.at.axis_end[x] = axis_end[x];
  a.at.amp = amplitude; a.at.sign = bwd ? -1.0 : 1.0;
  return a;
}

}  // namespace

extern "C" {

int prism_qk_norm_rotary(const void* q, const void* k, int dtype, int B, int64_t S, int Hq, int Hk, int D, int R,
                         const int64_t* strides, const void* wq, const void* wk, int wdtype, float eps,
                         const double* freqs, const void* pos, int pos64, const int64_t* pos_strides, int axes,
                         const int32_t* axis_end, int interleaved, float amplitude, void* out_q, void* out_k,
                         hipStream_t stream) {
  if (const int rc = check_heads("prism_qk_norm_rotary", dtype, wdtype, B, S, Hq, Hk, D, R, axes, eps)) return rc;
  if (B == 0 || S == 0 || Hq + Hk == 0) return PRISM_OK;
  PRISM_REQUIRE((!Hq || (q && out_q)) && (!Hk || (k && out_k)) && strides && freqs && pos && pos_strides && axis_end,
                "prism_qk_norm_rotary: null pointer");
  PRISM_REQUIRE(axis_end[axes - 1] == R / 2, "prism_qk_norm_rotary: the axes must share out all %d pairs", R / 2);
  HeadArgs a = head_args(wq, wk, wdtype, B, S, Hq, Hk, D, R, eps, freqs, pos, pos64, pos_strides, axes, axis_end, amplitude, false);
  a.x[0] = q; a.x[1] = k; a.o[0] = out_q; a.o[1] = out_k;
  for (int t = 0; t < 2; ++t) {
    const int64_t* s = strides + 6 * t;
    a.xb[t] = s[0]; a.xh[t] = s[1]; a.xs[t] = s[2]; a.ob[t] = s[3]; a.oh[t] = s[4]; a.os[t] = s[5];
  }
  if (dtype == PRISM_F32) launch_fwd<ElemF32>(a, interleaved != 0, stream);
  else if (dtype == PRISM_BF16) launch_fwd<ElemBf16>(a, interleaved != 0, stream);
  else launch_fwd<ElemF16>(a, interleaved != 0, stream);
  PRISM_LAUNCH_CHECK("prism_qk_norm_rotary");
  return PRISM_OK;
}

int prism_qk_norm_rotary_bwd(const void* dyq, const void* dyk, const void* q, const void* k, int dtype, int B, int64_t S,
                             int Hq, int Hk, int D, int R, const int64_t* strides, const void* wq, const void* wk,
                             int wdtype, float eps, const double* freqs, const void* pos, int pos64,
                             const int64_t* pos_strides, int axes, const int32_t* axis_end, int interleaved,
                             float amplitude, void* dq, void* dk, float* partial, void* dwq, void* dwk,
                             hipStream_t stream) {
  if (const int rc = check_heads("prism_qk_norm_rotary_bwd", dtype, wdtype, B, S, Hq, Hk, D, R, axes, eps)) return rc;
  if (B == 0 || S == 0 || Hq + Hk == 0) return PRISM_OK;
  PRISM_REQUIRE((!Hq || (q && dyq && dq)) && (!Hk || (k && dyk && dk)) && strides && freqs && pos && pos_strides && axis_end,
                "prism_qk_norm_rotary_bwd: null pointer");
  PRISM_REQUIRE(axis_end[axes - 1] == R / 2, "prism_qk_norm_rotary_bwd: the axes must share out all %d pairs", R / 2);
  PRISM_REQUIRE((!dwq && !dwk) || partial, "prism_qk_norm_rotary_bwd: null workspace");
  HeadArgs a = head_args(wq, wk, wdtype, B, S, Hq, Hk, D, R, eps, freqs, pos, pos64, pos_strides, axes, axis_end, amplitude, true);
  a.x[0] = q; a.x[1] = k; a.g[0] = dyq; a.g[1] = dyk; a.o[0] = dq; a.o[1] = dk;
  for (int t = 0; t < 2; ++t) {
    const int64_t* s = strides + 9 * t;
    a.gb[t] = s[0]; a.gh[t] = s[1]; a.gs[t] = s[2]; a.xb[t] = s[3]; a.xh[t] = s[4]; a.xs[t] = s[5];
    a.ob[t] = s[6]; a.oh[t] = s[7]; a.os[t] = s[8];
  }
  a.partial = dwq || dwk ? partial : nullptr;
  if (dtype == PRISM_F32) launch_bwd<ElemF32>(a, interleaved != 0, dwq, dwk, stream);
  else if (dtype == PRISM_BF16) launch_bwd<ElemBf16>(a, interleaved != 0, dwq, dwk, stream);
  else launch_bwd<ElemF16>(a, interleaved != 0, dwq, dwk, stream);
  PRISM_LAUNCH_CHECK("prism_qk_norm_rotary_bwd");
  return PRISM_OK;
}

}  // extern "C"
