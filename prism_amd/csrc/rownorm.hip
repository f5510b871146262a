// Root-mean-square norm of rows with the residual's addition, output in the
// input's type or in 8 bits with a scale per row, and its gradients (gfx950).
//
//   h = x + r (kept in x's type for the next layer), s = 1 / sqrt(mean(h^2) + eps), y = h s w
//   8 bits: scale = max(max_j |y_j| / qmax, 2^-126), q = round(y / scale)
//   dx = dr = s (g - xh mean(g xh)) + dh with g = dy w, xh = h s;  dw = sum over rows of dy xh
//
// What the layer around the attention runs between its residual stream and
// its projections (wan_video_dit.py:699-705 norms q and k so).
//
// Sums, the norm and the products are fp32; h is rounded to x's type only
// where it is stored (the forward norms the unrounded sum, the backward reads
// the stored one: half a step of h apart), y once.
//
// Bound: HBM, a few operations per element.  Every element is read once and
// held in registers between the sum and the product; a row of up to 64 vectors
// of 16 bytes times four goes to one wave (no barrier), a longer one to a
// workgroup of four or sixteen waves (one barrier per reduction).  Measured, bf16:
// 75,600 x 5,120 with residual to e4m3 499 us (5.4 TB/s); forward and backward of
// 14,040 x 5,120 with residual 234 us (eight tensors, 4.9 TB/s: the forward 5.8, the
// backward 4.4); 4 rows 5.6 us.
#include <type_traits>

#include "common.h"
#include "elements.h"

namespace {

constexpr int kMaxWidth = 16384;

struct NormArgs {
  const void *x, *r, *w;  // rows of x and r: xs, rs elements apart; r, w or null
  int64_t M, xs, rs;
  int N, w_f32, out;      // out: PRISM_* code of y, or PRISM_E4M3 / PRISM_I8
  float eps, inv_n;
  void *h, *y;            // [M, N]; h written where r is given
  float *scale, *inv;     // [M] or null
};

struct NormBwdArgs {
  const void *dy, *dh, *h, *w;  // rows dys, dhs, hs elements apart; dh, w or null
  int64_t M, dys, dhs, hs;
  int N, w_f32;
  float inv_n;
  const float* inv;             // [M]
  void* dx;                     // [M, N]
  float* partial;               // [gridDim.x, N] or null
};

template <class E, int VEC>
__device__ __forceinline__ void load_weight(float* wv, const void* w, int f32, int col) {
  if (!w) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) wv[k] = 1.0f;
  } else if (f32) {
    constexpr int V = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int c = 0; c < VEC; c += V) {
      const auto t = Pack<ElemF32, V>::load(w, col + c);
#pragma unroll
      for (int k = 0; k < V; ++k) wv[c + k] = t.get(k);
    }
  } else {
    const auto t = Pack<E, VEC>::load(w, col);
#pragma unroll
    for (int k = 0; k < VEC; ++k) wv[k] = t.get(k);
  }
}

// sum (or the largest bit pattern of non-negative floats: NaN above infinity
// above every number) over the WAVES waves of a row; red: WAVES words of LDS
// that no wave still reads
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum_xor(v);
  if (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) s += red[i];
  return s;
}
template <int WAVES>
__device__ __forceinline__ uint32_t row_umax(uint32_t v, uint32_t* red) {
  for (int off = 32; off >= 1; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, off, 64);
    v = o > v ? o : v;
  }
  if (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t s = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) s = red[i] > s ? red[i] : s;
  return s;
}

// VEC values y of one row as 8-bit codes of y / scale.  z stays within qmax up
// to the rounding of 1 / scale, which the clamp takes back; a NaN (rows with a
// NaN or an infinity, whose scale is not finite either) becomes e4m3's NaN and
// int8's 0.
template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t* q, const float* y, float rscale, int out) {
  union {
    typename Words<VEC >= 2 ? VEC : 2>::type w;
    uint8_t b[VEC >= 2 ? VEC : 2];
  } u;
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const float z = y[k] * rscale;
    if (out == PRISM_E4M3) {
      const float c = z != z ? z : __builtin_amdgcn_fmed3f(z, -448.0f, 448.0f);
      u.b[k] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false);
    } else {
      const float c = z != z ? 0.0f : __builtin_amdgcn_fmed3f(rintf(z), -127.0f, 127.0f);
      u.b[k] = (uint8_t)(int8_t)(int)c;
    }
  }
  if constexpr (VEC >= 2) *reinterpret_cast<decltype(u.w)*>(q) = u.w;
  else *q = u.b[0];
}

template <class E, int VEC, int ITEMS, int WAVES>
__global__ __launch_bounds__(WAVES == 16 ? 1024 : 256) void rms_norm_kernel(NormArgs a) {
  __shared__ float red[WAVES];
  __shared__ uint32_t redm[WAVES];
  const int tid = (int)threadIdx.x, lane = WAVES == 1 ? tid & 63 : tid;
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (tid >> 6) : (int64_t)blockIdx.x;
  if (row >= a.M) return;  // whole waves; with WAVES > 1 the grid is M
  float h[ITEMS][VEC];
  float ss = 0.0f;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int col = (it * 64 * WAVES + lane) * VEC;
    if (col < a.N) {
      const auto t = Pack<E, VEC>::load(a.x, row * a.xs + col);
#pragma unroll
      for (int k = 0; k < VEC; ++k) h[it][k] = t.get(k);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) h[it][k] = 0.0f;
    }
  }
  if (a.r) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * 64 * WAVES + lane) * VEC;
      if (col < a.N) {
        const auto t = Pack<E, VEC>::load(a.r, row * a.rs + col);
        Pack<E, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          h[it][k] += t.get(k);
          o.set(k, h[it][k]);
        }
        o.store(a.h, row * a.N + col);
      }
    }
  }
#pragma unroll
  for (int it = 0; it < ITEMS; ++it)
#pragma unroll
    for (int k = 0; k < VEC; ++k) ss = __builtin_fmaf(h[it][k], h[it][k], ss);
  const float s = 1.0f / sqrtf(__builtin_fmaf(row_sum<WAVES>(ss, red), a.inv_n, a.eps));
  if (a.inv && lane == 0) a.inv[row] = s;

  uint32_t top = 0;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int col = (it * 64 * WAVES + lane) * VEC;
    if (col < a.N) {
      float wv[VEC];
      load_weight<E, VEC>(wv, a.w, a.w_f32, col);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        h[it][k] = h[it][k] * s * wv[k];
        const uint32_t u = __float_as_uint(h[it][k]) & 0x7fffffffu;
        top = u > top ? u : top;
      }
      if (a.out < PRISM_E4M3) {
        Pack<E, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.set(k, h[it][k]);
        o.store(a.y, row * a.N + col);
      }
    }
  }
  if (a.out < PRISM_E4M3) return;
  const float amax = __uint_as_float(row_umax<WAVES>(top, redm));
  float scale = amax / (a.out == PRISM_E4M3 ? 448.0f : 127.0f);
  scale = scale < 1.17549435e-38f ? 1.17549435e-38f : scale;  // (rows of zeros; a NaN stays)
  const float rscale = 1.0f / scale;
  if (lane == 0) a.scale[row] = scale;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int col = (it * 64 * WAVES + lane) * VEC;
    if (col < a.N) store_codes<VEC>((uint8_t*)a.y + row * a.N + col, h[it], rscale, a.out);
  }
}

template <class E, int VEC, int ITEMS, int WAVES>
__global__ __launch_bounds__(WAVES == 16 ? 1024 : 256) void rms_norm_bwd_kernel(NormBwdArgs a) {
  constexpr int ROWS = WAVES == 1 ? 4 : 1;  // rows of a workgroup at a time
  __shared__ float red[2][WAVES];
  __shared__ float sums[WAVES == 1 ? 3 * 64 * VEC * ITEMS : 1];
  const int tid = (int)threadIdx.x, lane = WAVES == 1 ? tid & 63 : tid, sub = WAVES == 1 ? tid >> 6 : 0;
  float dw[ITEMS][VEC];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it)
#pragma unroll
    for (int k = 0; k < VEC; ++k) dw[it][k] = 0.0f;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < a.M; row += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    const float s = a.inv[row];
    Pack<E, VEC> hp[ITEMS], yp[ITEMS];
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * 64 * WAVES + lane) * VEC;
      if (col < a.N) {
        hp[it] = Pack<E, VEC>::load(a.h, row * a.hs + col);
        yp[it] = Pack<E, VEC>::load(a.dy, row * a.dys + col);
      }
    }
    float c = 0.0f;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * 64 * WAVES + lane) * VEC;
      if (col < a.N) {
        float wv[VEC];
        load_weight<E, VEC>(wv, a.w, a.w_f32, col);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float xh = hp[it].get(k) * s, dy = yp[it].get(k);
          dw[it][k] = __builtin_fmaf(dy, xh, dw[it][k]);
          c = __builtin_fmaf(dy * wv[k], xh, c);
        }
      }
    }
    // (the other parity's words are read before the barrier that this turn's
    // writers pass, so one barrier a row is enough)
    c = row_sum<WAVES>(c, red[turn]) * a.inv_n;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int col = (it * 64 * WAVES + lane) * VEC;
      if (col < a.N) {
        // (g and xh again from the packed row: half the registers of keeping them)
        Pack<E, VEC> o;
        float v[VEC];
        load_weight<E, VEC>(v, a.w, a.w_f32, col);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = s * __builtin_fmaf(-hp[it].get(k) * s, c, yp[it].get(k) * v[k]);
        if (a.dh) {
          const auto t = Pack<E, VEC>::load(a.dh, row * a.dhs + col);
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[k] += t.get(k);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.set(k, v[k]);
        o.store(a.dx, row * a.N + col);
      }
    }
  }
  if (!a.partial) return;
  if constexpr (WAVES == 1) {  // the four waves' sums, in wave order
    constexpr int W = 64 * VEC * ITEMS;
    if (sub > 0)
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sums[(sub - 1) * W + (it * VEC + k) * 64 + lane] = dw[it][k];
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dw[it][k] += sums[i * W + (it * VEC + k) * 64 + lane];
  }
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int col = (it * 64 * WAVES + lane) * VEC;
    if (col < a.N)
#pragma unroll
      for (int k = 0; k < VEC; ++k) a.partial[(int64_t)blockIdx.x * a.N + col + k] = dw[it][k];
  }
}

// dw[col] = sum of the workgroups' rows: 32 columns a workgroup, 32 threads a
// column, each a stripe of rows in order, the stripes added in order
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* __restrict__ partial, int parts, int N,
                                                            int dtype, void* dw) {
  __shared__ float sum[32][33];
  const int c = (int)threadIdx.x & 31, j = (int)threadIdx.x >> 5;
  const int col = (int)blockIdx.x * 32 + c;
  float s = 0.0f;
  if (col < N)
#pragma unroll 8
    for (int p = j; p < parts; p += 32) s += partial[(int64_t)p * N + col];
  sum[j][c] = s;
  __syncthreads();
  if (j || col >= N) return;
  for (int i = 1; i < 32; ++i) s += sum[i][c];
  if (dtype == PRISM_F32) ((float*)dw)[col] = s;
  else if (dtype == PRISM_BF16) ((__bf16*)dw)[col] = (__bf16)s;
  else ((_Float16*)dw)[col] = (_Float16)s;
}

// Waves per row and vectors per lane of a row of n vectors: one wave up to 4
// vectors a lane, four waves up to 4, sixteen beyond: what a lane holds (and in
// the backward, its column sums) fits the registers without spilling
struct RowShape {
  int waves, items;
};
RowShape row_shape(int n) {
  if (n <= 256) return {1, n <= 64 ? 1 : n <= 128 ? 2 : 4};
  if (n <= 1024) return {4, n <= 512 ? 2 : n <= 768 ? 3 : 4};
  const int per = (n + 1023) / 1024;
  return {16, per <= 2 ? 2 : per <= 4 ? 4 : per <= 8 ? 8 : 16};
}

template <class E, int VEC, class F>
void for_shape(int N, F f) {
  const RowShape s = row_shape((N + VEC - 1) / VEC);
#define PRISM_ROW_CASE(W, I) \
  if (s.waves == W && s.items == I) return f(std::integral_constant<int, W>{}, std::integral_constant<int, I>{});
  PRISM_ROW_CASE(1, 1)
  PRISM_ROW_CASE(1, 2)
  PRISM_ROW_CASE(1, 4)
  PRISM_ROW_CASE(4, 2)
  PRISM_ROW_CASE(4, 3)
  PRISM_ROW_CASE(4, 4)
  PRISM_ROW_CASE(16, 2)
  if constexpr (VEC <= 4) {
    PRISM_ROW_CASE(16, 4)
  }
  if constexpr (VEC == 1) {
    PRISM_ROW_CASE(16, 8)
    PRISM_ROW_CASE(16, 16)
  }
#undef PRISM_ROW_CASE
}

template <class E, int VEC>
void launch_norm(NormArgs a, hipStream_t stream) {
  for_shape<E, VEC>(a.N, [&](auto w, auto i) {
    constexpr int W = decltype(w)::value, I = decltype(i)::value;
    // (64 W threads a row: as many rows at a time as half of what a launch holds)
    constexpr int64_t most = PRISM_MAX_THREADS / 2 / (64 * W), es = sizeof(typename E::type);
    const int64_t oes = a.out < PRISM_E4M3 ? es : 1;
    for (int64_t left = a.M;; left -= most) {
      a.M = left < most ? left : most;
      const unsigned grid = (unsigned)(W == 1 ? (a.M + 3) / 4 : a.M);
      rms_norm_kernel<E, VEC, I, W><<<grid, W == 16 ? 1024 : 256, 0, stream>>>(a);
      if (left <= most) return;
      a.x = (const char*)a.x + most * a.xs * es;
      if (a.r) a.r = (const char*)a.r + most * a.rs * es;
      if (a.h) a.h = (char*)a.h + most * a.N * es;
      a.y = (char*)a.y + most * a.N * oes;
      if (a.scale) a.scale += most;
      if (a.inv) a.inv += most;
    }
  });
}
// up to `parts` workgroups, none without a row; returns how many
template <class E, int VEC>
int launch_norm_bwd(const NormBwdArgs& a, int parts, hipStream_t stream) {
  for_shape<E, VEC>(a.N, [&](auto w, auto i) {
    constexpr int W = decltype(w)::value, I = decltype(i)::value;
    const int64_t groups = W == 1 ? (a.M + 3) / 4 : a.M;
    parts = groups < parts ? (int)groups : parts;
    rms_norm_bwd_kernel<E, VEC, I, W><<<(unsigned)parts, W == 16 ? 1024 : 256, 0, stream>>>(a);
  });
  return parts;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" {

int prism_rms_norm(const void* x, int64_t x_stride, const void* r, int64_t r_stride, const void* w, int w_dtype,
                   int dtype, int64_t M, int N, float eps, void* h, void* y, int out_dtype, float* scale, float* inv,
                   hipStream_t stream) {
  PRISM_REQUIRE(dtype >= PRISM_F32 && dtype <= PRISM_F16, "prism_rms_norm: dtype code %d unknown", dtype);
  PRISM_REQUIRE(M >= 0 && M < (1ll << 31), "prism_rms_norm: M=%lld out of range", (long long)M);
  PRISM_REQUIRE(N >= 1 && N <= kMaxWidth, "prism_rms_norm: N=%d must be 1 to %d", N, kMaxWidth);
  PRISM_REQUIRE(eps >= 0.0f, "prism_rms_norm: eps must not be negative");
  PRISM_REQUIRE(out_dtype == dtype || out_dtype == PRISM_E4M3 || out_dtype == PRISM_I8,
                "prism_rms_norm: output code %d must be the input's or 8 bits", out_dtype);
  PRISM_REQUIRE(w_dtype == dtype || w_dtype == PRISM_F32, "prism_rms_norm: weight must have x's type or float32");
  if (M == 0) return PRISM_OK;
  PRISM_REQUIRE(x && y && (!r || h), "prism_rms_norm: null pointer");
  PRISM_REQUIRE(out_dtype == dtype || scale, "prism_rms_norm: 8-bit output needs scales");
  NormArgs a{x, r, w, M, x_stride, r_stride, N, w_dtype == PRISM_F32, out_dtype, eps, 1.0f / (float)N, h, y, scale, inv};
  const int vec = 16 / elem_size(dtype);
  const bool wide = N % vec == 0 && x_stride % vec == 0 && (!r || r_stride % vec == 0) && aligned16(x) && aligned16(r) &&
                    aligned16(w) && aligned16(h) && aligned16(y);
  if (dtype == PRISM_F32) wide ? launch_norm<ElemF32, 4>(a, stream) : launch_norm<ElemF32, 1>(a, stream);
  else if (dtype == PRISM_BF16) wide ? launch_norm<ElemBf16, 8>(a, stream) : launch_norm<ElemBf16, 1>(a, stream);
  else wide ? launch_norm<ElemF16, 8>(a, stream) : launch_norm<ElemF16, 1>(a, stream);
  PRISM_LAUNCH_CHECK("prism_rms_norm");
  return PRISM_OK;
}

// Workgroups of the backward at most, each of which walks rows and leaves a partial
// sum of dw; more of them keep the memory busy, fewer leave less to add.  Rows of 257 to
// 2,048 elements go to a wave or to a workgroup by their type and alignment, which the
// launch knows: it starts no workgroup without a row (launch_norm_bwd).  Measured (us, both kernels) with
// 256 / 512 / 1,024: 1,024 rows of 1,536 bf16 8.1 / 8.9 / 11.2; 4,096 of 4,096 36 / 26 /
// 25; 16,384 of 512 23 / 17 / 15, of 5,120 187 / 134 / 112; 1,024 rows of 16,384 (sixteen
// waves a row) 28 / 33 / 45.
int prism_rms_norm_parts(int64_t M, int N, int* parts) {
  PRISM_REQUIRE(M >= 1 && M < (1ll << 31) && N >= 1 && N <= kMaxWidth && parts, "prism_rms_norm_parts: bad argument");
  const int64_t groups = N <= 256 ? (M + 3) / 4 : M, most = N > 8192 ? 256 : M >= 8192 ? 1024 : 512;
  *parts = (int)(groups < most ? groups : most);
  return PRISM_OK;
}

int prism_rms_norm_bwd(const void* dy, int64_t dy_stride, const void* dh, int64_t dh_stride, const void* h,
                       int64_t h_stride, const void* w, int w_dtype, int dtype, int64_t M, int N, const float* inv,
                       void* dx, float* partial, int parts, void* dw, hipStream_t stream) {
  PRISM_REQUIRE(dtype >= PRISM_F32 && dtype <= PRISM_F16, "prism_rms_norm_bwd: dtype code %d unknown", dtype);
  PRISM_REQUIRE(M >= 1 && M < (1ll << 31), "prism_rms_norm_bwd: M=%lld out of range", (long long)M);
  PRISM_REQUIRE(N >= 1 && N <= kMaxWidth, "prism_rms_norm_bwd: N=%d must be 1 to %d", N, kMaxWidth);
  PRISM_REQUIRE(w_dtype == dtype || w_dtype == PRISM_F32, "prism_rms_norm_bwd: weight must have x's type or float32");
  PRISM_REQUIRE(dy && h && inv && dx && (!dw || partial), "prism_rms_norm_bwd: null pointer");
  PRISM_REQUIRE(parts >= 1, "prism_rms_norm_bwd: parts must be >= 1");
  NormBwdArgs a{dy, dh, h, w, M, dy_stride, dh_stride, h_stride, N, w_dtype == PRISM_F32, 1.0f / (float)N, inv, dx,
                dw ? partial : nullptr};
  const int vec = 16 / elem_size(dtype);
  const bool wide = N % vec == 0 && dy_stride % vec == 0 && (!dh || dh_stride % vec == 0) && h_stride % vec == 0 &&
                    aligned16(dy) && aligned16(dh) && aligned16(h) && aligned16(w) && aligned16(dx);
  if (dtype == PRISM_F32) parts = wide ? launch_norm_bwd<ElemF32, 4>(a, parts, stream) : launch_norm_bwd<ElemF32, 1>(a, parts, stream);
  else if (dtype == PRISM_BF16) parts = wide ? launch_norm_bwd<ElemBf16, 8>(a, parts, stream) : launch_norm_bwd<ElemBf16, 1>(a, parts, stream);
  else parts = wide ? launch_norm_bwd<ElemF16, 8>(a, parts, stream) : launch_norm_bwd<ElemF16, 1>(a, parts, stream);
  if (dw) rms_norm_dw_kernel<<<(unsigned)((N + 31) / 32), 1024, 0, stream>>>(partial, parts, N, w_dtype, dw);
  PRISM_LAUNCH_CHECK("prism_rms_norm_bwd");
  return PRISM_OK;
}

}  // extern "C"
