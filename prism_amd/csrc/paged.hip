// Appending to a paged cache, and reading sequences back from it (gfx950).
//
// append: token t of sequence b with n_b new tokens of kv_lens[b] in all stands at place
// kv_lens[b] - n_b + its number among them; its keys, turned by their position where
// frequencies are given (rotary.hip's rotation), and its values go to that place's page,
// rounded to the cache's 16 bits, or from there to 4 bits (paged.h).
// gather: the places 0 .. n_b - 1 of every sequence, one behind the other.
//
// Numbers: the rotation is formed in float64 and rounded (as float32, then) to 16 bits.  In
// 4 bits a rounding that goes the other way moves a value by a third, so a key beside a border
// between two codes has to fall on the side on which it stands; 16-bit caches hold the same bits.
//
// Bound: HBM for prompts, the launch for single tokens.  A lane takes 8 channels (16
// bytes) of a token's heads, keeps their angles, place and page and walks the heads, four
// in flight; four lanes share a scale's 32 channels.  Single tokens: one head per thread.
//
// Measured (bf16, D = 128): append of 16,001 tokens, 8 heads, 16 bits 30.6 us (131 MB, 4.3
// TB/s); 8,191 tokens, 8 heads to 4 bits, half a rotation apart, 22 to 24 us from HBM (43 MB: the
// float64 angles and products); with the angles in an LDS table 21.9 and, 16 bits, 32: each lane
// forms its own.  The same tensors again and again, from the last cache: 16.3 us, interleaved (four
// angles a lane in place of eight) 13.2, without a rotation 9.8.  Gather of
// 32,764 places, 4 bits 37 us (170 MB, 4.6 TB/s).  32 single tokens: 6.5 us.
#include <type_traits>

#include "angles.h"
#include "elements.h"
#include "paged.h"

namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  const void *k, *v;                // [T, Hk, D], channels adjacent
  int64_t kt, kh, vt, vh;           // strides in elements
  PagedSide kc, vc;
  PagedTable table;
  const int32_t *lens, *cu;         // cu: [B + 1], or null: each tokens a sequence
  int B, each, T, Hk, D, lanes, tpb, heads_per;
  int R;                            // channels that turn (0: none)
  Angles at;                        // at.pos null: the place
};
struct GatherArgs {
  void *k, *v;                      // [T, Hk, D], dense
  PagedSide kc, vc;
  PagedTable table;
  const int32_t* cu;
  int B, T, Hk, D, lanes, tpb, heads_per;
};

// the sequence that holds row t (first b with cu[b + 1] > t), or -1
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int t) {
  int lo = 0, hi = B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo < B && cu[lo] <= t ? lo : -1;
}

// the 8 values x (already of the cache's 16-bit type) of a lane as codes, written with their scale
__device__ __forceinline__ void store_codes(uint8_t* base, int place, int places, int D, int u, const float* x, bool live) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  for (int off = 1; off <= 2; off <<= 1) {
    const uint32_t b = (uint32_t)__shfl_xor((int)top, off, 64);
    top = b > top ? b : top;
  }
  const uint32_t byte = scale_byte(top);
  const float s = scale_of(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  if (!live) return;
  *reinterpret_cast<uint32_t*>(base + place * (D / 2) + 4 * u) = w;
  if ((u & 3) == 0) base[places * (D / 2) + place * (D / 32) + (u >> 2)] = (uint8_t)byte;
}

// a cos + b sin as float.  (Contraction off: with it the compiler may join this rounding
// and the following one to 16 bits, in some instances and not in others.)
__device__ __forceinline__ float turned(float a, float b, double cs, double sn) {
#pragma clang fp contract(off)
  return (float)((double)a * cs + (double)b * sn);
}

template <class E, int BITS, bool INTER>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  typedef Pack<E, 8> P;
  constexpr int NP = INTER ? 4 : 8;
  const int u = (int)threadIdx.x & (a.lanes - 1), c0 = 8 * u;
  const int row = (int)blockIdx.x * a.tpb + (int)threadIdx.x / a.lanes, t = row < a.T ? row : a.T - 1;
  const int b = a.cu ? sequence_of(a.cu, a.B, t) : t / a.each;
  int place = -1, page = -1;
  if (b >= 0) {
    const int first = a.cu ? a.cu[b] : b * a.each, count = a.cu ? a.cu[b + 1] - first : a.each;
    place = a.lens[b] - count + (t - first);
    page = place < 0 ? -1 : a.table.page(b, place >> a.table.lg);
  }
  const bool live = row < a.T && page >= 0;  // (every lane takes part in the exchanges)
  if (__builtin_amdgcn_ballot_w64(live) == 0) return;
  const int places = 1 << a.table.lg, at = place & (places - 1);
  // angles of the lane's pairs; half a rotation apart, the lane that holds the others
  const bool rot = c0 < a.R && live, upper = !INTER && c0 >= a.R / 2;
  int other = (int)threadIdx.x & 63;
  if (!INTER && c0 < a.R) other += upper ? -(a.R / 16) : a.R / 16;
  double cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    cs[i] = 1.0;
    sn[i] = 0.0;
    const int p = INTER ? c0 / 2 + i : c0 + i - (upper ? a.R / 2 : 0);
    if (rot && 2 * p < a.R) {  // (interleaved, the rotation may end inside the piece)
      a.at.turned(a.at.pos ? a.at.place(0, t, p) : (double)place, p, sn[i], cs[i]);
      if (!INTER && !upper) sn[i] = -sn[i];
    }
  }
  uint8_t* const kc = a.kc.p + (live ? page : 0) * a.kc.page;
  uint8_t* const vc = a.vc.p + (live ? page : 0) * a.vc.page;
  const int64_t ks = t * a.kt + c0, vs = t * a.vt + c0;
  int h = (int)blockIdx.y * a.heads_per;
  const int end = h + a.heads_per < a.Hk ? h + a.heads_per : a.Hk;
  auto some = [&](auto heads) {
    constexpr int C = decltype(heads)::value;
    P k[C], v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      k[i] = P::load(a.k, ks + (h + i) * a.kh);
      v[i] = P::load(a.v, vs + (h + i) * a.vh);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      P o = k[i];
      if (a.R) {
        if constexpr (INTER) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (c0 + 2 * x >= a.R) continue;
            const float p = k[i].get(2 * x), q = k[i].get(2 * x + 1);
            o.set(2 * x, turned(p, q, cs[x], -sn[x]));
            o.set(2 * x + 1, turned(q, p, cs[x], sn[x]));
          }
        } else {
          P q;
          q.w = make_uint4(__shfl(k[i].w.x, other, 64), __shfl(k[i].w.y, other, 64), __shfl(k[i].w.z, other, 64), __shfl(k[i].w.w, other, 64));
#pragma unroll
          for (int x = 0; x < 8; ++x) o.set(x, turned(k[i].get(x), q.get(x), cs[x], sn[x]));
        }
        if (!rot) o = k[i];  // (channels that do not turn, whatever they hold)
      }
      uint8_t* const kb = kc + (h + i) * a.kc.head;
      uint8_t* const vb = vc + (h + i) * a.vc.head;
      if constexpr (BITS == 16) {
        if (live) {
          o.store(kb + at * a.kc.row, c0);
          v[i].store(vb + at * a.vc.row, c0);
        }
      } else {
        float x[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = o.get(j);
          y[j] = v[i].get(j);
        }
        store_codes(kb, at, places, a.D, u, x, live);
        store_codes(vb, at, places, a.D, u, y, live);
      }
    }
  };
  for (; h + 4 <= end; h += 4) {
    some(std::integral_constant<int, 4>{});
  }
  for (; h < end; ++h) some(std::integral_constant<int, 1>{});
}

template <class E, int BITS>
__global__ __launch_bounds__(kThreads) void gather_kernel(GatherArgs a) {
  const int u = (int)threadIdx.x & (a.lanes - 1), t = (int)blockIdx.x * a.tpb + (int)threadIdx.x / a.lanes;
  if (t >= a.T) return;
  const int b = sequence_of(a.cu, a.B, t), place = b >= 0 ? t - a.cu[b] : 0;
  const int page = b >= 0 ? a.table.page(b, place >> a.table.lg) : -1;
  const int places = 1 << a.table.lg, at = place & (places - 1);
  const bool live = page >= 0;
  const uint8_t* const kc = a.kc.p + (live ? page : 0) * a.kc.page;
  const uint8_t* const vc = a.vc.p + (live ? page : 0) * a.vc.page;
  uint4* const ko = (uint4*)a.k + (int64_t)t * a.Hk * a.lanes + u;
  uint4* const vo = (uint4*)a.v + (int64_t)t * a.Hk * a.lanes + u;
  int h = (int)blockIdx.y * a.heads_per;
  const int end = h + a.heads_per < a.Hk ? h + a.heads_per : a.Hk;
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll 4
  for (; h < end; ++h) {
    const uint8_t* kb = kc + h * a.kc.head;
    const uint8_t* vb = vc + h * a.vc.head;
    uint4 x = none, y = none;
    if constexpr (BITS == 16) {
      if (live) {
        x = *reinterpret_cast<const uint4*>(kb + at * a.kc.row + 16 * u);
        y = *reinterpret_cast<const uint4*>(vb + at * a.vc.row + 16 * u);
      }
    } else if (live) {
      const int code = at * (a.D / 2) + 4 * u, scale = places * (a.D / 2) + at * (a.D / 32) + (u >> 2);
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(kb + code), vw = *reinterpret_cast<const uint32_t*>(vb + code);
      const float ksc = scale_of(kb[scale]), vsc = scale_of(vb[scale]);
      if constexpr (std::is_same<E, ElemBf16>::value) {
        x = bf16_of_codes(kw, ksc);
        y = bf16_of_codes(vw, vsc);
      } else {
        x = f16_of_codes(kw, ksc);
        y = f16_of_codes(vw, vsc);
      }
    }
    ko[(int64_t)h * a.lanes] = x;
    vo[(int64_t)h * a.lanes] = y;
  }
}

// lanes of a head, tokens of a workgroup, and heads per slice so that a launch has four
// workgroups a CU where it can (single tokens: one head a thread).  8,192 tokens, 8 heads of
// 128, 4 bits, the same tensors again and again (from the last cache), append / gather, us, at 512 / 1,024 / 2,048 workgroups: 16.4 / 17.0 / 22.9 (each
// slice forms the angles anew), 10.7 / 9.7 / 9.5; 3,000 tokens of 40 heads, 16 bits: 34 / 35 /
// 33, 25 / 23.5 / 23.3.
template <class A>
dim3 cut_tokens(A* a) {
  a->lanes = a->D / 8;
  a->tpb = kThreads / a->lanes;
  const int64_t gx = ((int64_t)a->T + a->tpb - 1) / a->tpb, want = 1024;
  const int64_t slices = gx >= want ? 1 : (want + gx - 1) / gx;
  a->heads_per = slices >= a->Hk ? 1 : (int)((a->Hk + slices - 1) / slices);
  return dim3((unsigned)gx, (unsigned)((a->Hk + a->heads_per - 1) / a->heads_per));
}

int append(const void* k, const void* v, int dtype, int64_t T, int Hk, int D, const int64_t* strides, void* k_cache,
           void* v_cache, int bits, int64_t pages, int page_size, const int64_t* cache_strides, const int32_t* table,
           int64_t table_stride, int64_t width, const int32_t* lens, int B, const int32_t* cu, const double* freqs, int R,
           int interleaved, const void* pos, int pos64, const int64_t* pos_strides, int axes, const int32_t* axis_end,
           double amplitude, hipStream_t stream) {
  if (const int rc = paged_check("prism_paged_append", dtype, bits, Hk, D, pages, page_size, cache_strides, k_cache, v_cache, width, B))
    return rc;
  PRISM_REQUIRE(T >= 0 && T < (1ll << 30), "prism_paged_append: too many tokens");
  PRISM_REQUIRE(cu || B == 0 || T % B == 0, "prism_paged_append: %lld tokens do not share out over %d sequences", (long long)T, B);
  if (T == 0 || B == 0) return PRISM_OK;
  PRISM_REQUIRE(k && v && strides && table && lens, "prism_paged_append: null pointer");
  PRISM_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0 && strides[0] % 8 == 0 && strides[1] % 8 == 0 &&
                    strides[2] % 8 == 0 && strides[3] % 8 == 0,
                "prism_paged_append: rows must be 16-byte aligned");
  AppendArgs a{};
  a.k = k; a.v = v;
  a.kt = strides[0]; a.kh = strides[1]; a.vt = strides[2]; a.vh = strides[3];
  paged_sides(&a.kc, &a.vc, bits, cache_strides, k_cache, v_cache);
  a.table = paged_table(table, table_stride, width, pages, page_size);
  a.lens = lens; a.cu = cu;
  a.B = B; a.each = (int)(T / B); a.T = (int)T; a.Hk = Hk; a.D = D;
  if (freqs) {
    PRISM_REQUIRE(R >= 2 && R <= D && R % 2 == 0 && (interleaved || R % 16 == 0),
                  "prism_paged_append: rotary dim %d must be even (not interleaved: a multiple of 16), 2 to the head dim", R);
    PRISM_REQUIRE(!pos || (pos_strides && axes >= 1 && axes <= kMaxAxes && axis_end && axis_end[axes - 1] == R / 2),
                  "prism_paged_append: the axes must share out all %d pairs", R / 2);
    a.R = R;
    a.at.freqs = freqs; a.at.pos = pos; a.at.pos64 = pos64;
    a.at.axes = 1;
    if (pos) {
      a.at.ps = pos_strides[0]; a.at.pa = pos_strides[1];
      a.at.axes = axes;
      for (int x = 0; x < axes; ++x) a.at.axis_end[x] = axis_end[x];
    }
    a.at.amp = amplitude; a.at.sign = 1.0;
  }
  const dim3 grid = cut_tokens(&a);
  PRISM_REQUIRE(grid.x < PRISM_MAX_THREADS / kThreads, "prism_paged_append: too many tokens");
  auto run = [&](auto e) {
    using E = decltype(e);
    if (bits == 16) {
      if (interleaved) append_kernel<E, 16, true><<<grid, kThreads, 0, stream>>>(a);
      else append_kernel<E, 16, false><<<grid, kThreads, 0, stream>>>(a);
    } else {
      if (interleaved) append_kernel<E, 4, true><<<grid, kThreads, 0, stream>>>(a);
      else append_kernel<E, 4, false><<<grid, kThreads, 0, stream>>>(a);
    }
  };
  if (dtype == PRISM_BF16) run(ElemBf16{});
  else run(ElemF16{});
  PRISM_LAUNCH_CHECK("prism_paged_append");
  return PRISM_OK;
}

}  // namespace

int paged_check(const char* name, int dtype, int bits, int Hk, int D, int64_t pages, int page_size, const int64_t* strides,
                const void* k_cache, const void* v_cache, int64_t width, int64_t B) {
  PRISM_REQUIRE(dtype == PRISM_BF16 || dtype == PRISM_F16, "%s: dtype code %d (bfloat16 or float16)", name, dtype);
  PRISM_REQUIRE(bits == 16 || bits == 4, "%s: a cache holds 16 or 4 bits, not %d", name, bits);
  PRISM_REQUIRE(D == 64 || D == 128, "%s: head_dim %d unsupported (64, 128)", name, D);
  PRISM_REQUIRE(Hk >= 1 && Hk < (1 << 16), "%s: heads out of range", name);
  PRISM_REQUIRE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
                "%s: page size %d must be 16, 32, 64, 128 or 256", name, page_size);
  PRISM_REQUIRE(pages >= 1 && pages < (1ll << 31) && width >= 1 && width * page_size < (1ll << 30) && B >= 0 && B < (1ll << 24),
                "%s: sizes out of range", name);
  PRISM_REQUIRE(strides && k_cache && v_cache, "%s: null pointer", name);
  PRISM_REQUIRE(((uintptr_t)k_cache & 15) == 0 && ((uintptr_t)v_cache & 15) == 0, "%s: caches must be 16-byte aligned", name);
  const int unit = bits == 16 ? 8 : 16;
  for (int i = 0; i < 6; ++i) {
    if (bits == 4 && i % 3 == 2) continue;
    PRISM_REQUIRE(strides[i] >= 0 && strides[i] % unit == 0 && (i % 3 != 2 || strides[i] < (1 << 24)),
                  "%s: a cache's strides must be whole 16 bytes, a place's below 2^24 elements", name);
  }
  return PRISM_OK;
}
void paged_sides(PagedSide* k, PagedSide* v, int bits, const int64_t* s, const void* k_cache, const void* v_cache) {
  const int es = bits == 16 ? 2 : 1;
  *k = {(uint8_t*)k_cache, s[0] * es, s[1] * es, s[2] * es};
  *v = {(uint8_t*)v_cache, s[3] * es, s[4] * es, s[5] * es};
}
PagedTable paged_table(const int32_t* table, int64_t stride, int64_t width, int64_t pages, int page_size) {
  return {table, stride, (int)width, (int)pages, __builtin_ctz((unsigned)page_size)};
}

extern "C" {

int prism_paged_append(const void* k, const void* v, int dtype, int64_t T, int Hk, int D, const int64_t* strides, void* k_cache,
                       void* v_cache, int bits, int64_t pages, int page_size, const int64_t* cache_strides,
                       const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lens, int B,
                       const int32_t* cu, const double* freqs, int R, int interleaved, const void* pos, int pos64,
                       const int64_t* pos_strides, int axes, const int32_t* axis_end, float amplitude, hipStream_t stream) {
  return append(k, v, dtype, T, Hk, D, strides, k_cache, v_cache, bits, pages, page_size, cache_strides, table, table_stride, width,
                lens, B, cu, freqs, R, interleaved, pos, pos64, pos_strides, axes, axis_end, (double)amplitude, stream);
}

int prism_paged_append_f64(const void* k, const void* v, int dtype, int64_t T, int Hk, int D, const int64_t* strides,
                           void* k_cache, void* v_cache, int bits, int64_t pages, int page_size,
                           const int64_t* cache_strides, const int32_t* table, int64_t table_stride, int64_t width,
                           const int32_t* lens, int B, const int32_t* cu, const double* freqs, int R, int interleaved,
                           const void* pos, int pos64, const int64_t* pos_strides, int axes, const int32_t* axis_end,
                           double amplitude, hipStream_t stream) {
  return append(k, v, dtype, T, Hk, D, strides, k_cache, v_cache, bits, pages, page_size, cache_strides, table, table_stride, width,
                lens, B, cu, freqs, R, interleaved, pos, pos64, pos_strides, axes, axis_end, amplitude, stream);
}

int prism_paged_gather(const void* k_cache, const void* v_cache, int dtype, int bits, int64_t pages, int page_size,
                       const int64_t* cache_strides, const int32_t* table, int64_t table_stride, int64_t width, int B,
                       const int32_t* cu, int64_t T, int Hk, int D, void* k, void* v, hipStream_t stream) {
  if (const int rc = paged_check("prism_paged_gather", dtype, bits, Hk, D, pages, page_size, cache_strides, k_cache, v_cache, width, B))
    return rc;
  PRISM_REQUIRE(T >= 0 && T < (1ll << 30), "prism_paged_gather: too many tokens");
  if (T == 0) return PRISM_OK;
  PRISM_REQUIRE(table && cu && k && v, "prism_paged_gather: null pointer");
  PRISM_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, "prism_paged_gather: outputs must be 16-byte aligned");
  GatherArgs a{};
  a.k = k; a.v = v;
  paged_sides(&a.kc, &a.vc, bits, cache_strides, k_cache, v_cache);
  a.table = paged_table(table, table_stride, width, pages, page_size);
  a.cu = cu;
  a.B = B; a.T = (int)T; a.Hk = Hk; a.D = D;
  const dim3 grid = cut_tokens(&a);
  PRISM_REQUIRE(grid.x < PRISM_MAX_THREADS / kThreads, "prism_paged_gather: too many tokens");
  auto run = [&](auto e) {
    using E = decltype(e);
    if (bits == 16) gather_kernel<E, 16><<<grid, kThreads, 0, stream>>>(a);
    else gather_kernel<E, 4><<<grid, kThreads, 0, stream>>>(a);
  };
  if (dtype == PRISM_BF16) run(ElemBf16{});
  else run(ElemF16{});
  PRISM_LAUNCH_CHECK("prism_paged_gather");
  return PRISM_OK;
}

}  // extern "C"
