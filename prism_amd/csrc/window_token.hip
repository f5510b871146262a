// Window attention of few query rows over a long cache (gfx950): single tokens
// of a stream and short runs of them.  The operation of window_fwd.hip where the
// rows of a (sequence, key head) are few, so the time is the read of the keys
// and values that they see.
//
// A tile of 32 rows (tokens x heads of the group, window.h) is taken by
// `splits` workgroups, each walking its share of the row tile's key list; in a
// workgroup each of the four waves walks every fourth tile of 32 keys by itself,
// with a double-buffered LDS stage of its own (its copies are awaited by its own
// vmcnt: no barrier until the end), so the CU keeps four waves' copies in flight.
// The four waves' sums are joined in LDS, the workgroups' in a second kernel, both
// in a fixed order.
//
// Bound: HBM.  Measured: 8 tokens, 32 heads over 8, D = 128, window 4,096: 25.3 + 4.1 us
// (5.3 TB/s in the first kernel); 2 tokens over 131,072 keys, fp16, caches laid out by
// token: 192 + 5 us (5.6 TB/s).
#include <type_traits>

#include "window.h"

namespace {

constexpr int kMaxSplits = 256;

template <int D>
struct TokenTiles {
  using RT = RowTile<D>;
  static constexpr int TILE = RT::BYTES / 2;     // 32 rows
  static constexpr int KB = TILE / 1024;         // copy instructions per tile
  static constexpr int STAGE = 2 * TILE;         // K, V
  static constexpr int LDS = 4 * 2 * STAGE;      // four waves, two stages
};

__device__ __forceinline__ void dma_b128_ordered(uint32_t voff, const void* base, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(m0) : "m0", "memory");
}
__device__ __forceinline__ void dma_b128_from_ordered(const void* src, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m0) : "m0", "memory");
}
// (a wave reads what it copied itself: the waits order its own accesses, and
// the memory clobbers keep the compiler's LDS reads on their side of them)
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <class E, int D>
__global__ __launch_bounds__(256, 1) void window_token_kernel(WinArgs a) {
  using T = TokenTiles<D>;
  using RT = typename T::RT;
  using RS = RowSource<D>;
  constexpr int NS = D / 16, NDT = D / 32, KB = T::KB, COUNT = 2 * KB;
  static_assert(KB % 4 == 0, "four lane offsets serve all copies of a tile");
  __shared__ __align__(1024) uint8_t smem[T::LDS];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  const int split = (int)blockIdx.x % a.splits, id = (int)blockIdx.x / a.splits;
  const int bh = id / a.tiles, tile = id - bh * a.tiles;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const SeqSpan sq = seq_span(a, b);
  const int rows = a.Sq * a.G, r0 = tile * 32, last = sq.n - 1;
  const int i0 = r0 / a.G, i1 = (r0 + 31) / a.G < last ? (r0 + 31) / a.G : last;
  const KeyList kl = key_list(a, sq, i0, i1);
  const int nt = (kl.n + 31) >> 5;
  const int t0 = (int)((int64_t)nt * split / a.splits), t1 = (int)((int64_t)nt * (split + 1) / a.splits);

  const uint8_t* kb = (const uint8_t*)uniform_ptr(a.k.p + b * a.k.b + hk * a.k.h);
  const uint8_t* vb = (const uint8_t*)uniform_ptr(a.v.p + b * a.v.b + hk * a.v.h);
  const int64_t kstep = 2 * a.k.s, vstep = 2 * a.v.s;
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    koff[x] = (uint32_t)RS::row(x, lane) * (uint32_t)kstep + (uint32_t)RS::byte(x, lane);
    voff[x] = (uint32_t)RS::row(x, lane) * (uint32_t)vstep + (uint32_t)RS::byte(x, lane);
  }
  uint8_t* const mine = smem + w * 2 * T::STAGE;
  const uint32_t lds0 = lds_addr(mine);
  auto issue = [&](int t, int st) {
    const int u0 = 32 * t;
    const uint32_t lds = lds0 + (uint32_t)(st * T::STAGE);
    if ((u0 >= kl.nsink || u0 + 31 < kl.nsink) && u0 + 31 < kl.n) {
      const int key0 = kl.key(u0);
      const uint8_t* kt = (const uint8_t*)uniform_ptr(kb + key0 * kstep);
      const uint8_t* vt = (const uint8_t*)uniform_ptr(vb + key0 * vstep);
#pragma unroll
      for (int i = 0; i < KB; ++i)
        dma_b128_ordered(koff[i & 3], kt + (i >> 2) * RS::ROWS4 * kstep, lds + (uint32_t)i * 1024u);
#pragma unroll
      for (int i = 0; i < KB; ++i)
        dma_b128_ordered(voff[i & 3], vt + (i >> 2) * RS::ROWS4 * vstep, lds + (uint32_t)(KB + i) * 1024u);
      return;
    }
#pragma unroll 1
    for (int i = 0; i < KB; ++i) {
      const int u = u0 + RS::row(i, lane), key = kl.key(u < kl.n ? u : kl.n - 1), at = RS::byte(i, lane);
      dma_b128_from_ordered(kb + key * kstep + at, uniform_u32(lds + (uint32_t)i * 1024u));
      dma_b128_from_ordered(vb + key * vstep + at, uniform_u32(lds + (uint32_t)(KB + i) * 1024u));
    }
  };

  // this lane's row, as in window_fwd_kernel
  const int r = r0 + l32, rc = r < rows ? r : rows - 1;
  const int i = rc / a.G, head = hk * a.G + (rc - i * a.G);
  const uint16_t* qp = a.q.p + b * a.q.b + head * a.q.h + i * a.q.s;
  bf16x8 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = ld_bf16x8(qp + 16 * s + 8 * g);
#pragma unroll
  for (int s = 0; s < NS; ++s) consume_regs(qf[s]);
  TokenSpan span = token_span(a, kl, i + sq.off);
  if (i > last) span = TokenSpan{1, 0, 0};
  const bool whole = (r0 + 31) / a.G <= last;
  WaveSpan ws;
  ws.init(a, kl, i0 + sq.off, i1 + sq.off);

  RowOperand kop;
  kop.init<RT>(0, l32, g);
  TrOperand vop;
  vop.init<RT>(0, lane);
  const float NINF = -__builtin_inff();
  f32x16 acc_o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = f32x16_zero();
  float m = NINF, l = 0.0f;

  if (t0 + w < t1) issue(t0 + w, 0);
  if (t0 + w + 4 < t1) issue(t0 + w + 4, 1);
  int st = 0;
  for (int t = t0 + w; t < t1; t += 4, st ^= 1) {
    if (t + 4 < t1) copies_wait<COUNT>();  // (the next tile's copies may be in flight)
    else copies_wait<0>();
    const uint8_t* sK = mine + st * T::STAGE;
    const uint8_t* sV = sK + T::TILE;
    const int u0 = 32 * t;
    bf16x8 kf[NS], vfr[2][NDT];
#pragma unroll
    for (int s = 0; s < NS; ++s) kf[s] = kop.load(sK, s);
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) vfr[tt][dt] = vop.load<RT>(sV, tt, dt);
    f32x16 sacc = f32x16_zero(), s2 = f32x16_zero();
#pragma unroll
    for (int s = 0; s < NS; s += 2) {
      sacc = E::mfma(kf[s], qf[s], sacc);
      s2 = E::mfma(kf[s + 1], qf[s + 1], s2);
    }
    reads_done();  // the stage is in registers: its next copy may land
    if (t + 8 < t1) issue(t + 8, st);
#pragma unroll
    for (int x = 0; x < 16; ++x) sacc[x] += s2[x];
    if (!whole || !ws.all(u0, u0 + 31)) {
      const uint32_t bits = (uint32_t)span_bits(span, u0) >> (4 * g);
#pragma unroll
      for (int x = 0; x < 16; ++x) sacc[x] = keep_or_ninf(sacc[x], bits, 8 * (x >> 2) + (x & 3));
    }
    float mx = sacc[0];
#pragma unroll
    for (int x = 1; x < 16; ++x) mx = fmax_nn(mx, sacc[x]);
    mx = xor32_max(mx) * a.scale_log2;
    const bool move = mx > m + (E::SHIFT + E::MARGIN) || (m == NINF && mx != NINF);
    const float m_new = move ? mx - E::SHIFT : m;
    const float alpha = move ? fast_exp2(m - m_new) : 1.0f;
    const float mb = m_new == NINF ? 0.0f : m_new;
    if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc_o[dt][x] *= alpha;
    }
    float ls = 0.0f;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float p = fast_exp2(__builtin_fmaf(sacc[x], a.scale_log2, -mb));
      sacc[x] = p;
      ls += p;
    }
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const bf16x8 pb = win_b_from_acc<E>(&sacc, tt);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = E::mfma(vfr[tt][dt], pb, acc_o[dt]);
    }
    l = __builtin_fmaf(l, alpha, xor32_add(ls));
    m = m_new;
  }

  if (win_not_finite<NDT>(acc_o, l, i <= last)) {
    // (the wave's tiles one after the other; a tile's partial sums join as the
    // waves' do)
    float mw = NINF, lw = 0.0f;
    f32x16 ow[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) ow[dt] = f32x16_zero();
#pragma unroll 1
    for (int t = t0 + w; t < t1; t += 4) {
      win_careful<E, D>(a, kl, span, 32 * t, 32 * t + 32 < kl.n ? 32 * t + 32 : kl.n, qp, kb, vb, kstep, vstep, g, acc_o, m, l);
      const float top = fmaxf(mw, m);
      const float f0 = mw == top ? 1.0f : fast_exp2(mw - top), f1 = m == NINF ? 0.0f : fast_exp2(m - top);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          ow[dt][x] = m == NINF && l == 0.0f ? ow[dt][x] : __builtin_fmaf(acc_o[dt][x], f1, ow[dt][x] * f0);
      lw = m == NINF && l == 0.0f ? lw : __builtin_fmaf(l, f1, lw * f0);
      mw = top;
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = ow[dt];
    m = mw;
    l = lw;
  }

  // join the four waves: every wave's sums on the largest reference, then wave w
  // adds a quarter of the channels (registers 4 NDT w ...) in wave order
  __shared__ float ml[4][2][32];
  if (g == 0) {
    ml[w][0][l32] = m;
    ml[w][1][l32] = l;
  }
  __syncthreads();  // (also: no wave reads its stages any more)
  float top = ml[0][0][l32];
#pragma unroll
  for (int x = 1; x < 4; ++x) top = fmaxf(top, ml[x][0][l32]);
  float lt = 0.0f;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float f = ml[x][0][l32] == NINF ? 0.0f : fast_exp2(ml[x][0][l32] - top);
    lt = __builtin_fmaf(ml[x][1][l32], f, lt);
  }
  const float f = m == NINF ? 0.0f : fast_exp2(m - top);
  float* red = reinterpret_cast<float*>(smem);
  constexpr int NR = NDT * 16, QR = NR / 4;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) red[(w * NR + dt * 16 + x) * 64 + lane] = acc_o[dt][x] * f;
  __syncthreads();
  float o[QR];
#pragma unroll
  for (int x = 0; x < QR; ++x) {
    o[x] = red[(w * QR + x) * 64 + lane];
#pragma unroll
    for (int y = 1; y < 4; ++y) o[x] += red[(y * NR + w * QR + x) * 64 + lane];
  }
  if (r >= rows) return;
#pragma unroll
  for (int x = 0; x < QR; x += 8) {
    const int reg = w * QR + x, d = 32 * (reg >> 4) + 8 * ((reg & 15) >> 2);
    const float4 u = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]), v = make_float4(o[x + 4], o[x + 5], o[x + 6], o[x + 7]);
    if (a.splits == 1) {
      const float inv = lt > 0.0f || lt != lt ? 1.0f / lt : 0.0f;
      win_store_o<E>(a, b * a.o.b + head * a.o.h + i * a.o.s + d, g, win_scaled(u, inv), win_scaled(v, inv));
    } else {
      float* at = a.part + (((int64_t)split * a.total + id) * 32 + l32) * D + d + 4 * g;
      *reinterpret_cast<float4*>(at) = u;
      *reinterpret_cast<float4*>(at + 8) = v;
    }
  }
  if (w == 0 && g == 0) {
    if (a.splits == 1) {
      if (a.lse)
        a.lse[((int64_t)b * a.Hk * a.G + head) * a.Sq + i] =
            lt > 0.0f || lt != lt ? (top + __log2f(lt)) * 0.6931471805599453f : NINF;
    } else {
      const int64_t at = ((int64_t)split * a.total + id) * 32 + l32;
      a.part_ml[2 * at] = top;
      a.part_ml[2 * at + 1] = lt;
    }
  }
}

// the splits' sums of a row, in order: one wave per row
template <class E, int D>
__global__ __launch_bounds__(256) void window_join_kernel(WinArgs a) {
  const int lane = threadIdx.x & 63, l32 = (int)(blockIdx.x & 7) * 4 + (int)(threadIdx.x >> 6);
  const int id = (int)(blockIdx.x >> 3), bh = id / a.tiles, r = (id - bh * a.tiles) * 32 + l32;
  if (r >= a.Sq * a.G) return;
  const int b = bh / a.Hk, hk = bh - b * a.Hk, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const float NINF = -__builtin_inff();
  const int64_t row = (int64_t)id * 32 + l32, step = (int64_t)a.total * 32;
  float m = NINF;
  for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[2 * (row + s * step)]);
  const float top = wave_max_xor(m);
  constexpr int C = D / 64;  // channels per lane
  typedef typename std::conditional<C == 2, float2, float>::type V;
  float o[2] = {0.0f, 0.0f}, l = 0.0f;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (row + s * step));
    const V p = *reinterpret_cast<const V*>(a.part + (row + s * step) * D + C * lane);
    const float f = ml.x == NINF ? 0.0f : fast_exp2(ml.x - top);  // (a part that sees nothing has sums of 0)
    l = __builtin_fmaf(ml.y, f, l);
    if constexpr (C == 2) {
      o[0] = __builtin_fmaf(p.x, f, o[0]);
      o[1] = __builtin_fmaf(p.y, f, o[1]);
    } else {
      o[0] = __builtin_fmaf(p, f, o[0]);
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const int64_t at = b * a.o.b + head * a.o.h + i * a.o.s + C * lane;
  auto put = [&](uint16_t* to, uint32_t u) {
    if constexpr (C > 1) *reinterpret_cast<uint32_t*>(to + at) = u;
    else to[at] = (uint16_t)u;
  };
  const uint32_t u = E::pack(o[0] * inv, o[1] * inv);
  put(a.o.p, u);
  if (a.rest) put(a.rest, E::pack(o[0] * inv - E::lo(u), o[1] * inv - E::hi(u)));
  if (a.lse && lane == 0)
    a.lse[((int64_t)b * a.Hk * a.G + head) * a.Sq + i] =
        l > 0.0f || l != l ? (top + __log2f(l)) * 0.6931471805599453f : NINF;
}

}  // namespace

extern "C" {

// Whether a call goes to these kernels, and over how many workgroups (splits) the
// keys of a row tile are cut.
//
// These kernels read the keys once per 32 rows, window_fwd_kernel once per 128:
// it wins where many row tiles see many keys.  Measured at D = 128, these /
// window_fwd_kernel (us), by row tiles of the launch and keys seen: 8 x 4,100: 13.6
// / 24; 64 x 4,100: 20.6 / 25; 128 x 4,100: 28 / 28 (sharing one sequence) and 48 /
// 35; 256 x 4,100: 82 / 39; 16 x 8,000: 16 / 37; 128 x 500: 15 / 19; 256 x 500: 17 /
// 19; 512 x 500: 30 / 20; 256 x 300: 11 / 14; 512 x 300: 19 / 14.
//
// Splits: a second kernel costs 2 us, and each part 0.05 of its work, so up to 512
// keys one workgroup, beyond that about sqrt(keys) / 2.5, and no more than give
// each CU one workgroup.  Measured, D = 128, 1 row tile of 300 keys: 8.3 us in one
// part, 10.2 in two; of 1,000: 13.3 in one, 9.6 in 8, 11.6 in 32; of 4,000: 37 in
// one, 11.5 in 16, 12.4 in 64; of 32,000: 41 in 8, 16.3 in 64, 25 in 256.  Caches
// read for the first time: 64 tiles of 4,100 keys 32.4 us in 3 parts, 33.4 in 4, 39
// in 6; 16 tiles of 131,000 185 in 12, 189 in 16, 217 in 20 (rows 2 KB apart: 202 in
// 12, 191 in 16); 128 tiles of 4,100 58.8 in one, 56.1 in two.
int prism_window_token_plan(int B, int Hq, int Hk, int64_t Sq, int64_t Sk, int64_t window, int64_t sinks, int causal,
                            int* splits, int64_t* floats) {
  PRISM_REQUIRE(B >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Sq >= 0 && Sk >= 0 && window >= 1 && sinks >= 0 &&
                    splits && floats,
                "prism_window_token_plan: bad argument");
  const int64_t G = Hq / Hk, tiles = (Sq * G + 31) / 32, items = (int64_t)B * Hk * tiles;
  const int64_t tokens = (32 + G - 1) / G < Sq ? (32 + G - 1) / G : Sq;
  const int64_t side = window < Sk ? (causal ? window : 2 * window) : Sk;
  const int64_t some = side + tokens + (sinks < Sk ? sinks : Sk), seen = some < Sk ? some : Sk;
  *floats = 0;
  *splits = 0;
  if (tiles > 1 && items > 64 && (items > 256 || seen > 1024)) return PRISM_OK;  // window_fwd_kernel's
  const int64_t by_chip = items ? 256 / items : 1;
  int64_t n = seen <= 512 ? 1 : (int64_t)(__builtin_sqrt((double)seen) / 2.5);
  n = n < by_chip ? n : by_chip;
  n = n < 1 ? 1 : n < kMaxSplits ? n : kMaxSplits;
  *splits = (int)n;
  if (n > 1) *floats = n * items * 32;
  return PRISM_OK;
}

int prism_window_token(const void* q, const void* k, const void* v, int dtype, int B, int Hq, int Hk, int64_t Sq,
                       int64_t Sk, int D, const int64_t* strides, int64_t window, int64_t sinks, int causal,
                       const int32_t* q_lens, const int32_t* kv_lens, float sm_scale, void* o, void* rest, float* lse,
                       int splits, float* part_o, float* part_ml, hipStream_t stream) {
  if (const int rc = win_check("prism_window_token", dtype, B, Hq, Hk, Sq, Sk, D, window, sinks, sm_scale, strides, 4,
                               {q, k, v, o, rest}))
    return rc;
  if (B == 0 || Sq == 0) return PRISM_OK;
  PRISM_REQUIRE(q && o && (Sk == 0 || (k && v)), "prism_window_token: null pointer");
  PRISM_REQUIRE(splits >= 1 && splits <= kMaxSplits && (splits == 1 || (part_o && part_ml)),
                "prism_window_token: bad splits or workspace");
  WinArgs a = win_args(q, k, v, o, B, Hq, Hk, Sq, Sk, strides, window, sinks, causal, q_lens, kv_lens, sm_scale);
  a.lse = lse;
  a.rest = (uint16_t*)rest;
  a.tiles = (int)((Sq * a.G + 31) / 32);
  const int64_t items = (int64_t)B * Hk * a.tiles;
  PRISM_REQUIRE(items < PRISM_MAX_THREADS / 256 && (splits == 1 || items * (splits > 8 ? splits : 8) < PRISM_MAX_THREADS / 256),
                "prism_window_token: too many row tiles");
  a.total = (int)items;
  a.splits = splits; a.part = part_o; a.part_ml = part_ml;
  const unsigned grid = (unsigned)(items * splits), join = (unsigned)(items * 8);
  auto run = [&](auto kernel, auto joiner) {
    kernel<<<grid, 256, 0, stream>>>(a);
    if (splits > 1) joiner<<<join, 256, 0, stream>>>(a);
  };
  if (dtype == PRISM_BF16) {
    if (D == 64) run(window_token_kernel<WinBf16, 64>, window_join_kernel<WinBf16, 64>);
    else run(window_token_kernel<WinBf16, 128>, window_join_kernel<WinBf16, 128>);
  } else {
    if (D == 64) run(window_token_kernel<WinF16, 64>, window_join_kernel<WinF16, 64>);
    else run(window_token_kernel<WinF16, 128>, window_join_kernel<WinF16, 128>);
  }
  PRISM_LAUNCH_CHECK("prism_window_token");
  return PRISM_OK;
}

}  // extern "C"
