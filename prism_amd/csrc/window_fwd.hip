// Window attention forward (gfx950, v_mfma_f32_32x32x16): query token at
// position p sees the keys p - W < j <= p (causal) or |p - j| < W, and the first
// `sinks` keys (causal: those at or before p), of its sequence's length.
//
//   o = sum_j softmax_j(scale q k_j) v_j over the seen keys; 0, and lse -inf, where there are none
//
// Prompts and training (window_fwd_kernel): one workgroup of four waves per 128
// rows, a wave per 32, two workgroups per CU, as the block-sparse forward over
// pairs (attn_fwd.hip): K and V tiles of 64 entries of the key list (window.h)
// are copied HBM -> LDS by global_load_lds_dwordx4 into two stages, S^T = K Q^T
// keeps one query per lane column, softmax in base 2 with a lazy running
// maximum, O^T += V^T P^T from the S^T accumulators.  Only tiles at the ends of a
// window (and the one where the sinks end) are masked, by a 64-bit word per lane
// made from three bounds; a wave skips tiles that none of its tokens sees.
//
// Numbers: scores, maximum, sum and output are fp32; P is rounded to the inputs'
// type for the product with V (half a step of each key's weight, in any direction;
// float16 at a reference that keeps small weights in its range, window.h), o once.
//
// Bound: the matrix cores and the exponentials' VALU beside each other, at D = 64
// the VALU (each score costs the same there for half the products).  Measured: 16,001
// tokens, 32 heads over 8, D = 128, window 4,096, 16 sinks 905-970 us (0.97-1.04
// PFLOP/s of seen pairs; matrix cores busy 55% of the cycles, VALU 53%); 14,040
// tokens, 5 heads, D = 128, 4,680 to both sides, 1,560 sinks 339-348 + 9 us.
#include "window.h"

namespace {

template <class E, int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void window_fwd_kernel(WinArgs a) {
  using T = WinTiles<D>;
  using RT = typename T::RT;
  constexpr int NS = D / 16, NDT = D / 32;
  __shared__ __align__(1024) uint8_t smem[2 * T::STAGE];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  const WinItem it = win_item(a, xcd_group_remap<8>((int)blockIdx.x, a.items));
  const int b = it.b, hk = it.hk, tile = it.tile;
  const SeqSpan sq = seq_span(a, b);
  const int rows = a.Sq * a.G, r0 = tile * 128, wr0 = r0 + 32 * w;
  const int last = sq.n - 1;
  auto token = [&](int r) { const int i = r / a.G; return i < last ? i : last; };
  const KeyList kl = r0 / a.G > last ? KeyList{0, 0, 0} : key_list(a, sq, r0 / a.G, token(r0 + 127));
  const int all = (kl.n + 63) >> 6;
  const int t0 = it.slot < 0 ? 0 : all * it.split / a.splits, t1 = it.slot < 0 ? all : all * (it.split + 1) / a.splits;

  const float NINF = -__builtin_inff();
  StageCopy<D> copy;
  copy.init(a, b, hk, w & 1, lane);
  const uint32_t lds0 = lds_addr(smem);
  if (w < 2 && t1 > t0) copy.issue(kl, 64 * t0, lds0 + (uint32_t)((t0 & 1) * T::STAGE));

  RowOperand kop;
  kop.init<RT>(0, l32, g);
  TrOperand vop;
  vop.init<RT>(0, lane);

  // this lane's row (rows past the end re-read the last one and are not stored)
  const int r = wr0 + l32, rc = r < rows ? r : rows - 1;
  const int i = rc / a.G, head = hk * a.G + (rc - i * a.G);
  const uint16_t* qp = a.q.p + b * a.q.b + head * a.q.h + i * a.q.s;
  bf16x8 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = ld_bf16x8(qp + 16 * s + 8 * g);
#pragma unroll
  for (int s = 0; s < NS; ++s) consume_regs(qf[s]);

  const bool live = i <= last;  // rows past the sequence's queries see nothing
  TokenSpan span = token_span(a, kl, i + sq.off);
  if (!live) span = TokenSpan{1, 0, 0};
  const int wi0 = (int)uniform_u32((uint32_t)(wr0 / a.G)), wi1 = (int)uniform_u32((uint32_t)token(wr0 + 31));
  const bool some = wi0 <= last && wr0 < rows;
  const bool whole = (wr0 + 31) / a.G <= last;  // every row of the wave is a query
  WaveSpan ws;
  ws.init(a, kl, wi0 + sq.off, wi1 + sq.off);

  f32x16 acc_o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = f32x16_zero();
  float m = NINF, l = 1.0f;

  for (int t = t0; t < t1; ++t) {
    dma_wait_all();
    __syncthreads();
    if (w < 2 && t + 1 < t1) copy.issue(kl, 64 * (t + 1), lds0 + (uint32_t)(((t + 1) & 1) * T::STAGE));
    const int u0 = 64 * t;
    if (!some || !ws.any(u0, u0 + 63)) continue;
    const uint8_t* sK = smem + (t & 1) * T::STAGE;
    const uint8_t* sV = sK + RT::BYTES;
    // S^T[key][q] = K Q^T, two 32-key halves as interleaved MFMA chains, the K
    // operands through a ring of four registers
    f32x16 sacc[2] = {f32x16_zero(), f32x16_zero()};
    {
      constexpr int NO = 2 * NS, RING = 4;
      bf16x8 kfr[RING];
      auto rd = [&](int x) { return kop.load(sK + RT::rows(32 * (x & 1)), x >> 1); };
#pragma unroll
      for (int x = 0; x + 1 < RING; ++x) kfr[x] = rd(x);
#pragma unroll
      for (int x = 0; x < NO; ++x) {
        if (x + RING - 1 < NO) kfr[(x + RING - 1) % RING] = rd(x + RING - 1);
        sacc[x & 1] = E::mfma(kfr[x % RING], qf[x >> 1], sacc[x & 1]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, RING - 1, 0);
#pragma unroll
      for (int x = 0; x + RING - 1 < NO; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, RING - 1, 0);
    }
    // V^T operands of the P V product, in flight while the softmax runs (at D = 64
    // those of two steps at a time: 128 registers let four workgroups share a CU)
    constexpr int VR = D == 64 ? 2 : 4;
    bf16x8 vfr[VR][NDT];
#pragma unroll
    for (int tt = 0; tt < VR; ++tt)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) vfr[tt][dt] = vop.load<RT>(sV, tt, dt);
    if (!whole || !ws.all(u0, u0 + 63)) {
      // this lane's entries are 32 kh + 8 j + 4 g + x: bit (32 kh + 8 j + x) of the word >> 4 g
      const uint64_t mm = span_bits(span, u0) >> (4 * g);
      const uint32_t lo = (uint32_t)mm, hi = (uint32_t)(mm >> 32);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int bit = 8 * (x >> 2) + (x & 3);
        sacc[0][x] = keep_or_ninf(sacc[0][x], lo, bit);
        sacc[1][x] = keep_or_ninf(sacc[1][x], hi, bit);
      }
    }
    __builtin_amdgcn_s_setprio(2);
    float mx = fmax_nn(sacc[0][0], sacc[1][0]);
#pragma unroll
    for (int x = 1; x < 16; ++x) mx = fmax_nn(fmax_nn(mx, sacc[0][x]), sacc[1][x]);
    mx = xor32_max(mx) * a.scale_log2;
    // the running reference moves only when the tile's maximum is far above it (window.h)
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
    __builtin_amdgcn_s_setprio(1);
    float ls = 0.0f;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int h = tt >> 1, x0 = 8 * (tt & 1);
#pragma unroll
      for (int x = x0; x < x0 + 8; ++x) {
        const float p = fast_exp2(__builtin_fmaf(sacc[h][x], a.scale_log2, -mb));
        sacc[h][x] = p;
        ls += p;
      }
      const bf16x8 pb = win_b_from_acc<E>(sacc, tt);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        acc_o[dt] = E::mfma(vfr[tt % VR][dt], pb, acc_o[dt]);
        if (tt + VR < 4) vfr[tt % VR][dt] = vop.load<RT>(sV, tt + VR, dt);
      }
    }
    if constexpr (VR == 4) {
      __builtin_amdgcn_sched_group_barrier(0x002, 28, 0);
#pragma unroll
      for (int x = 0; x < 3 * NDT; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 28 / NDT, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, NDT, 0);
    }
    ls = xor32_add(ls);
    l = __builtin_fmaf(l, alpha, ls);
    m = m_new;
    __builtin_amdgcn_s_setprio(0);
  }

  if (some && win_not_finite<NDT>(acc_o, l, live)) {
    win_careful<E, D>(a, kl, span, 64 * t0, 64 * t1 < kl.n ? 64 * t1 : kl.n, qp, copy.kb, copy.vb, copy.kstep, copy.vstep, g,
                      acc_o, m, l);
    if (m == NINF && l == 0.0f) l = 1.0f;  // saw nothing
  }
  if (it.slot >= 0) {  // a part: unnormalised sums in register order, reference and sum
    float4* pa = reinterpret_cast<float4*>(a.part) + ((int64_t)it.slot * 4 + w) * NDT * 256 + lane;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        pa[(dt * 4 + j) * 64] =
            make_float4(acc_o[dt][4 * j], acc_o[dt][4 * j + 1], acc_o[dt][4 * j + 2], acc_o[dt][4 * j + 3]);
    if (g == 0) reinterpret_cast<float2*>(a.part_ml)[((int64_t)it.slot * 4 + w) * 32 + l32] = make_float2(m, l);
    return;
  }
  // (the row again from the lane: nothing of it stays in a register over the loop)
  const int re = wr0 + (opaque_thread_id() & 31);
  if (re >= rows) return;
  const int ie = re / a.G, he = hk * a.G + (re - ie * a.G);
  const float inv = 1.0f / l;
  const int64_t at = b * a.o.b + he * a.o.h + ie * a.o.s;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; j += 2)
      win_store_o<E>(a, at + 32 * dt + 8 * j, g, win_scaled(acc_o[dt], j, inv), win_scaled(acc_o[dt], j + 1, inv));
  if (a.lse && g == 0)
    a.lse[((int64_t)b * a.Hk * a.G + he) * a.Sq + ie] = (m + __log2f(l)) * 0.6931471805599453f;
}

// the parts of a cut row tile, in order: one workgroup per tile and 32 channels,
// the lanes of window_fwd_kernel
template <class E, int D>
__global__ __launch_bounds__(256) void window_fwd_join_kernel(WinArgs a) {
  constexpr int NDT = D / 32;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, w = threadIdx.x >> 6, dt = (int)blockIdx.y;
  const WinItem it = win_tile(a, a.whole + (int)blockIdx.x, 0, 0);
  const int r = it.tile * 128 + 32 * w + l32;
  if (r >= a.Sq * a.G) return;
  const float NINF = -__builtin_inff();
  const int64_t first = (int64_t)blockIdx.x * a.splits * 4 + w;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first * 32 + l32;
  const float4* pa = reinterpret_cast<const float4*>(a.part) + (first * NDT + dt) * 256 + lane;
  float top = NINF;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[(int64_t)s * 128].x);
  float4 o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 1
  for (int s = 0; s < a.splits; s += 4) {  // (four parts in flight, past the end the last one again: 11.4 -> 8.5 us)
    float2 x[4];
    float4 v[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = s + k < a.splits ? s + k : a.splits - 1;
      x[k] = ml[t * 128];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = pa[t * 4 * NDT * 256 + j * 64];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = s + k < a.splits;
      const float f = x[k].x == NINF ? 0.0f : fast_exp2(x[k].x - top);  // (a part that sees nothing has sums of 0)
      l = in ? __builtin_fmaf(x[k].y, f, l) : l;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j].x = in ? __builtin_fmaf(v[k][j].x, f, o[j].x) : o[j].x;
        o[j].y = in ? __builtin_fmaf(v[k][j].y, f, o[j].y) : o[j].y;
        o[j].z = in ? __builtin_fmaf(v[k][j].z, f, o[j].z) : o[j].z;
        o[j].w = in ? __builtin_fmaf(v[k][j].w, f, o[j].w) : o[j].w;
      }
    }
  }
  const bool none = top == NINF && l == 0.0f;
  const float inv = none ? 0.0f : 1.0f / l;
  const int i = r / a.G, head = it.hk * a.G + (r - i * a.G);
  const int64_t at = it.b * a.o.b + head * a.o.h + i * a.o.s + 32 * dt;
#pragma unroll
  for (int j = 0; j < 4; j += 2) win_store_o<E>(a, at + 8 * j, g, win_scaled(o[j], inv), win_scaled(o[j + 1], inv));
  if (a.lse && g == 0 && dt == 0)
    a.lse[((int64_t)it.b * a.Hk * a.G + head) * a.Sq + i] = none ? NINF : (top + __log2f(l)) * 0.6931471805599453f;
}

}  // namespace

WinCut win_row_cut(int64_t slots, int B, int Hk, int64_t G, int64_t Sq, int64_t Sk, int D, int64_t window, int64_t sinks,
                   int causal) {
  const int64_t tokens = 128 / G + 1 < Sq ? 128 / G + 1 : Sq;
  const int64_t side = window < Sk ? (causal ? window : 2 * window) : Sk;
  const int64_t some = side + tokens + (sinks < Sk ? sinks : Sk), seen = some < Sk ? some : Sk;
  return win_cut((int64_t)B * Hk * ((Sq * G + 127) / 128), slots, (seen + 63) / 64, D);
}

int win_check(const char* name, int dtype, int B, int Hq, int Hk, int64_t Sq, int64_t Sk, int D, int64_t window,
              int64_t sinks, float sm_scale, const int64_t* strides, int tensors,
              std::initializer_list<const void*> pointers) {
  PRISM_REQUIRE(dtype == PRISM_BF16 || dtype == PRISM_F16, "%s: dtype code %d (bfloat16 or float16)", name, dtype);
  PRISM_REQUIRE(D == 64 || D == 128, "%s: head_dim %d unsupported (64, 128)", name, D);
  PRISM_REQUIRE(B >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0, "%s: %d query heads do not share %d key heads evenly", name,
                Hq, Hk);
  PRISM_REQUIRE(Sq >= 0 && Sk >= 0 && Sq < (1 << 29) && Sk < (1 << 29), "%s: lengths out of range", name);
  PRISM_REQUIRE(Sq * (Hq / Hk) < (1ll << 30), "%s: too many query rows", name);
  PRISM_REQUIRE(window >= 1 && sinks >= 0, "%s: window must be at least 1 and sinks at least 0", name);
  PRISM_REQUIRE(sm_scale > 0.0f && sm_scale < __builtin_inff(), "%s: sm_scale must be positive and finite", name);
  PRISM_REQUIRE(strides, "%s: null pointer", name);
  // rows are copied 16 bytes at a time at 32-bit offsets inside a tile
  for (int i = 0; i < tensors; ++i)
    PRISM_REQUIRE(strides[3 * i] % 8 == 0 && strides[3 * i + 1] % 8 == 0 && strides[3 * i + 2] % 8 == 0 &&
                      strides[3 * i + 2] >= 0 && strides[3 * i + 2] < (1 << 24),
                  "%s: strides must be multiples of 8 elements, a row's below 2^24", name);
  for (const void* p : pointers)
    PRISM_REQUIRE(((uintptr_t)p & 15) == 0, "%s: pointers must be 16-byte aligned", name);
  return PRISM_OK;
}

WinArgs win_args(const void* q, const void* k, const void* v, void* o, int B, int Hq, int Hk, int64_t Sq, int64_t Sk,
                 const int64_t* s, int64_t window, int64_t sinks, int causal, const int32_t* q_lens,
                 const int32_t* kv_lens, float sm_scale) {
  WinArgs a{};
  a.q = {(uint16_t*)q, s[0], s[1], s[2]};
  a.k = {(uint16_t*)k, s[3], s[4], s[5]};
  a.v = {(uint16_t*)v, s[6], s[7], s[8]};
  a.o = {(uint16_t*)o, s[9], s[10], s[11]};
  a.q_lens = q_lens; a.kv_lens = kv_lens;
  a.B = B; a.Hk = Hk; a.G = Hq / Hk; a.Sq = (int)Sq; a.Sk = (int)Sk;
  a.window = (int)(window < (1 << 29) ? window : 1 << 29);
  a.sinks = (int)(sinks < Sk ? sinks : Sk);
  a.causal = causal != 0;
  a.scale = sm_scale; a.scale_log2 = sm_scale * 1.4426950408889634f;
  return a;
}

// workgroups of window_fwd_kernel that the chip holds: two a CU at D = 128, four
// at 64 (registers)
static int64_t fwd_slots(int D) { return D == 128 ? 512 : 1024; }

extern "C" {

int prism_window_fwd_plan(int B, int Hq, int Hk, int64_t Sq, int64_t Sk, int D, int64_t window, int64_t sinks, int causal,
                          int64_t* floats) {
  PRISM_REQUIRE(B >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Sq >= 0 && Sk >= 0 && D >= 1 && window >= 1 &&
                    sinks >= 0 && floats,
                "prism_window_fwd_plan: bad argument");
  const int64_t G = Hq / Hk;
  const WinCut c = win_row_cut(fwd_slots(D), B, Hk, G, Sq, Sk, D, window, sinks, causal);
  *floats = ((int64_t)B * Hk * ((Sq * G + 127) / 128) - c.whole) * c.splits * 128 * (D + 2);
  return PRISM_OK;
}

int prism_window_rest(int64_t Sk, int64_t window, int64_t sinks, int causal) { return !win_few(Sk, window, sinks, causal); }

int prism_window_fwd(const void* q, const void* k, const void* v, int dtype, int B, int Hq, int Hk, int64_t Sq,
                     int64_t Sk, int D, const int64_t* strides, int64_t window, int64_t sinks, int causal,
                     const int32_t* q_lens, const int32_t* kv_lens, float sm_scale, void* o, void* rest, float* lse,
                     float* part, hipStream_t stream) {
  if (const int rc = win_check("prism_window_fwd", dtype, B, Hq, Hk, Sq, Sk, D, window, sinks, sm_scale, strides, 4,
                               {q, k, v, o, rest, part}))
    return rc;
  if (B == 0 || Sq == 0) return PRISM_OK;
  PRISM_REQUIRE(q && o && (Sk == 0 || (k && v)), "prism_window_fwd: null pointer");
  WinArgs a = win_args(q, k, v, o, B, Hq, Hk, Sq, Sk, strides, window, sinks, causal, q_lens, kv_lens, sm_scale);
  a.lse = lse;
  a.rest = (uint16_t*)rest;
  a.tiles = (int)((Sq * a.G + 127) / 128);
  const int64_t total = (int64_t)B * Hk * a.tiles;
  const WinCut c = win_row_cut(fwd_slots(D), B, Hk, a.G, Sq, Sk, D, window, sinks, causal);
  const int64_t cut = total - c.whole, items = c.whole + cut * c.splits;
  PRISM_REQUIRE(items < PRISM_MAX_THREADS / 256, "prism_window_fwd: too many row tiles");
  PRISM_REQUIRE(cut == 0 || part, "prism_window_fwd: null workspace");
  a.total = (int)total;
  a.whole = (int)c.whole; a.splits = (int)c.splits; a.items = (int)items;
  a.ranked = win_ranked(q_lens, B, a.tiles, total, fwd_slots(D));
  a.part = part;
  a.part_ml = part + cut * c.splits * 128 * D;
  auto run = [&](auto kernel, auto join) {
    kernel<<<(unsigned)items, 256, 0, stream>>>(a);
    if (cut) join<<<dim3((unsigned)cut, (unsigned)(D / 32)), 256, 0, stream>>>(a);
  };
  if (dtype == PRISM_BF16) {
    if (D == 64) run(window_fwd_kernel<WinBf16, 64>, window_fwd_join_kernel<WinBf16, 64>);
    else run(window_fwd_kernel<WinBf16, 128>, window_fwd_join_kernel<WinBf16, 128>);
  } else {
    if (D == 64) run(window_fwd_kernel<WinF16, 64>, window_fwd_join_kernel<WinF16, 64>);
    else run(window_fwd_kernel<WinF16, 128>, window_fwd_join_kernel<WinF16, 128>);
  }
  PRISM_LAUNCH_CHECK("prism_window_fwd");
  return PRISM_OK;
}

}  // extern "C"
