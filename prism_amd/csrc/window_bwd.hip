// Window attention backward (gfx950, v_mfma_f32_32x32x16), of window_fwd.hip:
//
//   P = exp(scale q k - lse),  delta = rowsum(o do),  dS = P (do v - delta)
//   dv = P^T do,  dk = scale dS^T q,  dq = scale dS k
//
// window_dq_kernel, by 128 rows, over the key list of the forward: S^T and dP^T
// keep one query per lane column, dQ^T += K^T dS^T.  It also forms delta and
// leaves (m2, delta) = (lse log2 e - GRAD, delta) of every row for the second kernel: from the
// rows of do, o and o's rest (what its rounding left off, kept by the forward: with
// the rounded o alone dq is 2.6e-3 off, norm-wise, bf16, with its rest 2.4e-3; of 235
// us of a step of 2 x 4,096 tokens at D = 64 writing and reading it take 7), or, where rows see 64 keys at most, as sum_j P_j dP_j in a pass over
// the tiles before (the fewer keys the larger delta's error beside dS: 3.0e-3 from the
// rounded o for rows that see 1 to 5 keys, 2.3e-3 with the pass).
// The pass costs no more than reading o: 14,040 tokens, 40 heads over 8, window 64,
// D = 128: 200 us with it, 240 without; 2 x 4,001 tokens, window 60 and 4 sinks 52 / 51.
// window_dkdv_kernel, by 128 keys (64 at D = 64), over the tokens that see them,
// one query head of the group after the other: the two halves of each 64-row
// query tile on different waves (partial sums added through LDS in a fixed
// order); of the eight waves at D = 128 the two of a SIMD run half an entry apart,
// as the block-sparse dK/dV (attn_bwd.hip).  The sinks' key tiles are seen by every later token: long
// lists, and all lists of a launch of few key tiles, are cut over several
// workgroups, whose fp32 sums window_merge_kernel adds in order.  No atomics: the
// same bits every time; sums over the heads that share a key head are fp32.
//
// Numbers: P and dS are rounded to the inputs' type for the products (float16: times
// 2^GRAD, window.h; a dS beyond 1,023 becomes infinite, which a loss scaler sees), the
// rest is fp32.
//
// Bound: the matrix cores at D = 128.  Measured: 14,040 tokens, 5 heads, D = 128, 4,680
// to both sides, 1,560 sinks: dQ 402-418 + 6 us, dK/dV 559-579 + 11 (matrix cores busy
// 71% and 68% of the cycles); 2 x 4,096 padded tokens (half to all of them), 16 heads
// over 4, D = 64, window 1,024: dQ 45-75 us, dK/dV 76-101 + 5.  There nothing is full
// (matrix cores 28% in dK/dV, 36% in dQ): launches of one round, whose tiles read
// their tokens and keys past the L2 (dK/dV 309 MB, dQ 173, of 42 MB of inputs).
#include <type_traits>

#include "window.h"

namespace {

struct WinBwdArgs {
  WinArgs w;                 // (w.o: the forward's output; w.lse: its lse)
  WinTensor do_, dq, dk, dv;
  float* m2;                 // [B Hq, Sq] lse log2 e - GRAD
  float* delta;              // [B Hq, Sq]
  // dK/dV items: the sink tiles of all heads, sink_splits pieces each, then the
  // other tiles, rest_whole whole and the others in rest_splits pieces; pieces of
  // a cut tile leave their sums in acc
  int sink_tiles, key_tiles, sink_splits, sink_items, rest_whole, rest_splits, items;
  int ranked;                // the other tiles by rank (rank_tile)
  int exact;                 // delta from P and dP instead of o (window_dq_kernel)
  float4* acc;
};

template <class E>
__device__ __forceinline__ float dot8(bf16x8 a, bf16x8 b, float s) {
  const uint4 x = __builtin_bit_cast(uint4, a), y = __builtin_bit_cast(uint4, b);
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = __builtin_fmaf(E::lo(xs[i]), E::lo(ys[i]), s);
    s = __builtin_fmaf(E::hi(xs[i]), E::hi(ys[i]), s);
  }
  return s;
}
__device__ __forceinline__ float keep_or_zero(float x, uint32_t bits, int b) {
  return __uint_as_float(__float_as_uint(x) & (uint32_t)__builtin_amdgcn_sbfe((int)bits, (uint32_t)b, 1u));
}

template <class E, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void window_dq_kernel(WinBwdArgs ba) {
  const WinArgs& a = ba.w;
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
  const int every = (kl.n + 63) >> 6;
  const int t0 = it.slot < 0 ? 0 : every * it.split / a.splits;
  const int t1 = it.slot < 0 ? every : every * (it.split + 1) / a.splits;

  StageCopy<D> copy;
  copy.init(a, b, hk, w & 1, lane);
  const uint32_t lds0 = lds_addr(smem);
  if (w < 2 && t1 > t0) copy.issue(kl, 64 * t0, lds0 + (uint32_t)((t0 & 1) * T::STAGE));

  RowOperand rop;  // K / V rows l32 (+ 32 kh as an immediate)
  rop.init<RT>(0, l32, g);
  TrOperand top;   // K^T over key rows 0 .. 63
  top.init<RT>(0, lane);

  const int r = wr0 + l32, rc = r < rows ? r : rows - 1;
  const int i = rc / a.G, head = hk * a.G + (rc - i * a.G);
  const int64_t lrow = ((int64_t)b * a.Hk * a.G + head) * a.Sq + i;
  const bool live = i <= last;
  bf16x8 qf[NS], df[NS];
  float dlt = 0.0f;
  {
    const uint16_t* qp = a.q.p + b * a.q.b + head * a.q.h + i * a.q.s + 8 * g;
    const uint16_t* dp = ba.do_.p + b * ba.do_.b + head * ba.do_.h + i * ba.do_.s + 8 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      qf[s] = ld_bf16x8(qp + 16 * s);
      df[s] = ld_bf16x8(dp + 16 * s);
    }
    if (!ba.exact) {  // (all loads of a branch before the first sum that waits for one)
      const int64_t at = b * a.o.b + head * a.o.h + i * a.o.s + 8 * g;
      bf16x8 of[NS], rf[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) of[s] = ld_bf16x8(a.o.p + at + 16 * s);
      if (a.rest) {
#pragma unroll
        for (int s = 0; s < NS; ++s) rf[s] = ld_bf16x8(a.rest + at + 16 * s);
#pragma unroll
        for (int s = 0; s < NS; ++s) dlt = dot8<E>(rf[s], df[s], dlt);
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) dlt = dot8<E>(of[s], df[s], dlt);
    }
  }
  const float lse = a.lse[lrow];
  // rows that see nothing: P = 2^(s - inf) = 0
  const float mq = lse == -__builtin_inff() ? __builtin_inff() : lse * 1.4426950408889634f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    consume_regs(qf[s]);
    consume_regs(df[s]);
  }
  consume_regs(mq);
  consume_regs(dlt);
  TokenSpan span = token_span(a, kl, i + sq.off);
  if (!live) span = TokenSpan{1, 0, 0};
  const int wi0 = (int)uniform_u32((uint32_t)(wr0 / a.G)), wi1 = (int)uniform_u32((uint32_t)token(wr0 + 31));
  const bool some = wi0 <= last && wr0 < rows;
  const bool whole = (wr0 + 31) / a.G <= last;
  WaveSpan ws;
  ws.init(a, kl, wi0 + sq.off, wi1 + sq.off);

  if (ba.exact) {  // (never cut: t0 .. t1 is the whole list)
    for (int t = t0; t < t1; ++t) {
      dma_wait_all();
      __syncthreads();
      if (w < 2 && t + 1 < t1) copy.issue(kl, 64 * (t + 1), lds0 + (uint32_t)(((t + 1) & 1) * T::STAGE));
      const uint8_t* sK = smem + (t & 1) * T::STAGE;
      f32x16 sacc[2] = {f32x16_zero(), f32x16_zero()}, pacc[2] = {f32x16_zero(), f32x16_zero()};
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          sacc[kh] = E::mfma(rop.load(sK + RT::rows(32 * kh), x), qf[x], sacc[kh]);
          pacc[kh] = E::mfma(rop.load(sK + RT::BYTES + RT::rows(32 * kh), x), df[x], pacc[kh]);
        }
      const uint64_t mm = span_bits(span, 64 * t) >> (4 * g);
      const uint32_t bits[2] = {(uint32_t)mm, (uint32_t)(mm >> 32)};
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float p = fast_exp2(__builtin_fmaf(sacc[kh][x], a.scale_log2, -mq));
          dlt += keep_or_zero(p * pacc[kh][x], bits[kh], 8 * (x >> 2) + (x & 3));
        }
    }
    __syncthreads();
    if (w < 2 && t1 > t0 + 1) copy.issue(kl, 64 * t0, lds0 + (uint32_t)((t0 & 1) * T::STAGE));
  }
  dlt = xor32_add(dlt);
  const float mg = mq - E::GRAD;  // P and dS from here on times 2^GRAD (window.h)
  if (r < rows && g == 0 && it.split == 0) {
    ba.m2[lrow] = mg;
    ba.delta[lrow] = dlt;
  }

  // the dP^T chains start from -delta (at D = 64 from 0, and delta is subtracted
  // after them: 168 registers let three workgroups share a CU)
  constexpr bool FROM = D != 64;
  f32x16 ndl;
#pragma unroll
  for (int x = 0; x < 16; ++x) ndl[x] = FROM ? -dlt : 0.0f;
  f32x16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = f32x16_zero();

  for (int t = t0; t < t1; ++t) {
    dma_wait_all();
    __syncthreads();
    if (w < 2 && t + 1 < t1) copy.issue(kl, 64 * (t + 1), lds0 + (uint32_t)(((t + 1) & 1) * T::STAGE));
    const int u0 = 64 * t;
    if (!some || !ws.any(u0, u0 + 63)) continue;
    const uint8_t* sK = smem + (t & 1) * T::STAGE;
    const uint8_t* sV = sK + RT::BYTES;
    f32x16 sacc[2] = {f32x16_zero(), f32x16_zero()}, pacc[2] = {ndl, ndl};
    {
      constexpr int NO = 4 * NS, RING = 4;
      bf16x8 op[RING];
      auto rd = [&](int x) { return rop.load(((x & 1) ? sV : sK) + RT::rows(32 * ((x >> 1) & 1)), x >> 2); };
#pragma unroll
      for (int x = 0; x + 1 < RING; ++x) op[x] = rd(x);
#pragma unroll
      for (int x = 0; x < NO; ++x) {
        if (x + RING - 1 < NO) op[(x + RING - 1) % RING] = rd(x + RING - 1);
        const int kh = (x >> 1) & 1;
        if (x & 1) pacc[kh] = E::mfma(op[x % RING], df[x >> 2], pacc[kh]);
        else sacc[kh] = E::mfma(op[x % RING], qf[x >> 2], sacc[kh]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, RING - 1, 0);
#pragma unroll
      for (int x = 0; x + RING - 1 < NO; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, RING - 1, 0);
    }
    constexpr int NQ = 4 * NDT, RQ = 4;
    bf16x8 kt[RQ];
    auto rdk = [&](int x) { return top.load<RT>(sK, x / NDT, x % NDT); };
#pragma unroll
    for (int x = 0; x + 1 < RQ; ++x) kt[x] = rdk(x);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float p = fast_exp2(__builtin_fmaf(sacc[kh][x], a.scale_log2, -mg));
        pacc[kh][x] = FROM ? p * pacc[kh][x] : p * (pacc[kh][x] - dlt);
      }
    if (!whole || !ws.all(u0, u0 + 63)) {
      // dS is 0 where the query does not see the key, whatever the unmasked
      // values were (after the exponentials, which so stay in one block with the
      // products before them)
      const uint64_t mm = span_bits(span, u0) >> (4 * g);
      const uint32_t bits[2] = {(uint32_t)mm, (uint32_t)(mm >> 32)};
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int x = 0; x < 16; ++x) pacc[kh][x] = keep_or_zero(pacc[kh][x], bits[kh], 8 * (x >> 2) + (x & 3));
    }
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const bf16x8 sb = win_b_from_acc<E>(pacc, tt);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const int x = tt * NDT + dt;
        if (x + RQ - 1 < NQ) kt[(x + RQ - 1) % RQ] = rdk(x + RQ - 1);
        dq[dt] = E::mfma(kt[x % RQ], sb, dq[dt]);
      }
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (x + RQ - 1 < NQ) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  if (it.slot >= 0) {
    float4* pa = reinterpret_cast<float4*>(a.part) + ((int64_t)it.slot * 4 + w) * NDT * 256 + lane;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj)
        pa[(dt * 4 + jj) * 64] = make_float4(dq[dt][4 * jj], dq[dt][4 * jj + 1], dq[dt][4 * jj + 2], dq[dt][4 * jj + 3]);
    return;
  }
  if (r >= rows) return;
  uint16_t* dqr = ba.dq.p + b * ba.dq.b + head * ba.dq.h + i * ba.dq.s;
  const float f = a.scale * E::BACK;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int jj = 0; jj < 4; jj += 2)
      win_store<E>(dqr + 32 * dt + 8 * jj, g, win_scaled(dq[dt], jj, f), win_scaled(dq[dt], jj + 1, f));
}

// ------------------------------------------------------------ dK / dV
// Tokens that see key j: i0 <= i <= i1
struct TokenRange {
  int i0, i1;
};
__device__ __forceinline__ TokenRange tokens_of(const WinArgs& a, const SeqSpan& s, int j) {
  if (j >= s.L) return {1, 0};
  const bool sink = j < a.sinks;
  const int p0 = a.causal ? j : sink ? s.off : j - a.window + 1;
  const int i0 = p0 - s.off, i1 = j + a.window - 1 - s.off, end = s.n - 1;
  return {i0 > 0 ? i0 : 0, sink || i1 > end ? end : i1};
}

// tokens that see some key of [j0, j0 + keys) (the first and the last key's, and the
// sinks' where it has some)
__device__ __forceinline__ TokenRange tile_tokens(const WinArgs& a, const SeqSpan& s, int j0, int keys) {
  if (j0 >= s.L || s.n == 0) return {0, -1};
  const int jl = j0 + keys - 1 < s.L - 1 ? j0 + keys - 1 : s.L - 1;
  const TokenRange f = tokens_of(a, s, j0), l = tokens_of(a, s, jl);
  return {f.i0 < l.i0 ? f.i0 : l.i0, f.i1 > l.i1 ? f.i1 : l.i1};
}

struct DkdvItem {
  int b, hk, tile, split, splits, slot;  // slot: workspace piece, -1: the whole list
};
// tile t of the rest: (sequence, key head, key tile), for tiles of `keys` keys
struct KeyTile {
  int b, hk, tile;
};
__device__ __forceinline__ KeyTile rest_tile(const WinBwdArgs& a, int t, int keys) {
  const int nrest = a.key_tiles - a.sink_tiles;
  if (a.ranked) {
    const int lane = (int)threadIdx.x & 63;
    int c = 0;
    if (lane < a.w.B) {
      c = (seq_span(a.w, lane).L + keys - 1) / keys - a.sink_tiles;
      c = c > 0 ? c : 0;
    }
    const RankedTile r = rank_tile(c, a.w.B, a.w.Hk, nrest, t);
    return {r.b, r.hk, a.sink_tiles + r.rank + (r.live ? 0 : __builtin_amdgcn_readlane(c, r.b))};
  }
  const int bh = t / nrest, b = bh / a.w.Hk;
  return {b, bh - b * a.w.Hk, a.sink_tiles + t - bh * nrest};
}
__device__ __forceinline__ DkdvItem dkdv_item(const WinBwdArgs& a, int id, int keys) {
  DkdvItem d;
  if (id < a.sink_items) {
    const int t = id / a.sink_splits, bh = t / a.sink_tiles;
    d.tile = t - bh * a.sink_tiles;
    d.b = bh / a.w.Hk;
    d.hk = bh - d.b * a.w.Hk;
    d.splits = a.sink_splits;
    d.split = id - t * a.sink_splits;
    d.slot = a.sink_splits > 1 ? id : -1;
  } else {
    const int y = id - a.sink_items, z = y - a.rest_whole;
    const KeyTile k = rest_tile(a, z < 0 ? y : a.rest_whole + z / a.rest_splits, keys);
    d.b = k.b;
    d.hk = k.hk;
    d.tile = k.tile;
    d.splits = z < 0 ? 1 : a.rest_splits;
    d.split = z < 0 ? 0 : z % a.rest_splits;
    d.slot = z < 0 || a.rest_splits == 1 ? -1 : (a.sink_splits > 1 ? a.sink_items : 0) + z;
  }
  return d;
}

// Keys of a workgroup.  D = 128: two tiles of 64, eight waves, all of a CU's
// registers.  D = 64: one tile, four waves, and three workgroups share a CU, whose
// phases drift apart by themselves.
constexpr int key_tiles_of(int D) { return D == 64 ? 1 : 2; }
constexpr int kAhead = 2;  // entry j + 2 is copied while j is multiplied

template <int D>
struct DkdvTiles {
  using RT = RowTile<D>;
  static constexpr int KT = key_tiles_of(D), KEYS = 64 * KT, THREADS = 256 * KT;
  static constexpr int STAGES = kAhead + KT;         // (the second tile's waves still read entry j - 1)
  static constexpr int STAGE = 2 * RT::BYTES + 512;  // Q, dO, m2 and delta
  static constexpr int NDT = D / 32;
  static constexpr int RED = 2 * KT * 64 * 2 * NDT * 16 * 4;
  static constexpr int LDS = STAGES * STAGE > RED ? STAGES * STAGE : RED;
};

template <class E, int D>
__global__ __launch_bounds__(DkdvTiles<D>::THREADS, D == 64 ? 3 : 1) void window_dkdv_kernel(WinBwdArgs ba) {
  const WinArgs& a = ba.w;
  using T = DkdvTiles<D>;
  using RT = RowTile<D>;
  using RS = RowSource<D>;
  constexpr int NS = D / 16, NDT = D / 32, SB = T::STAGE, COUNT = 2 * RT::KB / 4, KEYS = T::KEYS, STAGES = T::STAGES;
  __shared__ __align__(1024) uint8_t smem[T::LDS];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  const int kh = w & 1, qh = (w >> 1) & 1, tk = w >> 2;
  const DkdvItem it = dkdv_item(ba, xcd_group_remap<8>((int)blockIdx.x, ba.items), KEYS);
  const SeqSpan sq = seq_span(a, it.b);
  const int j0 = it.tile * KEYS;

  // the tile's tokens, as 64-token tiles of each head from lo on
  const TokenRange tokens = tile_tokens(a, sq, j0, KEYS);
  const int lo = tokens.i0, hi = tokens.i1;
  if (hi < lo && it.slot >= 0) return;  // (window_merge_kernel knows)
  const int nti = hi >= lo ? (hi - lo + 64) >> 6 : 0, all = nti * a.G;
  const int e0 = (int)((int64_t)all * it.split / it.splits), e1 = (int)((int64_t)all * (it.split + 1) / it.splits);
  const int n = e1 - e0;

  // copies: waves 0-3 issue KB-instructions w, w + 4, ... (Q then dO), wave 3
  // also the m2 row and wave 2 the delta row
  const uint32_t lds0 = lds_addr(smem);
  const int64_t qstep = 2 * a.q.s, dstep = 2 * ba.do_.s;
  // the next entry to copy: its head, token tile, and where its rows begin (one
  // tile on at every entry: the scalar unit stands between the barrier and the
  // first products)
  int copy_head = n > 0 ? e0 / nti : 0, copy_tile = n > 0 ? e0 - copy_head * nti : 0;
  const uint8_t *qcur, *dcur;
  const float* rcur;
  auto seek = [&] {
    const int t0 = lo + 64 * copy_tile, head = it.hk * a.G + copy_head;
    qcur = (const uint8_t*)uniform_ptr(a.q.p + it.b * a.q.b + head * a.q.h + t0 * a.q.s);
    dcur = (const uint8_t*)uniform_ptr(ba.do_.p + it.b * ba.do_.b + head * ba.do_.h + t0 * ba.do_.s);
    rcur = (const float*)uniform_ptr((w == 3 ? ba.m2 : ba.delta) + ((int64_t)it.b * a.Hk * a.G + head) * a.Sq + t0);
  };
  if (n > 0) seek();
  auto issue = [&](int st) {
    if (w >= 4) return;
    const int left = hi - (lo + 64 * copy_tile);  // rows past hi re-read it
    const uint32_t base = lds0 + (uint32_t)(st * SB) + 1024u * (uint32_t)w;
    // (lane offsets are formed anew for every entry: the products need every register)
    const int ln = opaque_thread_id() & 63, crow = RS::row(w & 3, ln), cbyte = RS::byte(w & 3, ln);
    if (left >= 63) {
      const uint32_t qoff = (uint32_t)crow * (uint32_t)qstep + (uint32_t)cbyte;
      const uint32_t doff = (uint32_t)crow * (uint32_t)dstep + (uint32_t)cbyte;
      const uint8_t *qb = qcur, *db = dcur;
#pragma unroll
      for (int m = 0; m < RT::KB / 4; ++m, qb += RS::ROWS4 * qstep) dma_b128(qoff, qb, base + 4096u * (uint32_t)m);
#pragma unroll
      for (int m = 0; m < RT::KB / 4; ++m, db += RS::ROWS4 * dstep)
        dma_b128(doff, db, base + RT::BYTES + 4096u * (uint32_t)m);
    } else {
#pragma unroll
      for (int s = 0; s < COUNT; ++s) {
        const int m = s % (RT::KB / 4), row = crow + m * RS::ROWS4, rr = row < left ? row : left;
        const bool isq = s < RT::KB / 4;
        const uint32_t off = (uint32_t)rr * (uint32_t)(isq ? qstep : dstep) + (uint32_t)cbyte;
        dma_b128(off, isq ? qcur : dcur, base + 4096u * (uint32_t)s);
      }
    }
    if (w >= 2)
      dma_b32(4u * (uint32_t)(ln < left ? ln : left), rcur, lds0 + (uint32_t)(st * SB) + 2u * RT::BYTES + (w == 3 ? 0u : 256u));
    if (++copy_tile == nti) {
      copy_tile = 0;
      if (++copy_head < a.G) seek();
    } else {
      qcur += 64 * qstep;
      dcur += 64 * dstep;
      rcur += 64;
    }
  };
  RowOperand rop;                // Q / dO rows 32 qh + l32
  rop.init<RT>(32 * qh, l32, g);
  TrOperand top;                 // Q^T / dO^T over query rows 32 qh .. 32 qh + 31
  top.init<RT>(32 * qh, lane);
#pragma unroll
  for (int x = 0; x < kAhead; ++x)
    if (x < n) issue(x);

  const int jw = j0 + 64 * tk + 32 * kh;
  bf16x8 kf[NS], vf[NS];
  {
    const int kc = jw + l32 < a.Sk ? jw + l32 : a.Sk - 1;
    const uint16_t* kp = a.k.p + it.b * a.k.b + it.hk * a.k.h + kc * a.k.s + 8 * g;
    const uint16_t* vp = a.v.p + it.b * a.v.b + it.hk * a.v.h + kc * a.v.s + 8 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      kf[s] = ld_bf16x8(kp + 16 * s);
      vf[s] = ld_bf16x8(vp + 16 * s);
    }
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    consume_regs(kf[s]);
    consume_regs(vf[s]);
  }
  // of the wave's 32 keys: tokens that see some, and all of them
  int any0, any1, all0, all1;
  {
    const int jl = jw + 31 < sq.L - 1 ? jw + 31 : sq.L - 1;
    const TokenRange f = tokens_of(a, sq, jw), l = tokens_of(a, sq, jl < jw ? jw : jl);
    any0 = f.i0 < l.i0 ? f.i0 : l.i0;
    any1 = f.i1 > l.i1 ? f.i1 : l.i1;
    all0 = f.i0 > l.i0 ? f.i0 : l.i0;
    all1 = f.i1 < l.i1 ? f.i1 : l.i1;
    if (jw + 31 >= sq.L) all1 = -1;  // (lanes past the keys)
    if (jw >= sq.L) any1 = -1;
    if (jw < a.sinks && jw + 31 >= a.sinks) {  // the first key past the sinks sees the earliest end
      const TokenRange x = tokens_of(a, sq, a.sinks);
      all0 = all0 > x.i0 ? all0 : x.i0;
      all1 = all1 < x.i1 ? all1 : x.i1;
    }
  }
  f32x16 dk[NDT], dv[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) { dk[dt] = f32x16_zero(); dv[dt] = f32x16_zero(); }

  // S = Q K^T and dP = dO V^T of one entry, then P and dS (B operands of the dV /
  // dK products: query rows 32 qh + 8 j + 4 g + i in register 4 j + i, column =
  // this lane's key); t0: the entry's first token of this wave's half
  auto sdp = [&](const uint8_t* sQ, int t0, bf16x8* pb, bf16x8* sb) {
    const uint8_t* sDO = sQ + RT::BYTES;
    const float* sM = reinterpret_cast<const float*>(sQ + 2 * RT::BYTES);
    const float* sDl = sM + 64;
    f32x16 sacc = f32x16_zero(), pacc = f32x16_zero();
    constexpr int NO = 2 * NS;
    bf16x8 op[3];
    auto rd = [&](int x) { return rop.load((x & 1) ? sDO : sQ, x >> 1); };
    op[0] = rd(0);
    op[1] = rd(1);
#pragma unroll
    for (int x = 0; x < NO; ++x) {
      if (x + 2 < NO) op[(x + 2) % 3] = rd(x + 2);
      if (x & 1) pacc = E::mfma(op[x % 3], vf[x >> 1], pacc);
      else sacc = E::mfma(op[x % 3], kf[x >> 1], sacc);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
    for (int x = 0; x + 3 < NO; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const float4 m4 = *reinterpret_cast<const float4*>(sM + 32 * qh + 8 * jj + 4 * g);
      const float4 d4 = *reinterpret_cast<const float4*>(sDl + 32 * qh + 8 * jj + 4 * g);
      const float mv[4] = {m4.x, m4.y, m4.z, m4.w}, dl4[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int rg = 4 * jj + x;
        const float p = fast_exp2(__builtin_fmaf(sacc[rg], a.scale_log2, -mv[x]));
        sacc[rg] = p;
        pacc[rg] = p * (pacc[rg] - dl4[x]);
      }
    }
    if (t0 < all0 || t0 + 31 > all1) {
      // rows that do not see the lane's key: P and dS are 0 there, whatever the
      // unmasked values were (the branch stands after the exponentials, which so
      // stay in one block with the products before them)
      const int ln = opaque_thread_id() & 63;
      const TokenRange mine = tokens_of(a, sq, jw + (ln & 31));
      const int b0 = mine.i0 - t0 > 0 ? mine.i0 - t0 : 0, b1 = mine.i1 - t0 < 31 ? mine.i1 - t0 : 31;
      uint32_t bits = b1 >= b0 ? (~0u << b0) & (~0u >> (31 - b1)) : 0u;
      bits >>= 4 * (ln >> 5);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int bit = 8 * (x >> 2) + (x & 3);
        sacc[x] = keep_or_zero(sacc[x], bits, bit);
        pacc[x] = keep_or_zero(pacc[x], bits, bit);
      }
    }
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) {
      pb[t2] = win_b_from_acc<E>(&sacc, t2);
      sb[t2] = win_b_from_acc<E>(&pacc, t2);
    }
  };
  // dV^T += dO^T P and dK^T += Q^T dS of one entry
  auto dvdk = [&](const uint8_t* sQ, const bf16x8* pb, const bf16x8* sb) {
    const uint8_t* sDO = sQ + RT::BYTES;
    constexpr int NO = 4 * NDT, RING = 4;
    bf16x8 op[RING];
    auto rd = [&](int x) { return top.load<RT>((x & 1) ? sQ : sDO, x / (2 * NDT), (x >> 1) % NDT); };
#pragma unroll
    for (int x = 0; x + 1 < RING; ++x) op[x] = rd(x);
#pragma unroll
    for (int x = 0; x < NO; ++x) {
      if (x + RING - 1 < NO) op[(x + RING - 1) % RING] = rd(x + RING - 1);
      const int t2 = x / (2 * NDT), dt = (x >> 1) % NDT;
      if (x & 1) dk[dt] = E::mfma(op[x % RING], sb[t2], dk[dt]);
      else dv[dt] = E::mfma(op[x % RING], pb[t2], dv[dt]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * (RING - 1), 0);
#pragma unroll
    for (int x = 0; x + RING - 1 < NO; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, RING - 1, 0);
  };

  // token tile of entry e, as it advances by one (no division in the loop)
  int tile_i = n > 0 ? e0 % nti : 0;
  auto half_of = [&] { return lo + 64 * tile_i + 32 * qh; };
  auto next_tile = [&] { tile_i = tile_i + 1 == nti ? 0 : tile_i + 1; };
  auto sees = [&](int t0) { return t0 + 31 >= any0 && t0 <= any1; };
  if (T::KT == 1 || tk == 0) {
    int st = 0;
    for (int x = 0; x < n; ++x) {
      if (w >= 2) stage_wait<kAhead + 1, COUNT + 1>(n - 1 - x);
      else stage_wait<kAhead + 1, COUNT>(n - 1 - x);
      __syncthreads();
      if (x + kAhead < n) issue((st + kAhead) % STAGES);
      const uint8_t* sQ = smem + st * SB;
      st = st + 1 == STAGES ? 0 : st + 1;
      const int t0 = half_of();
      next_tile();
      if (!sees(t0)) continue;
      bf16x8 pb[2], sb[2];
      sdp(sQ, t0, pb, sb);
      __builtin_amdgcn_s_setprio(1);
      dvdk(sQ, pb, sb);
      __builtin_amdgcn_s_setprio(0);
    }
  } else {
    int st = 0;
    bool pend = false;
    const uint8_t* sPrev = smem;
    bf16x8 pb[2], sb[2];
    for (int x = 0; x < n; ++x) {
      __syncthreads();
      const uint8_t* sQ = smem + st * SB;
      st = st + 1 == STAGES ? 0 : st + 1;
      const int t0 = half_of();
      next_tile();
      if (pend) dvdk(sPrev, pb, sb);
      pend = sees(t0);
      if (pend) {
        sdp(sQ, t0, pb, sb);
        sPrev = sQ;
      }
    }
    if (pend) dvdk(sPrev, pb, sb);
  }

  // add the two query-half partials in a fixed order (qh = 0 + qh = 1)
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  const int slot = kh | tk << 1;
  if (qh == 1) {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        red[((slot * 2 * NDT + dt) * 16 + x) * 64 + lane] = dk[dt][x];
        red[((slot * 2 * NDT + NDT + dt) * 16 + x) * 64 + lane] = dv[dt][x];
      }
  }
  __syncthreads();
  if (qh == 1) return;
  const int key = jw + (opaque_thread_id() & 31);
  uint16_t* dkr = ba.dk.p + it.b * ba.dk.b + it.hk * ba.dk.h + key * ba.dk.s;
  uint16_t* dvr = ba.dv.p + it.b * ba.dv.b + it.hk * ba.dv.h + key * ba.dv.s;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      dk[dt][x] += red[((slot * 2 * NDT + dt) * 16 + x) * 64 + lane];
      dv[dt][x] += red[((slot * 2 * NDT + NDT + dt) * 16 + x) * 64 + lane];
    }
    if (it.slot >= 0) {
      float4* pa = ba.acc + ((int64_t)it.slot * 2 * T::KT + slot) * 2 * NDT * 256 + lane;
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        pa[(dt * 4 + jj) * 64] = make_float4(dk[dt][4 * jj], dk[dt][4 * jj + 1], dk[dt][4 * jj + 2], dk[dt][4 * jj + 3]);
        pa[((NDT + dt) * 4 + jj) * 64] =
            make_float4(dv[dt][4 * jj], dv[dt][4 * jj + 1], dv[dt][4 * jj + 2], dv[dt][4 * jj + 3]);
      }
      continue;
    }
    if (key >= a.Sk) continue;
#pragma unroll
    for (int jj = 0; jj < 4; jj += 2) {
      const float f = a.scale * E::BACK;
      win_store<E>(dkr + 32 * dt + 8 * jj, g, win_scaled(dk[dt], jj, f), win_scaled(dk[dt], jj + 1, f));
      win_store<E>(dvr + 32 * dt + 8 * jj, g, win_scaled(dv[dt], jj, E::BACK), win_scaled(dv[dt], jj + 1, E::BACK));
    }
  }
}

// the parts of the row tiles of dQ that were cut, in order: one workgroup per
// tile and 32 channels, the lanes of window_dq_kernel
template <class E, int D>
__global__ __launch_bounds__(256) void window_dq_merge_kernel(WinBwdArgs ba) {
  constexpr int NDT = D / 32;
  const WinArgs& a = ba.w;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, w = threadIdx.x >> 6, dt = (int)blockIdx.y;
  const WinItem it = win_tile(a, a.whole + (int)blockIdx.x, 0, 0);
  const int r = it.tile * 128 + 32 * w + l32;
  if (r >= a.Sq * a.G) return;
  const float4* pa = reinterpret_cast<const float4*>(a.part) + (((int64_t)blockIdx.x * a.splits * 4 + w) * NDT + dt) * 256 + lane;
  float4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = pa[j * 64];
#pragma unroll 4
  for (int s = 1; s < a.splits; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = pa[(int64_t)s * 4 * NDT * 256 + j * 64];
      acc[j].x += v.x;
      acc[j].y += v.y;
      acc[j].z += v.z;
      acc[j].w += v.w;
    }
  const int i = r / a.G, head = it.hk * a.G + (r - i * a.G);
  uint16_t* out = ba.dq.p + it.b * ba.dq.b + head * ba.dq.h + i * ba.dq.s + 32 * dt;
#pragma unroll
  for (int j = 0; j < 4; j += 2)
    win_store<E>(out + 8 * j, g, win_scaled(acc[j], a.scale * E::BACK), win_scaled(acc[j + 1], a.scale * E::BACK));
}

// the pieces' sums of the cut key tiles (cut_sinks sink tiles, then the rest's),
// in order: one workgroup per tile and 32-column block of dK (blocks 0 .. NDT - 1)
// or dV; wave = 32 keys
template <class E, int D>
__global__ __launch_bounds__(128 * key_tiles_of(D)) void window_merge_kernel(WinBwdArgs a, int cut_sinks) {
  constexpr int NDT = D / 32, NB = 2 * NDT, KW = 2 * key_tiles_of(D);
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, w = threadIdx.x >> 6, blk = (int)blockIdx.y;
  const int x = (int)blockIdx.x, z = x - cut_sinks;
  const bool sink = z < 0;
  const int S = sink ? a.sink_splits : a.rest_splits;
  const int64_t first = sink ? (int64_t)x * S : (int64_t)cut_sinks * a.sink_splits + (int64_t)z * S;
  KeyTile kt;
  if (sink) {
    const int bh = x / a.sink_tiles;
    kt = {bh / a.w.Hk, bh % a.w.Hk, x - bh * a.sink_tiles};
  } else {
    kt = rest_tile(a, a.rest_whole + z, 32 * KW);
  }
  const int b = kt.b, hk = kt.hk, key = kt.tile * 32 * KW + 32 * w + l32;
  if (key >= a.w.Sk) return;
  const float4* pa = a.acc + ((first * KW + w) * NB + blk) * 256 + lane;
  const TokenRange tokens = tile_tokens(a.w, seq_span(a.w, b), kt.tile * 32 * KW, 32 * KW);
  const bool seen = tokens.i1 >= tokens.i0;  // else: no piece was left
  float4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = seen ? pa[j * 64] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int s = 1; s < (seen ? S : 1); ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = pa[(int64_t)s * KW * NB * 256 + j * 64];
      acc[j].x += v.x;
      acc[j].y += v.y;
      acc[j].z += v.z;
      acc[j].w += v.w;
    }
  const bool isk = blk < NDT;
  const WinTensor& t = isk ? a.dk : a.dv;
  const float f = (isk ? a.w.scale : 1.0f) * E::BACK;
  uint16_t* out = t.p + b * t.b + hk * t.h + key * t.s + 32 * (isk ? blk : blk - NDT);
#pragma unroll
  for (int j = 0; j < 4; j += 2) win_store<E>(out + 8 * j, g, win_scaled(acc[j], f), win_scaled(acc[j + 1], f));
}

// workgroups of window_dq_kernel that the chip holds: two a CU at D = 128, three
// at 64 (registers)
int64_t dq_slots(int D) { return D == 128 ? 512 : 768; }
// of window_dkdv_kernel: one a CU, three at D = 64
int64_t key_slots(int D) { return D == 128 ? 256 : 768; }

// How the dK/dV lists are cut, for one workgroup a CU (three at D = 64): the sinks' lists into
// pieces no longer than the others (or as two rounds of pieces allow), then the last
// round of tiles (win_cut).
struct DkdvPlan {
  int64_t sink_tiles, key_tiles, sink_splits, sink_items, rest_whole, rest_splits, rest_tiles, items, pieces;
};
DkdvPlan dkdv_plan(int B, int Hk, int64_t G, int64_t Sq, int64_t Sk, int D, int64_t window, int64_t sinks, int causal) {
  DkdvPlan p{};
  const int64_t keys = 64 * key_tiles_of(D);
  const int64_t BH = (int64_t)B * Hk, whole = G * ((Sq + 63) / 64);
  const int64_t span = window < Sq ? (causal ? window : 2 * window) + keys - 1 : Sq;
  p.key_tiles = (Sk + keys - 1) / keys;
  p.sink_tiles = ((sinks < Sk ? sinks : Sk) + keys - 1) / keys;
  int64_t rest = span < Sq ? G * ((span + 63) / 64) : whole;
  if (rest >= whole || p.sink_tiles == p.key_tiles) {  // all lists alike
    p.sink_tiles = 0;
    rest = whole;
  }
  const int64_t n = (rest > 8 ? rest : 8);
  p.rest_tiles = BH * (p.key_tiles - p.sink_tiles);
  const int64_t slots = key_slots(D), sinks_in = BH * p.sink_tiles;
  // Two rounds of the sinks' pieces at most: a piece's sums are 131 KB at D = 128 (33 at
  // 64), and pieces as short as the other lists would be terabytes of them where a
  // narrow window stands beside many sinks.  Measured, dK/dV and merge, D = 128, with
  // pieces of the others' length / up to eight rounds / four / two (us): 65,536 tokens,
  // 32 heads over 8, window 256, 1,024 sinks 3,375 / 2,825 / 2,790 / 2,805; 2 x 16,384,
  // window 64, 4,096 sinks 5,770 / 3,405 / 3,524 / 3,358; 20,000 tokens, 8 heads, window
  // 256, 640 sinks 295 / 285 / 248 / 220; 19 heads, 2,000 sinks 1,515 / 940 / 883 / 902.
  const int64_t most = sinks_in ? (2 * slots / sinks_in > 1 ? 2 * slots / sinks_in : 1) : 1;
  p.sink_splits = p.sink_tiles ? (whole + n - 1) / n < most ? (whole + n - 1) / n : most : 1;
  int64_t head = sinks_in * p.sink_splits;  // pieces before the rest's tiles
  const int64_t total = head + p.rest_tiles;
  const WinCut c = win_cut(total, slots, rest, D);
  p.rest_splits = c.splits;
  p.rest_whole = c.whole > head ? c.whole - head : 0;
  if (p.rest_whole > p.rest_tiles) p.rest_whole = p.rest_tiles;
  if (c.splits == 1) p.rest_whole = p.rest_tiles;
  if (c.whole == 0 && c.splits > 1 && p.sink_tiles) {  // less than a round: the sinks' pieces as short as the others
    const int64_t m = rest / c.splits > 8 ? rest / c.splits : 8;
    p.sink_splits = (whole + m - 1) / m < most ? (whole + m - 1) / m : most;
    head = sinks_in * p.sink_splits;
  }
  p.sink_items = head;
  p.items = head + p.rest_whole + (p.rest_tiles - p.rest_whole) * p.rest_splits;
  p.pieces = (p.sink_splits > 1 ? head : 0) + (p.rest_splits > 1 ? (p.rest_tiles - p.rest_whole) * p.rest_splits : 0);
  return p;
}
// float4-aligned workspace: dK/dV pieces, then dQ parts
int64_t bwd_floats(const DkdvPlan& p, const WinCut& c, int64_t row_tiles, int64_t D) {
  return p.pieces * 128 * key_tiles_of((int)D) * D + (row_tiles - c.whole) * c.splits * 128 * D;
}

}  // namespace

extern "C" {

int prism_window_bwd_plan(int B, int Hq, int Hk, int64_t Sq, int64_t Sk, int D, int64_t window, int64_t sinks, int causal,
                          int /*kv_lens*/, int64_t* floats) {
  PRISM_REQUIRE(B >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Sq >= 0 && Sk >= 0 && D >= 1 && window >= 1 &&
                    sinks >= 0 && floats,
                "prism_window_bwd_plan: bad argument");
  const int64_t G = Hq / Hk;
  *floats = bwd_floats(dkdv_plan(B, Hk, G, Sq, Sk, D, window, sinks, causal),
                       win_row_cut(dq_slots(D), B, Hk, G, Sq, Sk, D, window, sinks, causal), (int64_t)B * Hk * ((Sq * G + 127) / 128), D);
  return PRISM_OK;
}

int prism_window_bwd(const void* do_, const void* q, const void* k, const void* v, const void* o, const void* rest,
                     const float* lse, int dtype, int B, int Hq, int Hk, int64_t Sq, int64_t Sk, int D, const int64_t* strides,
                     int64_t window, int64_t sinks, int causal, const int32_t* q_lens, const int32_t* kv_lens,
                     float sm_scale, void* dq, void* dk, void* dv, float* rows, float* acc, hipStream_t stream) {
  if (const int rc = win_check("prism_window_bwd", dtype, B, Hq, Hk, Sq, Sk, D, window, sinks, sm_scale, strides, 8,
                               {q, k, v, o, rest, do_, dq, dk, dv, acc}))
    return rc;
  if (B == 0) return PRISM_OK;
  PRISM_REQUIRE(Sq == 0 || (q && o && do_ && lse && dq && rows), "prism_window_bwd: null pointer");
  PRISM_REQUIRE(Sk == 0 || (k && v && dk && dv), "prism_window_bwd: null pointer");
  WinBwdArgs a{};
  a.w = win_args(q, k, v, (void*)o, B, Hq, Hk, Sq, Sk, strides, window, sinks, causal, q_lens, kv_lens, sm_scale);
  a.w.lse = (float*)lse;
  a.w.rest = (uint16_t*)rest;
  const int64_t* s = strides + 12;
  a.do_ = {(uint16_t*)do_, s[0], s[1], s[2]};
  a.dq = {(uint16_t*)dq, s[3], s[4], s[5]};
  a.dk = {(uint16_t*)dk, s[6], s[7], s[8]};
  a.dv = {(uint16_t*)dv, s[9], s[10], s[11]};
  a.m2 = rows;
  a.delta = rows + (int64_t)B * Hq * Sq;
  a.w.tiles = (int)((Sq * a.w.G + 127) / 128);
  const int64_t total = (int64_t)B * Hk * a.w.tiles;
  const WinCut c = win_row_cut(dq_slots(D), B, Hk, a.w.G, Sq, Sk, D, window, sinks, causal);
  const DkdvPlan p = dkdv_plan(B, Hk, a.w.G, Sq, Sk, D, window, sinks, causal);
  const int64_t cut = total - c.whole, items = c.whole + cut * c.splits;
  PRISM_REQUIRE(items < PRISM_MAX_THREADS / 256 && p.items < PRISM_MAX_THREADS / (256 * key_tiles_of(D)),
                "prism_window_bwd: too many tiles");
  PRISM_REQUIRE(p.pieces + cut == 0 || acc, "prism_window_bwd: null workspace");
  a.w.total = (int)total;
  a.w.whole = (int)c.whole; a.w.splits = (int)c.splits; a.w.items = (int)items;
  a.w.ranked = win_ranked(q_lens, B, a.w.tiles, total, dq_slots(D));
  a.ranked = win_ranked(kv_lens, B, p.key_tiles, p.rest_tiles, key_slots(D));
  a.exact = cut == 0 && win_few(Sk, window, sinks, causal);
  a.w.part = acc + p.pieces * 128 * key_tiles_of(D) * D;
  a.sink_tiles = (int)p.sink_tiles; a.key_tiles = (int)p.key_tiles;
  a.sink_splits = (int)p.sink_splits; a.sink_items = (int)p.sink_items;
  a.rest_whole = (int)p.rest_whole; a.rest_splits = (int)p.rest_splits; a.items = (int)p.items;
  a.acc = (float4*)acc;
  const int cut_sinks = p.sink_splits > 1 ? B * Hk * a.sink_tiles : 0;
  const int64_t cut_keys = cut_sinks + (p.rest_splits > 1 ? p.rest_tiles - p.rest_whole : 0);
  auto run = [&](auto e, auto d) {
    using E = decltype(e);
    constexpr int DD = decltype(d)::value;
    if (items) window_dq_kernel<E, DD><<<(unsigned)items, 256, 0, stream>>>(a);
    if (cut) window_dq_merge_kernel<E, DD><<<dim3((unsigned)cut, DD / 32), 256, 0, stream>>>(a);
    if (p.items) window_dkdv_kernel<E, DD><<<(unsigned)p.items, DkdvTiles<DD>::THREADS, 0, stream>>>(a);
    if (cut_keys) window_merge_kernel<E, DD><<<dim3((unsigned)cut_keys, DD / 16), 128 * key_tiles_of(DD), 0, stream>>>(a, cut_sinks);
  };
  if (dtype == PRISM_BF16) {
    if (D == 64) run(WinBf16{}, std::integral_constant<int, 64>{});
    else run(WinBf16{}, std::integral_constant<int, 128>{});
  } else {
    if (D == 64) run(WinF16{}, std::integral_constant<int, 64>{});
    else run(WinF16{}, std::integral_constant<int, 128>{});
  }
  PRISM_LAUNCH_CHECK("prism_window_bwd");
  return PRISM_OK;
}

}  // extern "C"
