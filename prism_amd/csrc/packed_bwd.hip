// Attention of packed sequences, backward (gfx950, v_mfma_f32_32x32x16), of packed_fwd.hip:
//
//   P = exp(scale q k - lse),  delta = rowsum(o do),  dS = P (do v - delta)
//   dv = P^T do,  dk = scale dS^T q,  dq = scale dS k
//
// The inner loops are those of window_bwd.hip.  packed_dq_kernel, by 128 rows, over the
// keys of the forward; it forms delta from do, o and o's rest (what its rounding left off)
// and leaves (lse log2 e - GRAD, delta) of every row for packed_dkdv_kernel, by 128 keys (64
// at D = 64), over the tokens that see them, one query head of the group after the other.
// Both take their work from lists (packed.h): under the causal mask the first keys of a
// sequence are seen by all its tokens and the last by one, so blocks are taken longest first
// and the longest are cut, their fp32 sums added in order by a last kernel.  No atomics on
// results: the same bits every time; sums over the heads that share a key head are fp32.
//
// Bound: the matrix unit and its operands' reads from LDS (busy 46% in dQ and 55% in dK/dV of
// the time that includes the last, uneven round).  Measured (bf16, D = 128, causal, 8,191
// tokens of six sequences, 16 heads over 4): dQ 100 us (0.74 PFLOP/s), dK/dV 128 (0.77),
// the lists 5.6, the merge 6; before the keys were cut by a fair share of a round 163
// + 98.
//
// Numbers: P and dS are rounded to the inputs' type for the products (float16: times
// 2^GRAD, window.h; a dS beyond 1,023 becomes infinite, which a loss scaler sees), the
// rest is fp32.
#include <type_traits>

#include "packed.h"

namespace {

struct PackBwdArgs {
  PackArgs w;                // (w.o: the forward's output; w.lse: its lse; w.list, w.part: dQ's)
  PackTensor do_, dq, dk, dv;
  float* m2;                 // [Hq, Tq] lse log2 e - GRAD
  float* delta;              // [Hq, Tq]
  PackList keys;             // dK/dV's list
  float4* acc;               // and its pieces
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
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_dq_kernel(PackBwdArgs ba) {
  const PackArgs& a = ba.w;
  using T = WinTiles<D>;
  using RT = typename T::RT;
  constexpr int NS = D / 16, NDT = D / 32;
  __shared__ __align__(1024) uint8_t smem[2 * T::STAGE];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  PackItem it;
  it.init(a, pack_id(a.list, (int)blockIdx.x));
  if (!it.live) return;
  const int rows = it.s.n * a.G, r0 = it.tile * 128, wr0 = r0 + 32 * w;
  auto token = [&](int r) { return (r < rows ? r : rows - 1) / a.G; };
  const int nk = pack_keys(a, it.s, token(r0 + 127));
  const int every = (nk + 63) >> 6;
  const int t0 = it.first_of(every, it.part), t1 = it.first_of(every, it.part + 1);

  PackCopy<D> copy;
  copy.init(a, it, w & 1, lane);
  const uint32_t lds0 = lds_addr(smem);
  if (w < 2 && t1 > t0) copy.issue(nk, 64 * t0, lds0 + (uint32_t)((t0 & 1) * T::STAGE));

  RowOperand rop;  // K / V rows l32 (+ 32 kh as an immediate)
  rop.init<RT>(0, l32, g);
  TrOperand top;   // K^T over key rows 0 .. 63
  top.init<RT>(0, lane);

  const int r = wr0 + l32, rc = r < rows ? r : rows - 1;
  const int i = rc / a.G, head = it.hk * a.G + (rc - i * a.G);
  const int64_t lrow = (int64_t)head * a.Tq + it.s.q0 + i, row = it.s.q0 + i;
  bf16x8 qf[NS], df[NS];
  float dlt = 0.0f;
  {
    const uint16_t* qp = a.q.p + head * a.q.h + row * a.q.s + 8 * g;
    const uint16_t* dp = ba.do_.p + head * ba.do_.h + row * ba.do_.s + 8 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      qf[s] = ld_bf16x8(qp + 16 * s);
      df[s] = ld_bf16x8(dp + 16 * s);
    }
    // (all loads before the first sum that waits for one)
    const int64_t at = head * a.o.h + row * a.o.s + 8 * g;
    bf16x8 of[NS], rf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      of[s] = ld_bf16x8(a.o.p + at + 16 * s);
      rf[s] = ld_bf16x8(a.rest + at + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) dlt = dot8<E>(rf[s], df[s], dlt);
#pragma unroll
    for (int s = 0; s < NS; ++s) dlt = dot8<E>(of[s], df[s], dlt);
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
  const int last = pack_keys(a, it.s, i) - 1;  // the last key that the row sees (-1: none)
  const bool some = wr0 < rows;
  const int first_last = (int)uniform_u32((uint32_t)(pack_keys(a, it.s, token(wr0)) - 1));  // of the wave's first row
  const int wave_last = (int)uniform_u32((uint32_t)(pack_keys(a, it.s, token(wr0 + 31)) - 1));

  dlt = xor32_add(dlt);
  const float mg = mq - E::GRAD;  // P and dS from here on times 2^GRAD (window.h)
  if (r < rows && g == 0 && it.part == 0) {
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
    if (w < 2 && t + 1 < t1) copy.issue(nk, 64 * (t + 1), lds0 + (uint32_t)(((t + 1) & 1) * T::STAGE));
    const int u0 = 64 * t;
    if (!some || u0 > wave_last) continue;
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
    if (u0 + 63 > first_last) {
      // dS is 0 where the query does not see the key, whatever the unmasked
      // values were (after the exponentials, which so stay in one block with the
      // products before them)
      const uint64_t mm = upto_bits(last, u0) >> (4 * g);
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
  uint16_t* dqr = ba.dq.p + head * ba.dq.h + row * ba.dq.s;
  const float f = a.scale * E::BACK;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int jj = 0; jj < 4; jj += 2)
      win_store<E>(dqr + 32 * dt + 8 * jj, g, win_scaled(dq[dt], jj, f), win_scaled(dq[dt], jj + 1, f));
}

// ------------------------------------------------------------ dK / dV
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
__global__ __launch_bounds__(DkdvTiles<D>::THREADS, D == 64 ? 3 : 1) void packed_dkdv_kernel(PackBwdArgs ba) {
  const PackArgs& a = ba.w;
  using T = DkdvTiles<D>;
  using RT = RowTile<D>;
  using RS = RowSource<D>;
  constexpr int NS = D / 16, NDT = D / 32, SB = T::STAGE, COUNT = 2 * RT::KB / 4, KEYS = T::KEYS, STAGES = T::STAGES;
  __shared__ __align__(1024) uint8_t smem[T::LDS];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  const int kh = w & 1, qh = (w >> 1) & 1, tk = w >> 2;
  PackItem it;
  {
    PackArgs b = a;  // (the list of the keys)
    b.list = ba.keys;
    it.init(b, pack_id(ba.keys, (int)blockIdx.x));
  }
  if (!it.live) return;
  const int j0 = it.tile * KEYS, off = it.s.n - it.s.L;

  // the tile's tokens, as 64-token tiles of each head from lo on
  const int lo = pack_first(a, it.s, j0), hi = it.s.n - 1;
  const int nti = hi >= lo ? (hi - lo + 64) >> 6 : 0, all = nti * a.G;
  const int e0 = it.first_of(all, it.part), e1 = it.first_of(all, it.part + 1);
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
    const int64_t row = it.s.q0 + t0;
    qcur = (const uint8_t*)uniform_ptr(a.q.p + head * a.q.h + row * a.q.s);
    dcur = (const uint8_t*)uniform_ptr(ba.do_.p + head * ba.do_.h + row * ba.do_.s);
    rcur = (const float*)uniform_ptr((w == 3 ? ba.m2 : ba.delta) + (int64_t)head * a.Tq + row);
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
    const int64_t kc = it.s.k0 + (jw + l32 < it.s.L ? jw + l32 : it.s.L - 1);
    const uint16_t* kp = a.k.p + it.hk * a.k.h + kc * a.k.s + 8 * g;
    const uint16_t* vp = a.v.p + it.hk * a.v.h + kc * a.v.s + 8 * g;
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
  // of the wave's 32 keys: the first token that sees some, and the first that sees all (past
  // the end: none does)
  const int any0 = jw < it.s.L ? pack_first(a, it.s, jw) : it.s.n;
  const int all0 = jw + 31 < it.s.L ? pack_first(a, it.s, jw + 31) : it.s.n;
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
    if (t0 < all0 || t0 + 31 > hi) {
      // rows that do not see the lane's key: P and dS are 0 there, whatever the
      // unmasked values were (the branch stands after the exponentials, which so
      // stay in one block with the products before them)
      const int ln = opaque_thread_id() & 63, key = jw + (ln & 31);
      const int from = key >= it.s.L ? it.s.n : a.causal && key + off > 0 ? key + off : 0;
      const int b0 = from - t0 > 0 ? from - t0 : 0, b1 = hi - t0 < 31 ? hi - t0 : 31;
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
  auto sees = [&](int t0) { return t0 + 31 >= any0 && t0 <= hi && any0 <= hi; };
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
  uint16_t* dkr = ba.dk.p + it.hk * ba.dk.h + (int64_t)(it.s.k0 + key) * ba.dk.s;
  uint16_t* dvr = ba.dv.p + it.hk * ba.dv.h + (int64_t)(it.s.k0 + key) * ba.dv.s;
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
    if (key >= it.s.L) continue;
#pragma unroll
    for (int jj = 0; jj < 4; jj += 2) {
      const float f = a.scale * E::BACK;
      win_store<E>(dkr + 32 * dt + 8 * jj, g, win_scaled(dk[dt], jj, f), win_scaled(dk[dt], jj + 1, f));
      win_store<E>(dvr + 32 * dt + 8 * jj, g, win_scaled(dv[dt], jj, E::BACK), win_scaled(dv[dt], jj + 1, E::BACK));
    }
  }
}

// the parts of the row tiles of dQ that were cut, in order: one workgroup per
// tile and 32 channels, the lanes of packed_dq_kernel
template <class E, int D>
__global__ __launch_bounds__(256) void packed_dq_merge_kernel(PackBwdArgs ba) {
  constexpr int NDT = D / 32;
  const PackArgs& a = ba.w;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, w = threadIdx.x >> 6, dt = (int)blockIdx.y;
  PackItem it;
  it.init_cut(a, (int)blockIdx.x);
  if (!it.live) return;
  const int r = it.tile * 128 + 32 * w + l32;
  if (r >= it.s.n * a.G) return;
  const float4* pa = reinterpret_cast<const float4*>(a.part) + (((int64_t)it.slot * 4 + w) * NDT + dt) * 256 + lane;
  float4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = pa[j * 64];
#pragma unroll 4
  for (int s = 1; s < it.parts; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = pa[(int64_t)s * 4 * NDT * 256 + j * 64];
      acc[j].x += v.x;
      acc[j].y += v.y;
      acc[j].z += v.z;
      acc[j].w += v.w;
    }
  const int i = r / a.G, head = it.hk * a.G + (r - i * a.G);
  uint16_t* out = ba.dq.p + head * ba.dq.h + (int64_t)(it.s.q0 + i) * ba.dq.s + 32 * dt;
#pragma unroll
  for (int j = 0; j < 4; j += 2)
    win_store<E>(out + 8 * j, g, win_scaled(acc[j], a.scale * E::BACK), win_scaled(acc[j + 1], a.scale * E::BACK));
}

// the pieces' sums of the cut key tiles, in order: one workgroup per tile and
// 32-column block of dK (blocks 0 .. NDT - 1) or dV; wave = 32 keys
template <class E, int D>
__global__ __launch_bounds__(128 * key_tiles_of(D)) void packed_merge_kernel(PackBwdArgs ba) {
  constexpr int NDT = D / 32, NB = 2 * NDT, KW = 2 * key_tiles_of(D);
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, w = threadIdx.x >> 6, blk = (int)blockIdx.y;
  PackItem it;
  {
    PackArgs b = ba.w;
    b.list = ba.keys;
    it.init_cut(b, (int)blockIdx.x);
  }
  if (!it.live) return;
  const int key = it.tile * 32 * KW + 32 * w + l32;
  if (key >= it.s.L) return;
  const float4* pa = ba.acc + (((int64_t)it.slot * KW + w) * NB + blk) * 256 + lane;
  float4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = pa[j * 64];
#pragma unroll 4
  for (int s = 1; s < it.parts; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = pa[(int64_t)s * KW * NB * 256 + j * 64];
      acc[j].x += v.x;
      acc[j].y += v.y;
      acc[j].z += v.z;
      acc[j].w += v.w;
    }
  const bool isk = blk < NDT;
  const PackTensor& t = isk ? ba.dk : ba.dv;
  const float f = (isk ? ba.w.scale : 1.0f) * E::BACK;
  uint16_t* out = t.p + it.hk * t.h + (int64_t)(it.s.k0 + key) * t.s + 32 * (isk ? blk : blk - NDT);
#pragma unroll
  for (int j = 0; j < 4; j += 2) win_store<E>(out + 8 * j, g, win_scaled(acc[j], f), win_scaled(acc[j + 1], f));
}

// workgroups of packed_dq_kernel that the chip holds: two a CU at D = 128, three
// at 64 (registers); of packed_dkdv_kernel one, three at 64
PackCut dq_cut(int B, int64_t G, int Hk, int64_t Tq, int64_t Tk, int D) {
  return pack_cut(Tq * G, 128, B, Hk, D == 128 ? 512 : 768, (Tk + 63) / 64, 0, 4);
}
PackCut dkdv_cut(int B, int64_t G, int Hk, int64_t Tq, int64_t Tk, int D) {
  return pack_cut(Tk, 64 * key_tiles_of(D), B, Hk, D == 128 ? 256 : 768, G * ((Tq + 63) / 64), 1, 8);
}
int64_t dkdv_piece(int D) { return 128ll * key_tiles_of(D) * D; }  // floats

}  // namespace

extern "C" {

int prism_packed_bwd_plan(int B, int Hq, int Hk, int64_t Tq, int64_t Tk, int D, int64_t* ints, int64_t* floats) {
  PRISM_REQUIRE(B >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Tq >= 0 && Tk >= 0 && D >= 1 && ints && floats,
                "prism_packed_bwd_plan: bad argument");
  const int64_t G = Hq / Hk;
  const PackCut c = dq_cut(B, G, Hk, Tq, Tk, D), k = dkdv_cut(B, G, Hk, Tq, Tk, D);
  *ints = pack_ints(c) + pack_ints(k);
  *floats = c.pieces * 128 * D + k.pieces * dkdv_piece(D);
  return PRISM_OK;
}

int prism_packed_bwd(const void* do_, const void* q, const void* k, const void* v, const void* o, const void* rest,
                     const float* lse, int dtype, int B, int Hq, int Hk, int64_t Tq, int64_t Tk, int D,
                     const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int causal, float sm_scale, void* dq,
                     void* dk, void* dv, float* rows, int32_t* plan, float* part, hipStream_t stream) {
  if (const int rc = pack_check("prism_packed_bwd", dtype, B, Hq, Hk, Tq, Tk, D, sm_scale, strides, 8,
                                {q, k, v, o, rest, do_, dq, dk, dv, plan, part}))
    return rc;
  PRISM_REQUIRE(cu_q && cu_k && (Tq == 0 || (q && o && rest && do_ && lse && dq && rows)), "prism_packed_bwd: null pointer");
  PRISM_REQUIRE(Tk == 0 || (k && v && dk && dv), "prism_packed_bwd: null pointer");
  PackBwdArgs a{};
  a.w = pack_args(q, k, v, (void*)o, B, Hq, Hk, Tq, Tk, strides, cu_q, cu_k, causal, sm_scale);
  a.w.lse = (float*)lse;
  a.w.rest = (uint16_t*)rest;
  const int64_t* s = strides + 8;
  a.do_ = {(uint16_t*)do_, s[0], s[1]};
  a.dq = {(uint16_t*)dq, s[2], s[3]};
  a.dk = {(uint16_t*)dk, s[4], s[5]};
  a.dv = {(uint16_t*)dv, s[6], s[7]};
  a.m2 = rows;
  a.delta = rows + (int64_t)Hq * Tq;
  PackCut c = dq_cut(B, a.w.G, Hk, Tq, Tk, D), y = dkdv_cut(B, a.w.G, Hk, Tq, Tk, D);
  PRISM_REQUIRE(c.list.items < PRISM_MAX_THREADS / 256 && y.list.items < PRISM_MAX_THREADS / (256 * key_tiles_of(D)),
                "prism_packed_bwd: too many tiles");
  PRISM_REQUIRE((!c.list.entries && !y.list.entries) || plan, "prism_packed_bwd: null workspace");
  PRISM_REQUIRE(c.pieces + y.pieces == 0 || part, "prism_packed_bwd: null workspace");
  pack_place(&c, plan);
  pack_place(&y, plan + pack_ints(c));
  a.w.list = c.list;
  a.keys = y.list;
  a.w.part = part;
  a.acc = (float4*)(part + c.pieces * 128 * D);
  if (Tq == 0) a.w.list.entries = nullptr;
  pack_plan(a.w, Tk ? &a.keys : nullptr, stream);
  auto run = [&](auto e, auto d) {
    using E = decltype(e);
    constexpr int DD = decltype(d)::value;
    if (Tq) packed_dq_kernel<E, DD><<<(unsigned)a.w.list.items, 256, 0, stream>>>(a);
    if (Tq && c.cuts) packed_dq_merge_kernel<E, DD><<<dim3((unsigned)(c.cuts * c.list.per), DD / 32), 256, 0, stream>>>(a);
    if (Tk) packed_dkdv_kernel<E, DD><<<(unsigned)a.keys.items, DkdvTiles<DD>::THREADS, 0, stream>>>(a);
    if (Tk && y.cuts) packed_merge_kernel<E, DD><<<dim3((unsigned)(y.cuts * y.list.per), DD / 16), 128 * key_tiles_of(DD), 0, stream>>>(a);
  };
  if (dtype == PRISM_BF16) {
    if (D == 64) run(WinBf16{}, std::integral_constant<int, 64>{});
    else run(WinBf16{}, std::integral_constant<int, 128>{});
  } else {
    if (D == 64) run(WinF16{}, std::integral_constant<int, 64>{});
    else run(WinF16{}, std::integral_constant<int, 128>{});
  }
  PRISM_LAUNCH_CHECK("prism_packed_bwd");
  return PRISM_OK;
}

}  // extern "C"
