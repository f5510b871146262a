// Attention of packed sequences, forward (gfx950, v_mfma_f32_32x32x16): token i of a
// sequence with L keys and n queries sees its keys j <= i + L - n (causal), or all.
//
//   o = sum_j softmax_j(scale q k_j) v_j over the seen keys; 0, and lse -inf, where there are none
//
// The inner loop is that of window_fwd.hip: one workgroup of four waves per 128 rows, K
// and V tiles of 64 keys copied HBM -> LDS into two stages, S^T = K Q^T with one query
// per lane column, softmax in base 2 with a lazy running maximum, O^T += V^T P^T from the
// S^T accumulators; only tiles on the diagonal and at a sequence's end are masked.  What
// each workgroup takes stands in a list that a first kernel makes from the lengths
// (packed.h).
//
// Numbers: as window_fwd.hip (scores, maximum, sum and output fp32; P rounded to the
// inputs' type for its product, o once).
//
// Bound: the matrix and vector units together (58 and 55% busy, D = 128).  Measured (bf16,
// D = 128, causal): 16,001 tokens of three sequences, 32 heads over 8: 0.72 to 0.87 ms as the
// clocks allow, 1.05 PFLOP/s at best (a library product of 8,192^3 reaches 1.29), the list
// 6 us of it; 8,191 of six, 16 over 4: 79 us (0.63 PFLOP/s: two rounds of unequal blocks);
// 301 of seven, 32 over 8, without a list: 8.1 us.
#include "packed.h"

namespace {

template <class E>
__device__ __forceinline__ void pack_store_o(const PackArgs& a, int64_t at, int g, float4 x, float4 y) {
  const uint2 u = win_pack4<E>(x), v = win_pack4<E>(y);
  *reinterpret_cast<uint4*>(a.o.p + at + 8 * g) = win_join_halves(u, v);
  if (a.rest) win_store<E>(a.rest + at, g, win_left<E>(x, u), win_left<E>(y, v));
}

template <class E, int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void packed_fwd_kernel(PackArgs a) {
  using T = WinTiles<D>;
  using RT = typename T::RT;
  constexpr int NS = D / 16, NDT = D / 32;
  __shared__ __align__(1024) uint8_t smem[2 * T::STAGE];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  PackItem it;
  it.init(a, pack_id(a.list, (int)blockIdx.x));
  if (!it.live) return;
  const int rows = it.s.n * a.G, r0 = it.tile * 128, wr0 = r0 + 32 * w, off = it.s.L - it.s.n;
  auto token = [&](int r) { return (r < rows ? r : rows - 1) / a.G; };
  const int nk = pack_keys(a, it.s, token(r0 + 127));
  const int all = (nk + 63) >> 6;
  const int t0 = it.first_of(all, it.part), t1 = it.first_of(all, it.part + 1);

  const float NINF = -__builtin_inff();
  PackCopy<D> copy;
  copy.init(a, it, w & 1, lane);
  const uint32_t lds0 = lds_addr(smem);
  if (w < 2 && t1 > t0) copy.issue(nk, 64 * t0, lds0 + (uint32_t)((t0 & 1) * T::STAGE));

  RowOperand kop;
  kop.init<RT>(0, l32, g);
  TrOperand vop;
  vop.init<RT>(0, lane);

  // this lane's row (rows past the end re-read the last one and are not stored)
  const int r = wr0 + l32, rc = r < rows ? r : rows - 1;
  const int i = rc / a.G, head = it.hk * a.G + (rc - i * a.G);
  const uint16_t* qp = a.q.p + head * a.q.h + (it.s.q0 + i) * a.q.s;
  bf16x8 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = ld_bf16x8(qp + 16 * s + 8 * g);
#pragma unroll
  for (int s = 0; s < NS; ++s) consume_regs(qf[s]);

  const int last = pack_keys(a, it.s, i) - 1;  // the last key that the row sees (-1: none)
  const bool some = wr0 < rows;
  const int first_last = (int)uniform_u32((uint32_t)(pack_keys(a, it.s, token(wr0)) - 1));  // of the wave's first row
  const int wave_last = (int)uniform_u32((uint32_t)(pack_keys(a, it.s, token(wr0 + 31)) - 1));

  f32x16 acc_o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = f32x16_zero();
  float m = NINF, l = 1.0f;

  for (int t = t0; t < t1; ++t) {
    dma_wait_all();
    __syncthreads();
    if (w < 2 && t + 1 < t1) copy.issue(nk, 64 * (t + 1), lds0 + (uint32_t)(((t + 1) & 1) * T::STAGE));
    const int u0 = 64 * t;
    if (!some || u0 > wave_last) continue;
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
    if (u0 + 63 > first_last) {
      // this lane's keys are 32 kh + 8 j + 4 g + x: bit (32 kh + 8 j + x) of the word >> 4 g
      const uint64_t mm = upto_bits(last, u0) >> (4 * g);
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

  if (some && win_not_finite<NDT>(acc_o, l, r < rows)) {
    WinArgs wa{};
    wa.scale_log2 = a.scale_log2;
    win_careful<E, D>(wa, KeyList{0, 0, nk}, TokenSpan{0, last, 0}, 64 * t0, 64 * t1 < nk ? 64 * t1 : nk, qp, copy.kb, copy.vb,
                      copy.kstep, copy.vstep, g, acc_o, m, l);
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
  const int ie = re / a.G, he = it.hk * a.G + (re - ie * a.G);
  const float inv = 1.0f / l;
  const int64_t at = he * a.o.h + (it.s.q0 + ie) * a.o.s;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; j += 2)
      pack_store_o<E>(a, at + 32 * dt + 8 * j, g, win_scaled(acc_o[dt], j, inv), win_scaled(acc_o[dt], j + 1, inv));
  if (a.lse && g == 0) a.lse[(int64_t)he * a.Tq + it.s.q0 + ie] = (m + __log2f(l)) * 0.6931471805599453f;
}

// the parts of a cut row tile, in order: one workgroup per tile and 32 channels, the
// lanes of packed_fwd_kernel (as window_fwd_join_kernel)
template <class E, int D>
__global__ __launch_bounds__(256) void packed_fwd_join_kernel(PackArgs a) {
  constexpr int NDT = D / 32;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, w = threadIdx.x >> 6, dt = (int)blockIdx.y;
  PackItem it;
  it.init_cut(a, (int)blockIdx.x);
  if (!it.live) return;
  const int r = it.tile * 128 + 32 * w + l32;
  if (r >= it.s.n * a.G) return;
  const float NINF = -__builtin_inff();
  const int64_t first = (int64_t)it.slot * 4 + w;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first * 32 + l32;
  const float4* pa = reinterpret_cast<const float4*>(a.part) + (first * NDT + dt) * 256 + lane;
  float top = NINF;
#pragma unroll 8
  for (int s = 0; s < it.parts; ++s) top = fmaxf(top, ml[(int64_t)s * 128].x);
  float4 o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 1
  for (int s = 0; s < it.parts; s += 4) {  // (four parts in flight, past the end the last one again)
    float2 x[4];
    float4 v[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = s + k < it.parts ? s + k : it.parts - 1;
      x[k] = ml[t * 128];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = pa[t * 4 * NDT * 256 + j * 64];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = s + k < it.parts;
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
  const int64_t at = head * a.o.h + (it.s.q0 + i) * a.o.s + 32 * dt;
#pragma unroll
  for (int j = 0; j < 4; j += 2) pack_store_o<E>(a, at + 8 * j, g, win_scaled(o[j], inv), win_scaled(o[j + 1], inv));
  if (a.lse && g == 0 && dt == 0)
    a.lse[(int64_t)head * a.Tq + it.s.q0 + i] = none ? NINF : (top + __log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------ the work list
constexpr int kPlanThreads = 1024, kBins = 512;

// A block's length in list tiles, of its longest tile
__device__ __forceinline__ int pack_cost(const PackArgs& a, const PackList& l, const PackSeq& s, int tile, int tiles) {
  if (l.keys) {
    const int n = s.n - pack_first(a, s, tile * l.unit);
    return ((n + 63) >> 6) * a.G;
  }
  const int end = (tile + l.gs < tiles ? tile + l.gs : tiles), r = end * l.unit - 1, rows = s.n * a.G;
  return (pack_keys(a, s, (r < rows ? r : rows - 1) / a.G) + 63) >> 6;
}

// One workgroup per list: the blocks' lengths in all, then how many stand in each of
// kBins lengths, then every block (or its parts) at its place, longest first.  (Which of
// two equally long blocks stands first varies; results do not depend on it.)
__global__ __launch_bounds__(kPlanThreads) void pack_plan_kernel(PackArgs a, PackList second) {
  const PackList l = blockIdx.x == 0 ? a.list : second;
  a.list = l;
  __shared__ unsigned long long total;
  __shared__ int longest, cuts, pieces, at[kBins], sums[kBins / 64];
  const int tid = (int)threadIdx.x;
  // lanes of a sequence: as many as leave one sequence for each group
  int lanes = 64;
  while (lanes > 1 && (kPlanThreads / lanes) < a.B + 2) lanes >>= 1;
  const int group = tid / lanes, sub = tid & (lanes - 1), groups = kPlanThreads / lanes;
  // (three walks over the blocks; the group's first sequence, and a thread's first block of it,
  // often its only ones, are looked up once)
  PackSeq mine{0, 0, 0, 0};
  if (group < a.B + 2) mine = pack_seq(a, group, l.keys);
  const int my_tiles = pack_tiles(a, mine);
  const int my_cost = sub * l.gs < my_tiles ? pack_cost(a, l, mine, sub * l.gs, my_tiles) : 0;
  // (no thread walks more blocks than sequences that do not overlap can have in all)
  auto blocks = [&](auto visit) {
    int left = l.max_entries;
    if (sub * l.gs < my_tiles) visit(mine, sub * l.gs, my_cost);
    for (int t = (sub + lanes) * l.gs; t < my_tiles && left > 0; t += lanes * l.gs, --left)
      visit(mine, t, pack_cost(a, l, mine, t, my_tiles));
    for (int s = group + groups; s < a.B + 2; s += groups) {
      const PackSeq q = pack_seq(a, s, l.keys);
      const int tiles = pack_tiles(a, q);
      for (int t = sub * l.gs; t < tiles && left > 0; t += lanes * l.gs, --left) visit(q, t, pack_cost(a, l, q, t, tiles));
    }
  };
  if (tid == 0) {
    total = 0;
    longest = 1;
    cuts = pieces = 0;
  }
  for (int x = tid; x < kBins; x += kPlanThreads) at[x] = 0;
  __syncthreads();
  {
    unsigned long long sum = 0;
    int top = 0;
    blocks([&](const PackSeq&, int, int c) {
      sum += (unsigned long long)c;
      top = c > top ? c : top;
    });
    for (int off = 32; off >= 1; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
    sum = wave_sum_u64(sum);
    if ((tid & 63) == 0) {
      atomicAdd(&total, sum);
      atomicMax(&longest, top);
    }
  }
  __syncthreads();
  // a part's length, about; without cuts, the longest block's
  const int whole = longest;
  int share = whole;
  if (l.want) {
    const double fair = ceil((double)total / (double)l.want);
    share = fair < (double)whole ? (int)fair : whole;
    share = share > l.least ? share : l.least;
  }
  auto parts_of = [&](int c) {
    return l.want == 0 || 4 * c <= l.from * share ? 1 : (4 * c - (l.from - 4) * share + 4 * share - 1) / (4 * share);
  };
  const float per_bin = (float)(kBins - 1) / (float)whole;
  auto bin_of = [&](int c, int parts) {  // longest first
    const int bin = kBins - 1 - (int)((float)c * per_bin / (float)parts);
    return bin < 0 ? 0 : bin < kBins ? bin : kBins - 1;
  };
  blocks([&](const PackSeq&, int, int c) {
    const int p = parts_of(c);
    atomicAdd(&at[bin_of(c, p)], p);
  });
  __syncthreads();
  // the bins' first places (exclusive sums)
  int count = 0, upto = 0;
  if (tid < kBins) {
    count = at[tid];
    upto = (int)wave_incl_scan_u32((uint32_t)count, tid & 63);
    if ((tid & 63) == 63) sums[tid >> 6] = upto;
  }
  __syncthreads();
  if (tid < kBins) {
    for (int x = 0; x < (tid >> 6); ++x) upto += sums[x];
    at[tid] = upto - count;
    if (tid == kBins - 1) l.counts[0] = (uint32_t)upto < (uint32_t)l.max_entries ? upto : l.max_entries;
  }
  __syncthreads();
  blocks([&](const PackSeq& q, int t, int c) {
    const int p = parts_of(c), first = atomicAdd(&at[bin_of(c, p)], p);
    int slot = -1;
    if (p > 1) {
      const int x = atomicAdd(&cuts, 1);
      slot = atomicAdd(&pieces, p * l.per);
      // (pack_cut's room is enough for any bounds, as the shares come from the same lengths; a block
      // without room would be dropped, and its place among the cuts, which are counted, hold nothing)
      const bool room = (uint32_t)x < (uint32_t)l.max_cuts && slot >= 0 && slot <= l.max_pieces - p * l.per;
      if ((uint32_t)x < (uint32_t)l.max_cuts)
        l.cuts[x] = room ? PackEntry{q.q0, q.n, q.k0, q.L, t, 0, p, slot} : PackEntry{0, 0, 0, 0, 0, 0, 1, -1};
      if (!room) slot = -2;
    }
    for (int y = 0; y < p; ++y)
      if ((uint32_t)(first + y) < (uint32_t)l.max_entries)
        l.entries[first + y] = slot == -2 ? PackEntry{0, 0, 0, 0, 0, 0, 1, -1} : PackEntry{q.q0, q.n, q.k0, q.L, t, y, p, slot};
  });
  __syncthreads();
  if (tid == 0) {
    l.counts[1] = (uint32_t)cuts < (uint32_t)l.max_cuts ? cuts : l.max_cuts;
    l.counts[2] = pieces;
  }
}

// workgroups of packed_fwd_kernel that the chip holds: two a CU at D = 128, four
// at 64 (registers)
int64_t fwd_slots(int D) { return D == 128 ? 512 : 1024; }
PackCut fwd_cut(int B, int64_t G, int Hk, int64_t Tq, int64_t Tk, int D) {
  return pack_cut(Tq * G, 128, B, Hk, fwd_slots(D), (Tk + 63) / 64, 0, 4);
}

}  // namespace

PackCut pack_cut(int64_t rows, int unit, int64_t B, int64_t Hk, int64_t slots, int64_t longest, int keys, int least) {
  PackCut c{};
  const int64_t mean = rows / unit / (B > 0 ? B : 1), tiles = rows / unit + B + 2;
  c.list.unit = unit;
  c.list.keys = keys;
  c.list.least = least;
  if (B <= 62 && tiles * Hk <= slots && longest <= 2 * least) {
    c.list.gs = 1;
    c.list.per = (int)Hk;
    c.list.items = (int)(tiles * Hk);
    return c;
  }
  // Blocks of eight tiles where sequences have many (16,001 tokens of three, 32 heads over 8:
  // 737 us, of four 755, of two 769, single ones 797); of two tiles of keys, which are longer and
  // are cut (eight of 12,000: dQ and dK/dV 614 us, of eight 654).
  int gs = keys ? 2 : 8;
  while (gs > 1 && mean < 2 * gs) gs /= 2;
  const int64_t per = gs * Hk, blocks = rows / (unit * gs) + B + 2;
  // Parts.  Rows: as many as make one round of the chip with the tiles, none where the tiles
  // fill it: a part's sums are written and read (66 KB at D = 128).  Measured (us, uncut / one
  // round / two rounds of parts), forward, D = 128: one sequence of 4,000, 2 heads 77 / 37 / 41;
  // 2,047, 32 heads over 8 (one round uncut) 58 / 59 / 76; six of 8,191 in all, 16 over 4, (two
  // rounds) 73 / 75 / 103.  Keys, whose lists differ most and whose workgroups have a CU each: of
  // 17 twentieths of a round, from 1.25 such lengths on.  dQ and dK/dV (uncut / three quarters /
  // nine tenths / 1.2 rounds, all from 1.5 on): the same 125 / 81 / 78 / 85, 231 / 175 / 163 / 179,
  // 257 / 260 / 238 / 235; four of 5,000 without the mask, 10 over 5, 155 / 160 / 162 / 179.  (0.9
  // from 1.5 / 0.9 from 1.25 / 0.85 from 1.25 / 0.8 from 1.125: 79 / 78 / 78 / 78, 163 / 171 / 159 /
  // 159, 240 / 225 / 228 / 227, 160 / 171 / 161 / 177.)
  const int64_t fill = slots > tiles * Hk ? slots - tiles * Hk : 0;
  const int64_t want = keys ? (tiles * Hk > 6 * slots ? 0 : (slots * 17 / 20 + per - 1) / per) : fill / per;
  c.list.from = keys ? 5 : 6;
  c.list.gs = gs;
  c.list.per = (int)per;
  c.list.want = (int)want;
  // A block is cut from f = from / 4 shares on, into length / share - f + 1 parts, rounded up, the
  // shares being `want` at most in all: no more than want / f are cut, into no more than 2 want / f
  c.entries = blocks + want;
  c.cuts = (4 * want + c.list.from - 1) / c.list.from;
  c.pieces = (8 * want + c.list.from - 1) / c.list.from * per;
  c.list.max_entries = (int)c.entries;
  c.list.max_cuts = (int)c.cuts;
  c.list.max_pieces = (int)c.pieces;
  c.list.items = (int)(c.entries * per < (1ll << 30) ? c.entries * per : 1ll << 30);  // (more are refused)
  c.list.entries = (PackEntry*)1;  // (pack_place)
  return c;
}
void pack_place(PackCut* c, int32_t* buffer) {
  if (!c->list.entries) return;
  c->list.counts = buffer;
  c->list.entries = (PackEntry*)(buffer + 8);
  c->list.cuts = c->list.entries + c->entries;
}

int pack_check(const char* name, int dtype, int B, int Hq, int Hk, int64_t Tq, int64_t Tk, int D, float sm_scale,
               const int64_t* strides, int tensors, std::initializer_list<const void*> pointers) {
  PRISM_REQUIRE(dtype == PRISM_BF16 || dtype == PRISM_F16, "%s: dtype code %d (bfloat16 or float16)", name, dtype);
  PRISM_REQUIRE(D == 64 || D == 128, "%s: head_dim %d unsupported (64, 128)", name, D);
  PRISM_REQUIRE(B >= 0 && B < (1 << 24) && Hk >= 1 && Hq >= Hk && Hq % Hk == 0,
                "%s: %d query heads do not share %d key heads evenly", name, Hq, Hk);
  PRISM_REQUIRE(Tq >= 0 && Tk >= 0 && Tq < (1 << 29) && Tk < (1 << 29) && Tq * (Hq / Hk) < (1ll << 30),
                "%s: too many tokens", name);
  PRISM_REQUIRE(sm_scale > 0.0f && sm_scale < __builtin_inff(), "%s: sm_scale must be positive and finite", name);
  PRISM_REQUIRE(strides, "%s: null pointer", name);
  // rows are copied 16 bytes at a time at 32-bit offsets inside a tile
  for (int i = 0; i < tensors; ++i)
    PRISM_REQUIRE(strides[2 * i] % 8 == 0 && strides[2 * i + 1] % 8 == 0 && strides[2 * i + 1] >= 0 &&
                      strides[2 * i + 1] < (1 << 24),
                  "%s: strides must be multiples of 8 elements, a row's below 2^24", name);
  for (const void* p : pointers)
    PRISM_REQUIRE(((uintptr_t)p & 15) == 0, "%s: pointers must be 16-byte aligned", name);
  return PRISM_OK;
}

PackArgs pack_args(const void* q, const void* k, const void* v, void* o, int B, int Hq, int Hk, int64_t Tq, int64_t Tk,
                   const int64_t* s, const int32_t* cu_q, const int32_t* cu_k, int causal, float sm_scale) {
  PackArgs a{};
  a.q = {(uint16_t*)q, s[0], s[1]};
  a.k = {(uint16_t*)k, s[2], s[3]};
  a.v = {(uint16_t*)v, s[4], s[5]};
  a.o = {(uint16_t*)o, s[6], s[7]};
  a.cu_q = cu_q; a.cu_k = cu_k;
  a.B = B; a.Hk = Hk; a.G = Hq / Hk; a.Tq = (int)Tq; a.Tk = (int)Tk;
  a.causal = causal != 0;
  a.scale = sm_scale; a.scale_log2 = sm_scale * 1.4426950408889634f;
  return a;
}

void pack_plan(const PackArgs& a, const PackList* b, hipStream_t stream) {
  const bool first = a.list.entries, other = b && b->entries;
  if (first) pack_plan_kernel<<<other ? 2 : 1, kPlanThreads, 0, stream>>>(a, other ? *b : a.list);
  else if (other) {
    PackArgs c = a;
    c.list = *b;
    pack_plan_kernel<<<1, kPlanThreads, 0, stream>>>(c, *b);
  }
}

extern "C" {

int prism_packed_fwd_plan(int B, int Hq, int Hk, int64_t Tq, int64_t Tk, int D, int64_t* ints, int64_t* floats) {
  PRISM_REQUIRE(B >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Tq >= 0 && Tk >= 0 && D >= 1 && ints && floats,
                "prism_packed_fwd_plan: bad argument");
  const PackCut c = fwd_cut(B, Hq / Hk, Hk, Tq, Tk, D);
  *ints = pack_ints(c);
  *floats = c.pieces * 128 * (D + 2);
  return PRISM_OK;
}

int prism_packed_fwd(const void* q, const void* k, const void* v, int dtype, int B, int Hq, int Hk, int64_t Tq, int64_t Tk,
                     int D, const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int causal, float sm_scale,
                     void* o, void* rest, float* lse, int32_t* plan, float* part, hipStream_t stream) {
  if (const int rc = pack_check("prism_packed_fwd", dtype, B, Hq, Hk, Tq, Tk, D, sm_scale, strides, 4, {q, k, v, o, rest, plan, part}))
    return rc;
  if (Tq == 0) return PRISM_OK;
  PRISM_REQUIRE(q && o && cu_q && cu_k && (Tk == 0 || (k && v)), "prism_packed_fwd: null pointer");
  PackArgs a = pack_args(q, k, v, o, B, Hq, Hk, Tq, Tk, strides, cu_q, cu_k, causal, sm_scale);
  a.lse = lse;
  a.rest = (uint16_t*)rest;
  PackCut c = fwd_cut(B, a.G, Hk, Tq, Tk, D);
  PRISM_REQUIRE(c.list.items < PRISM_MAX_THREADS / 256, "prism_packed_fwd: too many row tiles");
  PRISM_REQUIRE((!c.list.entries || plan) && (!c.pieces || part), "prism_packed_fwd: null workspace");
  pack_place(&c, plan);
  a.list = c.list;
  a.part = part;
  a.part_ml = part + c.pieces * 128 * D;
  pack_plan(a, nullptr, stream);
  auto run = [&](auto kernel, auto join) {
    kernel<<<(unsigned)a.list.items, 256, 0, stream>>>(a);
    if (c.cuts) join<<<dim3((unsigned)(c.cuts * c.list.per), (unsigned)(D / 32)), 256, 0, stream>>>(a);
  };
  if (dtype == PRISM_BF16) {
    if (D == 64) run(packed_fwd_kernel<WinBf16, 64>, packed_fwd_join_kernel<WinBf16, 64>);
    else run(packed_fwd_kernel<WinBf16, 128>, packed_fwd_join_kernel<WinBf16, 128>);
  } else {
    if (D == 64) run(packed_fwd_kernel<WinF16, 64>, packed_fwd_join_kernel<WinF16, 64>);
    else run(packed_fwd_kernel<WinF16, 128>, packed_fwd_join_kernel<WinF16, 128>);
  }
  PRISM_LAUNCH_CHECK("prism_packed_fwd");
  return PRISM_OK;
}

}  // extern "C"
