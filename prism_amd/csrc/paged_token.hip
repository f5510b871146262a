// Attention of few new tokens over a paged cache (gfx950): the n queries of a sequence
// are its last n tokens, query i of L keys sees keys j <= i + L - n.
//
//   o = sum_j softmax_j(scale q k_j) v_j over the seen keys; 0, and lse -inf, where there are none
//
// The time is the read of the cache.  The rows of a (sequence, key head), tokens x heads of
// the group, are cut into tiles, and a tile's keys over `splits` workgroups (as many of them
// as its length asks for do something); in a workgroup each of the four waves walks every
// fourth tile of keys by itself.  The waves' sums are joined in LDS, the workgroups' in a
// second kernel, both in a fixed order.  The pages of a workgroup's keys are looked up in LDS,
// where they are put first (4,096 keys' or more at a time).
//
// 16 bits (paged16_kernel): 32 rows, tiles of 32 keys, K and V copied to a double-buffered LDS
// stage of each wave, as window_token.hip.
//
// 4 bits (paged4_kernel): 16 rows (or 32), tiles of 64 keys.  K's codes go from memory to
// the lanes that multiply them: v_mfma_f32_16x16x32 sums over channels in any order that Q
// shares, so a lane takes one key's 16 adjacent bytes (a scale's 32 channels) and makes each
// word of them an operand (four instructions a word).  V's codes go through LDS, whose
// transposing read gives a lane 16 keys of one channel; their scales, one for each key, are
// multiplied into P instead, once for each 32 channels.  Row r of the S tile t is key 16 (r /
// 4) + 4 t + r % 4, so that a lane's P are 16 adjacent keys, the same ones that it reads of V.
//
// Measured (bf16, 32 heads over 8, D = 128): 16 sequences of up to 8,192 keys in pages of 16, 16
// bits: 80 us and 5 for the join (404 MB: 5.1 TB/s, a copy runs at 4.8).  8 of up to 131,072,
// 4 bits, pages of 64: 168 to 181 us and 5 (840 MB, 4.8 TB/s), the vector unit issuing 79% of the time.
// With V's values made once and passed through LDS as bfloat16 instead of the codes it issues
// 57% and waits for LDS: 184 us; with parts dealt by length over all sequences 183, and small
// calls slower (4 x 2,000 keys: 9.5 us, 12.6).
//
// Numbers: scores, maximum, sum and output fp32.  16 bits: P rounded to the inputs' type,
// o once, as window_token.hip.  4 bits: K's and V's values are exact in the operands (K
// beside float16 queries: as float16), P times V's scale is rounded to bfloat16, whose
// range holds any scale; beside float16 queries to two of them, 16 bits in all (with one,
// o is 1.6e-3 off, norm-wise, for float16's own 2e-4).  Over 32 rows at D = 128 the second takes 16
// registers more than there are, which are spilled: 16 x 8,192 keys, 5 tokens x 64 heads over 8, 97 us, beside
// bfloat16 queries 65.
#include <type_traits>

#include "paged.h"
#include "window.h"

namespace {

constexpr int kMaxSplits = 256, kIds = 2048;  // page ids in LDS at a time

struct PagedArgs {
  const uint16_t* q;
  uint16_t* o;
  int64_t qt, qh, ot, oh;  // strides in elements: token, head
  PagedSide k, v;
  PagedTable table;
  const int32_t* lens;
  int B, Hk, G, n, rows;   // rows: of a (sequence, key head), n G
  float scale_log2;
  float* lse;              // [Hk G, B n], or null
  int tiles, total;        // row tiles of a (sequence, key head), of the launch
  int splits, least;       // key tiles that a part has at least
  float *part, *part_ml;
};

// keys of sequence b
__device__ __forceinline__ int keys_of(const PagedArgs& a, int b) {
  const int x = a.lens[b], most = a.table.width << a.table.lg;
  return x < 0 ? 0 : x < most ? x : most;
}
// parts of `tiles` key tiles
__device__ __forceinline__ int parts_of(const PagedArgs& a, int tiles) {
  const int p = tiles / a.least;
  return p < 1 ? 1 : p < a.splits ? p : a.splits;
}
// What a workgroup takes: rows r0 .. of a (sequence, key head), key tiles t0 .. t1 of KEYS
template <int ROWS, int KEYS>
struct PagedItem {
  int id, b, hk, r0, L, nk, parts, part, t0, t1;
  __device__ __forceinline__ void init(const PagedArgs& a, int block) {
    part = block % a.splits;
    id = block / a.splits;
    const int bh = id / a.tiles;
    r0 = (id - bh * a.tiles) * ROWS;
    b = bh / a.Hk;
    hk = bh - b * a.Hk;
    L = (int)uniform_u32((uint32_t)keys_of(a, b));
    const int last = (r0 + ROWS < a.rows ? r0 + ROWS : a.rows) - 1;
    nk = last / a.G + L - a.n + 1;
    nk = nk < 0 ? 0 : nk < L ? nk : L;
    const int tiles = (nk + KEYS - 1) / KEYS;
    parts = parts_of(a, tiles);
    t0 = part < parts ? (int)((int64_t)tiles * part / parts) : 0;
    t1 = part < parts ? (int)((int64_t)tiles * (part + 1) / parts) : 0;
  }
  // the last key that row r sees (-1: none)
  __device__ __forceinline__ int last_of(const PagedArgs& a, int r) const {
    const int x = (r < a.rows ? r : a.rows - 1) / a.G + L - a.n;
    return x < -1 ? -1 : x < L - 1 ? x : L - 1;
  }
};
// ids[x] = page of table entry p0 + x, x < count, by the whole workgroup
__device__ __forceinline__ void put_pages(const PagedArgs& a, int b, int p0, int count, int* ids) {
  __syncthreads();  // (nobody reads the last ones any more)
  for (int x = (int)threadIdx.x; x < count; x += 256) ids[x] = a.table.page(b, p0 + x);
  __syncthreads();
}

// the four waves' sums of ROWS rows: top and l over all waves of the lane's row of tile rb
// (16 rows each), and the factor for this wave's own sums
struct WaveJoin {
  float top, l, f;
};
template <int ROWS>
__device__ __forceinline__ WaveJoin join_waves(float (*ml)[2][ROWS], int row, float m) {
  const float NINF = -__builtin_inff();
  WaveJoin j;
  j.top = ml[0][0][row];
#pragma unroll
  for (int x = 1; x < 4; ++x) j.top = fmaxf(j.top, ml[x][0][row]);
  j.l = 0.0f;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float f = ml[x][0][row] == NINF ? 0.0f : fast_exp2(ml[x][0][row] - j.top);
    j.l = __builtin_fmaf(ml[x][1][row], f, j.l);
  }
  j.f = m == NINF ? 0.0f : fast_exp2(m - j.top);
  return j;
}
__device__ __forceinline__ bool has_weight(float l) { return l > 0.0f || l != l; }

// ------------------------------------------------------------ 16 bits
template <int D>
struct Paged16Tiles {
  using RT = RowTile<D>;
  static constexpr int TILE = RT::BYTES / 2;     // 32 rows
  static constexpr int KB = TILE / 1024;         // copy instructions per tile
  static constexpr int STAGE = 2 * TILE;         // K, V
  static constexpr int LDS = 4 * 2 * STAGE;      // four waves, two stages
};
__device__ __forceinline__ void copy_b128(uint32_t voff, const void* base, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(m0) : "m0", "memory");
}
__device__ __forceinline__ void copy_b128_from(const void* src, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m0) : "m0", "memory");
}
// (a wave reads what it copied itself: the waits order its own accesses, and
// the memory clobbers keep the compiler's LDS reads on their side of them)
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// acc, m, l of the lane's row (channels 32 dt + 8 j + 4 g + x in acc[dt][4 j + x]) go on over
// keys u0 .. u1 - 1, adding only what the row sees (win_careful of window.h)
template <class E, int D>
__device__ __forceinline__ void paged_careful(const PagedArgs& a, const PagedItem<32, 32>& it, int last, int u0, int u1,
                                              const uint16_t* q, int g, f32x16* acc, float& m, float& l) {
  constexpr int NDT = D / 32;
  const float NINF = -__builtin_inff();
#pragma unroll 1
  for (int u = u0; u < u1; ++u) {
    const int page = a.table.page(it.b, u >> a.table.lg), at = u & ((1 << a.table.lg) - 1);
    if (page < 0) continue;
    const uint16_t* k = (const uint16_t*)(a.k.p + page * a.k.page + it.hk * a.k.head + at * a.k.row) + 4 * g;
    const uint16_t* v = (const uint16_t*)(a.v.p + page * a.v.page + it.hk * a.v.head + at * a.v.row) + 4 * g;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const uint2 x = *reinterpret_cast<const uint2*>(q + 4 * g + 8 * c), y = *reinterpret_cast<const uint2*>(k + 8 * c);
      s = __builtin_fmaf(E::lo(x.x), E::lo(y.x), s);
      s = __builtin_fmaf(E::hi(x.x), E::hi(y.x), s);
      s = __builtin_fmaf(E::lo(x.y), E::lo(y.y), s);
      s = __builtin_fmaf(E::hi(x.y), E::hi(y.y), s);
    }
    s = xor32_add(s) * a.scale_log2;
    const bool sees = u <= last;
    const float top = sees ? fmaxf(m, s) : m;
    const float alpha = m == top ? 1.0f : fast_exp2(m - top), p = fast_exp2(s - (top == NINF ? 0.0f : top));
    m = top;
    if (sees) l = __builtin_fmaf(l, alpha, p);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 y = *reinterpret_cast<const uint2*>(v + 32 * dt + 8 * j);
        const float w[4] = {E::lo(y.x), E::hi(y.x), E::lo(y.y), E::hi(y.y)};
#pragma unroll
        for (int x = 0; x < 4; ++x)
          acc[dt][4 * j + x] = sees ? __builtin_fmaf(p, w[x], acc[dt][4 * j + x] * alpha) : acc[dt][4 * j + x];
      }
  }
}

template <class E, int D>
__global__ __launch_bounds__(256, 1) void paged16_kernel(PagedArgs a) {
  using T = Paged16Tiles<D>;
  using RT = typename T::RT;
  using RS = RowSource<D>;
  constexpr int NS = D / 16, NDT = D / 32, KB = T::KB, COUNT = 2 * KB;
  static_assert(KB % 4 == 0, "four lane offsets serve all copies of a tile");
  __shared__ __align__(1024) uint8_t smem[T::LDS];
  __shared__ int ids[kIds + 1];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  PagedItem<32, 32> it;
  it.init(a, (int)blockIdx.x);
  if (it.part >= it.parts) return;
  const int lg = a.table.lg, mask = (1 << lg) - 1, nk = it.nk;
  const uint8_t* kb = (const uint8_t*)uniform_ptr(a.k.p + it.hk * a.k.head);
  const uint8_t* vb = (const uint8_t*)uniform_ptr(a.v.p + it.hk * a.v.head);
  const int64_t kstep = a.k.row, vstep = a.v.row;
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    koff[x] = (uint32_t)RS::row(x, lane) * (uint32_t)kstep + (uint32_t)RS::byte(x, lane);
    voff[x] = (uint32_t)RS::row(x, lane) * (uint32_t)vstep + (uint32_t)RS::byte(x, lane);
  }
  uint8_t* const mine = smem + w * 2 * T::STAGE;
  const uint32_t lds0 = lds_addr(mine);
  int p0 = 0;  // table entry of ids[0]
  // page of key u (past the list its last one's)
  auto page_of = [&](int u) { return ids[((u < nk ? u : nk - 1) >> lg) - p0]; };
  auto issue = [&](int t, int st) {
    const int u0 = 32 * t;
    const uint32_t lds = lds0 + (uint32_t)(st * T::STAGE);
    if (u0 + 31 < nk) {
      // (each half of the tile, 16 keys, stands in one page; a page that is none: page 0, and masked)
      const int i0 = (int)uniform_u32((uint32_t)page_of(u0)), i1 = (int)uniform_u32((uint32_t)page_of(u0 + 16));
      const int64_t x0 = i0 < 0 ? 0 : i0, x1 = i1 < 0 ? 0 : i1;
      const uint8_t* kh[2] = {kb + x0 * a.k.page + (u0 & mask) * kstep, kb + x1 * a.k.page + (((u0 + 16) & mask) - 16) * kstep};
      const uint8_t* vh[2] = {vb + x0 * a.v.page + (u0 & mask) * vstep, vb + x1 * a.v.page + (((u0 + 16) & mask) - 16) * vstep};
#pragma unroll
      for (int i = 0; i < KB; ++i)
        copy_b128(koff[i & 3], kh[2 * i / KB] + (i >> 2) * RS::ROWS4 * kstep, lds + (uint32_t)i * 1024u);
#pragma unroll
      for (int i = 0; i < KB; ++i)
        copy_b128(voff[i & 3], vh[2 * i / KB] + (i >> 2) * RS::ROWS4 * vstep, lds + (uint32_t)(KB + i) * 1024u);
      return;
    }
#pragma unroll 4
    for (int i = 0; i < KB; ++i) {
      const int u = u0 + RS::row(i, lane), key = u < nk ? u : nk - 1, at = RS::byte(i, lane), id = page_of(key);
      const int64_t x = id < 0 ? 0 : id;
      copy_b128_from(kb + x * a.k.page + (key & mask) * kstep + at, uniform_u32(lds + (uint32_t)i * 1024u));
      copy_b128_from(vb + x * a.v.page + (key & mask) * vstep + at, uniform_u32(lds + (uint32_t)(KB + i) * 1024u));
    }
  };

  // this lane's row (rows past the end re-read the last one and are not stored)
  const int r = it.r0 + l32, rc = r < a.rows ? r : a.rows - 1;
  const int i = rc / a.G, head = it.hk * a.G + (rc - i * a.G);
  const int64_t token = (int64_t)it.b * a.n + i;
  const uint16_t* qp = a.q + token * a.qt + head * a.qh;
  bf16x8 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = ld_bf16x8(qp + 16 * s + 8 * g);
#pragma unroll
  for (int s = 0; s < NS; ++s) consume_regs(qf[s]);
  const int last = it.last_of(a, r), first_last = (int)uniform_u32((uint32_t)it.last_of(a, it.r0));

  RowOperand kop;
  kop.init<RT>(0, l32, g);
  TrOperand vop;
  vop.init<RT>(0, lane);
  const float NINF = -__builtin_inff();
  f32x16 acc_o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = f32x16_zero();
  float m = NINF, l = 0.0f;

  const int chunk = (kIds << lg) >> 5;  // key tiles whose pages stand in LDS at a time
#pragma unroll 1
  for (int c0 = it.t0; c0 < it.t1; c0 += chunk) {
    const int c1 = c0 + chunk < it.t1 ? c0 + chunk : it.t1;
    p0 = (32 * c0) >> lg;
    const int end = 32 * c1 < nk ? 32 * c1 : nk;
    put_pages(a, it.b, p0, ((end - 1) >> lg) - p0 + 1, ids);
    if (c0 + w < c1) issue(c0 + w, 0);
    if (c0 + w + 4 < c1) issue(c0 + w + 4, 1);
    int st = 0;
    for (int t = c0 + w; t < c1; t += 4, st ^= 1) {
      const int u0 = 32 * t;
      const bool there0 = page_of(u0) >= 0, there1 = page_of(u0 + 16) >= 0;
      if (t + 4 < c1) copies_wait<COUNT>();  // (the next tile's copies may be in flight)
      else copies_wait<0>();
      const uint8_t* sK = mine + st * T::STAGE;
      const uint8_t* sV = sK + T::TILE;
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
      if (t + 8 < c1) issue(t + 8, st);
#pragma unroll
      for (int x = 0; x < 16; ++x) sacc[x] += s2[x];
      if (u0 + 31 > first_last || !there0 || !there1) {
        uint32_t bits = (uint32_t)(last - u0 >= 31 ? ~0u : last < u0 ? 0u : (2u << (last - u0)) - 1);
        bits &= (there0 ? 0xffffu : 0u) | (there1 ? 0xffff0000u : 0u);
        bits >>= 4 * g;
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
  }

  if (win_not_finite<NDT>(acc_o, l, r < a.rows)) {  // (window.h: the wave's rows again, key by key)
    m = NINF;
    l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc_o[dt] = f32x16_zero();
#pragma unroll 1
    for (int c0 = it.t0; c0 < it.t1; c0 += chunk)
#pragma unroll 1
      for (int t = c0 + w; t < it.t1 && t < c0 + chunk; t += 4)
        paged_careful<E, D>(a, it, last, 32 * t, 32 * t + 32 < nk ? 32 * t + 32 : nk, qp, g, acc_o, m, l);
  }

  // join the four waves: every wave's sums on the largest reference, then wave w
  // adds a quarter of the channels (registers 4 NDT w ...) in wave order
  __shared__ float ml[4][2][32];
  if (g == 0) {
    ml[w][0][l32] = m;
    ml[w][1][l32] = l;
  }
  __syncthreads();  // (also: no wave reads its stages any more)
  const WaveJoin j = join_waves<32>(ml, l32, m);
  float* red = reinterpret_cast<float*>(smem);
  constexpr int NR = NDT * 16, QR = NR / 4;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) red[(w * NR + dt * 16 + x) * 64 + lane] = acc_o[dt][x] * j.f;
  __syncthreads();
  float o[QR];
#pragma unroll
  for (int x = 0; x < QR; ++x) {
    o[x] = red[(w * QR + x) * 64 + lane];
#pragma unroll
    for (int y = 1; y < 4; ++y) o[x] += red[(y * NR + w * QR + x) * 64 + lane];
  }
  if (r >= a.rows) return;
  const int64_t at = ((int64_t)it.part * a.total + it.id) * 32 + l32;
#pragma unroll
  for (int x = 0; x < QR; x += 8) {
    const int reg = w * QR + x, d = 32 * (reg >> 4) + 8 * ((reg & 15) >> 2);
    const float4 u = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]), v = make_float4(o[x + 4], o[x + 5], o[x + 6], o[x + 7]);
    if (it.parts == 1) {
      const float inv = has_weight(j.l) ? 1.0f / j.l : 0.0f;
      win_store<E>(a.o + token * a.ot + head * a.oh + d, g, win_scaled(u, inv), win_scaled(v, inv));
    } else {
      float* to = a.part + at * D + d + 4 * g;
      *reinterpret_cast<float4*>(to) = u;
      *reinterpret_cast<float4*>(to + 8) = v;
    }
  }
  if (w == 0 && g == 0) {
    if (it.parts == 1) {
      if (a.lse)
        a.lse[(int64_t)head * a.B * a.n + token] = has_weight(j.l) ? (j.top + __log2f(j.l)) * 0.6931471805599453f : NINF;
    } else {
      a.part_ml[2 * at] = j.top;
      a.part_ml[2 * at + 1] = j.l;
    }
  }
}

// ------------------------------------------------------------ 4 bits
typedef int paged_v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) paged_v2i paged_lds_v2i;

// S (16 keys x 16 rows) of 32 channels: for float16 queries K's values as float16
// (SPLIT: P times V's scale as two bfloat16s, what the first leaves off in the second)
struct Paged4Bf16 {
  static constexpr bool SPLIT = false;
  static __device__ __forceinline__ f32x4 mfma(uint4 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint4 values(uint32_t w, float s) { return bf16_of_codes(w, s); }
  using Out = WinBf16;
};
struct Paged4F16 {
  static constexpr bool SPLIT = true;
  static __device__ __forceinline__ f32x4 mfma(uint4 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint4 values(uint32_t w, float s) { return f16_of_codes(w, s); }
  using Out = WinF16;
};
// a b, and 0 where either is 0 (v_mul_legacy_f32: 0 times an infinity or a NaN is 0); the
// compiler has no builtin for the instruction, so its intrinsic is declared by name
extern "C" __device__ __attribute__((const)) float prism_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
// max and sum over the four lanes l16, l16 + 16, .. that share a row
__device__ __forceinline__ float rows_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xor32_max(fmax_nn(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float rows_add(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xor32_add(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

template <class E, int D, int NR>
__global__ __launch_bounds__(256, 2) void paged4_kernel(PagedArgs a) {
  constexpr int ROWS = 16 * NR, NS = D / 32, NC = D / 16, HB = D / 2;  // k-steps, 16-channel blocks, bytes of a place's codes
  constexpr int NV = 64 * HB / 1024;                                   // 1 KB of V's codes an instruction
  constexpr int VS = D / 32;                                           // 16-byte words of 16 places' scales
  typedef typename std::conditional<D == 128, uint4, uint2>::type KWord;
  constexpr int VLDS = 64 * HB, RED = 4 * NR * NC * 4 * 64 * 4;
  __shared__ __align__(1024) uint8_t smem[4 * VLDS > RED ? 4 * VLDS : RED];
  __shared__ int ids[kIds + 1];
  __shared__ float ml[4][2][ROWS];
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int w = (int)uniform_u32(threadIdx.x >> 6);
  PagedItem<ROWS, 64> it;
  it.init(a, (int)blockIdx.x);
  if (it.part >= it.parts) return;
  const int lg = a.table.lg, mask = (1 << lg) - 1, nk = it.nk;
  const uint8_t* kb = a.k.p + it.hk * a.k.head;
  const uint8_t* vb = a.v.p + it.hk * a.v.head;
  const int scales = HB << lg;  // byte of a page's first scale
  uint8_t* const mine = smem + w * VLDS;

  // rows l16 of each row tile
  bf16x8 qf[NR][NS];
  int last[NR];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const int r = it.r0 + 16 * x + l16, rc = r < a.rows ? r : a.rows - 1;
    const int i = rc / a.G, head = it.hk * a.G + (rc - i * a.G);
    const uint16_t* qp = a.q + ((int64_t)it.b * a.n + i) * a.qt + head * a.qh;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[x][s] = ld_bf16x8(qp + (D / 4) * g + 8 * s);
    last[x] = it.last_of(a, r);
  }
  const int first_last = (int)uniform_u32((uint32_t)it.last_of(a, it.r0));

  // a tile's codes and scales
  struct Tile {
    KWord k[4];
    uint32_t ks[4];
    uint4 v[NV], vs[VS];
    int there;  // page of the lane's 16 keys
  };
  int p0 = 0;
  auto page_of = [&](int u) { return ids[((u < nk ? u : nk - 1) >> lg) - p0]; };
  auto load = [&](int t, Tile& c) {
    const int u0 = 64 * t;
    {
      const int u = u0 + 16 * (l16 >> 2), id = page_of(u);
      const uint8_t* p = kb + (int64_t)(id < 0 ? 0 : id) * a.k.page;
      const int at = (u & mask) + (l16 & 3);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        c.k[x] = *reinterpret_cast<const KWord*>(p + (at + 4 * x) * HB + (HB / 4) * g);
        c.ks[x] = p[scales + (at + 4 * x) * (D / 32) + (D == 128 ? g : g >> 1)];
      }
    }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const int row = x * (1024 / HB) + lane / (HB / 16), u = u0 + (row & ~15), id = page_of(u);
      const uint8_t* p = vb + (int64_t)(id < 0 ? 0 : id) * a.v.page;
      c.v[x] = *reinterpret_cast<const uint4*>(p + ((u & mask) + (row & 15)) * HB + 16 * (lane % (HB / 16)));
    }
    const int u = u0 + 16 * g, id = page_of(u);
    const uint8_t* p = vb + (int64_t)(id < 0 ? 0 : id) * a.v.page + scales + (u & mask) * (D / 32);
#pragma unroll
    for (int x = 0; x < VS; ++x) c.vs[x] = *reinterpret_cast<const uint4*>(p + 16 * x);
    c.there = id;
  };
  // V's codes in LDS: 16-byte pieces of a place swizzled so that the transposing read of 16
  // places takes all banks
  auto piece = [](int row, int c) { return row * HB + 16 * (c ^ (D == 128 ? (row >> 2) & 3 : (row >> 3) & 1)); };

  const float NINF = -__builtin_inff();
  f32x4 acc[NR][NC];
  float m[NR], l[NR];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    m[x] = NINF;
    l[x] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[x][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int chunk = (kIds << lg) >> 6;  // key tiles whose pages stand in LDS at a time
#pragma unroll 1
  for (int c0 = it.t0; c0 < it.t1; c0 += chunk) {
    const int c1 = c0 + chunk < it.t1 ? c0 + chunk : it.t1;
    p0 = (64 * c0) >> lg;
    const int end = 64 * c1 < nk ? 64 * c1 : nk;
    put_pages(a, it.b, p0, ((end - 1) >> lg) - p0 + 1, ids);
    Tile next;
    if (c0 + w < c1) load(c0 + w, next);
#pragma unroll 1
    for (int t = c0 + w; t < c1; t += 4) {
      const Tile c = next;
      const int u0 = 64 * t;
#pragma unroll
      for (int x = 0; x < NV; ++x)
        *reinterpret_cast<uint4*>(mine + piece(x * (1024 / HB) + lane / (HB / 16), lane % (HB / 16))) = c.v[x];
      if (t + 4 < c1) load(t + 4, next);
      f32x4 s[NR][4];
#pragma unroll
      for (int x = 0; x < NR; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[x][y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        uint32_t kw[4];
        if constexpr (D == 128) { kw[0] = c.k[y].x; kw[1] = c.k[y].y; kw[2] = c.k[y].z; kw[3] = c.k[y].w; }
        else { kw[0] = c.k[y].x; kw[1] = c.k[y].y; }
        const float ksc = scale_of(c.ks[y]);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const uint4 kv = E::values(kw[st], ksc);
#pragma unroll
          for (int x = 0; x < NR; ++x) s[x][y] = E::mfma(kv, qf[x][st], s[x][y]);
        }
      }
      if (u0 + 63 > first_last || __builtin_amdgcn_ballot_w64(c.there < 0)) {
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          const int end16 = last[x] - (u0 + 16 * g);
          const uint32_t bits = c.there < 0 || end16 < 0 ? 0u : end16 >= 15 ? 0xffffu : (2u << end16) - 1;
#pragma unroll
          for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int z = 0; z < 4; ++z) s[x][y][z] = keep_or_ninf(s[x][y][z], bits, 4 * y + z);
        }
      }
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        float mx = s[x][0][0];
#pragma unroll
        for (int y = 1; y < 16; ++y) mx = fmax_nn(mx, s[x][y >> 2][y & 3]);
        mx = rows_max(mx) * a.scale_log2;
        const bool move = mx > m[x] + WinBf16::MARGIN || (m[x] == NINF && mx != NINF);
        const float m_new = move ? mx : m[x];
        const float alpha = move ? fast_exp2(m[x] - m_new) : 1.0f;
        const float mb = m_new == NINF ? 0.0f : m_new;
        if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
          for (int cb = 0; cb < NC; ++cb)
#pragma unroll
            for (int z = 0; z < 4; ++z) acc[x][cb][z] *= alpha;
        }
        float ls = 0.0f;
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          const float p = fast_exp2(__builtin_fmaf(s[x][y >> 2][y & 3], a.scale_log2, -mb));
          s[x][y >> 2][y & 3] = p;
          ls += p;
        }
        l[x] = __builtin_fmaf(l[x], alpha, ls);  // (this lane's keys alone: added up at the end)
        m[x] = m_new;
      }
      // O^T += V^T P^T, 32 channels (one scale) at a time.  (A key that a row does not see has
      // P = 0, and 0 times any scale, 255's too, is 0 here.  A key that it sees and whose scale is
      // 255 makes its sums infinite or NaN: see behind the loop.)
#pragma unroll
      for (int blk = 0; blk < NS; ++blk) {
        bf16x8 pb[NR][2], pl[NR][2];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          float f[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const int byte = (8 * st + y) * (D / 32) + blk;  // of the 16 places' scales
            const uint4 word = c.vs[byte >> 4];
            const uint32_t d = (byte >> 2 & 3) == 0 ? word.x : (byte >> 2 & 3) == 1 ? word.y : (byte >> 2 & 3) == 2 ? word.z : word.w;
            f[y] = scale_of((d >> (8 * (byte & 3))) & 0xffu);
          }
#pragma unroll
          for (int x = 0; x < NR; ++x) {
            float p[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) p[y] = prism_mul_legacy(s[x][2 * st + (y >> 2)][y & 3], f[y]);
            const uint4 hi = make_uint4(pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7]));
            pb[x][st] = as_bf16x8(hi);
            if constexpr (E::SPLIT) {
              const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
              uint32_t lo[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) lo[y] = pack_bf16(p[2 * y] - WinBf16::lo(h[y]), p[2 * y + 1] - WinBf16::hi(h[y]));
              pl[x][st] = as_bf16x8(make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int cb = 2 * blk + half;
          const paged_v2i vt = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
              (paged_lds_v2i*)(mine + piece(16 * g + l16, cb >> 1) + 8 * (cb & 1)));
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const bf16x8 vv = as_bf16x8(bf16_of_codes((uint32_t)vt[st], 1.0f));
#pragma unroll
            for (int x = 0; x < NR; ++x) {
              acc[x][cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, pb[x][st], acc[x][cb], 0, 0, 0);
              if constexpr (E::SPLIT) acc[x][cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, pl[x][st], acc[x][cb], 0, 0, 0);
            }
          }
        }
      }
    }
  }

  // V's scale 255 stands for NaN, but enters P as an infinity (exponent bits alone), and so do the
  // sums where a code beside it is not 0.  Telling it in the loop would take two instructions for each
  // of a tile's 16 D / 32 scales of a lane; where a sum is infinite the wave looks at its keys' scales
  // again instead (the sums of values of 2^100 and more, which may be infinite too, stay as they are):
  // 8 sequences of 131,072 keys 206 us, with a NaN in one 239; 64 of them 1,772 and 1,900.
  bool endless = false;
#pragma unroll
  for (int x = 0; x < NR; ++x)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int z = 0; z < 4; ++z) endless = endless || __builtin_fabsf(acc[x][c][z]) == __builtin_inff();
  if (__builtin_amdgcn_ballot_w64(endless)) {
#pragma unroll 1
    for (int c0 = it.t0; c0 < it.t1; c0 += chunk)
#pragma unroll 1
      for (int t = c0 + w; t < it.t1 && t < c0 + chunk; t += 4) {
        // a key for each lane; of a block's first NaN on, whoever sees further has it
        const int u = 64 * t + lane, page = u < nk ? a.table.page(it.b, u >> lg) : -1;
        const uint8_t* const of_u = vb + (int64_t)(page < 0 ? 0 : page) * a.v.page + scales + (u & mask) * (D / 32);
#pragma unroll
        for (int blk = 0; blk < NS; ++blk) {
          const uint64_t hit = __builtin_amdgcn_ballot_w64(page >= 0 && of_u[blk] == 255);
          const int first = hit ? 64 * t + (int)__builtin_ctzll(hit) : nk;
#pragma unroll
          for (int x = 0; x < NR; ++x)
#pragma unroll
            for (int z = 0; z < 8; ++z)
              if (first <= last[x]) acc[x][2 * blk + (z >> 2)][z & 3] = __builtin_nanf("");
        }
      }
  }

  // join the four waves, as in paged16_kernel: wave w adds a quarter of the blocks
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    l[x] = rows_add(l[x]);
    if (g == 0) {
      ml[w][0][16 * x + l16] = m[x];
      ml[w][1][16 * x + l16] = l[x];
    }
  }
  __syncthreads();
  float4* red = reinterpret_cast<float4*>(smem);
  WaveJoin j[NR];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    j[x] = join_waves<ROWS>(ml, 16 * x + l16, m[x]);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      red[((w * NR + x) * NC + c) * 64 + lane] =
          make_float4(acc[x][c][0] * j[x].f, acc[x][c][1] * j[x].f, acc[x][c][2] * j[x].f, acc[x][c][3] * j[x].f);
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const int r = it.r0 + 16 * x + l16;
    if (r >= a.rows) continue;
    const int i = r / a.G, head = it.hk * a.G + (r - i * a.G);
    const int64_t token = (int64_t)it.b * a.n + i, at = ((int64_t)it.part * a.total + it.id) * ROWS + 16 * x + l16;
#pragma unroll
    for (int y = 0; y < NC / 4; ++y) {
      const int c = w * (NC / 4) + y, d = 16 * c + 4 * g;
      float4 o = red[(x * NC + c) * 64 + lane];
#pragma unroll
      for (int z = 1; z < 4; ++z) {
        const float4 v = red[((z * NR + x) * NC + c) * 64 + lane];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      }
      if (it.parts == 1) {
        const float inv = has_weight(j[x].l) ? 1.0f / j[x].l : 0.0f;
        *reinterpret_cast<uint2*>(a.o + token * a.ot + head * a.oh + d) = win_pack4<typename E::Out>(win_scaled(o, inv));
      } else {
        *reinterpret_cast<float4*>(a.part + at * D + d) = o;
      }
    }
    if (w == 0 && g == 0) {
      if (it.parts == 1) {
        if (a.lse)
          a.lse[(int64_t)head * a.B * a.n + token] = has_weight(j[x].l) ? (j[x].top + __log2f(j[x].l)) * 0.6931471805599453f : NINF;
      } else {
        a.part_ml[2 * at] = j[x].top;
        a.part_ml[2 * at + 1] = j[x].l;
      }
    }
  }
}

// the parts' sums of a row, in order: one wave per row (ROWS, KEYS: those of the kernel before)
template <class E, int D, int ROWS, int KEYS>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  const int lane = threadIdx.x & 63, x = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), row = x % ROWS;
  const int id = x / ROWS;
  if (id >= a.total) return;
  PagedItem<ROWS, KEYS> it;
  it.init(a, id * a.splits);
  const int r = it.r0 + row;
  if (r >= a.rows || it.parts == 1) return;
  const int i = r / a.G, head = it.hk * a.G + (r - i * a.G);
  const int64_t token = (int64_t)it.b * a.n + i, first = (int64_t)id * ROWS + row, step = (int64_t)a.total * ROWS;
  const float NINF = -__builtin_inff();
  float m = NINF;
  for (int s = lane; s < it.parts; s += 64) m = fmaxf(m, a.part_ml[2 * (first + s * step)]);
  const float top = wave_max_xor(m);
  constexpr int C = D / 64;  // channels per lane
  typedef typename std::conditional<C == 2, float2, float>::type V;
  float o[2] = {0.0f, 0.0f}, l = 0.0f;
#pragma unroll 8
  for (int s = 0; s < it.parts; ++s) {
    const float2 v = *reinterpret_cast<const float2*>(a.part_ml + 2 * (first + s * step));
    const V p = *reinterpret_cast<const V*>(a.part + (first + s * step) * D + C * lane);
    const float f = v.x == NINF ? 0.0f : fast_exp2(v.x - top);  // (a part that sees nothing has sums of 0)
    l = __builtin_fmaf(v.y, f, l);
    if constexpr (C == 2) {
      o[0] = __builtin_fmaf(p.x, f, o[0]);
      o[1] = __builtin_fmaf(p.y, f, o[1]);
    } else {
      o[0] = __builtin_fmaf(p, f, o[0]);
    }
  }
  const float inv = has_weight(l) ? 1.0f / l : 0.0f;
  uint16_t* to = a.o + token * a.ot + head * a.oh + C * lane;
  const uint32_t u = E::pack(o[0] * inv, o[1] * inv);
  if constexpr (C > 1) *reinterpret_cast<uint32_t*>(to) = u;
  else *to = (uint16_t)u;
  if (a.lse && lane == 0)
    a.lse[(int64_t)head * a.B * a.n + token] = has_weight(l) ? (top + __log2f(l)) * 0.6931471805599453f : NINF;
}

// How a call is cut: rows of a tile, keys of a tile, and over how many workgroups at most.
//
// One round of the chip at most (one workgroup a CU over 16 bits, two over 4: what fits at D =
// 128; at 64 twice as many would), about sqrt(keys) / 2.5 parts (4 bits, tiles twice as long: / 5) of
// the longest sequence that the table could hold, one up to 512 keys, and no part of a sequence
// below two tiles.  Measured (us, 32 heads over 8, D = 128, pages of 16 or 64; lengths from half
// to all of the stated): 16 bits, 256 / 512 / 1,024 workgroups: 1 x 32,768 26 / 33 / 34; 16 x
// 8,192 84 / 85 / 91; 64 x 2,048 82 / 82 / 97; 8 x 131,072 561 / 543 / 537.  4 bits: 18 / 21 /
// 21; 39 / 35 / 38; 33 / 33 / 42; 209 / 183 / 179; 2 x 131,072 46 / 45 / 52.  Parts of 2 / 8 / 16
// tiles at least: 1 x 1,000 12.1 / 14.0 / 16.2 (4 bits 10.7 / 12.1 / 12.8), 1 x 4,096 14.8 / 14.7
// / 17.9 (12.1 / 14.0 / 17.3).  The parts are rounded down, so that counts between are not cut and
// wait for their longest sequence (TB/s): 16 bits, 16 / 17 / 20 / 24 / 31 / 32 / 33 / 48 sequences of up to 8,192
// 4.8 / 4.5 / 4.8 / 5.1 / 5.4 / 5.2 / 4.7 / 5.3, D = 64, 16 / 24 / 32 / 48 4.5 / 4.7 / 5.1 / 4.8; 4 bits, 32
// / 33 / 48 / 64 / 70 of up to 16,384 4.1 / 3.2 / 4.0 / 4.8 / 4.2, D = 64, 32 / 48 / 64 3.9 / 3.3 / 3.9, and 64 / 70
// of 8,192 with 4 key heads 4.4 / 2.9.  Tables sixteen times as wide as the lengths: 4 x 4,096 19.5 us and 19.7
// (4 bits 16.0 and 13.4).
struct PagedCut {
  int rows, keys, least;
  int64_t tiles, total, splits;
};
PagedCut paged_cut(int B, int64_t n, int Hk, int64_t G, int64_t places, int bits) {
  PagedCut c{};
  const int64_t rows = n * G;
  c.rows = bits == 16 || rows > 16 ? 32 : 16;
  c.keys = bits == 16 ? 32 : 64;
  c.least = 2;
  c.tiles = (rows + c.rows - 1) / c.rows;
  c.total = (int64_t)B * Hk * c.tiles;
  const int64_t slots = bits == 16 ? 256 : 512;
  const int64_t by_chip = c.total ? slots / c.total : 1;
  int64_t s = places <= 512 ? 1 : (int64_t)(__builtin_sqrt((double)places) / (bits == 16 ? 2.5 : 5.0));
  s = s < by_chip ? s : by_chip;
  c.splits = s < 1 ? 1 : s < kMaxSplits ? s : kMaxSplits;
  return c;
}

}  // namespace

extern "C" {

int prism_paged_plan(int B, int64_t n, int Hq, int Hk, int D, int bits, int64_t places, int64_t* floats) {
  PRISM_REQUIRE(B >= 0 && n >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && D >= 1 && (bits == 16 || bits == 4) && places >= 0 && floats,
                "prism_paged_plan: bad argument");
  const PagedCut c = paged_cut(B, n, Hk, Hq / Hk, places, bits);
  *floats = c.splits > 1 ? c.splits * c.total * c.rows * (D + 2) : 0;
  return PRISM_OK;
}

int prism_paged_fwd(const void* q, int dtype, int B, int64_t n, int Hq, int Hk, int D, const int64_t* strides,
                    const void* k_cache, const void* v_cache, int bits, int64_t pages, int page_size,
                    const int64_t* cache_strides, const int32_t* table, int64_t table_stride, int64_t width,
                    const int32_t* lens, float sm_scale, void* o, float* lse, float* part, hipStream_t stream) {
  if (const int rc = paged_check("prism_paged_fwd", dtype, bits, Hk, D, pages, page_size, cache_strides, k_cache, v_cache, width, B))
    return rc;
  PRISM_REQUIRE(Hq >= Hk && Hq % Hk == 0 && Hq < (1 << 16), "prism_paged_fwd: %d query heads do not share %d key heads evenly", Hq, Hk);
  PRISM_REQUIRE(n >= 0 && n * (Hq / Hk) < (1ll << 30) && B * n < (1ll << 30), "prism_paged_fwd: too many query rows");
  PRISM_REQUIRE(sm_scale > 0.0f && sm_scale < __builtin_inff(), "prism_paged_fwd: sm_scale must be positive and finite");
  if (B == 0 || n == 0) return PRISM_OK;
  PRISM_REQUIRE(q && o && strides && table && lens, "prism_paged_fwd: null pointer");
  PRISM_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)o & 15) == 0 && ((uintptr_t)part & 15) == 0,
                "prism_paged_fwd: pointers must be 16-byte aligned");
  for (int i = 0; i < 4; ++i) PRISM_REQUIRE(strides[i] % 8 == 0, "prism_paged_fwd: strides must be multiples of 8 elements");
  PagedArgs a{};
  a.q = (const uint16_t*)q; a.o = (uint16_t*)o;
  a.qt = strides[0]; a.qh = strides[1]; a.ot = strides[2]; a.oh = strides[3];
  paged_sides(&a.k, &a.v, bits, cache_strides, k_cache, v_cache);
  a.table = paged_table(table, table_stride, width, pages, page_size);
  a.lens = lens;
  a.B = B; a.Hk = Hk; a.G = Hq / Hk; a.n = (int)n; a.rows = (int)(n * a.G);
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.lse = lse;
  const PagedCut c = paged_cut(B, n, Hk, a.G, width * page_size, bits);
  PRISM_REQUIRE(c.total * c.splits < PRISM_MAX_THREADS / 256 && c.total * c.rows / 4 < PRISM_MAX_THREADS / 256,
                "prism_paged_fwd: too many row tiles");
  PRISM_REQUIRE(c.splits == 1 || part, "prism_paged_fwd: null workspace");
  a.tiles = (int)c.tiles; a.total = (int)c.total; a.splits = (int)c.splits; a.least = c.least;
  a.part = part;
  a.part_ml = part + c.splits * c.total * c.rows * D;
  const unsigned grid = (unsigned)(c.total * c.splits), join = (unsigned)(c.total * c.rows / 4);
  auto run = [&](auto kernel, auto joiner) {
    kernel<<<grid, 256, 0, stream>>>(a);
    if (c.splits > 1) joiner<<<join, 256, 0, stream>>>(a);
  };
  auto with = [&](auto e, auto four, auto d) {
    using E = decltype(e);
    using F = decltype(four);
    constexpr int DD = decltype(d)::value;
    if (bits == 16) run(paged16_kernel<E, DD>, paged_join_kernel<E, DD, 32, 32>);
    else if (c.rows == 16) run(paged4_kernel<F, DD, 1>, paged_join_kernel<E, DD, 16, 64>);
    else run(paged4_kernel<F, DD, 2>, paged_join_kernel<E, DD, 32, 64>);
  };
  if (dtype == PRISM_BF16) {
    if (D == 64) with(WinBf16{}, Paged4Bf16{}, std::integral_constant<int, 64>{});
    else with(WinBf16{}, Paged4Bf16{}, std::integral_constant<int, 128>{});
  } else {
    if (D == 64) with(WinF16{}, Paged4F16{}, std::integral_constant<int, 64>{});
    else with(WinF16{}, Paged4F16{}, std::integral_constant<int, 128>{});
  }
  PRISM_LAUNCH_CHECK("prism_paged_fwd");
  return PRISM_OK;
}

}  // extern "C"
