// What the window attention kernels share (gfx950): which keys a run of query
// rows sees, the copies of their K and V rows into LDS, element types.
//
// Rows.  The G query heads that share a key head are one set of rows: row r of
// a (sequence, key head) is token r / G of query head hk G + r % G, so a tile of
// rows covers few tokens and each staged K / V tile serves all heads of the
// group.
//
// Keys.  Token i of a sequence with L keys and n queries stands at p = i + L -
// n.  A run of tokens sees the sinks [0, nsink) and the keys [ws, hi] of its
// windows: a virtual list u = 0 .. n - 1 with key(u) = u for u < nsink, u + shift
// beyond.  Tiles of 64 (or 32) entries of that list are staged, so a few sinks
// cost no tile of their own, and rows of memory that no query of the run sees
// are never read (an entry past the end re-reads the last one): what stands in
// unused cache rows, NaN included, cannot reach a result.  Entry u is visible to
// the token at p where a <= u <= b or u < c (TokenSpan).
#pragma once
#include <initializer_list>

#include "common.h"
#include "mfma.h"
#include "tile_dma.h"

// ------------------------------------------------------------ element types
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Softmax reference.  P = 2^(score - m) is rounded to the type for its product with
// V.  m is SHIFT below the largest score when it was last moved, and moves when a
// score is more than MARGIN above that one, so P <= 2^(SHIFT + MARGIN); o = acc / l and
// lse = m + log2 l do not depend on it.  bfloat16 has float's range: any reference
// will do, and one that moves rarely costs least.  float16 loses bits below 2^-14 and
// everything below 2^-25, while l sums P unrounded: a long tail far below one large
// score would not weigh what it does (one list of 65,000 keys 17.0 nats below a sink:
// o 0.0039 for 0.0027 with m at the largest score).  P up to 2^15 keeps all of a key's bits down to 2^-26
// of the largest weight (18 nats) and some down to 2^-37; a margin of 3 moves the
// reference no more than a few times in a list.
//
// Gradients.  The backward takes P, and with it dS = P (dP - delta), times 2^GRAD, and
// the products' fp32 sums back by BACK: a float16 dS of 4,096 seen keys and do of 1e-3
// is subnormal (dq and dk 5e-3 off norm-wise, 5e-2 at 1e-4).  With 2^6 what is lost
// there stays below half of what dq's and dk's own rounding to float16 loses (2e-4 and
// 8e-4; at 32,768 keys 7e-4 and 7e-3, beside 2e-3 and 2e-2), and dS may be up to 1,023
// before it becomes infinite; 2^8 would bring little and leave 255.
struct WinBf16 {
  static constexpr float SHIFT = 0.0f, MARGIN = 8.0f, GRAD = 0.0f, BACK = 1.0f;
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
// (operands travel as bf16x8: eight 16-bit values whatever their type)
struct WinF16 {
  static constexpr float SHIFT = 12.0f, MARGIN = 3.0f, GRAD = 6.0f, BACK = 0x1p-6f;
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
  static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
};

// B operand of k-step tt from an accumulator of 32-row blocks (b_from_acc for either type)
template <class E>
__device__ __forceinline__ bf16x8 win_b_from_acc(const f32x16* acc, int tt) {
  const int h = tt >> 1, j0 = 2 * (tt & 1);
  uint4 pb;
  pb.x = E::pack(acc[h][4 * j0 + 0], acc[h][4 * j0 + 1]);
  pb.y = E::pack(acc[h][4 * j0 + 2], acc[h][4 * j0 + 3]);
  pb.z = E::pack(acc[h][4 * j0 + 4], acc[h][4 * j0 + 5]);
  pb.w = E::pack(acc[h][4 * j0 + 6], acc[h][4 * j0 + 7]);
  return as_bf16x8(pb);
}

// ------------------------------------------------------------ arguments
struct WinTensor {  // [B, H, S, D], channels adjacent; strides in elements
  uint16_t* p;
  int64_t b, h, s;
};
struct WinArgs {
  WinTensor q, k, v, o;
  const int32_t *q_lens, *kv_lens;  // [B] or null
  int B, Hk, G, Sq, Sk;
  int window, sinks, causal;
  float scale, scale_log2;
  uint16_t* rest;                   // what o's rounding left off, at o's strides (win_store_o); or null
  float* lse;                       // [B, Hk G, Sq] natural log, -inf for rows that see nothing; or null
  int tiles;                        // row tiles of a (sequence, key head)
  int total;                        // row tiles of the launch
  // Work items: the first `whole` row tiles one each, every later one `splits`,
  // item i of which takes the i-th part of its key list (single tokens: whole =
  // 0) and leaves its sums in part (and m and l in part_ml)
  int whole, splits, items;
  float *part, *part_ml;
  int ranked;                       // tiles by rank (rank_tile)
};

// ------------------------------------------------------------ spans
struct SeqSpan {
  int L, n, off;  // keys, queries, position of token 0
};
__device__ __forceinline__ SeqSpan seq_span(const WinArgs& a, int b) {
  SeqSpan s;
  s.L = a.Sk;
  s.n = a.Sq;
  if (a.kv_lens) {  // (lengths outside the tensors are cut to them)
    const int x = a.kv_lens[b];
    s.L = x < 0 ? 0 : x < a.Sk ? x : a.Sk;
  }
  if (a.q_lens) {
    const int x = a.q_lens[b];
    s.n = x < 0 ? 0 : x < a.Sq ? x : a.Sq;
  }
  s.off = s.L - s.n;
  return s;
}

// the virtual key list of tokens i0 .. i1 (i0 > i1: none)
struct KeyList {
  int nsink, shift, n;
  __device__ __forceinline__ int key(int u) const { return u < nsink ? u : u + shift; }
};
__device__ __forceinline__ KeyList key_list(const WinArgs& a, const SeqSpan& s, int i0, int i1) {
  KeyList k;
  const int pmin = i0 + s.off, pmax = i1 + s.off;
  const int top = a.causal ? pmax : pmax + a.window - 1;
  const int hi = top < s.L - 1 ? top : s.L - 1;
  int ns = a.causal ? (a.sinks < pmax + 1 ? a.sinks : pmax + 1) : a.sinks;
  ns = ns < s.L ? ns : s.L;
  ns = ns > 0 ? ns : 0;
  const int lo = pmin - a.window + 1;
  const int ws = lo > ns ? lo : ns;
  k.nsink = ns;
  k.shift = ws - ns;
  k.n = ns + (hi >= ws ? hi - ws + 1 : 0);
  if (i0 > i1) k.n = k.nsink = 0;
  return k;
}

// entries of the list that the token at p sees: a <= u <= b or u < c
struct TokenSpan {
  int a, b, c;
};
__device__ __forceinline__ TokenSpan token_span(const WinArgs& a, const KeyList& k, int p) {
  TokenSpan t;
  const int lo = p - a.window + 1 - k.shift, hi = (a.causal ? p : p + a.window - 1) - k.shift;
  t.a = lo > k.nsink ? lo : k.nsink;
  t.b = hi < k.n - 1 ? hi : k.n - 1;
  t.c = a.causal && p + 1 < k.nsink ? p + 1 : k.nsink;
  return t;
}
// bit j of the result: entry u0 + j is visible, j < 64
__device__ __forceinline__ uint64_t span_bits(const TokenSpan& t, int u0) {
  const int lo = t.a - u0 > 0 ? t.a - u0 : 0, hi = t.b - u0 < 63 ? t.b - u0 : 63;
  uint64_t m = hi >= lo ? (~0ull << lo) & (~0ull >> (63 - hi)) : 0ull;
  const int c = t.c - u0;
  m |= c >= 64 ? ~0ull : c > 0 ? (1ull << c) - 1 : 0ull;
  return m;
}

// Which entries the tokens p0 .. p1 of a wave see: some of [u0, u1], all of it.
// (token_span's bounds grow with p, so the ends of the run give them.)
struct WaveSpan {
  int a_any, b_any, c_any, a_all, b_all, c_all;
  __device__ __forceinline__ void init(const WinArgs& w, const KeyList& k, int p0, int p1) {
    const TokenSpan f = token_span(w, k, p0), l = token_span(w, k, p1);
    a_any = f.a; b_any = l.b; c_any = l.c;
    a_all = l.a; b_all = f.b; c_all = f.c;
  }
  __device__ __forceinline__ bool any(int u0, int u1) const { return (u1 >= a_any && u0 <= b_any) || u0 < c_any; }
  __device__ __forceinline__ bool all(int u0, int u1) const { return (u0 >= a_all && u1 <= b_all) || u1 < c_all; }
};

// ------------------------------------------------------------ copies
// 16 bytes per lane from a 64-bit address of its own: LDS[m0 + 16 lane] <- *src
__device__ __forceinline__ void dma_b128_from(const void* src, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m0) : "m0");
}

// Row and byte of the row that lane `lane` of KB-instruction i of a row tile
// fetches (RowTile::src_offset for rows that are not adjacent in memory).
// Instruction i + 4m is 4096 m / W rows further on, at the same byte.
template <int D>
struct RowSource {
  using RT = RowTile<D>;
  static constexpr int ROWS4 = 4096 / RT::W;
  static __device__ __forceinline__ int row(int i, int lane) {
    const int pos = 1024 * i + 16 * lane;
    return 4 * (pos / RT::Q) + (((pos % RT::Q) >> 6) & 3);
  }
  static __device__ __forceinline__ int byte(int i, int lane) {
    const int pos = 1024 * i + 16 * lane, rq = pos / RT::Q, rem = pos - rq * RT::Q;
    return 16 * (4 * (rem >> 8) + (((rem >> 4) & 3) ^ (rq & 3)));
  }
};

template <int D>
struct WinTiles {
  using RT = RowTile<D>;
  static constexpr int STAGE = 2 * RT::BYTES, STAGE_KB = 2 * RT::KB;
};

// The tile copies of a 64-entry stage (K then V) by two waves (wid 0, 1).  At D =
// 64 the lane offsets are formed anew for every tile, since registers decide how
// many workgroups share a CU there; at D = 128 they are kept (dQ 423 -> 411 us,
// forward 348 -> 336 us of a 480p step).
template <int D>
struct StageCopy {
  using RT = RowTile<D>;
  using RS = RowSource<D>;
  static constexpr int COUNT = RT::KB;  // instructions per wave and stage
  const uint8_t *kb, *vb;               // K and V of the (sequence, key head)
  int64_t kstep, vstep;                 // bytes per row
  int wid;
  uint32_t koff[2], voff[2];            // lane offsets of instructions wid, wid + 2 (D = 128)
  __device__ __forceinline__ void offsets(int lane, uint32_t* ko, uint32_t* vo) const {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = RS::row(wid + 2 * x, lane), c = RS::byte(wid + 2 * x, lane);
      ko[x] = (uint32_t)r * (uint32_t)kstep + (uint32_t)c;
      vo[x] = (uint32_t)r * (uint32_t)vstep + (uint32_t)c;
    }
  }
  __device__ __forceinline__ void init(const WinArgs& a, int b, int hk, int wid_, int lane) {
    wid = wid_;
    kb = (const uint8_t*)uniform_ptr(a.k.p + b * a.k.b + hk * a.k.h);
    vb = (const uint8_t*)uniform_ptr(a.v.p + b * a.v.b + hk * a.v.h);
    kstep = 2 * a.k.s;
    vstep = 2 * a.v.s;
    if constexpr (D == 128) offsets(lane, koff, voff);
  }
  __device__ __forceinline__ void issue(const KeyList& k, int u0, uint32_t lds) const {
    const int lane = opaque_thread_id() & 63;
    if ((u0 >= k.nsink || u0 + 63 < k.nsink) && u0 + 63 < k.n) {  // 64 adjacent keys
      const int key0 = k.key(u0);
      const uint8_t* kt = (const uint8_t*)uniform_ptr(kb + key0 * kstep);
      const uint8_t* vt = (const uint8_t*)uniform_ptr(vb + key0 * vstep);
      uint32_t ko[2], vo[2];
      if constexpr (D == 128) {
        ko[0] = koff[0]; ko[1] = koff[1]; vo[0] = voff[0]; vo[1] = voff[1];
      } else {
        offsets(lane, ko, vo);
      }
#pragma unroll
      for (int s = 0; s < COUNT; ++s) {
        const int i = wid + 2 * s;
        const bool isk = 2 * s < RT::KB;
        const int m = ((2 * s) % RT::KB) >> 2;  // (instruction wid + 2 (s & 1) + 4 m of its tile)
        const uint8_t* base = isk ? kt + m * RS::ROWS4 * kstep : vt + m * RS::ROWS4 * vstep;
        dma_b128(isk ? ko[s & 1] : vo[s & 1], base, lds + (uint32_t)i * 1024u);
      }
      return;
    }
#pragma unroll 1
    for (int s = 0; s < COUNT; ++s) {
      const int i = wid + 2 * s, t = i < RT::KB ? i : i - RT::KB;
      const int u = u0 + RS::row(t, lane), key = k.key(u < k.n ? u : k.n - 1);
      const uint8_t* src = (i < RT::KB ? kb + key * kstep : vb + key * vstep) + RS::byte(t, lane);
      dma_b128_from(src, uniform_u32(lds + (uint32_t)i * 1024u));
    }
  }
};

// Sequences of different lengths (right-padded batches): the tiles of a launch
// by rank, the first of every sequence and key head, then the second of each,
// and so on, and behind them the tiles past the sequences' ends.  In a launch of
// one or two rounds every CU gets a like share of the heavy tiles so, and the empty
// ones end the launch; in the order by sequences some CUs hold four full tiles and
// others four empty ones.  Measured (us, by sequences / by rank): 2,598 and 2,306
// tokens of 4,096, 16 heads over 4, D = 64, window 1,024: forward 46 / 35, dQ 50 /
// 42, dK/dV 88 / 76; three sequences of 1,500 to 2,700, 12 heads over 4, D = 128,
// window 2,000: forward 86 / 61, dQ 107 / 77.  (With as many heads as an XCD group has
// items, tiles that share tokens stand in different XCDs: dK/dV of the first case
// reads 309 MB for 42 MB of inputs.)
struct RankedTile {
  int b, hk, rank;
  bool live;  // else the rank-th of the tiles past the end
};
// c: the tiles of sequence `lane` (B <= 64, tiles <= 4,096); all lanes active
__device__ __forceinline__ RankedTile rank_tile(int c, int B, int Hk, int tiles, int index) {
  const int lane = (int)threadIdx.x & 63;
  auto before = [&](int r) {  // tiles of ranks below r
    int n = 0;
    for (int b = 0; b < B; ++b) {
      const int x = __builtin_amdgcn_readlane(c, b);
      n += x < r ? x : r;
    }
    return n * Hk;
  };
  RankedTile t;
  const int live = (int)uniform_u32((uint32_t)before(tiles));
  t.live = index < live;
  if (!t.live) {
    c = tiles - c;
    index -= live;
  }
  // the last rank with no more than `index` tiles before it: by 64, then by one
  int r = 64 * (__popcll(__builtin_amdgcn_ballot_w64(before(64 * lane) <= index)) - 1);
  r += __popcll(__builtin_amdgcn_ballot_w64(before(r + lane) <= index)) - 1;
  t.rank = r;
  const int j = (int)uniform_u32((uint32_t)(index - before(r)));
  uint64_t who = __builtin_amdgcn_ballot_w64(lane < B && c > r);
  for (int x = j / Hk; x > 0; --x) who &= who - 1;
  t.b = who ? (int)__builtin_ctzll(who) : 0;
  t.hk = j % Hk;
  return t;
}

// Work item -> (sequence, key head, row tile), part of its list and workspace
// slot (-1: whole).  Row tiles of one key head are neighbours (their windows
// overlap in an XCD's L2), the last ones, whose causal lists are longest, first.
// (Without the causal mask the longest lists are in the middle: neither this order nor
// the choice of the cut tiles goes by length there, and launches end less evenly.)
struct WinItem {
  int b, hk, tile, split, slot;
};
__device__ __forceinline__ WinItem win_tile(const WinArgs& a, int index, int split, int slot) {
  WinItem it;
  it.split = split;
  it.slot = slot;
  if (a.ranked) {
    const int lane = (int)threadIdx.x & 63;
    int c = 0;
    if (lane < a.B) c = (seq_span(a, lane).n * a.G + 127) >> 7;
    const RankedTile t = rank_tile(c, a.B, a.Hk, a.tiles, index);
    c = __builtin_amdgcn_readlane(c, t.b);
    it.b = t.b;
    it.hk = t.hk;
    it.tile = t.live ? c - 1 - t.rank : c + t.rank;
    return it;
  }
  const int bh = index / a.tiles;
  it.tile = a.tiles - 1 - (index - bh * a.tiles);
  it.b = bh / a.Hk;
  it.hk = bh - it.b * a.Hk;
  return it;
}
__device__ __forceinline__ WinItem win_item(const WinArgs& a, int id) {
  const int y = id - a.whole, q = y / a.splits;
  return id < a.whole ? win_tile(a, id, 0, -1) : win_tile(a, a.whole + q, y - q * a.splits, a.splits == 1 ? -1 : y);
}

// ------------------------------------------------------------ values that are not finite
// A product over a tile multiplies the values that a row does not see by 0, and 0
// times a NaN or an infinity is a NaN.  The kernels therefore look at their sums
// once, at the end: where one of a wave's 32 rows is not finite, the wave computes
// its rows again key by key, adding only what each row sees.  (Rows that do see
// such a value keep it; the others get what they would have without it.)  Slow, 0.5
// to 1.5 us for each key of the list (4,000 queries of 8 heads over 4,000 keys, one NaN:
// 80 us become 6.2 ms at D = 128, 52 become 2.2 at 64), and free otherwise.
template <int NDT>
__device__ __forceinline__ bool win_not_finite(const f32x16* acc, float l, bool live) {
  float t = 0.0f * l;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) t = __builtin_fmaf(acc[dt][x], 0.0f, t);
  return __builtin_amdgcn_ballot_w64(live && t != t) != 0;
}
// acc, m, l of the lane's row (channels 32 dt + 8 j + 4 g + x in acc[dt][4 j + x]) over entries u0 .. u1 - 1
template <class E, int D>
__device__ __forceinline__ void win_careful(const WinArgs& a, const KeyList& kl, const TokenSpan& span, int u0, int u1,
                                            const uint16_t* q, const uint8_t* kb, const uint8_t* vb, int64_t kstep,
                                            int64_t vstep, int g, f32x16* acc, float& m, float& l) {
  constexpr int NDT = D / 32;
  const float NINF = -__builtin_inff();
  m = NINF;
  l = 0.0f;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) acc[dt] = f32x16_zero();
#pragma unroll 1
  for (int u = u0; u < u1; ++u) {
    const int key = kl.key(u);
    const uint16_t* k = (const uint16_t*)(kb + key * kstep) + 4 * g;
    const uint16_t* v = (const uint16_t*)(vb + key * vstep) + 4 * g;
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
    const bool sees = (u >= span.a && u <= span.b) || u < span.c;
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

// ------------------------------------------------------------ output
// Lanes l and l + 32 hold channels 8 j + 0 .. 3 and 8 j + 4 .. 7 of the same row (u for
// block j, v for j + 1, packed): all of block j for the lower half, of j + 1 for the
// upper, so that a lane stores 16 bytes (2 x 4,096 tokens, 16 heads over 4, D = 64,
// window 1,024: forward 55 -> 52 us, against stores of 8).
__device__ __forceinline__ uint4 win_join_halves(uint2 u, uint2 v) {
  const auto x = __builtin_amdgcn_permlane32_swap(u.x, v.x, false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(u.y, v.y, false, false);
  return make_uint4(x[0], y[0], x[1], y[1]);
}
template <class E>
__device__ __forceinline__ uint2 win_pack4(float4 x) {
  return make_uint2(E::pack(x.x, x.y), E::pack(x.z, x.w));
}
// blocks j (x) and j + 1 (y) of a row whose block j begins at p; both halves of the wave
template <class E>
__device__ __forceinline__ void win_store(uint16_t* p, int g, float4 x, float4 y) {
  *reinterpret_cast<uint4*>(p + 8 * g) = win_join_halves(win_pack4<E>(x), win_pack4<E>(y));
}
// what rounding to u leaves off x
template <class E>
__device__ __forceinline__ float4 win_left(float4 x, uint2 u) {
  return make_float4(x.x - E::lo(u.x), x.y - E::hi(u.x), x.z - E::lo(u.y), x.w - E::hi(u.y));
}
// the same for o at element `at`, and its rest where the call asks for it
template <class E>
__device__ __forceinline__ void win_store_o(const WinArgs& a, int64_t at, int g, float4 x, float4 y) {
  const uint2 u = win_pack4<E>(x), v = win_pack4<E>(y);
  *reinterpret_cast<uint4*>(a.o.p + at + 8 * g) = win_join_halves(u, v);
  if (a.rest) win_store<E>(a.rest + at, g, win_left<E>(x, u), win_left<E>(y, v));
}
__device__ __forceinline__ float4 win_scaled(f32x16 v, int j, float f) {
  return make_float4(v[4 * j] * f, v[4 * j + 1] * f, v[4 * j + 2] * f, v[4 * j + 3] * f);
}
__device__ __forceinline__ float4 win_scaled(float4 v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }

// ------------------------------------------------------------ host side (window_fwd.hip)
// Whether rows see so few keys that the backward forms delta from P and dP
// (window_dq_kernel): it needs neither o nor its rest then
inline bool win_few(int64_t Sk, int64_t window, int64_t sinks, int causal) {
  const int64_t near = window < Sk ? window : Sk, keys = (causal ? near : 2 * near - 1) + (sinks < Sk ? sinks : Sk);
  return (keys < Sk ? keys : Sk) <= 64;
}
// PRISM_OK if the sizes, strides (3 per tensor) and pointers are what the kernels assume
int win_check(const char* name, int dtype, int B, int Hq, int Hk, int64_t Sq, int64_t Sk, int D, int64_t window,
              int64_t sinks, float sm_scale, const int64_t* strides, int tensors,
              std::initializer_list<const void*> pointers);
// the arguments that all launches share (strides: q, k, v, o)
WinArgs win_args(const void* q, const void* k, const void* v, void* o, int B, int Hq, int Hk, int64_t Sq, int64_t Sk,
                 const int64_t* strides, int64_t window, int64_t sinks, int causal, const int32_t* q_lens,
                 const int32_t* kv_lens, float sm_scale);

// How a launch of `total` tiles (of about `units` list entries each) is cut so
// that it ends evenly on `slots` workgroups at a time: whole rounds as they are,
// and the tiles of the last round in the number of parts that takes least time
// by this model, in entries of a full round: a part takes its entries and 3 more;
// a round that fills a share x of the slots 0.5 + 0.5 x of a full one (fewer
// workgroups on a CU each run faster); the second kernel 2, and 0.015 (D = 64:
// 0.005) for each part's sums, written and read.  Measured, both kernels: 550
// tiles of 133 entries over 512 slots at D = 128, uncut / 38 of them in 13 parts:
// forward 428 / 357 us; 1,024 tiles of 17 entries over 768 slots at D = 64, uncut
// / 256 of them in 3 parts: dQ 59 / 66 us.
struct WinCut {
  int64_t whole, splits;
};
inline WinCut win_cut(int64_t total, int64_t slots, int64_t units, int D) {
  WinCut c{total / slots * slots, 1};
  const int64_t rest = total - c.whole;
  double best = 0;
  for (int64_t s = 1; s <= 32 && (s == 1 || units >= 4 * s); ++s) {
    const double full = (double)(rest * s / slots), x = (double)(rest * s % slots) / (double)slots;
    const double rounds = full + (x > 0 ? 0.5 + 0.5 * x : 0);
    const double cost = rounds * ((double)units / (double)s + 3) + (s > 1 ? 2 + (D == 64 ? 0.005 : 0.015) * (double)(rest * s) : 0);
    if (s == 1 || cost < best) {
      best = cost;
      c.splits = s;
    }
  }
  if (c.splits == 1) c.whole = total;
  return c;
}
// Whether a launch of `total` tiles goes by rank (rank_tile): sequences of their
// own lengths, several workgroups a CU (dK/dV at D = 128 has one: 150 us by
// sequences, 152 by rank), more tiles than CUs, and no more than two rounds (beyond
// them the order by sequences is better: neighbours share keys in an XCD's L2, and a
// CU that ends early takes the next tile).
inline int win_ranked(const int32_t* lens, int B, int64_t tiles, int64_t total, int64_t slots) {
  return lens && B > 1 && B <= 64 && tiles <= 4096 && slots > 256 && total > 256 && total <= 2 * slots;
}
// the cut of a launch over row tiles of 128 (forward, dQ)
WinCut win_row_cut(int64_t slots, int B, int Hk, int64_t G, int64_t Sq, int64_t Sk, int D, int64_t window, int64_t sinks,
                   int causal);
