// What the kernels of packed batches share (gfx950): sequences of a batch standing
// behind one another in [tokens, heads, D] tensors, bounded by cu_seqlens on the
// device; how a launch finds its work; element types, copies and stores of window.h.
//
// Rows.  As in window.h, row r of a (sequence, key head) is token r / G of query head
// hk G + r % G.  Token i of a sequence with L keys and n queries stands at p = i + L -
// n and sees keys 0 .. p (causal) or all L.  Rows before the first sequence and behind
// the last are taken as two more sequences without keys (s = 0 and B + 1): they give 0.
//
// Work lists.  The lengths stand on the device, so the host knows only bounds: a launch
// has as many workgroups as any lengths could need, and those past the list end at
// once.  A first kernel of one workgroup (pack_plan_kernel) writes the list: blocks of
// gs neighbouring tiles of a sequence (they read the same keys at about the same time,
// and ids in groups of eight share an XCD's L2), longest first, so that the launch ends
// evenly; blocks longer than a fair share of a slot's work are cut into parts along
// their key (or token) list, whose fp32 sums a last kernel adds in order.  Launches of
// one round over short sequences do without a list (PackItem::direct).
#pragma once
#include "window.h"

struct PackTensor {  // [T, H, D], channels adjacent; strides in elements
  uint16_t* p;
  int64_t h, s;
};

// an entry of the work list: a part of a block of tiles (all key heads)
struct PackEntry {
  int q0, n, k0, L, tile, part, parts, slot;  // slot: of the block's first piece in the workspace; -1: not cut
};
struct PackList {
  PackEntry* entries;   // null: direct
  PackEntry* cuts;      // blocks that were cut (part = 0)
  int* counts;          // entries, cuts, pieces
  int max_entries, max_cuts, max_pieces;
  int gs, per;          // tiles of a block; items of an entry: gs Hk
  int unit;             // rows (of tokens x G, or keys) of a tile
  int keys;             // tiles of keys (dK/dV), else of rows
  int want, least;      // parts: as many as this of equal length in all (0: never cut), of so many list tiles at least
  int from;             // blocks longer than from / 4 of such a length are cut
  int items;            // workgroups of the launch
};
struct PackArgs {
  PackTensor q, k, v, o;
  const int32_t *cu_q, *cu_k;  // [B + 1]
  int B, Hk, G, Tq, Tk, causal;
  float scale, scale_log2;
  uint16_t* rest;       // what o's rounding left off, at o's strides; or null
  float* lse;           // [Hk G, Tq] natural log, -inf for rows that see nothing; or null
  PackList list;
  float *part, *part_ml;
};

// sequence s of 0 .. B + 1, cut to the tensors (bounds that decrease: empty)
struct PackSeq {
  int q0, n, k0, L;
};
__device__ __forceinline__ PackSeq pack_seq(const PackArgs& a, int s, bool keys) {
  auto bound = [](const int32_t* cu, int i, int T) { const int x = cu[i]; return x < 0 ? 0 : x < T ? x : T; };
  PackSeq q;
  q.q0 = s == 0 ? 0 : bound(a.cu_q, s - 1, a.Tq);
  q.k0 = s == 0 ? 0 : bound(a.cu_k, s - 1, a.Tk);
  q.n = (s == a.B + 1 ? a.Tq : bound(a.cu_q, s, a.Tq)) - q.q0;
  q.L = (s == a.B + 1 ? a.Tk : bound(a.cu_k, s, a.Tk)) - q.k0;
  q.n = q.n > 0 ? q.n : 0;
  q.L = q.L > 0 ? q.L : 0;
  if (s == 0 || s == a.B + 1) (keys ? q.n : q.L) = 0;
  return q;
}
__device__ __forceinline__ int pack_tiles(const PackArgs& a, const PackSeq& s) {
  return a.list.keys ? (s.L + a.list.unit - 1) / a.list.unit : (int)(((int64_t)s.n * a.G + a.list.unit - 1) / a.list.unit);
}
// keys that tokens up to i1 see
__device__ __forceinline__ int pack_keys(const PackArgs& a, const PackSeq& s, int i1) {
  if (!a.causal) return s.L;
  const int x = i1 + s.L - s.n + 1;
  return x < 0 ? 0 : x < s.L ? x : s.L;
}
// the first token that sees some key from j0 on (n: none)
__device__ __forceinline__ int pack_first(const PackArgs& a, const PackSeq& s, int j0) {
  if (!a.causal) return s.L > 0 ? 0 : s.n;
  const int x = j0 + s.n - s.L;
  return x < 0 ? 0 : x < s.n ? x : s.n;
}

// The item of workgroup id: as xcd_group_remap<8>, but every second run of 64 goes to the XCDs
// the other way round: the list is sorted by length, and the first XCD would have the longest of
// each run (dQ and dK/dV of 16,001 tokens of three sequences, 32 heads over 8: 2,275 us, so 2,235;
// of 8,191 of six, 16 over 4: 243, 237; others within 1%).
__device__ __forceinline__ int pack_id(const PackList& l, int id) {
  if (id >= (l.items & ~63)) return id;
  const int run = id >> 6, xcd = id & 7, slot = (id >> 3) & 7;
  return run * 64 + (run & 1 ? 7 - xcd : xcd) * 8 + slot;
}

struct PackItem {
  PackSeq s;
  int hk, tile, part, parts, slot;  // slot: workspace piece, -1: the whole list
  bool live;
  // the first of `all` list tiles that part p takes (all x parts may pass 32 bits)
  __device__ __forceinline__ int first_of(int all, int p) const {
    return slot < 0 ? (p ? all : 0) : (int)((int64_t)all * p / parts);
  }
  // without a list: sequences in order, tile by tile (B <= 62; all lanes active)
  __device__ __forceinline__ void direct(const PackArgs& a, int id) {
    const int lane = (int)threadIdx.x & 63, x = id / a.Hk;
    hk = id - x * a.Hk;
    PackSeq mine{0, 0, 0, 0};
    if (lane < a.B + 2) mine = pack_seq(a, lane, a.list.keys);
    const int count = pack_tiles(a, mine);
    const int upto = (int)wave_incl_scan_u32((uint32_t)count, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > x);
    live = past != 0;
    const int who = live ? (int)__builtin_ctzll(past) : 0;
    s.q0 = __builtin_amdgcn_readlane(mine.q0, who);
    s.n = __builtin_amdgcn_readlane(mine.n, who);
    s.k0 = __builtin_amdgcn_readlane(mine.k0, who);
    s.L = __builtin_amdgcn_readlane(mine.L, who);
    tile = x - (__builtin_amdgcn_readlane(upto, who) - __builtin_amdgcn_readlane(count, who));
    part = 0;
    parts = 1;
    slot = -1;
  }
  __device__ __forceinline__ void of_entry(const PackArgs& a, const PackEntry& e, int r) {
    auto u = [](int x) { return (int)uniform_u32((uint32_t)x); };
    s.q0 = u(e.q0); s.n = u(e.n); s.k0 = u(e.k0); s.L = u(e.L);
    hk = r / a.list.gs;
    const int x = r - hk * a.list.gs;
    tile = u(e.tile) + x;
    part = u(e.part); parts = u(e.parts); slot = u(e.slot);
    if (slot >= 0) slot += (hk * a.list.gs + x) * parts + part;
    live = tile < pack_tiles(a, s);
  }
  __device__ __forceinline__ void init(const PackArgs& a, int id) {
    if (!a.list.entries) {
      direct(a, id);
      return;
    }
    const int blk = id / a.list.per;
    const PackEntry e = a.list.entries[blk];  // (beside the count, which says whether it holds something)
    live = blk < (int)uniform_u32((uint32_t)a.list.counts[0]);
    if (live) of_entry(a, e, id - blk * a.list.per);
  }
  // block of the join's workgroup id
  __device__ __forceinline__ void init_cut(const PackArgs& a, int id) {
    const int blk = id / a.list.per;
    live = blk < (int)uniform_u32((uint32_t)a.list.counts[1]);
    if (live) of_entry(a, a.list.cuts[blk], id - blk * a.list.per);
  }
};

// The tile copies of a 64-key stage (K then V) by two waves, as StageCopy of window.h
template <int D>
struct PackCopy {
  using RT = RowTile<D>;
  using RS = RowSource<D>;
  static constexpr int COUNT = RT::KB;
  const uint8_t *kb, *vb;  // K and V of the (sequence, key head)
  int64_t kstep, vstep;    // bytes per row
  int wid;
  uint32_t koff[2], voff[2];
  __device__ __forceinline__ void offsets(int lane, uint32_t* ko, uint32_t* vo) const {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = RS::row(wid + 2 * x, lane), c = RS::byte(wid + 2 * x, lane);
      ko[x] = (uint32_t)r * (uint32_t)kstep + (uint32_t)c;
      vo[x] = (uint32_t)r * (uint32_t)vstep + (uint32_t)c;
    }
  }
  __device__ __forceinline__ void init(const PackArgs& a, const PackItem& it, int wid_, int lane) {
    wid = wid_;
    kb = (const uint8_t*)uniform_ptr(a.k.p + it.hk * a.k.h + it.s.k0 * a.k.s);
    vb = (const uint8_t*)uniform_ptr(a.v.p + it.hk * a.v.h + it.s.k0 * a.v.s);
    kstep = 2 * a.k.s;
    vstep = 2 * a.v.s;
    if constexpr (D == 128) offsets(lane, koff, voff);
  }
  // keys u0 .. u0 + 63 of n (past the end the last one again: a later sequence's rows are never read)
  __device__ __forceinline__ void issue(int n, int u0, uint32_t lds) const {
    const int lane = opaque_thread_id() & 63;
    if (u0 + 63 < n) {
      const uint8_t* kt = (const uint8_t*)uniform_ptr(kb + u0 * kstep);
      const uint8_t* vt = (const uint8_t*)uniform_ptr(vb + u0 * vstep);
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
        const int m = ((2 * s) % RT::KB) >> 2;
        const uint8_t* base = isk ? kt + m * RS::ROWS4 * kstep : vt + m * RS::ROWS4 * vstep;
        dma_b128(isk ? ko[s & 1] : vo[s & 1], base, lds + (uint32_t)i * 1024u);
      }
      return;
    }
#pragma unroll 1
    for (int s = 0; s < COUNT; ++s) {
      const int i = wid + 2 * s, t = i < RT::KB ? i : i - RT::KB;
      const int u = u0 + RS::row(t, lane), key = u < n ? u : n - 1;
      const uint8_t* src = (i < RT::KB ? kb + key * kstep : vb + key * vstep) + RS::byte(t, lane);
      dma_b128_from(src, uniform_u32(lds + (uint32_t)i * 1024u));
    }
  }
};

// bit j: key u0 + j is at or before `last`
__device__ __forceinline__ uint64_t upto_bits(int last, int u0) {
  const int b = last - u0;
  return b >= 63 ? ~0ull : b < 0 ? 0ull : (2ull << b) - 1;
}

// ------------------------------------------------------------ host side (packed_fwd.hip)
// How a launch is listed: tiles of `unit` rows (rows: of all sequences together), `slots`
// workgroups on the chip at a time; longest: rows of the longest list that any lengths
// could give, in list tiles
struct PackCut {
  PackList list;
  int64_t entries, cuts, pieces;
};
PackCut pack_cut(int64_t rows, int unit, int64_t B, int64_t Hk, int64_t slots, int64_t longest, int keys, int least);
inline int64_t pack_ints(const PackCut& c) {  // ints of the list's buffer
  return c.list.entries ? 8 + 8 * (c.entries + c.cuts) : 0;
}
// the list's place in its buffer
void pack_place(PackCut* c, int32_t* buffer);
int pack_check(const char* name, int dtype, int B, int Hq, int Hk, int64_t Tq, int64_t Tk, int D, float sm_scale,
               const int64_t* strides, int tensors, std::initializer_list<const void*> pointers);
PackArgs pack_args(const void* q, const void* k, const void* v, void* o, int B, int Hq, int Hk, int64_t Tq, int64_t Tk,
                   const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int causal, float sm_scale);
// the list kernel over one or two launches' lists (b: null or the same batch's other list)
void pack_plan(const PackArgs& a, const PackList* b, hipStream_t stream);
