// Paged caches (gfx950): the keys (or values) of many sequences in pages of a power of
// two of places, each sequence's pages listed in a row of a table.
//
// 16 bits: rows [page][head][place], channels adjacent, any strides of whole 16 bytes.
// 4 bits: for each (page, head) the codes of its places, D / 2 bytes each (an even
// channel in the low half of its byte), then their scales, D / 32 bytes each.  A code is
// a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (the hardware's 4-bit float), a scale byte
// e stands for 2^(e - 127), shared by 32 channels: the least that keeps them within 6, so
// nothing is cut off, 1 at least; 255 where one of them is not finite (all 32 are then
// read as NaN).  Powers of two make code x scale exact in bfloat16, and one instruction
// makes two such values.
//
// Table entries outside [0, pages) are no pages: what would stand there is not stored and
// not seen.
#pragma once
#include "common.h"
#include "mfma.h"

struct PagedSide {
  uint8_t* p;
  int64_t page, head, row;  // strides in bytes (row: 16 bits only)
};
struct PagedTable {
  const int32_t* table;  // [B, width] at rows `stride` apart
  int64_t stride;
  int width, pages, lg;  // lg: log2 of the places of a page
  // page of `index` of sequence b, or -1
  __device__ __forceinline__ int page(int b, int index) const {
    if (index < 0 || index >= width) return -1;
    const int x = table[(int64_t)b * stride + index];
    return x < 0 || x >= pages ? -1 : x;
  }
};

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// scale byte of 32 channels whose largest magnitude has these bits
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u);  // top <= 6 2^(e - 127)
  return (uint32_t)(e < 1 ? 1 : e);
}

// the eight values of a word of codes, times a scale
__device__ __forceinline__ uint4 bf16_of_codes(uint32_t w, float s) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
  return r;
}
__device__ __forceinline__ uint4 f16_of_codes(uint32_t w, float s) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
  return r;
}

// ------------------------------------------------------------ host side (paged.hip)
// what the kernels assume of a cache; strides (host): page, head, place of keys, then of
// values, in elements (4 bits: bytes; the places' are not read)
int paged_check(const char* name, int dtype, int bits, int Hk, int D, int64_t pages, int page_size, const int64_t* strides,
                const void* k_cache, const void* v_cache, int64_t width, int64_t B);
void paged_sides(PagedSide* k, PagedSide* v, int bits, const int64_t* strides, const void* k_cache, const void* v_cache);
PagedTable paged_table(const int32_t* table, int64_t stride, int64_t width, int64_t pages, int page_size);
