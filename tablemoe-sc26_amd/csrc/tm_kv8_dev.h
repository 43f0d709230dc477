// Device pieces shared by the kernels that read the 8-bit cache.
#pragma once

#include "tm_kv8.h"

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Value of the lane 32 away.
__device__ __forceinline__ float tm_other_half(float v) { return __shfl_xor(v, 32, 64); }

// Where a tile of 32 tokens of one head lies.
struct Kv8Place {
  int64_t slot;  // page * heads + head
  int tile;      // within the page
  bool there;
};
// The page of a tile, as its sequence's row of the table names it (-1: past the table's width).  Loaded a round before
// the tile itself: the bytes wait for it.
__device__ __forceinline__ int tm_kv8_page(const tm_kv8_batch &bt, const int32_t *row, int tile, int page_log2) {
  const int p = tile >> (page_log2 - 5);  // (max_pages < 2^24: a tile's number fits 32 bits)
  const int id = row[p < bt.max_pages ? p : bt.max_pages - 1];
  return p < bt.max_pages ? id : -1;
}
__device__ __forceinline__ Kv8Place tm_kv8_place(const tm_kv8_cache &c, int id, int h, int tile, int page_log2) {
  Kv8Place r;
  r.there = id >= 0 && id < c.n_pages;
  r.slot = (int64_t)(r.there ? id : 0) * c.n_kv_heads + h;
  r.tile = tile & ((1 << (page_log2 - 5)) - 1);
  return r;
}

// A lane's share of a tile's K (or V): D / 32 pieces of 16 bytes.
template <int N>
__device__ __forceinline__ void tm_kv8_load(const void *base, const Kv8Place &w, int page_log2, int lane, uint4 (&r)[N]) {
  const uint8_t *p = static_cast<const uint8_t *>(base) +
                     (((w.slot << (page_log2 - 5)) + w.tile) * (int64_t)(N * 1024)) + lane * 16;
#pragma unroll
  for (int j = 0; j < N; ++j) r[j] = *reinterpret_cast<const uint4 *>(p + j * 1024);
}

// Exponent of a power of two.
__device__ __forceinline__ int tm_exponent(float s) { return (int)(__float_as_uint(s) >> 23 & 0xff) - 127; }
