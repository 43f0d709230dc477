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
__device__ __forceinline__ Kv8Place tm_kv8_place(const tm_kv8_cache &c, const tm_kv8_batch &bt, int64_t b, int h,
                                                 int64_t tile, int page_log2) {
  const int tl = page_log2 - 5;  // tiles of a page: 1 << tl
  const int64_t p = tile >> tl;
  Kv8Place r;
  int64_t id = p < bt.max_pages ? bt.table[b * bt.ld_table + p] : -1;
  r.there = id >= 0 && id < c.n_pages;
  id = r.there ? id : 0;
  r.slot = id * c.n_kv_heads + h;
  r.tile = (int)(tile & ((1 << tl) - 1));
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
__device__ __forceinline__ float tm_exponent(float s) { return (float)((int)(__float_as_uint(s) >> 23 & 0xff) - 127); }
