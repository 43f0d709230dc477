// The paged key/value cache in 8 bits: its layout, and what the kernels that
// write and read it share.
//
// A page holds 32, 64 or 128 tokens of one sequence.  Per page and key head
// there is one power-of-two scale for K and one for V (the rule of tm_fp8_dev.h,
// never below 2^-100), and the values as tiles of 32 tokens by 32 columns, 1 KiB
// each, in the order in which the 32x32x16 matrix instruction wants its
// operands: lane l's 16 bytes are two k-steps of 8.
//   K tile j: byte e of lane l is token l % 32, column 32 j + 16 (l / 32) + e.
//   V tile j: byte e of lane l is column 32 j + l % 32, token
//             16 (e / 8) + 8 (e / 4 % 2) + 4 (l / 32) + e % 4.
// The tokens of V stand in the order in which K Q^T leaves its rows in a lane's
// registers, so the probabilities of a tile are an operand of the second product
// as they come out of the first: nothing is exchanged between lanes or goes
// through LDS.
#pragma once

#include "tm_fp8_dev.h"
#include "tm_mfma.h"

constexpr int kKv8Tile = 32;
constexpr int64_t kKv8MaxGrid = (int64_t)1 << 24;  // workgroups of 256: a launch holds under 2^32 threads in a direction
constexpr float kKv8MinScale = 0x1p-100f;

// A batch's sequence: its new tokens are [first, first + n) of the caller's rows,
// the last n of its `len` positions.  Whatever the lists hold, the ranges lie
// within the rows; pages are checked where they are looked up.
struct Kv8Seq {
  int64_t first, n, len;
};
__device__ __forceinline__ Kv8Seq tm_kv8_seq(const tm_kv8_batch &bt, int64_t b) {
  Kv8Seq s;
  int64_t lo = b, hi = b + 1;
  if (bt.starts != nullptr) {
    lo = bt.starts[b];
    hi = bt.starts[b + 1];
  }
  lo = lo < 0 ? 0 : lo > bt.n_tokens ? bt.n_tokens : lo;
  hi = hi < lo ? lo : hi > bt.n_tokens ? bt.n_tokens : hi;
  s.first = lo;
  s.n = hi - lo;
  const int64_t len = bt.lengths[b];
  s.len = len < 0 ? 0 : len;
  return s;
}

// The sequence that owns unit u where sequence b's units begin at
// starts[b] * num / den + more * b: the last b that begins at or before u.
__device__ __forceinline__ int64_t tm_kv8_unit(const tm_kv8_batch &bt, int64_t u, int64_t num, int64_t den, int64_t more,
                                               int64_t &in) {
  int64_t lo = 0, hi = bt.n_seqs - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if ((int64_t)bt.starts[mid] * num / den + more * mid <= u) lo = mid;
    else hi = mid - 1;
  }
  in = u - ((int64_t)bt.starts[lo] * num / den + more * lo);
  return lo;
}

// Eight e4m3 values as an operand of DT (exact in both: 4 significant bits, 2^-9 to 448).
template <int DT>
__device__ __forceinline__ uint4 tm_kv8_operand(uint32_t lo, uint32_t hi) {
  if constexpr (DT == TM_DT_BF16) {
    return tm_fp8_to_bf16x8(lo, hi);
  } else {
    uint4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
    return r;
  }
}

// What the entry points refuse about a cache and a batch (host).
int tm_kv8_check(const char *what, const tm_kv8_cache *c, const tm_kv8_batch *b) __attribute__((visibility("hidden")));

// How a call's keys are cut up for workgroups: at most `splits` parts, of at least `least` tiles of 32.
struct Kv8Cut {
  int splits, least;
};
// Cut of the keys of a call with one query per sequence (`groups` heads to a key head), and the softmax
// statistics of its rows: stats[row][split] = (reference in units of log2, sum), the
// first ceil(tiles / per) of them written, with tiles of 32 keys and per as
// tm_kv8_per gives it.  Arguments as checked by tm_kv8_importance.
__attribute__((visibility("hidden"))) Kv8Cut tm_internal_kv8_cut(const tm_kv8_cache *c, const tm_kv8_batch *b, int groups);
__attribute__((visibility("hidden"))) int tm_internal_kv8_stats(const tm_kv8_cache *cache, const tm_kv8_batch *batch,
                                                                int32_t dtype, const void *q, int64_t qs_b, int64_t qs_h,
                                                                int32_t n_heads, float scale, float2 *stats,
                                                                hipStream_t s);
// Tiles of a part: whole rounds of a workgroup's four waves.
__device__ __forceinline__ int64_t tm_kv8_per(int64_t tiles, Kv8Cut cut) {
  const int64_t n = ((tiles + cut.splits - 1) / cut.splits + 3) / 4 * 4;
  return n > cut.least ? n : cut.least;
}
