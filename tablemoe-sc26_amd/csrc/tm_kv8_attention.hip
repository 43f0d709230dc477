// Attention over the 8-bit cache (layout: tm_kv8.h): tm_kv8_attention.
//
// Rows of a sequence are its (new token, query head of one key head) pairs, so a
// key head's keys serve all its query heads.  A workgroup owns R x 32 rows; its
// four waves take every fourth tile of 32 keys and join through LDS.  Per tile and
// 32 rows:
//   S^T = K Q^T on the 16-bit instructions (a byte of K is exact in 16 bits), a
//   lane holding 16 keys of one row;  x = S^T sk scale log2(e) + log2(sv);
//   P = 2^(x - m) under a reference m of the row, so that the values' scale
//   rides in P and V enters as the bytes stand;  O^T += V^T P.
// With l = sum P / sv the result is O / l and log sum exp = (m + log2 l) ln 2.  sv is
// 2^-100 to 2^120 and l stays in range, but a factor of it may not: where P falls
// under fp32's smallest number for sv's sake, or a reference moves that far, l is
// taken apart from P or in two factors.
// m is set 2^8 under the first tile's largest x and raised only where the
// probabilities of a lane's 16 keys sum to more than 2^15: no maximum is taken of
// the other tiles, and O is seldom scaled again.  P is rounded to fp16 for the
// second product whatever the queries' type, and V's bytes become fp16 (exact):
// half a step is 2^-11 of a probability at most, where bf16 would leave 2^-8 (an output's
// error against 64 bits 1.9e-3 of its size instead of 1.6e-3, which is its own
// rounding); what lies under 2^-33 of a row's largest is lost.  All sums are fp32; l
// takes the probabilities before that rounding (log sum exp has no other), so an
// output's weights sum to 1 up to 2^-11.
//
// A long prompt is bound by instructions: per 32 keys and 64 rows the products take 1024
// cycles of the matrix units, of which about half keep the vector units from
// issuing, and the conversions of K and V (64, 5 cycles each), exponentials (32, 8.5)
// and the rest (about 110, 3 to 6) another 1000.  So a long prompt's waves own 64 rows,
// which share the conversions, with the queries' operands in LDS (in registers they
// would leave one wave per SIMD, which issues a vector instruction every 5 to 12
// cycles where two issue one every 3).  Tried and slower: the tile converted once per
// workgroup into LDS; one wave per SIMD with the next tile's scores among this tile's exponentials.
// A decode step is bound by HBM; where rows alone do not fill the device, the keys
// are split over workgroups too, and a second launch joins their parts.
#include "tm_internal.h"
#include "tm_kv8_dev.h"

#include <type_traits>

namespace {

typedef float tm_f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 tm_f16x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kMaxSplits = 128;
constexpr int kRoom = 8;  // log2 of the first maximum's P
// What the probabilities of 16 keys may sum to before the reference is raised (each is rounded to fp16: at most 65504).
constexpr float kMost = 32768.f;
constexpr int kFar = 80;  // of 126: what is left to P is 2^-46 of its row's largest

struct AttArgs {
  tm_kv8_cache c;
  tm_kv8_batch b;
  const void *q;
  int64_t qs_t, qs_h;
  void *out;
  int64_t os_t, os_h;
  float *lse;
  float2 *stats;  // [row of the call][split]: reference, sum
  float *part;    // [row of the call][split][v_dim]
  float scale;
  Kv8Cut cut;
  int32_t heads, groups, page_log2, causal, tiles1, rows, early, turn;  // tiles1: row tiles of one token; rows: of a tile
};

// l 2^x, where 2^x alone may be too small for fp32.
__device__ __forceinline__ float scaled(float l, float x) {
  const float root = __builtin_amdgcn_exp2f(0.5f * x);
  return l * root * root;
}

// A row tile: rows [r0, r0 + rows) of sequence b (tokens times heads of a key head: under 2^31).
struct RowTile {
  Kv8Seq s;
  int64_t b;
  uint32_t r0;
  int rows;
  int64_t end;    // keys that its last row sees
  int64_t tiles;  // of 32 keys
  int64_t per;    // tiles of a split
};
__device__ __forceinline__ int64_t visible(const AttArgs &a, const Kv8Seq &s, uint32_t token) {
  const int64_t cap = (int64_t)a.b.max_pages << a.page_log2;
  int64_t e = a.causal ? s.len - s.n + token + 1 : s.len;
  e = e < cap ? e : cap;
  return e < 0 ? 0 : e;
}
// Row tile j of sequence t.b (false: it has no such rows).
template <int ROWS = 32>
__device__ __forceinline__ bool tile_at(const AttArgs &a, int64_t j, RowTile &t) {
  t.s = tm_kv8_seq(a.b, t.b);
  const int64_t all = t.s.n * a.groups;
  if (j < 0 || j * ROWS >= all) return false;
  t.r0 = (uint32_t)(j * ROWS);
  t.rows = (int)(all - t.r0 < ROWS ? all - t.r0 : ROWS);
  const uint32_t last = a.b.starts != nullptr ? (t.r0 + t.rows - 1) / (uint32_t)a.groups : 0;  // the tile's last token
  t.end = visible(a, t.s, last);
  t.tiles = (t.end + 31) >> 5;
  const bool fills = a.cut.least > 4 && all * a.c.n_kv_heads >= 256 * 32;  // one workgroup per CU of its own
  t.per = a.cut.splits == 1 || fills ? t.tiles + 3 : tm_kv8_per(t.tiles, a.cut);
  return true;
}
// Row tile u of the call.
template <int ROWS = 32>
__device__ __forceinline__ bool row_tile(const AttArgs &a, int64_t u, RowTile &t) {
  int64_t j = 0;
  if (a.b.starts == nullptr) {
    t.b = a.tiles1 == 1 ? (uint32_t)u : (uint32_t)u / (uint32_t)a.tiles1;
    j = u - t.b * a.tiles1;
  } else {
    t.b = tm_kv8_unit(a.b, u, a.groups, ROWS, 1, j);
  }
  return tile_at<ROWS>(a, j, t);
}
// A row's token (of its sequence) and its head among the key head's.
__device__ __forceinline__ uint32_t token_of(const AttArgs &a, uint32_t row) {
  return a.b.starts == nullptr ? 0 : row / (uint32_t)a.groups;
}

// DV = 0: the statistics alone.
template <int DT, int D, int DV, int R>
__global__ __launch_bounds__(kThreads, R == 2 || D + DV > 320 ? 2 : 3) void attend_kernel(AttArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int NK = D / 32, NV = DV / 32;
  constexpr int kChunk = 64;  // columns joined at a time
  constexpr size_t kQ = R * NK * 2 * 64 * 16, kJoin = DV ? sizeof(float) * kWaves * 32 * (kChunk + 4) : 0;
  __shared__ __align__(16) uint8_t lds[kQ > kJoin ? kQ : kJoin];  // the queries' operands, then the parts to join
  __shared__ float2 join[kWaves][32];
  __shared__ float inv_s[32];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int c = lane & 31, g = lane >> 5;
  // The last tokens see most: they go first.  (A call with starts counts up to twice the tiles that there are: with the
  // tiles first, one sequence of 4 tokens of 131071 keys kept to half of the XCDs, 44 us, 36 so.)
  const uint32_t heads = a.c.n_kv_heads, splits = a.cut.splits;
  uint32_t block = gridDim.x - 1 - blockIdx.x, split = 0;
  if (splits > 1) {
    const uint32_t by = a.cut.least == 4 ? splits : gridDim.x / splits, quot = block / by;
    if (a.cut.least == 4) {  // every tile is split: its parts one after the other, over all XCDs
      split = block - quot * by;
      block = quot;
    } else {
      block = block - quot * by;
      split = splits - 1 - quot;
    }
  }
  if (a.turn) {  // what has work may come at steps of 8, which is one XCD: these are turned against each other
    const uint32_t units = gridDim.x / splits;
    if (block < (units & ~7u)) block = (block & ~7u) | ((block + (block >> 3) + split) & 7);
  }
  block = __builtin_amdgcn_readfirstlane(block);
  split = __builtin_amdgcn_readfirstlane(split);
  const int h = (int)(block % heads);
  RowTile t;
  if (!row_tile<32 * R>(a, block / heads, t)) return;
  const int t0 = (int)((int64_t)split * t.per < t.tiles ? split * t.per : t.tiles), n = (int)(t0 + t.per < t.tiles ? t0 + t.per : t.tiles);
  if (t0 >= n && split > 0) return;
  const bool whole = t.per >= t.tiles;  // nothing to join with other workgroups
  auto head_of = [&](uint32_t row, uint32_t token) { return (int64_t)h * a.groups + (row - token * a.groups); };

  const float unit = a.scale * kLog2e;
  const int seen_whole = (int)(visible(a, t.s, token_of(a, t.r0)) >> 5);  // tiles that every row sees whole
  const int32_t *const pages = a.b.table + t.b * a.b.ld_table;
  auto page_of = [&](int tile) { return tm_kv8_page(a.b, pages, tile < n ? tile : n - 1, a.page_log2); };
  auto place = [&](int tile, int id) { return tm_kv8_place(a.c, id, h, tile < n ? tile : n - 1, a.page_log2); };

  // the first tile of the wave is on its way while the queries are laid out
  uint4 kf[NK], vf[NV ? NV : 1];
  const int begin = t0 + wave;
  Kv8Place w = {};
  int id = -1;
  float sk = 1.f, sv = 1.f;
  if (begin < n) {
    w = place(begin, page_of(begin));
    id = page_of(begin + kWaves);
    tm_kv8_load<NK>(a.c.k, w, a.page_log2, lane, kf);
    if constexpr (NV > 0) tm_kv8_load<NV>(a.c.v, w, a.page_log2, lane, vf);
    sk = a.c.k_scale[w.slot];
    if constexpr (NV > 0) sv = a.c.v_scale[w.slot];
  }

  uint4(*const qs)[64] = reinterpret_cast<uint4(*)[64]>(lds);  // [r][j][e]
  int64_t limit[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t in = 32 * r + c, row = t.r0 + (in < (uint32_t)t.rows ? in : t.rows - 1), token = token_of(a, row);
    limit[r] = visible(a, t.s, token);
    const T *const q = static_cast<const T *>(a.q) + (t.s.first + token) * a.qs_t + head_of(row, token) * a.qs_h + 16 * g;
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = (r * NK + j) * 2 + e;
        if (at % kWaves == wave) qs[at][lane] = *reinterpret_cast<const uint4 *>(q + 32 * j + 8 * e);
      }
  }
  __syncthreads();
  tm_f32x16 o[R][NV ? NV : 1];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -__builtin_huge_valf();
    l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[r][j][i] = 0.f;
  }
  int most = -127;  // log2 of the largest value scale so far
  bool first = true;      // some row has no reference yet, or may have none
  bool seen_nan = false;  // among values that some row does not see
#pragma unroll 1
  for (int tile = begin; tile < n; tile += kWaves) {
    tm_f32x16 s[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[r][i] = 0.f;
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 k = e ? tm_kv8_operand<DT>(kf[j].z, kf[j].w) : tm_kv8_operand<DT>(kf[j].x, kf[j].y);
#pragma unroll
        for (int r = 0; r < R; ++r) {
        s[r] = tm_mfma32x32x16<DT>(k, qs[(r * NK + j) * 2 + e][lane], s[r]);
        }
      }
    const Kv8Place wn = place(tile + kWaves, id);
    id = page_of(tile + 2 * kWaves);
    tm_kv8_load<NK>(a.c.k, wn, a.page_log2, lane, kf);
    const int power = w.there ? tm_exponent(sv) : 0;
    const float mul = (w.there ? sk : 1.f) * unit, add = (float)power;
    sk = a.c.k_scale[wn.slot];
    if constexpr (NV > 0) sv = a.c.v_scale[wn.slot];
    if (!w.there || tile >= seen_whole) {
      first = true;
      uint32_t nan = 0;  // a NaN among values that some row does not see stays out of the product
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint32_t *const p = reinterpret_cast<uint32_t *>(&vf[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = ((p[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // 0x80 where a byte is NaN
          nan |= x;
          p[e] &= ~((x >> 7) * 0xffu);
        }
      }
      seen_nan = seen_nan || nan != 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t left = (w.there ? limit[r] : 0) - (int64_t)tile * 32;
        int lim = left > 32 ? 32 : left < 0 ? 0 : (int)left;
        asm volatile("" : "+v"(lim));  // (what follows stays in this branch)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[r][i] = 8 * (i / 4) + 4 * g + i % 4 < lim ? s[r][i] : -__builtin_huge_valf();
      }
    }
    w = wn;
    const bool low = power < most - kFar;  // P may vanish where P / sv counts
    most = power > most ? power : most;
    bool none = false;
    uint4 p[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      auto settle = [&] {  // the row's reference 2^8 under its largest score so far
        float top = s[r][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[r][i]);
        top = fmaf(top, mul, add);
        top = fmaxf(top, tm_other_half(top));
        const float to = fmaxf(m[r], top - kRoom);
        const float root = m[r] == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(0.5f * (m[r] - to)), f = root * root;
        m[r] = to;
        l[r] = l[r] * root * root;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[r][j][i] *= f;
      };
      if (first) {
        settle();
        none = none || m[r] == -__builtin_huge_valf();
      }
      float sum;
      auto probabilities = [&] {
        const float off = add - (m[r] == -__builtin_huge_valf() ? 0.f : m[r]);
        uint32_t pf[8];
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const tm_f32x2 x = {__builtin_amdgcn_exp2f(fmaf(s[r][i], mul, off)), __builtin_amdgcn_exp2f(fmaf(s[r][i + 1], mul, off))};
          sum += x.x + x.y;
          pf[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, tm_f16x2));
        }
        p[r][0] = make_uint4(pf[0], pf[1], pf[2], pf[3]);
        p[r][1] = make_uint4(pf[4], pf[5], pf[6], pf[7]);
      };
      probabilities();
      if (__any(sum > kMost)) {
        settle();
        probabilities();
      }
      if (low) {
        float top = s[r][0], apart = 0.f;
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[r][i]);
        top = top == -__builtin_huge_valf() ? 0.f : top * mul;
#pragma unroll
        for (int i = 0; i < 16; ++i) apart += __builtin_amdgcn_exp2f(fmaf(s[r][i], mul, -top));
        l[r] += scaled(apart, top - (m[r] == -__builtin_huge_valf() ? 0.f : m[r]) - kRoom);
      } else {
        l[r] += __builtin_ldexpf(sum, -kRoom - power);
      }
    }
    if (first) first = __any(none);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 v = e ? tm_kv8_operand<TM_DT_F16>(vf[j].z, vf[j].w) : tm_kv8_operand<TM_DT_F16>(vf[j].x, vf[j].y);
#pragma unroll
        for (int r = 0; r < R; ++r) o[r][j] = tm_mfma32x32x16<TM_DT_F16>(v, p[r][e], o[r][j]);
      }
    if constexpr (NV > 0) tm_kv8_load<NV>(a.c.v, w, a.page_log2, lane, vf);
  }
  const bool patch = __syncthreads_or(seen_nan) != 0;  // (the queries are done with, too)
  float(*const obuf)[32][kChunk + 4] = reinterpret_cast<float(*)[32][kChunk + 4]>(lds);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (32 * r >= t.rows) break;
    const float total_w = l[r] + tm_other_half(l[r]), mw = m[r] + kRoom;  // (O stands for 2^kRoom times its sum)
    if (r > 0) __syncthreads();
    if (g == 0) join[wave][c] = make_float2(mw, total_w);
    __syncthreads();
    float top = -__builtin_huge_valf(), total = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) top = fmaxf(top, join[x][c].x);
    const float base = top == -__builtin_huge_valf() ? 0.f : top;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) total += scaled(join[x][c].y, join[x][c].x - base);
    const float f = __builtin_amdgcn_exp2f(mw - base);
    const int rows = t.rows - 32 * r < 32 ? t.rows - 32 * r : 32;
    if (wave == 0 && g == 0) {
      if (NV > 0) inv_s[c] = total == 0.f ? 0.f : __builtin_amdgcn_exp2f(-(float)kRoom) / total;
      if (c < rows) {
        const uint32_t row = t.r0 + 32 * r + c, token = token_of(a, row);
        const int64_t at = (t.s.first + token) * a.heads + head_of(row, token);
        if (NV == 0 || !whole) a.stats[at * a.cut.splits + split] = make_float2(top, total);
        else if (a.lse) a.lse[at] = total == 0.f ? -__builtin_huge_valf() : (top + __builtin_amdgcn_logf(total)) * kLn2;
      }
    }
    if constexpr (NV > 0) {
#pragma unroll
      for (int part = 0; part < DV / kChunk; ++part) {
        if (part) __syncthreads();
#pragma unroll
        for (int jj = 0; jj < kChunk / 32; ++jj)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const tm_f32x16 &v = o[r][part * (kChunk / 32) + jj];
            *reinterpret_cast<float4 *>(&obuf[wave][c][32 * jj + 2 * i + 4 * g]) =
                make_float4(v[i] * f, v[i + 1] * f, v[i + 2] * f, v[i + 3] * f);
          }
        __syncthreads();
        for (int e = threadIdx.x; e < rows * (kChunk / 8); e += kThreads) {
          const int rr = e / (kChunk / 8), col = e % (kChunk / 8) * 8;
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = 0.f;
#pragma unroll
          for (int x = 0; x < kWaves; ++x)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += obuf[x][rr][col + k];
          const uint32_t row = t.r0 + 32 * r + rr, token = token_of(a, row);
          if (patch) {  // the NaN that this row does see: columns of NaN
            const int64_t seen = visible(a, t.s, token);
            const int end = seen < (int64_t)n * 32 ? (int)seen : n * 32;
            for (int key = (seen_whole > t0 ? seen_whole : t0) * 32; key < end; ++key) {
              const Kv8Place at = place(key >> 5, page_of(key >> 5));
              if (!at.there) continue;
              const int in = key & 31;
              const uint8_t *const vb = static_cast<const uint8_t *>(a.c.v) +
                                        ((at.slot << (a.page_log2 - 5)) + at.tile) * (int64_t)(NV * 1024) +
                                        (in / 4 % 2) * 512 + in / 16 * 8 + in / 8 % 2 * 4 + in % 4;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int to = part * kChunk + col + k;
                if ((vb[to / 32 * 1024 + to % 32 * 16] & 0x7f) == 0x7f) v[k] = __builtin_nanf("");
              }
            }
          }
          if (whole) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= inv_s[rr];
            tm_store8<DT>(static_cast<T *>(a.out) + (t.s.first + token) * a.os_t + head_of(row, token) * a.os_h +
                              part * kChunk + col, v);
          } else {
            tm_store8<TM_DT_F32>(a.part + (((t.s.first + token) * a.heads + head_of(row, token)) * a.cut.splits + split) * DV +
                                     part * kChunk + col, v);
          }
        }
      }
    }
  }
}

// Joins the splits of rows: a workgroup takes a row at a time, a thread 4 columns of some splits, whose
// parts are requested together with the statistics.
template <int DT, int DV, int OWN>
__global__ __launch_bounds__(kThreads) void join_kernel(AttArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int kCols = DV / 4, kSets = kThreads / kCols;  // OWN: splits of a thread
  __shared__ float fac[kMaxSplits];
  __shared__ __align__(16) float4 red[kSets][kCols];
  const int h = blockIdx.y;
  const int col = threadIdx.x % kCols, set = threadIdx.x / kCols, lane = threadIdx.x & 63;
  float4 v[OWN];
  float2 s0, s1;
  auto request = [&](int64_t row) {  // (parts that were not written are read, not used)
    const float *const p = a.part + row * a.cut.splits * DV + col * 4;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int s = set + i * kSets;
      v[i] = *reinterpret_cast<const float4 *>(p + (int64_t)(s < a.cut.splits ? s : 0) * DV);
    }
    const float2 *const st = a.stats + row * a.cut.splits;
    s0 = st[lane < a.cut.splits ? lane : 0], s1 = st[lane + 64 < a.cut.splits ? lane + 64 : 0];
  };
  auto join = [&](int64_t tok, int64_t head, int n) {
    const float2 none = make_float2(-__builtin_huge_valf(), 0.f);
    const float2 x0 = lane < n ? s0 : none, x1 = lane + 64 < n ? s1 : none;
    const float top = tm_wave_max(fmaxf(x0.x, x1.x));
    const float base = top == -__builtin_huge_valf() ? 0.f : top;
    const float f0 = __builtin_amdgcn_exp2f(x0.x - base), f1 = __builtin_amdgcn_exp2f(x1.x - base);
    const float total = tm_wave_sum(scaled(x0.y, x0.x - base) + scaled(x1.y, x1.x - base));
    if (threadIdx.x < 64) {
      fac[lane] = f0;
      fac[lane + 64] = f1;
    }
    __syncthreads();
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (set < kSets) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int s = set + i * kSets;
        if (s < n) {
          const float f = fac[s];
          y.x = fmaf(v[i].x, f, y.x), y.y = fmaf(v[i].y, f, y.y), y.z = fmaf(v[i].z, f, y.z), y.w = fmaf(v[i].w, f, y.w);
        }
      }
      red[set][col] = y;
    }
    __syncthreads();
    if (set != 0) return;
#pragma unroll
    for (int s = 1; s < kSets; ++s) {
      const float4 x = red[s][col];
      y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
    }
    const float inv = total == 0.f ? 0.f : __builtin_amdgcn_exp2f(-(float)kRoom) / total;
    T o[4] = {Elem<DT>::from_f(y.x * inv), Elem<DT>::from_f(y.y * inv), Elem<DT>::from_f(y.z * inv), Elem<DT>::from_f(y.w * inv)};
    __builtin_memcpy(static_cast<T *>(a.out) + tok * a.os_t + head * a.os_h + col * 4, o, 8);
    if (a.lse && threadIdx.x == 0)
      a.lse[tok * a.heads + head] = total == 0.f ? -__builtin_huge_valf() : (top + __builtin_amdgcn_logf(total)) * kLn2;
  };
  auto parts = [](const RowTile &t) { return (int)((t.tiles + t.per - 1) / t.per); };
  RowTile t = {};
  if (a.early) {
    // Most rows have parts: they are on their way before the lists are read.
    const uint32_t tok = blockIdx.x / (uint32_t)a.groups, in = blockIdx.x - tok * a.groups;
    const int64_t head = h * a.groups + in;
    request((int64_t)tok * a.heads + head);
    int64_t at = 0;
    t.b = a.b.starts == nullptr ? tok : tm_kv8_unit(a.b, tok, 1, 1, 0, at);
    if (!tile_at(a, (at * a.groups + in) / 32, t) || at < 0 || at >= t.s.n || t.per >= t.tiles) return;
    join(tok, head, parts(t));
    return;
  }
  const bool any = a.rows == 64 ? row_tile<64>(a, blockIdx.x, t) : row_tile(a, blockIdx.x, t);
  if (!any || t.per >= t.tiles) return;
  for (int r = blockIdx.z; r < t.rows; r += gridDim.z) {
    const uint32_t rr = t.r0 + r, in = token_of(a, rr);
    const int64_t tok = t.s.first + in, head = h * a.groups + (rr - in * a.groups);
    request(tok * a.heads + head);
    if (r >= (int)gridDim.z) __syncthreads();  // (the row before is summed)
    join(tok, head, parts(t));
  }
}

// How a call is cut up: R x 32 rows a workgroup, at most `tiles` of these per key head, keys split `splits` times.
struct Plan {
  int r;
  Kv8Cut cut;
  int64_t tiles;
  bool turn;  // workgroups with work are not evenly spread
};
Plan plan_of(const tm_kv8_cache *c, const tm_kv8_batch *b, int groups) {
  const int64_t rows = b->n_tokens * groups, heads = c->n_kv_heads;
  Plan p = {1, {1, 4}, b->starts ? rows / 32 + b->n_seqs : b->n_seqs * tm_cdiv(groups, 32), false};
  const int64_t keys = (int64_t)b->max_pages * c->page_size / kKv8Tile;
  // workgroups that have rows, if the sequences have as many each
  const int64_t units = b->n_seqs > 0 ? b->n_seqs * tm_cdiv(tm_cdiv(rows, b->n_seqs), 32) * heads : 0;
  int64_t s = 1;
  // 64 rows a wave where that leaves four workgroups for each that a CU holds (32 heads on 4, us with 32 and 64 rows:
  // 2048 tokens 53, 58; 4099 173, 167; 8192 599, 554); wider values leave no registers for them
  if (b->starts && c->v_dim <= 128 && rows / 64 * heads >= 2048) {
    p.r = 2;
    p.tiles = rows / 64 + b->n_seqs;
  } else if (units > 0 && keys > 32) {
    // Up to 1024 keys (eight rounds of the four waves) one launch: a round is 0.7 us, joining parts 3 of the host's and 2
    // of the device's.  Then one workgroup per CU, from 4096 keys on two (32 heads on 4, one sequence, us by splits: 4000
    // keys 1 28, 4 13.6, 16 9.4; eight sequences of 4000: 1 29, 4 14.7, 8 11.9, 16 12.4).
    s = (keys <= 128 ? 256 : 512) / units;
    s = s < keys / kWaves ? s : keys / kWaves;
    s = s < 1 ? 1 : s;
  }
  // Sequences of one table may differ much: a part has about 4096 keys of the longest, from two workgroups per CU on
  // 8192, and a short sequence no more parts than above (32 heads on 4, us before and now: one of 65536 among 31 of 1000
  // keys 153, 60, among 127 434, 98, 31 of 65536 beside a prompt of 1024 tokens 707, 438; but 128 of 500 in a table of 65536
  // 16.7, 24, of 2000 46, 52).  Sequences whose rows fill the device stay whole (row_tile); the parts of all rows take
  // 512 MiB at most.
  int64_t most = keys / (units >= 512 ? 256 : 128);
  if (b->n_seqs > 1 && most > s) {
    const int64_t fit = ((int64_t)1 << 29) / (rows * heads * (c->v_dim + 2) * (int64_t)sizeof(float) + 1);
    most = most < fit ? most : fit;
    if (most > s) {
      p.cut.least = (int)(units >= 512 ? 64 : (units + 31) / 32 * 4);
      s = most;
    }
  }
  p.cut.splits = (int)(s > kMaxSplits ? kMaxSplits : s);
  // (Prompts are not turned: a head's tiles share an XCD's L2; three pieces of 1024 tokens of 16 heads 216 us, 244 turned.)
  p.turn = b->starts ? p.cut.splits == 1 && 2 * p.tiles * heads >= 3 * units : p.cut.least > 4;
  return p;
}

AttArgs args_of(const tm_kv8_cache *c, const tm_kv8_batch *b, const void *q, int64_t qs_t, int64_t qs_h, int n_heads,
                float scale, const Plan &p) {
  AttArgs a = {};
  a.c = *c;
  a.b = *b;
  a.q = q, a.qs_t = qs_t, a.qs_h = qs_h;
  a.scale = scale;
  a.heads = n_heads;
  a.groups = n_heads / c->n_kv_heads;
  a.cut = p.cut;
  a.page_log2 = c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  a.tiles1 = (int)tm_cdiv(a.groups, 32);
  a.rows = 32 * p.r;
  a.turn = p.turn;
  return a;
}

template <int DT, int D, int DV, int R>
void launch(const AttArgs &a, const Plan &p, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles * a.c.n_kv_heads * p.cut.splits));
  hipLaunchKernelGGL((attend_kernel<DT, D, DV, R>), grid, dim3(kThreads), 0, s, a);
}

}  // namespace

Kv8Cut tm_internal_kv8_cut(const tm_kv8_cache *c, const tm_kv8_batch *b, int groups) {
  return plan_of(c, b, groups).cut;
}
int tm_internal_kv8_stats(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t dtype, const void *q, int64_t qs_b,
                          int64_t qs_h, int32_t n_heads, float scale, float2 *stats, hipStream_t s) {
  const Plan p = plan_of(cache, batch, n_heads / cache->n_kv_heads);
  AttArgs a = args_of(cache, batch, q, qs_b, qs_h, n_heads, scale, p);
  a.stats = stats;
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    switch (cache->head_dim) {
      case 64: launch<DT, 64, 0, 1>(a, p, s); break;
      case 128: launch<DT, 128, 0, 1>(a, p, s); break;
      case 192: launch<DT, 192, 0, 1>(a, p, s); break;
      default: launch<DT, 256, 0, 1>(a, p, s); break;
    }
  };
  if (dtype == TM_DT_F16) run(std::integral_constant<int, TM_DT_F16>{});
  else run(std::integral_constant<int, TM_DT_BF16>{});
  TM_LAUNCH_CHECK("tm_kv8_importance(statistics)");
  return TM_OK;
}

extern "C" size_t tm_kv8_attention_workspace_size(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t n_heads) {
  if (!cache || !batch || n_heads < 1 || cache->n_kv_heads < 1 || n_heads % cache->n_kv_heads || batch->n_tokens <= 0)
    return 0;
  const int s = plan_of(cache, batch, n_heads / cache->n_kv_heads).cut.splits;
  if (s == 1) return 0;
  return (size_t)batch->n_tokens * n_heads * s * (cache->v_dim + 2) * sizeof(float) + 16;
}

extern "C" int tm_kv8_attention(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t dtype, const void *q,
                                int64_t qs_t, int64_t qs_h, int32_t n_heads, float scale, int32_t causal, void *out,
                                int64_t os_t, int64_t os_h, float *lse, void *workspace, size_t workspace_bytes,
                                tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE, "tm_kv8_attention: unsupported dtype tag %d",
             (int)dtype);
  const int bad = tm_kv8_check("tm_kv8_attention", cache, batch);
  if (bad != TM_OK) return bad;
  TM_REQUIRE(n_heads >= 1 && n_heads <= 4096 && n_heads % cache->n_kv_heads == 0, TM_EINVAL_SHAPE,
             "tm_kv8_attention: %d query heads on %d key heads", n_heads, cache->n_kv_heads);
  TM_REQUIRE(scale > 0.f && scale < __builtin_huge_valf(), TM_EINVAL_ARG, "tm_kv8_attention: scale must be positive and finite");
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return TM_OK;
  TM_REQUIRE(q && out, TM_EINVAL_ARG, "tm_kv8_attention: null pointer");
  if (batch->n_tokens == 1) qs_t = os_t = 0;  // (the stride of a single row means nothing)
  if (n_heads == 1) qs_h = os_h = 0;
  TM_REQUIRE(tm_aligned16(q) && tm_aligned16(out) && qs_t % 8 == 0 && qs_h % 8 == 0 && os_t % 8 == 0 && os_h % 8 == 0,
             TM_EINVAL_SHAPE, "tm_kv8_attention: rows of q and out must be 16-byte aligned, strides multiples of 8 elements");
  const int groups = n_heads / cache->n_kv_heads;
  const Plan p = plan_of(cache, batch, groups);
  TM_REQUIRE(p.tiles * cache->n_kv_heads * p.cut.splits < kKv8MaxGrid && batch->n_tokens * groups < ((int64_t)1 << 31), TM_EINVAL_SHAPE,
             "tm_kv8_attention: too many rows");
  const size_t need = tm_kv8_attention_workspace_size(cache, batch, n_heads);
  TM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && tm_aligned16(workspace)), TM_EWORKSPACE,
             "tm_kv8_attention: workspace %zu bytes < %zu", workspace_bytes, need);
  AttArgs a = args_of(cache, batch, q, qs_t, qs_h, n_heads, scale, p);
  if (cache->n_pages == 0) a.b.max_pages = 0;  // no page is there
  a.out = out, a.os_t = os_t, a.os_h = os_h;
  a.lse = lse;
  a.causal = causal != 0;
  a.part = static_cast<float *>(workspace);
  a.stats = reinterpret_cast<float2 *>(a.part + batch->n_tokens * n_heads * p.cut.splits * cache->v_dim);
  hipStream_t s = tm_hip_stream(stream);
  auto run = [&](auto dt, auto d, auto dv) {
    constexpr int DT = decltype(dt)::value, D = decltype(d)::value, DV = decltype(dv)::value;
    if constexpr (DV <= 128) {
      if (p.r == 2) launch<DT, D, DV, 2>(a, p, s);
      else launch<DT, D, DV, 1>(a, p, s);
    } else {
      launch<DT, D, DV, 1>(a, p, s);
    }
    TM_LAUNCH_CHECK("tm_kv8_attention");
    if (p.cut.splits > 1) {
      // A workgroup per row.  Where prompts may stay whole, two a tile (a workgroup that ends at once takes 1.2 ns: three
      // pieces of 1024 tokens on 30000 keys 1682 us with 32, 1632 with 2).
      const bool early = p.cut.least == 4;
      a.early = early;
      const dim3 grid((unsigned)(early ? batch->n_tokens * groups : p.tiles), (unsigned)cache->n_kv_heads,
                      early ? 1u : batch->starts ? 2u : (unsigned)(groups < 32 ? groups : 32));
      constexpr int kSets = kThreads / (DV / 4);
      if (p.cut.splits <= 4 * kSets) hipLaunchKernelGGL((join_kernel<DT, DV, 4>), grid, dim3(kThreads), 0, s, a);
      else hipLaunchKernelGGL((join_kernel<DT, DV, (kMaxSplits + kSets - 1) / kSets>), grid, dim3(kThreads), 0, s, a);
      TM_LAUNCH_CHECK("tm_kv8_attention(join)");
    }
    return TM_OK;
  };
  auto columns = [&](auto dt) {
    using std::integral_constant;
    if (cache->head_dim == 64) return run(dt, integral_constant<int, 64>{}, integral_constant<int, 64>{});
    if (cache->head_dim == 128) return run(dt, integral_constant<int, 128>{}, integral_constant<int, 128>{});
    if (cache->head_dim == 256) return run(dt, integral_constant<int, 256>{}, integral_constant<int, 256>{});
    if (cache->v_dim == 128) return run(dt, integral_constant<int, 192>{}, integral_constant<int, 128>{});
    return run(dt, integral_constant<int, 192>{}, integral_constant<int, 192>{});
  };
  if (dtype == TM_DT_F16) return columns(std::integral_constant<int, TM_DT_F16>{});
  return columns(std::integral_constant<int, TM_DT_BF16>{});
}
