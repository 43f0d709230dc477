// Attention over the 8-bit cache (layout: tm_kv8.h): tm_kv8_attention.
//
// Rows of a sequence are its (new token, query head of one key head) pairs, 32 a
// tile, so a key head's tile of keys serves all its query heads.  Per 32 keys:
//   S^T = K Q^T on the 16-bit instructions (a byte of K is exact in 16 bits), a
//   lane holding 16 keys of one row;  x = S^T sk scale log2(e) + log2(sv);
//   P = 2^(x - m) under a running reference m of the row, so that the values'
//   scale rides in P and V enters as the bytes stand;  O^T += V^T P.
// With l = sum P / sv the result is O / l and log sum exp = (m + log2 l) ln 2 (sv >=
// 2^-100: l stays in range).
// m is 2^8 under a running maximum of x and follows it only when that has grown by
// more than 2^6, so O is seldom scaled again and P lies in [0, 2^14].  P is rounded
// to fp16 for the second product whatever the queries' type, and V's bytes become
// fp16 (exact): half a step is 2^-12 of a probability, where bf16 would leave
// 2^-9 (an output's error against 64 bits 1.9e-3 of its size instead of 1.6e-3, which
// is its own rounding); what lies under 2^-33 of a row's largest is lost.  All
// sums are fp32.
//
// The four waves of a workgroup take every fourth tile of keys and join through
// LDS.  Where rows alone do not fill the device, the keys are split over
// workgroups as well, and a second launch joins their parts.
#include "tm_internal.h"
#include "tm_kv8_dev.h"

#include <type_traits>

namespace {

constexpr int kAttThreads = 256;
constexpr int kWaves = kAttThreads / 64;
constexpr int kMaxSplits = 128;
typedef float tm_f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 tm_f16x2 __attribute__((ext_vector_type(2)));

constexpr float kRoom = 8.f, kGrow = 6.f;  // log2 of a new maximum's P, of what it may grow by

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
  int32_t heads, groups, splits, page_log2, causal, tiles1;  // tiles1: row tiles of one token
};

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
__device__ __forceinline__ bool row_tile(const AttArgs &a, int64_t u, RowTile &t) {
  int64_t j = 0;
  uint32_t last = 0;  // the tile's last token
  if (a.b.starts == nullptr) {
    t.b = a.tiles1 == 1 ? (uint32_t)u : (uint32_t)u / (uint32_t)a.tiles1;
    j = u - t.b * a.tiles1;
  } else {
    t.b = tm_kv8_unit(a.b, u, a.groups, 32, 1, j);
  }
  t.s = tm_kv8_seq(a.b, t.b);
  const int64_t all = t.s.n * a.groups;
  if (j < 0 || j * 32 >= all) return false;
  t.r0 = (uint32_t)(j * 32);
  t.rows = (int)(all - t.r0 < 32 ? all - t.r0 : 32);
  if (a.b.starts != nullptr) last = (t.r0 + t.rows - 1) / (uint32_t)a.groups;
  t.end = visible(a, t.s, last);
  t.tiles = (t.end + 31) >> 5;
  t.per = a.splits == 1 ? t.tiles + 3 : tm_kv8_per(t.tiles, a.splits);
  return true;
}
// A row's token (of its sequence) and its head among the key head's.
__device__ __forceinline__ uint32_t token_of(const AttArgs &a, uint32_t row) {
  return a.b.starts == nullptr ? 0 : row / (uint32_t)a.groups;
}

// DV = 0: the statistics alone.
template <int DT, int D, int DV>
__global__ __launch_bounds__(kAttThreads, D + DV > 320 ? 1 : 2) void attend_kernel(AttArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int NK = D / 32, NV = DV / 32;
  constexpr int kChunk = 64;  // columns joined at a time
  __shared__ float2 join[kWaves][32];
  __shared__ __align__(16) float obuf[DV ? kWaves : 1][32][kChunk + 4];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int c = lane & 31, g = lane >> 5;
  const int h = blockIdx.y, split = blockIdx.z;
  RowTile t;
  if (!row_tile(a, gridDim.x - 1 - blockIdx.x, t)) return;  // the last tokens of a prompt see most: they go first
  const int64_t t0 = split * t.per, t1 = t0 + t.per < t.tiles ? t0 + t.per : t.tiles;
  if (t0 >= t1 && split > 0) return;
  const uint32_t row = t.r0 + (c < t.rows ? c : t.rows - 1);
  const uint32_t token = token_of(a, row);
  const int64_t call_row = (t.s.first + token) * a.heads + h * a.groups + (row - token * a.groups);
  const int64_t limit = visible(a, t.s, token), first_limit = visible(a, t.s, token_of(a, t.r0));

  uint4 qf[NK][2];
  {
    const T *const q = static_cast<const T *>(a.q) + (t.s.first + token) * a.qs_t +
                       (h * a.groups + (row - token * a.groups)) * a.qs_h + 16 * g;
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      qf[j][0] = *reinterpret_cast<const uint4 *>(q + 32 * j);
      qf[j][1] = *reinterpret_cast<const uint4 *>(q + 32 * j + 8);
    }
  }
  tm_f32x16 o[NV ? NV : 1];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[j][i] = 0.f;
  float m = -__builtin_huge_valf(), l = 0.f;
  const float unit = a.scale * kLog2e;

  auto step = [&](int64_t tile, const Kv8Place &w, const uint4 (&kf)[NK], uint4 (&vf)[NV ? NV : 1], float sk, float sv) {
    tm_f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      s = tm_mfma32x32x16<DT>(tm_kv8_operand<DT>(kf[j].x, kf[j].y), qf[j][0], s);
      s = tm_mfma32x32x16<DT>(tm_kv8_operand<DT>(kf[j].z, kf[j].w), qf[j][1], s);
    }
    const int64_t k0 = tile * 32;
    const bool edge = !w.there || k0 + 32 > first_limit;
    uint32_t nan_bytes = 0;
    if (edge) {
      const int64_t lim = w.there ? limit : 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int64_t key = k0 + 8 * (i / 4) + 4 * g + i % 4;
        s[i] = key < lim ? s[i] : -__builtin_huge_valf();
      }
      // a NaN among values that some row does not see stays out of the product
      if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          uint32_t *const p = reinterpret_cast<uint32_t *>(&vf[j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = p[e] & 0x7f7f7f7fu;
            const uint32_t n = (x + 0x01010101u) & 0x80808080u;  // 0x80 where a byte is 0x7f
            nan_bytes |= n;
            p[e] &= ~((n >> 7) * 0xffu);
          }
        }
      }
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    const float mul = (w.there ? sk : 1.f) * unit, add = w.there ? tm_exponent(sv) : 0.f;
    top = fmaf(top, mul, add);
    top = fmaxf(top, tm_other_half(top));
    if (__any(top > m + (kRoom + kGrow) || (m == -__builtin_huge_valf() && top > m))) {
      const float to = fmaxf(m, top - kRoom);
      const float f = m == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[j][i] *= f;
    }
    const float off = add - (m == -__builtin_huge_valf() ? 0.f : m);
    float sum = 0.f;
    uint32_t pf[8];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s[i], mul, off)), y = __builtin_amdgcn_exp2f(fmaf(s[i + 1], mul, off));
      sum += x + y;
      if constexpr (NV > 0) {
        pf[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(tm_f32x2{x, y}, tm_f16x2));
      }
    }
    l = fmaf(sum, __builtin_amdgcn_exp2f(-add - kRoom), l);
    if constexpr (NV > 0) {
      const uint4 p0 = make_uint4(pf[0], pf[1], pf[2], pf[3]), p1 = make_uint4(pf[4], pf[5], pf[6], pf[7]);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        o[j] = tm_mfma32x32x16<TM_DT_F16>(tm_kv8_operand<TM_DT_F16>(vf[j].x, vf[j].y), p0, o[j]);
        o[j] = tm_mfma32x32x16<TM_DT_F16>(tm_kv8_operand<TM_DT_F16>(vf[j].z, vf[j].w), p1, o[j]);
      }
      if (edge && __any(nan_bytes != 0)) {  // those that a row does see make its column NaN
        const uint8_t *const vb = static_cast<const uint8_t *>(a.c.v) +
                                  ((w.slot << (a.page_log2 - 5)) + w.tile) * (int64_t)(NV * 1024);
        const int64_t lim = w.there ? limit : 0;
        for (int key = 0; key < 32 && k0 + key < lim; ++key)
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int col = 8 * (i / 4) + 4 * g + i % 4;
              const uint8_t x = vb[j * 1024 + ((key / 4 % 2) * 32 + col) * 16 + key / 16 * 8 + key / 8 % 2 * 4 + key % 4];
              if ((x & 0x7f) == 0x7f) o[j][i] = __builtin_nanf("");
            }
      }
    }
  };

  const int64_t begin = t0 + wave;
  if (begin < t1) {
    uint4 ka[NK], va[NV ? NV : 1], kb[NK], vb[NV ? NV : 1];
    const int32_t *const pages = a.b.table + t.b * a.b.ld_table;
    auto page_of = [&](int64_t tile) { return tm_kv8_page(a.b, pages, tile < t1 ? tile : t1 - 1, a.page_log2); };
    auto fetch = [&](int64_t tile, int id, Kv8Place &w, uint4 (&kf)[NK], uint4 (&vf)[NV ? NV : 1], float &sk, float &sv) {
      w = tm_kv8_place(a.c, id, h, tile < t1 ? tile : t1 - 1, a.page_log2);
      tm_kv8_load<NK>(a.c.k, w, a.page_log2, lane, kf);
      if constexpr (NV > 0) tm_kv8_load<NV>(a.c.v, w, a.page_log2, lane, vf);
      sk = a.c.k_scale[w.slot];
      sv = NV ? a.c.v_scale[w.slot] : 1.f;
    };
    Kv8Place wa, wb;
    float ska, sva, skb, svb;
    int ida = page_of(begin), idb = page_of(begin + kWaves);
    fetch(begin, ida, wa, ka, va, ska, sva);
    for (int64_t tile = begin; tile < t1; tile += 2 * kWaves) {
      ida = page_of(tile + 2 * kWaves);
      fetch(tile + kWaves, idb, wb, kb, vb, skb, svb);
      step(tile, wa, ka, va, ska, sva);
      if (tile + kWaves >= t1) break;
      idb = page_of(tile + 3 * kWaves);
      fetch(tile + 2 * kWaves, ida, wa, ka, va, ska, sva);
      step(tile + kWaves, wb, kb, vb, skb, svb);
    }
  }
  l += tm_other_half(l);
  m += kRoom;  // (a P of 1 stands for 2^(x - m) now, O for 2^kRoom times its sum)
  if (g == 0) join[wave][c] = make_float2(m, l);
  __syncthreads();
  float top = -__builtin_huge_valf(), total = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, join[w][c].x);
  const float base = top == -__builtin_huge_valf() ? 0.f : top;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += join[w][c].y * __builtin_amdgcn_exp2f(join[w][c].x - base);
  const float f = __builtin_amdgcn_exp2f(m - base);
  const bool whole = t.per >= t.tiles;  // nothing to join with other workgroups
  if (wave == 0 && g == 0 && c < t.rows) {
    if (DV == 0 || !whole) a.stats[call_row * a.splits + split] = make_float2(top, total);
    if (whole && a.lse) a.lse[call_row] = total == 0.f ? -__builtin_huge_valf() : (top + __builtin_amdgcn_logf(total)) * kLn2;
  }
  if constexpr (NV > 0) {
    __shared__ float inv[32];
    if (wave == 0 && g == 0) inv[c] = total == 0.f ? 0.f : __builtin_amdgcn_exp2f(-kRoom) / total;
#pragma unroll
    for (int half = 0; half < DV / kChunk; ++half) {
#pragma unroll
      for (int jj = 0; jj < kChunk / 32; ++jj)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const tm_f32x16 &v = o[half * (kChunk / 32) + jj];
          *reinterpret_cast<float4 *>(&obuf[wave][c][32 * jj + 2 * i + 4 * g]) =
              make_float4(v[i] * f, v[i + 1] * f, v[i + 2] * f, v[i + 3] * f);
        }
      __syncthreads();
      for (int e = threadIdx.x; e < t.rows * (kChunk / 4); e += kAttThreads) {
        const int r = e / (kChunk / 4), col = e % (kChunk / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float4 x = *reinterpret_cast<const float4 *>(&obuf[w][r][col]);
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        }
        const uint32_t rr = t.r0 + r, tok = token_of(a, rr);
        const int64_t head = h * a.groups + (rr - tok * a.groups);
        const int to = half * kChunk + col;
        if (whole) {
          T y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = Elem<DT>::from_f(v[k] * inv[r]);
          __builtin_memcpy(static_cast<T *>(a.out) + (t.s.first + tok) * a.os_t + head * a.os_h + to, y, 8);
        } else {
          *reinterpret_cast<float4 *>(a.part + (((t.s.first + tok) * a.heads + head) * a.splits + split) * DV + to) =
              make_float4(v[0], v[1], v[2], v[3]);
        }
      }
      if (half + 1 < DV / kChunk) __syncthreads();
    }
  }
}

// Joins the splits of a row: a workgroup per row, a thread owning 4 columns of some splits, whose
// parts are requested together with the statistics.
template <int DT, int DV, int OWN>
__global__ __launch_bounds__(kAttThreads) void join_kernel(AttArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int kCols = DV / 4, kSets = kAttThreads / kCols;  // OWN: splits of a thread
  __shared__ float fac[kMaxSplits];
  __shared__ __align__(16) float4 red[kSets][kCols];
  const int h = blockIdx.y;
  RowTile t;
  if (!row_tile(a, blockIdx.x, t) || t.per >= t.tiles || (int)blockIdx.z >= t.rows) return;
  const int n = (int)((t.tiles + t.per - 1) / t.per);
  const uint32_t rr = t.r0 + blockIdx.z, tok = token_of(a, rr);
  const int64_t head = h * a.groups + (rr - tok * a.groups);
  const int64_t row = (t.s.first + tok) * a.heads + head;
  const int col = threadIdx.x % kCols, set = threadIdx.x / kCols, lane = threadIdx.x & 63;
  const float *const p = a.part + row * a.splits * DV + col * 4;
  float4 v[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int s = set + i * kSets;
    v[i] = *reinterpret_cast<const float4 *>(p + (int64_t)(s < n ? s : 0) * DV);
  }
  const float2 *const st = a.stats + row * a.splits;
  const float2 none = make_float2(-__builtin_huge_valf(), 0.f);
  const float2 x0 = lane < n ? st[lane] : none, x1 = lane + 64 < n ? st[lane + 64] : none;
  const float top = tm_wave_max(fmaxf(x0.x, x1.x));
  const float base = top == -__builtin_huge_valf() ? 0.f : top;
  const float f0 = __builtin_amdgcn_exp2f(x0.x - base), f1 = __builtin_amdgcn_exp2f(x1.x - base);
  const float total = tm_wave_sum(x0.y * f0 + x1.y * f1);
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
  const float inv = total == 0.f ? 0.f : __builtin_amdgcn_exp2f(-kRoom) / total;
  T o[4] = {Elem<DT>::from_f(y.x * inv), Elem<DT>::from_f(y.y * inv), Elem<DT>::from_f(y.z * inv), Elem<DT>::from_f(y.w * inv)};
  __builtin_memcpy(static_cast<T *>(a.out) + (t.s.first + tok) * a.os_t + head * a.os_h + col * 4, o, 8);
  if (a.lse && threadIdx.x == 0) a.lse[row] = total == 0.f ? -__builtin_huge_valf() : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

int page_log2(int page) { return page == 32 ? 5 : page == 64 ? 6 : 7; }

// Row tiles of a call (an upper bound), and the splits of the keys.
int64_t row_tiles(const tm_kv8_batch *b, int groups) {
  return b->starts ? b->n_tokens * groups / 32 + b->n_seqs : b->n_seqs * tm_cdiv(groups, 32);
}
int key_splits(const tm_kv8_cache *c, const tm_kv8_batch *b, int64_t tiles) {
  const int64_t units = tiles * c->n_kv_heads, keys = (int64_t)b->max_pages * c->page_size / 32;
  if (units <= 0) return 1;
  int64_t s = 512 / units;  // two workgroups per CU
  s = s < keys / 8 ? s : keys / 8;
  return (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
}

}  // namespace

int tm_internal_kv8_splits(const tm_kv8_cache *c, const tm_kv8_batch *b, int groups) {
  return key_splits(c, b, row_tiles(b, groups));
}
int tm_internal_kv8_stats(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t dtype, const void *q, int64_t qs_b,
                          int64_t qs_h, int32_t n_heads, float scale, float2 *stats, hipStream_t s) {
  AttArgs a = {};
  a.c = *cache;
  a.b = *batch;
  a.groups = n_heads / cache->n_kv_heads;
  const int64_t tiles = row_tiles(batch, a.groups);
  a.splits = key_splits(cache, batch, tiles);
  a.q = q, a.qs_t = qs_b, a.qs_h = qs_h;
  a.stats = stats;
  a.scale = scale;
  a.heads = n_heads;
  a.page_log2 = page_log2(cache->page_size);
  a.tiles1 = (int)tm_cdiv(a.groups, 32);
  const dim3 grid((unsigned)tiles, (unsigned)cache->n_kv_heads, (unsigned)a.splits);
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    switch (cache->head_dim) {
      case 64: hipLaunchKernelGGL((attend_kernel<DT, 64, 0>), grid, dim3(kAttThreads), 0, s, a); break;
      case 128: hipLaunchKernelGGL((attend_kernel<DT, 128, 0>), grid, dim3(kAttThreads), 0, s, a); break;
      case 192: hipLaunchKernelGGL((attend_kernel<DT, 192, 0>), grid, dim3(kAttThreads), 0, s, a); break;
      default: hipLaunchKernelGGL((attend_kernel<DT, 256, 0>), grid, dim3(kAttThreads), 0, s, a); break;
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
  const int s = key_splits(cache, batch, row_tiles(batch, n_heads / cache->n_kv_heads));
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
  AttArgs a = {};
  a.c = *cache;
  a.b = *batch;
  if (cache->n_pages == 0) a.b.max_pages = 0;  // no page is there
  a.groups = n_heads / cache->n_kv_heads;
  const int64_t tiles = row_tiles(batch, a.groups);
  TM_REQUIRE(batch->n_tokens * a.groups + 32 * batch->n_seqs < ((int64_t)1 << 31), TM_EINVAL_SHAPE,
             "tm_kv8_attention: too many rows");
  a.splits = key_splits(cache, batch, tiles);
  const size_t need = tm_kv8_attention_workspace_size(cache, batch, n_heads);
  TM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && tm_aligned16(workspace)), TM_EWORKSPACE,
             "tm_kv8_attention: workspace %zu bytes < %zu", workspace_bytes, need);
  a.q = q, a.qs_t = qs_t, a.qs_h = qs_h;
  a.out = out, a.os_t = os_t, a.os_h = os_h;
  a.lse = lse;
  const int64_t rows = batch->n_tokens * n_heads * a.splits;
  a.part = static_cast<float *>(workspace);
  a.stats = reinterpret_cast<float2 *>(a.part + rows * cache->v_dim);
  a.scale = scale;
  a.heads = n_heads;
  a.page_log2 = page_log2(cache->page_size);
  a.causal = causal != 0;
  a.tiles1 = (int)tm_cdiv(a.groups, 32);
  hipStream_t s = tm_hip_stream(stream);
  auto run = [&](auto dt, auto d, auto dv) {
    constexpr int DT = decltype(dt)::value, D = decltype(d)::value, DV = decltype(dv)::value;
    hipLaunchKernelGGL((attend_kernel<DT, D, DV>), dim3((unsigned)tiles, (unsigned)cache->n_kv_heads, (unsigned)a.splits),
                       dim3(kAttThreads), 0, s, a);
    TM_LAUNCH_CHECK("tm_kv8_attention");
    if (a.splits > 1) {
      // (rows of a tile: one token's heads, or 32 of several tokens)
      const dim3 grid((unsigned)tiles, (unsigned)cache->n_kv_heads, (unsigned)(!batch->starts && a.groups < 32 ? a.groups : 32));
      constexpr int kSets = kAttThreads / (DV / 4);
      if (a.splits <= 4 * kSets) hipLaunchKernelGGL((join_kernel<DT, DV, 4>), grid, dim3(kAttThreads), 0, s, a);
      else hipLaunchKernelGGL((join_kernel<DT, DV, (kMaxSplits + kSets - 1) / kSets>), grid, dim3(kAttThreads), 0, s, a);
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
