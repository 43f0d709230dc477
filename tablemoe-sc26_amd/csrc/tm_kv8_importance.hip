// Importance over the 8-bit cache: tm_kv8_importance.
//
// out[t] = 1/H sum over heads of exp(scale q_h . k_t - lse_h): with the rows'
// log sum exp at hand (from the attention of the same query, or from a first
// launch that reads K for the statistics alone) K is read once and nothing is
// kept between.  Per 32 keys and key head one 32x32 product S = Q K^T, rows =
// that head's queries: a lane has 16 rows of one key and adds them itself.  The
// waves of a workgroup take the key heads and tiles of its keys between them and
// join through LDS in a fixed order.
//
// Written by position of each sequence, or by row of the call's new tokens (the
// last positions of each sequence): then only these tokens' tiles are computed.
//
// Bound by HBM and the last cache: 131071 keys of 4 heads of 128 (67 MB) with the log sum exp at hand
// 13.7 us, 4.9 TB/s, a large copy's rate; 4099 keys without it 5.5 + 5.3 us, two launches of a few memory
// round trips each (averages under the profiler).
#include "tm_internal.h"
#include "tm_kv8_dev.h"

#include <type_traits>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxHeads = 256;
constexpr int kMaxPer = 16;  // tiles of a workgroup

struct ImpArgs {
  tm_kv8_cache c;
  tm_kv8_batch b;
  const void *q;
  int64_t qs_b, qs_h;
  const float *lse;
  int64_t ld_lse;
  const float2 *stats;
  float *out;
  int64_t ld_out, out_len;
  float scale;
  Kv8Cut cut;
  int32_t heads, groups, page_log2, per, head_waves, lanes_log2;
};

// BY_ROW: `out` by row of the new tokens (a form of its own: by position a lane then has 128 registers and a SIMD four
// waves, 131071 keys 13.6 us, with both in one 15.1).
template <int DT, int D, bool BY_ROW>
__global__ __launch_bounds__(kThreads) void importance_kernel(ImpArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int NK = D / 32;
  __shared__ float norm[kMaxHeads];                // the rows' log2 sum exp
  __shared__ float acc[kWaves][kMaxPer][32];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c = lane & 31, g = lane >> 5;
  int64_t b = blockIdx.y;
  int tile0 = (int)(blockIdx.x * a.per);
  Kv8Seq s = {};
  if constexpr (BY_ROW) {
    // a sequence of n new tokens touches at most (n - 2) / 32 + 2 tiles: at most n / (32 per) + 2 workgroups
    int64_t j = 0;
    b = blockIdx.x;
    if (a.b.starts != nullptr) b = tm_kv8_unit(a.b, blockIdx.x, 1, 32 * a.per, 2, j);
    s = tm_kv8_seq(a.b, b);
    const int64_t old = s.len - s.n, at = ((old > 0 ? old : 0) >> 5) + j * a.per;
    if (j < 0 || s.n == 0 || at * 32 >= s.len) return;
    tile0 = (int)at;
  }
  const int64_t cap = (int64_t)a.b.max_pages << a.page_log2;
  int64_t len = a.b.lengths[b];
  len = len < 0 ? 0 : len < cap ? len : cap;
  const int tiles = (int)((len + 31) >> 5);
  const int end = tile0 + a.per < tiles ? tile0 + a.per : tiles;  // tiles to compute
  if (tile0 < tiles) {
    if (a.lse != nullptr) {
      if (tid < a.heads) norm[tid] = a.lse[b * a.ld_lse + tid] * kLog2e;
    } else {
      const int lanes = 1 << a.lanes_log2, at = tid & (lanes - 1);
      const int used = (int)((tiles + tm_kv8_per(tiles, a.cut) - 1) / tm_kv8_per(tiles, a.cut));
      for (int h0 = 0; h0 < a.heads; h0 += kThreads >> a.lanes_log2) {
        const int h = h0 + (tid >> a.lanes_log2);
        const float2 *const st = a.stats + (b * a.heads + (h < a.heads ? h : a.heads - 1)) * a.cut.splits;
        float m = -__builtin_huge_valf(), l = 0.f;
        for (int s = at; s < used; s += lanes) {
          const float2 x = st[s];
          const float to = fmaxf(m, x.x), base = to == -__builtin_huge_valf() ? 0.f : to;
          l = l * __builtin_amdgcn_exp2f(m - base) + x.y * __builtin_amdgcn_exp2f(x.x - base);
          m = to;
        }
        for (int o = 1; o < lanes; o <<= 1) {
          const float om = __shfl_xor(m, o, 64), ol = __shfl_xor(l, o, 64);
          const float to = fmaxf(m, om), base = to == -__builtin_huge_valf() ? 0.f : to;
          l = l * __builtin_amdgcn_exp2f(m - base) + ol * __builtin_amdgcn_exp2f(om - base);
          m = to;
        }
        if (at == 0 && h < a.heads) norm[h] = m + __builtin_amdgcn_logf(l);
      }
    }
  }
  for (int i = tid; i < kWaves * kMaxPer * 32; i += kThreads) (&acc[0][0][0])[i] = 0.f;
  __syncthreads();

  const int hw = a.head_waves;  // waves that share a tile's heads
  const int my_head = wave % hw, my_tile = wave / hw, tile_waves = kWaves / hw;
  const float unit = a.scale * kLog2e;
  if (tile0 + my_tile < end)
    for (int h = my_head; h < a.c.n_kv_heads; h += hw)
      for (int r0 = 0; r0 < a.groups; r0 += 32) {
        uint4 qf[NK][2];
        const int row = r0 + c < a.groups ? r0 + c : a.groups - 1;
        const T *const q = static_cast<const T *>(a.q) + b * a.qs_b + (h * a.groups + row) * a.qs_h + 16 * g;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          qf[j][0] = *reinterpret_cast<const uint4 *>(q + 32 * j);
          qf[j][1] = *reinterpret_cast<const uint4 *>(q + 32 * j + 8);
        }
        float nr[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = r0 + 8 * (i / 4) + 4 * g + i % 4;
          nr[i] = norm[h * a.groups + (r < a.groups ? r : a.groups - 1)];
        }
        const int32_t *const pages = a.b.table + b * a.b.ld_table;
        auto page_of = [&](int tile) { return tm_kv8_page(a.b, pages, tile < end ? tile : end - 1, a.page_log2); };
        auto place = [&](int tile, int id) { return tm_kv8_place(a.c, id, h, tile < end ? tile : end - 1, a.page_log2); };
        uint4 kf[NK];
        Kv8Place w = place(tile0 + my_tile, page_of(tile0 + my_tile));
        int id = page_of(tile0 + my_tile + tile_waves);
        tm_kv8_load<NK>(a.c.k, w, a.page_log2, lane, kf);
        float sk = a.c.k_scale[w.slot];
#pragma unroll 1
        for (int tile = tile0 + my_tile; tile < end; tile += tile_waves) {
          tm_f32x16 s;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
          for (int j = 0; j < NK; ++j) {
            s = tm_mfma32x32x16<DT>(qf[j][0], tm_kv8_operand<DT>(kf[j].x, kf[j].y), s);
            s = tm_mfma32x32x16<DT>(qf[j][1], tm_kv8_operand<DT>(kf[j].z, kf[j].w), s);
          }
          const bool there = w.there;
          const float mul = there ? sk * unit : unit;
          w = place(tile + tile_waves, id);
          id = page_of(tile + 2 * tile_waves);
          tm_kv8_load<NK>(a.c.k, w, a.page_log2, lane, kf);
          sk = a.c.k_scale[w.slot];
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i], mul, -nr[i]));
            sum += r0 + 8 * (i / 4) + 4 * g + i % 4 < a.groups ? p : 0.f;
          }
          sum += tm_other_half(sum);
          if (g == 0 && there) acc[wave][tile - tile0][c] += sum;
        }
      }
  __syncthreads();
  for (int i = tid; i < a.per * 32; i += kThreads) {
    const int64_t t = (int64_t)tile0 * 32 + i;
    if (BY_ROW ? t >= s.len : t >= a.out_len) break;
    if (BY_ROW && t < s.len - s.n) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += acc[w][i >> 5][i & 31];
    a.out[BY_ROW ? s.first + t - (s.len - s.n) : b * a.ld_out + t] = t < len ? v / (float)a.heads : 0.f;
  }
}

}  // namespace

extern "C" size_t tm_kv8_importance_workspace_size(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t n_heads) {
  if (!cache || !batch || n_heads < 1 || cache->n_kv_heads < 1 || n_heads % cache->n_kv_heads || batch->n_seqs <= 0)
    return 0;
  tm_kv8_batch one = *batch;
  one.starts = nullptr;
  one.n_tokens = one.n_seqs;
  return (size_t)batch->n_seqs * n_heads * tm_internal_kv8_cut(cache, &one, n_heads / cache->n_kv_heads).splits * sizeof(float2);
}

// What the entry points share: `batch` has starts only where out goes by row.
static int importance(const char *what, const tm_kv8_cache *cache, const tm_kv8_batch *batch, bool by_row, int32_t dtype,
                      const void *q, int64_t qs_b, int64_t qs_h, int32_t n_heads, float scale, const float *lse,
                      int64_t ld_lse, int64_t out_len, float *out, int64_t ld_out, void *workspace,
                      size_t workspace_bytes, tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE, "%s: unsupported dtype tag %d", what, (int)dtype);
  const int bad = tm_kv8_check(what, cache, batch);
  if (bad != TM_OK) return bad;
  tm_kv8_batch one = *batch;  // one query per sequence
  one.starts = nullptr;
  one.n_tokens = one.n_seqs;
  TM_REQUIRE(n_heads >= 1 && n_heads <= kMaxHeads && n_heads % cache->n_kv_heads == 0, TM_EINVAL_SHAPE,
             "%s: %d query heads (at most %d) on %d key heads", what, n_heads, kMaxHeads, cache->n_kv_heads);
  TM_REQUIRE(scale > 0.f && scale < __builtin_huge_valf(), TM_EINVAL_ARG, "%s: scale must be positive and finite", what);
  TM_REQUIRE(out_len >= 0 && out_len < ((int64_t)1 << 31) && ld_out >= out_len && batch->n_seqs < 65536 &&
                 (lse == nullptr || ld_lse >= n_heads),
             TM_EINVAL_SHAPE, "%s: bad sizes (out_len %lld, %lld sequences)", what, (long long)out_len,
             (long long)batch->n_seqs);
  if (batch->n_seqs == 0 || out_len == 0) return TM_OK;
  TM_REQUIRE(q && out, TM_EINVAL_ARG, "%s: null pointer", what);
  if (batch->n_seqs == 1) qs_b = 0;  // (the stride of a single row means nothing)
  if (n_heads == 1) qs_h = 0;
  TM_REQUIRE(tm_aligned16(q) && qs_b % 8 == 0 && qs_h % 8 == 0, TM_EINVAL_SHAPE,
             "%s: rows of q must be 16-byte aligned, strides multiples of 8 elements", what);
  ImpArgs a = {};
  a.c = *cache;
  if (cache->n_pages == 0) one.max_pages = 0;
  a.b = one;
  if (by_row) a.b.starts = batch->starts, a.b.n_tokens = batch->n_tokens;
  a.groups = n_heads / cache->n_kv_heads;
  hipStream_t s = tm_hip_stream(stream);
  a.cut = tm_internal_kv8_cut(cache, &one, a.groups);
  if (lse == nullptr) {
    const size_t need = tm_kv8_importance_workspace_size(cache, batch, n_heads);
    TM_REQUIRE(workspace && workspace_bytes >= need && tm_aligned16(workspace), TM_EWORKSPACE,
               "%s: workspace %zu bytes < %zu", what, workspace_bytes, need);
    a.stats = static_cast<const float2 *>(workspace);
    const int st = tm_internal_kv8_stats(cache, &one, dtype, q, qs_b, qs_h, n_heads, scale,
                                         static_cast<float2 *>(workspace), s);
    if (st != TM_OK) return st;
  }
  a.q = q, a.qs_b = qs_b, a.qs_h = qs_h;
  a.lse = lse, a.ld_lse = ld_lse;
  a.out = out, a.ld_out = ld_out, a.out_len = out_len;
  a.scale = scale;
  a.heads = n_heads;
  a.page_log2 = cache->page_size == 32 ? 5 : cache->page_size == 64 ? 6 : 7;
  a.head_waves = cache->n_kv_heads >= 4 ? 4 : cache->n_kv_heads >= 2 ? 2 : 1;
  while (a.lanes_log2 < 6 && (kThreads >> (a.lanes_log2 + 1)) >= n_heads) ++a.lanes_log2;
  const int64_t tiles = tm_cdiv(out_len, 32);
  int64_t per = tm_cdiv(by_row ? tiles + one.n_seqs : tiles * one.n_seqs, 1024);
  const int tile_waves = kWaves / a.head_waves;
  per = tm_cdiv(per, tile_waves) * tile_waves;
  a.per = (int)(per > kMaxPer ? kMaxPer : per);
  const dim3 grid = !by_row ? dim3((unsigned)tm_cdiv(tiles, a.per), (unsigned)one.n_seqs)
                            : dim3((unsigned)(batch->starts ? out_len / (32 * a.per) + 2 * one.n_seqs : one.n_seqs));
  auto run = [&](auto dt, auto rows) {
    constexpr int DT = decltype(dt)::value;
    constexpr bool ROWS = decltype(rows)::value;
    switch (cache->head_dim) {
      case 64: hipLaunchKernelGGL((importance_kernel<DT, 64, ROWS>), grid, dim3(kThreads), 0, s, a); break;
      case 128: hipLaunchKernelGGL((importance_kernel<DT, 128, ROWS>), grid, dim3(kThreads), 0, s, a); break;
      case 192: hipLaunchKernelGGL((importance_kernel<DT, 192, ROWS>), grid, dim3(kThreads), 0, s, a); break;
      default: hipLaunchKernelGGL((importance_kernel<DT, 256, ROWS>), grid, dim3(kThreads), 0, s, a); break;
    }
  };
  auto type = [&](auto rows) {
    if (dtype == TM_DT_F16) run(std::integral_constant<int, TM_DT_F16>{}, rows);
    else run(std::integral_constant<int, TM_DT_BF16>{}, rows);
  };
  if (by_row) type(std::true_type{});
  else type(std::false_type{});
  TM_LAUNCH_CHECK(what);
  return TM_OK;
}

extern "C" int tm_kv8_importance(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t dtype, const void *q,
                                 int64_t qs_b, int64_t qs_h, int32_t n_heads, float scale, const float *lse,
                                 int64_t ld_lse, int64_t out_len, float *out, int64_t ld_out, void *workspace,
                                 size_t workspace_bytes, tm_stream_t stream) {
  TM_REQUIRE(cache && batch, TM_EINVAL_ARG, "tm_kv8_importance: null pointer");
  tm_kv8_batch one = *batch;
  one.starts = nullptr;
  return importance("tm_kv8_importance", cache, &one, false, dtype, q, qs_b, qs_h, n_heads, scale, lse, ld_lse, out_len,
                    out, ld_out, workspace, workspace_bytes, stream);
}

extern "C" int tm_kv8_importance_rows(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t dtype, const void *q,
                                      int64_t qs_b, int64_t qs_h, int32_t n_heads, float scale, const float *lse,
                                      int64_t ld_lse, float *out, void *workspace, size_t workspace_bytes,
                                      tm_stream_t stream) {
  TM_REQUIRE(cache && batch, TM_EINVAL_ARG, "tm_kv8_importance_rows: null pointer");
  return importance("tm_kv8_importance_rows", cache, batch, true, dtype, q, qs_b, qs_h, n_heads, scale, lse, ld_lse,
                    batch->n_tokens, out, batch->n_tokens, workspace, workspace_bytes, stream);
}
