// Writing into the 8-bit cache (layout and batch: tm_kv8.h): tm_kv8_append.
//
// A workgroup owns one page that a sequence writes to, one key head, and its K
// or V: the maximum of the new rows, the scale, the bytes.  Where the page held
// tokens before, its scale can only rise; what they hold is then rounded again.
#include "tm_kv8.h"
#include "tm_internal.h"

#include <type_traits>

namespace {

constexpr int kAppThreads = 256;

struct AppArgs {
  tm_kv8_cache c;
  tm_kv8_batch b;
  const void *src[2];
  int64_t s_t[2], s_h[2];
};

// Four e4m3 values times a power of two, rounded.
__device__ __forceinline__ uint32_t rescale4(uint32_t v, float f) {
  const float a = __builtin_amdgcn_cvt_f32_fp8((int)v, 0), b = __builtin_amdgcn_cvt_f32_fp8((int)v, 1);
  const float c = __builtin_amdgcn_cvt_f32_fp8((int)v, 2), d = __builtin_amdgcn_cvt_f32_fp8((int)v, 3);
  return tm_fp8_pack4(a * f, b * f, c * f, d * f);
}
__device__ __forceinline__ uint4 rescale16(uint4 v, float f) {
  return make_uint4(rescale4(v.x, f), rescale4(v.y, f), rescale4(v.z, f), rescale4(v.w, f));
}

// K: the rows [lo, hi) of the page from src (row 0 = the page's first token), the rows before lo times f.
template <int DT, int D>
__device__ void write_k(const typename Elem<DT>::T *src, int64_t s_t, int lo, int hi, float inv, float f,
                        uint8_t *__restrict__ page) {
  constexpr int kPieces = D / 16;  // of 16 columns
  auto at = [&](int row, int p) {
    return reinterpret_cast<uint4 *>(page + ((int64_t)(row >> 5) * (D / 32) + (p >> 1)) * 1024 + (p & 1) * 512 + (row & 31) * 16);
  };
  if (f != 1.f)
    for (int i = threadIdx.x; i < lo * kPieces; i += kAppThreads) {
      uint4 *const w = at(i / kPieces, i % kPieces);
      *w = rescale16(*w, f);
    }
  for (int i = threadIdx.x; i < (hi - lo) * kPieces; i += kAppThreads) {
    const int row = lo + i / kPieces, p = i % kPieces;
    float a[8], b[8];
    tm_load8<DT>(src + row * s_t + p * 16, a);
    tm_load8<DT>(src + row * s_t + p * 16 + 8, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = tm_fp8_quot(a[e], inv);
      b[e] = tm_fp8_quot(b[e], inv);
    }
    *at(row, p) = make_uint4(tm_fp8_pack4(a[0], a[1], a[2], a[3]), tm_fp8_pack4(a[4], a[5], a[6], a[7]),
                             tm_fp8_pack4(b[0], b[1], b[2], b[3]), tm_fp8_pack4(b[4], b[5], b[6], b[7]));
  }
}

// V: a thread's 16 bytes hold 16 tokens of one column.
template <int DT, int D>
__device__ void write_v(const typename Elem<DT>::T *src, int64_t s_t, int lo, int hi, float inv, float f,
                        uint8_t *__restrict__ page) {
  const int t0 = f != 1.f ? 0 : lo >> 5, t1 = (hi + 31) >> 5;
  for (int i = threadIdx.x; i < (t1 - t0) * D * 2; i += kAppThreads) {
    const int tile = t0 + i / (D * 2), lane = i & 63, col = (i % (D * 2) >> 6) * 32 + (lane & 31), g = lane >> 5;
    const int first = tile * 32 + 4 * g;  // byte e: token first + 16 (e / 8) + 8 (e / 4 % 2) + e % 4
    uint4 *const w = reinterpret_cast<uint4 *>(page + ((int64_t)tile * (D / 32) + (col >> 5)) * 1024 + lane * 16);
    // the tokens of this piece: [first, first + 28)
    const bool whole = first >= lo && first + 28 <= hi;
    if (!whole && (first >= hi || (first + 28 <= lo && f == 1.f))) continue;
    uint4 old = make_uint4(0, 0, 0, 0);
    if (!whole) old = *w;
    uint32_t r[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int tq = first + 8 * q;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = tq + e;
        v[e] = t >= lo && t < hi ? tm_fp8_quot(Elem<DT>::to_f(src[t * s_t + col]), inv) : 0.f;
      }
      const uint32_t now = tm_fp8_pack4(v[0], v[1], v[2], v[3]);
      const uint32_t was = f != 1.f ? rescale4(r[q], f) : r[q];
      uint32_t out = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = tq + e;
        out |= (t < lo ? was : t < hi ? now : r[q]) & (0xffu << (8 * e));
      }
      r[q] = out;
    }
    *w = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

template <int DT, int D, bool V>
__device__ void write_page(const typename Elem<DT>::T *src, int64_t s_t, int lo, int hi, uint8_t *page, float *scale) {
  __shared__ uint32_t top[kAppThreads / 64];
  constexpr int kVecs = D / 8;
  uint32_t m = 0;
  for (int i = threadIdx.x; i < (hi - lo) * kVecs; i += kAppThreads) {
    float v[8];
    tm_load8<DT>(src + (lo + i / kVecs) * s_t + i % kVecs * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = tm_fp8_amax(m, v[e]);
  }
  const float before = *scale;
  m = tm_wave_max_u32(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();  // (every thread has read the scale)
  m = max(max(top[0], top[1]), max(top[2], top[3]));
  float inv;
  float s = fmaxf(tm_fp8_scale(m, inv), kKv8MinScale);
  float f = 1.f;
  if (lo > 0) {
    if (before > s) s = before;
    else f = before / s;  // powers of two
  }
  inv = 1.f / s;
  if (threadIdx.x == 0) *scale = s;
  if constexpr (V) write_v<DT, D>(src, s_t, lo, hi, inv, f, page);
  else write_k<DT, D>(src, s_t, lo, hi, inv, f, page);
}

template <int DT, int D, int DV>
__global__ __launch_bounds__(kAppThreads) void append_kernel(AppArgs a) {
  using T = typename Elem<DT>::T;
  const int h = blockIdx.y;
  const bool vals = blockIdx.z != 0;
  const int page = a.c.page_size;
  int64_t b = blockIdx.x, j = 0;
  if (a.b.starts != nullptr) b = tm_kv8_unit(a.b, blockIdx.x, 1, page, 2, j);
  const Kv8Seq s = tm_kv8_seq(a.b, b);
  if (j < 0 || s.n == 0) return;
  const int64_t old = s.len - s.n;  // position of the first new token
  const int64_t p = (old > 0 ? old / page : 0) + j;
  const int64_t p0 = p * page;
  if (p >= a.b.max_pages || p0 >= s.len) return;
  const int64_t id = a.b.table[b * a.b.ld_table + p];
  if (id < 0 || id >= a.c.n_pages) return;
  const int lo = (int)(old > p0 ? old - p0 : 0), hi = (int)(s.len - p0 < page ? s.len - p0 : page);
  const int64_t row0 = s.first + p0 - old;  // the page's first token as a row (before the new ones: not read)
  const int64_t at = id * a.c.n_kv_heads + h;
  if (vals) {
    const T *const src = static_cast<const T *>(a.src[1]) + row0 * a.s_t[1] + h * a.s_h[1];
    write_page<DT, DV, true>(src, a.s_t[1], lo, hi, static_cast<uint8_t *>(a.c.v) + at * page * DV, a.c.v_scale + at);
  } else {
    const T *const src = static_cast<const T *>(a.src[0]) + row0 * a.s_t[0] + h * a.s_h[0];
    write_page<DT, D, false>(src, a.s_t[0], lo, hi, static_cast<uint8_t *>(a.c.k) + at * page * D, a.c.k_scale + at);
  }
}

}  // namespace

int tm_kv8_check(const char *what, const tm_kv8_cache *c, const tm_kv8_batch *b) {
  TM_REQUIRE(c && b, TM_EINVAL_ARG, "%s: null pointer", what);
  const int d = c->head_dim, dv = c->v_dim;
  TM_REQUIRE(c->n_pages >= 0 && c->n_pages < ((int64_t)1 << 31) && c->n_kv_heads >= 1 && c->n_kv_heads <= 1024 &&
                 (c->page_size == 32 || c->page_size == 64 || c->page_size == 128),
             TM_EINVAL_SHAPE, "%s: bad cache (%lld pages of %d tokens, %d heads)", what, (long long)c->n_pages,
             c->page_size, c->n_kv_heads);
  TM_REQUIRE((d == dv && (d == 64 || d == 128 || d == 192 || d == 256)) || (d == 192 && dv == 128), TM_EINVAL_SHAPE,
             "%s: columns (%d, %d) not in (64, 64), (128, 128), (192, 128), (192, 192), (256, 256)", what, d, dv);
  TM_REQUIRE(b->n_seqs >= 0 && b->n_seqs < ((int64_t)1 << 24) && b->n_tokens >= 0 && b->n_tokens < ((int64_t)1 << 31) &&
                 b->max_pages >= 0 && b->max_pages < (1 << 24) && b->ld_table >= b->max_pages &&
                 (b->starts != nullptr || b->n_tokens == b->n_seqs),
             TM_EINVAL_SHAPE, "%s: bad batch (%lld sequences, %lld tokens, %d pages)", what, (long long)b->n_seqs,
             (long long)b->n_tokens, b->max_pages);
  if (b->n_seqs == 0) return TM_OK;
  TM_REQUIRE((c->n_pages == 0 || (c->k && c->v && c->k_scale && c->v_scale)) && b->lengths &&
                 (b->table || b->max_pages == 0),
             TM_EINVAL_ARG, "%s: null pointer", what);
  TM_REQUIRE(tm_aligned16(c->k) && tm_aligned16(c->v), TM_EINVAL_SHAPE, "%s: k and v must be 16-byte aligned", what);
  return TM_OK;
}

extern "C" int tm_kv8_append(const tm_kv8_cache *cache, const tm_kv8_batch *batch, int32_t dtype, const void *k,
                             int64_t ks_t, int64_t ks_h, const void *v, int64_t vs_t, int64_t vs_h, tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F32 || dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE,
             "tm_kv8_append: unsupported dtype tag %d", (int)dtype);
  const int bad = tm_kv8_check("tm_kv8_append", cache, batch);
  if (bad != TM_OK) return bad;
  if (batch->n_tokens == 0 || batch->n_seqs == 0 || cache->n_pages == 0 || batch->max_pages == 0) return TM_OK;
  TM_REQUIRE(k && v, TM_EINVAL_ARG, "tm_kv8_append: null pointer");
  TM_REQUIRE(tm_aligned16(k) && tm_aligned16(v) && ks_t % 8 == 0 && ks_h % 8 == 0 && vs_t % 8 == 0 && vs_h % 8 == 0,
             TM_EINVAL_SHAPE, "tm_kv8_append: rows of k and v must be 16-byte aligned, strides multiples of 8 elements");
  AppArgs a = {*cache, *batch, {k, v}, {ks_t, vs_t}, {ks_h, vs_h}};
  // a sequence of n new tokens touches at most (n - 2) / page + 2 pages
  const int64_t units = batch->starts ? batch->n_tokens / cache->page_size + 2 * batch->n_seqs : batch->n_seqs;
  TM_REQUIRE(units < ((int64_t)1 << 31), TM_EINVAL_SHAPE, "tm_kv8_append: too many pages");
  const dim3 grid((unsigned)units, (unsigned)cache->n_kv_heads, 2);
  hipStream_t s = tm_hip_stream(stream);
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    auto launch = [&](auto d, auto dv) {
      hipLaunchKernelGGL((append_kernel<DT, decltype(d)::value, decltype(dv)::value>), grid, dim3(kAppThreads), 0, s, a);
    };
    using std::integral_constant;
    if (cache->head_dim == 64) launch(integral_constant<int, 64>{}, integral_constant<int, 64>{});
    else if (cache->head_dim == 128) launch(integral_constant<int, 128>{}, integral_constant<int, 128>{});
    else if (cache->head_dim == 256) launch(integral_constant<int, 256>{}, integral_constant<int, 256>{});
    else if (cache->v_dim == 128) launch(integral_constant<int, 192>{}, integral_constant<int, 128>{});
    else launch(integral_constant<int, 192>{}, integral_constant<int, 192>{});
    TM_LAUNCH_CHECK("tm_kv8_append");
    return TM_OK;
  });
}
