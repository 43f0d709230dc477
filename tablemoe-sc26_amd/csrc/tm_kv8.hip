// Writing into the 8-bit cache (layout and batch: tm_kv8.h): tm_kv8_append.
//
// A workgroup owns one page that a sequence writes to, one key head, and its K
// or V: the maximum of the new rows, the scale, the bytes.  Where the page held
// tokens before, its scale can only rise; what they hold is then rounded again.
// (A scale per token would need no such rounding and a scale for every key in the
// attention's inner loop.)
//
// Bound by HBM and latency: 9936 tokens of 4 heads of 128 in fp16 (30.5 MB) 10.9 us; one
// token for each of 32 sequences 4.8 us, a chain of look-ups, rows, maximum and the
// pieces to be merged (averages under the profiler).
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

// Whether one of the page's tokens before `lo` holds a value other than 0 and NaN, which are the same bytes under any scale.
template <int D, bool V>
__device__ __forceinline__ bool holds_values(const uint8_t *page, int lo) {
  uint32_t any = 0;
  for (int i = threadIdx.x; i < ((lo + 31) >> 5) * (2 * D); i += kAppThreads) {
    const uint4 w = reinterpret_cast<const uint4 *>(page)[i];
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
    const int lane = i & 63, t = i / (2 * D) * 32;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t x = d[q] & 0x7f7f7f7fu;
      const uint32_t is = (x + 0x7f7f7f7fu) & ~(x + 0x01010101u) & 0x80808080u;  // 0x80: neither 0 nor 0x7f
      // the dword's bytes before lo: a key's are all of one token, a value's of tokens one after the other
      const int left = V ? lo - (t + 4 * (lane >> 5) + 8 * q) : (t + (lane & 31) < lo ? 4 : 0);
      any |= left >= 4 ? is : left <= 0 ? 0u : is & (0xffffffffu >> (32 - 8 * left));
    }
  }
  return __syncthreads_or(any != 0) != 0;
}

// The new rows [lo, hi) of a page from src (row 0: the page's first token).  A thread owns four consecutive tokens by
// 8 columns, read once and kept in registers over the search for the maximum: as bytes they are whole dwords of
// V's pieces and halves of K's.  These meet in an image of the page in LDS, and what changes goes out as 16-byte pieces.
template <int DT, int PAGE, int D, bool V>
__device__ __forceinline__ void write_page(const typename Elem<DT>::T *src, int64_t s_t, int lo, int hi, uint8_t *image,
                                           uint8_t *__restrict__ page, float *scale) {
  using T = typename Elem<DT>::T;
  __shared__ uint32_t top[kAppThreads / 64];
  constexpr int kCols = D / 8, kItems = PAGE / 4 * kCols, kOwn = (kItems + kAppThreads - 1) / kAppThreads;
  struct alignas(16) Eight {
    T v[8];
  };
  Eight r[kOwn][4];
  uint32_t m = 0;
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int i = o * kAppThreads + threadIdx.x, t = i / kCols * 4, c = i % kCols * 8;
    if (i >= kItems || t >= hi || t + 4 <= lo) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // (a row that is not new: one that is again)
      const int row = t + e < lo ? lo : t + e < hi ? t + e : hi - 1;
      r[o][e] = *reinterpret_cast<const Eight *>(src + row * s_t + c);
    }
  }
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int i = o * kAppThreads + threadIdx.x, t = i / kCols * 4;
    if (i >= kItems || t >= hi || t + 4 <= lo) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int x = 0; x < 8; ++x) m = tm_fp8_amax(m, Elem<DT>::to_f(r[o][e].v[x]));
  }
  const float before = *scale;
  m = tm_wave_max_u32(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();  // (every thread has read the scale)
  m = max(max(top[0], top[1]), max(top[2], top[3]));
  float inv;
  float s = fmaxf(tm_fp8_scale(m, inv), kKv8MinScale);
  float f = 1.f;  // what the page held is taken times this
  if (lo > 0) {
    // New rows of zeros and non-finite values alone ask for no scale; nor does the 1 that such rows left where they
    // came first (an outlier's page may have 1, too, so its bytes are read: 32 tokens, captured, 4.6 us instead of 4.0).
    if (m == 0 && before > 0.f) s = before;  // (0: storage that nobody has written to)
    else if (before > s) s = before == 1.f && !holds_values<D, V>(page, lo) ? s : before;
    else f = before / s;  // powers of two
  }
  inv = 1.f / s;
  if (threadIdx.x == 0) *scale = s;
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int i = o * kAppThreads + threadIdx.x, t = i / kCols * 4, c = i % kCols * 8;
    if (i >= kItems || t >= hi || t + 4 <= lo) continue;
    uint8_t *const tile = image + (t >> 5) * (32 * D) + (c >> 5) * 1024;
    auto q = [&](int e, int x) { return tm_fp8_quot(Elem<DT>::to_f(r[o][e].v[x]), inv); };
    if constexpr (V) {
      uint8_t *const at = tile + ((t >> 2 & 1) * 32 + (c & 31)) * 16 + (t >> 3 & 3) * 4;
#pragma unroll
      for (int x = 0; x < 8; ++x)
        *reinterpret_cast<uint32_t *>(at + x * 16) = tm_fp8_pack4(q(0, x), q(1, x), q(2, x), q(3, x));
    } else {
      uint8_t *const at = tile + ((c >> 4 & 1) * 32 + (t & 31)) * 16 + (c & 8);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<uint2 *>(at + e * 16) = make_uint2(tm_fp8_pack4(q(e, 0), q(e, 1), q(e, 2), q(e, 3)),
                                                            tm_fp8_pack4(q(e, 4), q(e, 5), q(e, 6), q(e, 7)));
    }
  }
  __syncthreads();
  // the tiles with new tokens, those before them too where they are rounded again
  const int first = f != 1.f ? 0 : lo >> 5, last = (hi - 1) >> 5;
  for (int i = first * (2 * D) + threadIdx.x; i < (last + 1) * (2 * D); i += kAppThreads) {
    const int lane = i & 63, t = i / (2 * D) * 32;
    uint4 *const w = reinterpret_cast<uint4 *>(page) + i;
    const uint4 now = reinterpret_cast<const uint4 *>(image)[i];
    if constexpr (!V) {
      const int row = t + (lane & 31);
      if (row >= hi || (row < lo && f == 1.f)) continue;
      *w = row < lo ? rescale16(*w, f) : now;
    } else {
      const int t0 = t + 4 * (lane >> 5);  // dword q: tokens t0 + 8 q ..+3
      if (t0 >= lo && t0 + 28 <= hi) {
        *w = now;
        continue;
      }
      if (t0 >= hi || (t0 + 28 <= lo && f == 1.f)) continue;
      const uint4 old = *w;
      const uint32_t o[4] = {old.x, old.y, old.z, old.w}, n[4] = {now.x, now.y, now.z, now.w};
      uint32_t out[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t was = f != 1.f ? rescale4(o[q], f) : o[q];
        out[q] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = t0 + 8 * q + e;
          out[q] |= (x < lo ? was : x < hi ? n[q] : o[q]) & (0xffu << (8 * e));
        }
      }
      *w = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

template <int DT, int PAGE, int D, int DV>
__global__ __launch_bounds__(kAppThreads) void append_kernel(AppArgs a) {
  using T = typename Elem<DT>::T;
  const int h = blockIdx.y;
  const bool vals = blockIdx.z != 0;
  __shared__ __align__(16) uint8_t image[PAGE * (D > DV ? D : DV)];
  constexpr int page = PAGE;
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
    write_page<DT, PAGE, DV, true>(src, a.s_t[1], lo, hi, image, static_cast<uint8_t *>(a.c.v) + at * page * DV, a.c.v_scale + at);
  } else {
    const T *const src = static_cast<const T *>(a.src[0]) + row0 * a.s_t[0] + h * a.s_h[0];
    write_page<DT, PAGE, D, false>(src, a.s_t[0], lo, hi, image, static_cast<uint8_t *>(a.c.k) + at * page * D, a.c.k_scale + at);
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
  if (batch->n_tokens == 1) ks_t = vs_t = 0;  // (the stride of a single row means nothing)
  if (cache->n_kv_heads == 1) ks_h = vs_h = 0;
  TM_REQUIRE(tm_aligned16(k) && tm_aligned16(v) && ks_t % 8 == 0 && ks_h % 8 == 0 && vs_t % 8 == 0 && vs_h % 8 == 0,
             TM_EINVAL_SHAPE, "tm_kv8_append: rows of k and v must be 16-byte aligned, strides multiples of 8 elements");
  AppArgs a = {*cache, *batch, {k, v}, {ks_t, vs_t}, {ks_h, vs_h}};
  // a sequence of n new tokens touches at most (n - 2) / page + 2 pages
  const int64_t units = batch->starts ? batch->n_tokens / cache->page_size + 2 * batch->n_seqs : batch->n_seqs;
  TM_REQUIRE(units < kKv8MaxGrid, TM_EINVAL_SHAPE, "tm_kv8_append: too many pages");
  const dim3 grid((unsigned)units, (unsigned)cache->n_kv_heads, 2);
  hipStream_t s = tm_hip_stream(stream);
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    using std::integral_constant;
    auto launch = [&](auto d, auto dv) {
      auto go = [&](auto page) {
        hipLaunchKernelGGL((append_kernel<DT, decltype(page)::value, decltype(d)::value, decltype(dv)::value>), grid,
                           dim3(kAppThreads), 0, s, a);
      };
      if (cache->page_size == 32) go(integral_constant<int, 32>{});
      else if (cache->page_size == 64) go(integral_constant<int, 64>{});
      else go(integral_constant<int, 128>{});
    };
    if (cache->head_dim == 64) launch(integral_constant<int, 64>{}, integral_constant<int, 64>{});
    else if (cache->head_dim == 128) launch(integral_constant<int, 128>{}, integral_constant<int, 128>{});
    else if (cache->head_dim == 256) launch(integral_constant<int, 256>{}, integral_constant<int, 256>{});
    else if (cache->v_dim == 128) launch(integral_constant<int, 192>{}, integral_constant<int, 128>{});
    else launch(integral_constant<int, 192>{}, integral_constant<int, 192>{});
    TM_LAUNCH_CHECK("tm_kv8_append");
    return TM_OK;
  });
}
