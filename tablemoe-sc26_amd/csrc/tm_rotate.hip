// Rotary positions with several axes (text, images, video): tm_rotate_positions.
//
// For frequency i of axis a(i): turns = position * inv_freq[i] / 2 pi in 64 bits,
// less the whole turns, then sine and cosine of what is left in 32 bits (a far
// position's angle has lost 2^-24 of its own size in 32 bits, 0.01 rad at 10^5);
// each pair of columns is turned in fp32 and rounded once.
//
// A workgroup owns four tokens (fewer where rotary_dim exceeds 512): their sines and
// cosines go to LDS once (the heads share them), then its threads walk (token, head,
// 8 pairs) by 16-byte pieces, or pair by pair where sizes, strides or pointers are
// no multiples of 8 elements.
//
// Bound by HBM: 36 heads of 128, 30011 tokens in fp16 (554 MB) 117 us, 4.7 TB/s; 4099 in
// bf16 (76 MB) 13.9 us, 5.4 TB/s; 8 tokens 5 us, of which the 64-bit angle and
// sine and cosine about 2.
#include "tm_internal.h"

#include <type_traits>

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotPairs = 1024;  // sines and cosines that a workgroup holds
constexpr int kRotMaxAxes = 4;
constexpr int64_t kMaxGrid = (int64_t)1 << 24;  // workgroups: a launch holds under 2^32 threads in a direction

struct RotArgs {
  const void *in[2];
  void *out[2];
  int64_t in_t[2], in_h[2], out_t[2], out_h[2];
  int32_t heads[2];
  int64_t n;
  const int64_t *pos;
  int64_t ld_pos;
  const float *inv;
  int32_t half, dim, tokens, axes, interleaved;
  int32_t sections[kRotMaxAxes];
  float sign;
};

__device__ __forceinline__ int axis_of(const RotArgs &a, int i) {
  int at = 0;
  if (a.interleaved) {
    at = i % a.axes;
    int end = 0;
#pragma unroll
    for (int k = 0; k < kRotMaxAxes; ++k) end = k == at ? a.sections[k] : end;
    return i < a.axes * end ? at : 0;
  }
  int end = 0;
#pragma unroll
  for (int k = 0; k < kRotMaxAxes; ++k) {
    end += a.sections[k];
    at += (k + 1 < a.axes && i >= end) ? 1 : 0;
  }
  return at;
}

// VEC columns at a time (8, or 1 where sizes, strides or pointers are not multiples of 8 elements).
template <int DT, int VEC>
__device__ __forceinline__ void load_cols(const typename Elem<DT>::T *p, float (&v)[VEC]) {
  if constexpr (VEC == 8) tm_load8<DT>(p, v);
  else v[0] = Elem<DT>::to_f(p[0]);
}
template <int DT, int VEC>
__device__ __forceinline__ void store_cols(typename Elem<DT>::T *p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) tm_store8<DT>(p, v);
  else p[0] = Elem<DT>::from_f(v[0]);
}

template <int DT, int VEC, bool ADJ>
__global__ __launch_bounds__(kRotThreads) void rotate_kernel(RotArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ __align__(16) float cs[kRotPairs], sn[kRotPairs];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)(a.n - t0 < a.tokens ? a.n - t0 : a.tokens);
  for (int p = threadIdx.x; p < nt * a.half; p += kRotThreads) {
    const int tok = p / a.half, i = p - tok * a.half;
    const double turns = (double)a.pos[axis_of(a, i) * a.ld_pos + t0 + tok] * ((double)a.inv[i] * 0.15915494309189535);
    const float part = (float)(2.0 * (turns - rint(turns)));  // of half a turn
    float s, c;
    sincospif(part, &s, &c);
    cs[p] = c;
    sn[p] = s * a.sign;
  }
  __syncthreads();
  // items: a pair of column pieces that turn, then the pieces that are copied
  const int turn = a.half / VEC, per = turn + (a.dim - 2 * a.half) / VEC;
  const int heads = a.heads[0] + a.heads[1];
  const int items = nt * heads * per;
  for (int it = threadIdx.x; it < items; it += kRotThreads) {
    const int row = it / per, j = it - row * per;
    const int tok = row / heads;
    int h = row - tok * heads;
    const int which = h >= a.heads[0] ? 1 : 0;
    h -= which ? a.heads[0] : 0;
    const T *const src = static_cast<const T *>(which ? a.in[1] : a.in[0]) + (t0 + tok) * (which ? a.in_t[1] : a.in_t[0]) +
                         h * (which ? a.in_h[1] : a.in_h[0]);
    T *const dst = static_cast<T *>(which ? a.out[1] : a.out[0]) + (t0 + tok) * (which ? a.out_t[1] : a.out_t[0]) +
                   h * (which ? a.out_h[1] : a.out_h[0]);
    if (j >= turn) {
      if (src == dst) continue;
      float v[VEC];
      const int c = 2 * a.half + (j - turn) * VEC;
      load_cols<DT, VEC>(src + c, v);
      store_cols<DT, VEC>(dst + c, v);
      continue;
    }
    float x[VEC], y[VEC], cv[VEC], sv[VEC];
    const int lo = ADJ ? 2 * j * VEC : j * VEC, hi = ADJ ? lo + VEC : a.half + lo;
    load_cols<DT, VEC>(src + lo, x);
    load_cols<DT, VEC>(src + hi, y);
    const int p = tok * a.half + j * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      cv[e] = cs[p + e];
      sv[e] = sn[p + e];
    }
    if constexpr (ADJ && VEC == 8) {
      // x: pairs 0 to 3 of the piece, y: pairs 4 to 7
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float(&w)[8] = e < 4 ? x : y;
        const int o = 2 * (e & 3);
        const float u = w[o], v = w[o + 1];
        w[o] = u * cv[e] - v * sv[e];
        w[o + 1] = v * cv[e] + u * sv[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float u = x[e], v = y[e];
        x[e] = u * cv[e] - v * sv[e];
        y[e] = v * cv[e] + u * sv[e];
      }
    }
    store_cols<DT, VEC>(dst + lo, x);
    store_cols<DT, VEC>(dst + hi, y);
  }
}

}  // namespace

extern "C" int tm_rotate_positions(int32_t dtype, const void *q, int64_t n_tokens, int32_t n_heads, int64_t qs_t,
                                   int64_t qs_h, const void *k, int32_t n_kv_heads, int64_t ks_t, int64_t ks_h,
                                   int32_t head_dim, int32_t rotary_dim, const int64_t *positions, int64_t ld_positions,
                                   int32_t n_axes, const int32_t *sections, int32_t interleaved, int32_t adjacent,
                                   int32_t inverse, const float *inv_freq, void *q_out, int64_t qo_t, int64_t qo_h,
                                   void *k_out, int64_t ko_t, int64_t ko_h, tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F32 || dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE,
             "tm_rotate_positions: unsupported dtype tag %d", (int)dtype);
  TM_REQUIRE(n_tokens >= 0 && n_tokens < ((int64_t)1 << 31) && n_heads >= 1 && n_heads <= 4096 && head_dim >= 1 &&
                 head_dim <= 1024,
             TM_EINVAL_SHAPE, "tm_rotate_positions: bad sizes (tokens %lld, heads %d, head_dim %d)", (long long)n_tokens,
             n_heads, head_dim);
  TM_REQUIRE(k == nullptr || (n_kv_heads >= 1 && n_kv_heads <= 4096), TM_EINVAL_SHAPE,
             "tm_rotate_positions: bad number of key heads %d", n_kv_heads);
  TM_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, TM_EINVAL_SHAPE,
             "tm_rotate_positions: rotary_dim %d must be even, at most head_dim %d", rotary_dim, head_dim);
  TM_REQUIRE(n_axes >= 1 && n_axes <= kRotMaxAxes && ld_positions >= n_tokens, TM_EINVAL_SHAPE,
             "tm_rotate_positions: 1 to %d axes, rows of positions at least n_tokens long", kRotMaxAxes);
  TM_REQUIRE(sections, TM_EINVAL_ARG, "tm_rotate_positions: null pointer");
  int64_t sum = 0;
  for (int i = 0; i < n_axes; ++i) {
    TM_REQUIRE(sections[i] >= 0, TM_EINVAL_SHAPE, "tm_rotate_positions: a negative section");
    sum += sections[i];
  }
  TM_REQUIRE(sum == rotary_dim / 2, TM_EINVAL_SHAPE, "tm_rotate_positions: sections sum to %lld, not to %d",
             (long long)sum, rotary_dim / 2);
  if (n_tokens == 0) return TM_OK;
  TM_REQUIRE(q && positions && inv_freq && q_out && (k == nullptr || k_out), TM_EINVAL_ARG,
             "tm_rotate_positions: null pointer");
  RotArgs a = {};
  a.in[0] = q, a.in[1] = k;
  a.out[0] = q_out, a.out[1] = k_out;
  a.heads[0] = n_heads, a.heads[1] = k ? n_kv_heads : 0;
  const int64_t in_t[2] = {qs_t, ks_t}, in_h[2] = {qs_h, ks_h}, out_t[2] = {qo_t, ko_t}, out_h[2] = {qo_h, ko_h};
  for (int w = 0; w < 2; ++w) {  // (the stride of a single token or head means nothing)
    a.in_t[w] = n_tokens > 1 ? in_t[w] : 0, a.in_h[w] = a.heads[w] > 1 ? in_h[w] : 0;
    a.out_t[w] = n_tokens > 1 ? out_t[w] : 0, a.out_h[w] = a.heads[w] > 1 ? out_h[w] : 0;
  }
  a.n = n_tokens;
  a.pos = positions, a.ld_pos = ld_positions, a.inv = inv_freq;
  a.half = rotary_dim / 2, a.dim = head_dim, a.axes = n_axes, a.interleaved = interleaved != 0;
  for (int i = 0; i < n_axes; ++i) a.sections[i] = sections[i];
  a.sign = inverse ? -1.f : 1.f;
  bool wide = a.half % 8 == 0 && head_dim % 8 == 0;
  for (int w = 0; w < (k ? 2 : 1); ++w)
    wide = wide && tm_aligned16(a.in[w]) && tm_aligned16(a.out[w]) && a.in_t[w] % 8 == 0 && a.in_h[w] % 8 == 0 &&
           a.out_t[w] % 8 == 0 && a.out_h[w] % 8 == 0;
  a.tokens = 4;
  while (a.tokens > 1 && a.tokens * a.half > kRotPairs) --a.tokens;
  TM_REQUIRE(tm_cdiv(n_tokens, a.tokens) < kMaxGrid, TM_EINVAL_SHAPE, "tm_rotate_positions: too many tokens");
  const dim3 grid((unsigned)tm_cdiv(n_tokens, a.tokens));
  hipStream_t s = tm_hip_stream(stream);
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    auto launch = [&](auto vec, auto adj) {
      hipLaunchKernelGGL((rotate_kernel<DT, decltype(vec)::value, decltype(adj)::value>), grid, dim3(kRotThreads), 0, s, a);
    };
    auto pairs = [&](auto vec) {
      if (adjacent) launch(vec, std::true_type{});
      else launch(vec, std::false_type{});
    };
    if (wide) pairs(std::integral_constant<int, 8>{});
    else pairs(std::integral_constant<int, 1>{});
    TM_LAUNCH_CHECK("tm_rotate_positions");
    return TM_OK;
  });
}
