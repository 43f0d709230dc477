// Quantisation to 8 bits in blocks of 128 (the rule: tm_fp8_dev.h).
//
// Rows: 16 lanes own one block of one row, 8 columns each, loaded as 16-byte
// pieces; the block's maximum is three DPP exchanges and a row_mirror away and
// the values stay in registers until they are scaled, so a row is read once.
// Weights: a workgroup holds a block of 128 x 128 in registers between its
// maximum and its scaling.
//
// Bound by HBM: 64 matrices of 1536 x 2560 in bf16 (755 MB) take 138 us, 5.5 TB/s (150
// when each load waited for the one before); 4099 rows of 2048 (25 MB) 7.4 us, of which
// a launch is a third.
#include "tm_fp8_dev.h"
#include "tm_fp8.h"

#include <type_traits>

namespace {

constexpr int kQThreads = 256;

// Columns [c, c + 8) of a row of k columns, zero past k.  A full piece is one
// 16-byte load (fp32: two) at whatever alignment the rows have (element by
// element, 4099 rows of 2049 in bf16 took 13.1 us, this way 7.5).
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T *row, int64_t c, int64_t k, float (&v)[8]) {
  if (c + 8 <= k) {
    typename Elem<DT>::T e[8];
    __builtin_memcpy(e, row + c, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<DT>::to_f(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < k ? Elem<DT>::to_f(row[c + i]) : 0.f;
  }
}

template <int DT>
__global__ __launch_bounds__(kQThreads) void quantize_rows_kernel(const typename Elem<DT>::T *__restrict__ x, int64_t n,
                                                                 int64_t k, int64_t ld_x, int blocks,
                                                                 uint8_t *__restrict__ q, int64_t ld_q,
                                                                 float *__restrict__ scale, int64_t ld_s) {
  const int64_t item = ((int64_t)blockIdx.x * kQThreads + threadIdx.x) >> 4;  // (row, block)
  const int64_t row = item / blocks;
  const int b = (int)(item - row * blocks);
  if (row >= n) return;  // whole 16-lane groups
  const int sub = threadIdx.x & 15;
  const int64_t c = (int64_t)b * kFp8Block + sub * 8;
  float v[8];
  load8<DT>(x + row * ld_x, c, k, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = tm_fp8_amax(m, v[i]);
  m = tm_row16_max(m);
  float inv;
  const float s = tm_fp8_scale(m, inv);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = tm_fp8_quot(v[i], inv);
  const uint32_t lo = tm_fp8_pack4(v[0], v[1], v[2], v[3]), hi = tm_fp8_pack4(v[4], v[5], v[6], v[7]);
  *reinterpret_cast<uint2 *>(q + row * ld_q + c) = make_uint2(lo, hi);
  if (sub == 0) scale[row * ld_s + b] = s;
}

// One workgroup per 128 x 128 block: thread t holds rows t / 16 + 16 j, 8
// columns each.
template <int DT>
__global__ __launch_bounds__(kQThreads) void quantize_weight_kernel(const typename Elem<DT>::T *__restrict__ w,
                                                                   int64_t n, int64_t k, int nb, int kb,
                                                                   uint8_t *__restrict__ q, int64_t ld_q,
                                                                   float *__restrict__ scale) {
  __shared__ uint32_t top[kQThreads / 64];
  const int64_t blk = blockIdx.x;
  const int bc = (int)(blk % kb);
  const int64_t t = blk / kb;
  const int br = (int)(t % nb);
  const int64_t mat = t / nb;
  const int64_t c = (int64_t)bc * kFp8Block + (threadIdx.x & 15) * 8;
  const int64_t r0 = (int64_t)br * kFp8Block + (threadIdx.x >> 4);
  const typename Elem<DT>::T *const wm = w + mat * n * k;
  float v[8][8];
  auto load = [&](auto whole) {  // whole: no row ends inside the block, so no branch keeps the loads apart
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t r = r0 + 16 * j;
      const auto *const row = wm + (r < n ? r : n - 1) * k;  // (a row past n: the last one again, not stored)
      load8<DT>(row, c, decltype(whole)::value ? c + 8 : k, v[j]);
    }
  };
  if ((int64_t)(bc + 1) * kFp8Block <= k) load(std::true_type{});
  else load(std::false_type{});
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = tm_fp8_amax(m, v[j][i]);
  m = tm_wave_max_u32(m);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(top[0], top[1]), max(top[2], top[3]));
  float inv;
  const float s = tm_fp8_scale(m, inv);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = r0 + 16 * j;
    if (r >= n) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = tm_fp8_quot(v[j][i], inv);
    *reinterpret_cast<uint2 *>(q + (mat * n + r) * ld_q + c) =
        make_uint2(tm_fp8_pack4(v[j][0], v[j][1], v[j][2], v[j][3]), tm_fp8_pack4(v[j][4], v[j][5], v[j][6], v[j][7]));
  }
  if (threadIdx.x == 0) scale[blk] = s;
}

}  // namespace

int tm_internal_fp8_rows(int32_t dtype, const void *x, int64_t n, int64_t k, int64_t ld_x, void *q, int64_t ld_q,
                         float *scale, int64_t ld_s, hipStream_t s) {
  const int64_t blocks = tm_cdiv(k, kFp8Block);
  constexpr int kPer = kQThreads / 16;  // (row, block) pairs of a workgroup
  TM_REQUIRE(n <= (((int64_t)1 << 31) - 1) * kPer / blocks, TM_EINVAL_SHAPE, "tm_fp8_quantize_rows: too many rows");
  const int64_t grid = tm_cdiv(n * blocks, kPer);
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    const auto *const p = static_cast<const typename Elem<DT>::T *>(x);
    auto *const out = static_cast<uint8_t *>(q);
    hipLaunchKernelGGL((quantize_rows_kernel<DT>), dim3((unsigned)grid), dim3(kQThreads), 0, s, p, n, k, ld_x,
                       (int)blocks, out, ld_q, scale, ld_s);
    TM_LAUNCH_CHECK("tm_fp8_quantize_rows");
    return TM_OK;
  });
}

extern "C" int tm_fp8_quantize_rows(int32_t dtype, const void *x, int64_t n_rows, int64_t k, int64_t ld_x, void *q,
                                    int64_t ld_q, float *scale, int64_t ld_scale, tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F32 || dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE,
             "tm_fp8_quantize_rows: unsupported dtype tag %d", (int)dtype);
  TM_REQUIRE(n_rows >= 0 && k >= 1 && k < ((int64_t)1 << 31) && ld_x >= k, TM_EINVAL_SHAPE,
             "tm_fp8_quantize_rows: bad sizes (rows %lld, columns %lld, row stride %lld)", (long long)n_rows,
             (long long)k, (long long)ld_x);
  const int64_t blocks = tm_cdiv(k, kFp8Block);
  TM_REQUIRE(ld_q >= blocks * kFp8Block && ld_q % 16 == 0 && ld_scale >= blocks, TM_EINVAL_SHAPE,
             "tm_fp8_quantize_rows: a row of q takes %lld bytes (a multiple of 16), of scale %lld",
             (long long)(blocks * kFp8Block), (long long)blocks);
  if (n_rows == 0) return TM_OK;
  TM_REQUIRE(x && q && scale, TM_EINVAL_ARG, "tm_fp8_quantize_rows: null pointer");
  TM_REQUIRE(tm_aligned16(q), TM_EINVAL_SHAPE, "tm_fp8_quantize_rows: q must be 16-byte aligned");
  return tm_internal_fp8_rows(dtype, x, n_rows, k, ld_x, q, ld_q, scale, ld_scale, tm_hip_stream(stream));
}

extern "C" int tm_fp8_quantize_weight(int32_t dtype, const void *w, int64_t n_mats, int64_t n_rows, int64_t k, void *q,
                                      int64_t ld_q, float *scale, tm_stream_t stream) {
  TM_REQUIRE(n_mats >= 0 && n_rows >= 1 && k >= 1 && n_rows < ((int64_t)1 << 31) && k < ((int64_t)1 << 31),
             TM_EINVAL_SHAPE, "tm_fp8_quantize_weight: bad sizes (%lld matrices of %lld x %lld)", (long long)n_mats,
             (long long)n_rows, (long long)k);
  const int64_t nb = tm_cdiv(n_rows, kFp8Block), kb = tm_cdiv(k, kFp8Block);
  TM_REQUIRE(ld_q >= kb * kFp8Block && ld_q % 16 == 0, TM_EINVAL_SHAPE,
             "tm_fp8_quantize_weight: a row of q takes %lld bytes (a multiple of 16)", (long long)(kb * kFp8Block));
  TM_REQUIRE(n_mats < ((int64_t)1 << 31) / (nb * kb) + 1 && n_mats * nb * kb < ((int64_t)1 << 31), TM_EINVAL_SHAPE,
             "tm_fp8_quantize_weight: too many blocks");
  if (n_mats == 0) return TM_OK;
  TM_REQUIRE(w && q && scale, TM_EINVAL_ARG, "tm_fp8_quantize_weight: null pointer");
  TM_REQUIRE(tm_aligned16(q), TM_EINVAL_SHAPE, "tm_fp8_quantize_weight: q must be 16-byte aligned");
  const dim3 grid((unsigned)(n_mats * nb * kb));
  hipStream_t s = tm_hip_stream(stream);
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    using T = typename Elem<DT>::T;
    hipLaunchKernelGGL((quantize_weight_kernel<DT>), grid, dim3(kQThreads), 0, s, static_cast<const T *>(w), n_rows, k,
                       (int)nb, (int)kb, static_cast<uint8_t *>(q), ld_q, scale);
    TM_LAUNCH_CHECK("tm_fp8_quantize_weight");
    return TM_OK;
  });
}
