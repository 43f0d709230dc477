// Products with 8-bit weights (e4m3, one fp32 scale per 128 x 128 block) and
// activations quantised in blocks of 128 columns of a row: a linear layer and
// the SwiGLU MLP of experts.
//
//   y[r][c] = sum_b sx[r][b] sw[c / 128][b] sum_{k in block b} x[r][k] w[c][k]
//
// The MLP: g = x W1^T, u = x W3^T (fp32), f = silu(g) u (fp32, not rounded),
// f quantised in blocks of 128 columns, y = f W2^T (one rounding).
//
// Arithmetic.  The 8-bit matrix instructions truncate their products against
// the largest of a group: sums over 128 columns of normal data come out 1.5e-5
// to 6e-5 of their size off, whichever instruction (16x16x32 and 16x16x128 give
// the same bits), where the 16-bit ones are off by 1e-8.  e4m3 values are exact
// as bf16, so products whose result is kept in fp32 or is quantised again (g
// and u: an error of 3e-5 there turns roundings of f over, which costs y as much
// as its rounding to bf16) run on the bf16 instructions, and those that are
// rounded to 16 bits once at the end on the 8-bit ones.
#include "tm_fp8.h"
#include "tm_fp8_dev.h"

namespace {

enum { kUp = 0, kOut = 1 };
constexpr int kE4M3 = TM_DT_E4M3;  // activations that are quantised already

// Rows of a call: every row (dense), the (token, slot) pairs of a small batch
// found in the launch itself (slots), or the lists tm_group_slots writes.
struct Fp8Rows {
  int64_t n;  // dense: rows; slots: tokens
  const int64_t *ids;
  int64_t ld_ids;
  const uint8_t *mask;
  int64_t ms_b, ms_s;
  int32_t top_k, n_experts;
  const int32_t *offsets, *row_token;
  const int64_t *row_out;
};

// Activations: element (row, k) at x[row * ld + k]; kE4M3: with scale[row * ld_s + k / 128].
struct Fp8Src {
  const void *x;
  int64_t ld, k;
  const float *scale;
  int64_t ld_s;
};

struct Fp8Mat {
  const uint8_t *w;  // [experts][n][ld_w], rows padded to whole blocks
  const float *s;    // [experts][ceil(n / 128)][ceil(k / 128)]
};

struct Fp8Dst {
  void *y;
  int64_t ld;           // dense rows
  int64_t so_b, so_s;   // slots
  const void *add;      // bias [n] (ld_add 0) or addend [rows][n], nullable
  int64_t ld_add;
};

template <int DT>
__device__ __forceinline__ float at_f(const void *p, int64_t i) {
  return Elem<DT>::to_f(static_cast<const typename Elem<DT>::T *>(p)[i]);
}

// Four columns c .. c + 3 of a row of n columns.
template <int DT>
__device__ __forceinline__ void store4(void *y, int64_t at, const float (&v)[4], int c, int n, bool vec) {
  using T = typename Elem<DT>::T;
  T *const p = static_cast<T *>(y) + at + c;
  if (vec && c + 4 <= n) {
    if constexpr (DT == TM_DT_F32) {
      *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint2 r;
      T *e = reinterpret_cast<T *>(&r);
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = Elem<DT>::from_f(v[i]);
      *reinterpret_cast<uint2 *>(p) = r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < n) p[i] = Elem<DT>::from_f(v[i]);
  }
}

// ---------------------------------------------------------------------------
// Few rows: a stream of the weights.
//
// A workgroup of S waves owns 16 weight rows (up: of W1 and of W3); wave w
// holds their blocks [w KPW, (w + 1) KPW) in registers, loaded at once, and
// multiplies them with the workgroup's rows, 16 at a time, on the bf16
// instructions (K of more than S KPW blocks: in passes, loaded again for each
// 16 rows); the waves' sums are added in wave order through LDS.  Each lane
// quantises its own piece of a row on the way (32 columns of each block), so
// neither the activations nor, in the down product, f needs a launch before.
// ---------------------------------------------------------------------------
constexpr int kMaxSlots = 1024;  // (token, slot) pairs of a call that are found in the launch
constexpr int kMaxWaves = 8;

template <int DTX>
__device__ __forceinline__ void load_x(const Fp8Src &src, int64_t row, int kb, int g, bool live, float (&v)[4][8]) {
  using T = typename Elem<DTX>::T;
  const T *const p = static_cast<const T *>(src.x) + row * src.ld;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t c = (int64_t)kb * kFp8Block + 64 * (j >> 1) + 16 * g + 8 * (j & 1);
    if (live && c + 8 <= src.k) {
      tm_load8<DTX>(p + c, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = live && c + i < src.k ? Elem<DTX>::to_f(p[c + i]) : 0.f;
    }
  }
}

// B operands of block kb: this lane's 32 columns of its row, quantised, as
// bf16 values q * s.
template <int DTX>
__device__ __forceinline__ void quantised_frag(const float (&v)[4][8], uint4 (&b)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = tm_fp8_amax(m, v[j][i]);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  float inv;
  const float s = tm_fp8_scale(m, inv);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = tm_fp8_quot(v[j][i], inv);
    const uint2 lo = tm_fp8_scaled_bf16x4(tm_fp8_pack4(t[0], t[1], t[2], t[3]), s);
    const uint2 hi = tm_fp8_scaled_bf16x4(tm_fp8_pack4(t[4], t[5], t[6], t[7]), s);
    b[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}

template <int DT, int DTX, int MODE, int KPW>
__global__ __launch_bounds__(64 * kMaxWaves) void stream_kernel(Fp8Src src, Fp8Rows rows, Fp8Mat m0, Fp8Mat m1, int n_out,
                                                                int ld_w, int KT, int n_groups, Fp8Dst dst,
                                                                bool vec_out) {
  constexpr int NM = MODE == kUp ? 2 : 1;
  __shared__ float4 red[kMaxWaves][NM][64];
  __shared__ int list[kMaxSlots];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = (int)blockDim.x >> 6;
  const int t = lane & 15, g = lane >> 4;
  const int n0 = (int)(blockIdx.x % n_groups) * 16;
  const int64_t item = blockIdx.x / n_groups;
  int e = 0;
  int64_t first = 0, count = rows.n;
  if (rows.ids != nullptr) {
    // Slot `item` leads if its expert has no earlier slot; the leader's
    // workgroups take all of the expert's slots, in order.
    const int total = (int)rows.n * rows.top_k;
    auto expert_of = [&](int p) {
      const int b = p / rows.top_k, s = p - b * rows.top_k;
      const int64_t id = rows.ids[b * rows.ld_ids + s];
      return rows.mask[b * rows.ms_b + s * rows.ms_s] && id >= 0 && id < rows.n_experts ? (int)id : -1;
    };
    e = expert_of((int)item);
    if (e < 0) return;  // uniform
    if (wave == 0) {
      int c = 0;
      for (int p0 = 0; p0 < total; p0 += 64) {
        const int p = p0 + lane;
        const bool mine = p < total && expert_of(p) == e;
        const uint64_t all = __ballot(mine);
        if (mine) list[c + __popcll(all & ((1ull << lane) - 1))] = p;
        c += __popcll(all);
      }
      if (lane == 0) s_count = c;
    }
    __syncthreads();
    if (list[0] != (int)item) return;  // uniform
    count = s_count;
  } else if (rows.offsets != nullptr) {
    e = (int)item;
    first = rows.offsets[e];
    count = rows.offsets[e + 1] - first;
    if (count == 0) return;  // uniform
  }

  uint4 w[NM][KPW][2];
  float sw[NM][KPW];
  const int nb = (n_out + kFp8Block - 1) / kFp8Block;
  auto load_w = [&](int kb0) {
    const int r = n0 + t < n_out ? n0 + t : n_out - 1;  // (a row past n_out: the last one again, not stored)
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const Fp8Mat &mat = m == 0 ? m0 : m1;
      const uint8_t *const p = mat.w + ((int64_t)e * n_out + r) * ld_w + 16 * g;
      const float *const ps = mat.s + ((int64_t)e * nb + n0 / kFp8Block) * KT;
#pragma unroll
      for (int j = 0; j < KPW; ++j) {
        const int kb = kb0 + j;
        if (kb < KT) {  // uniform
          w[m][j][0] = *reinterpret_cast<const uint4 *>(p + (int64_t)kb * kFp8Block);
          w[m][j][1] = *reinterpret_cast<const uint4 *>(p + (int64_t)kb * kFp8Block + 64);
          sw[m][j] = ps[kb];
        }
      }
    }
  };
  const bool once = KT <= S * KPW;
  if (once) load_w(wave * KPW);
  for (int64_t c0 = 0; c0 < count; c0 += 16) {
    const bool live = c0 + t < count;
    int64_t xr = c0 + t;
    if (rows.ids != nullptr) xr = live ? (MODE == kUp ? list[c0 + t] / rows.top_k : list[c0 + t]) : 0;
    else if (rows.offsets != nullptr) xr = live ? (MODE == kUp ? (int64_t)rows.row_token[first + c0 + t] : first + c0 + t) : 0;
    else if (!live) xr = 0;
    tm_f32x4 acc[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) acc[m] = tm_f32x4{};
    for (int kb0 = wave * KPW; kb0 < KT; kb0 += S * KPW) {
    if (!once) load_w(kb0);
#pragma unroll
    for (int j = 0; j < KPW; ++j) {
      const int kb = kb0 + j;
      if (kb >= KT) continue;  // uniform
      uint4 b[4];
      float sx = 1.f;
      if constexpr (DTX == kE4M3) {
        const uint8_t *const p = static_cast<const uint8_t *>(src.x) + xr * src.ld + (int64_t)kb * kFp8Block + 16 * g;
        uint4 q0 = make_uint4(0, 0, 0, 0), q1 = q0;
        if (live) {
          q0 = *reinterpret_cast<const uint4 *>(p);
          q1 = *reinterpret_cast<const uint4 *>(p + 64);
          sx = src.scale[xr * src.ld_s + kb];
        }
        b[0] = tm_fp8_to_bf16x8(q0.x, q0.y);
        b[1] = tm_fp8_to_bf16x8(q0.z, q0.w);
        b[2] = tm_fp8_to_bf16x8(q1.x, q1.y);
        b[3] = tm_fp8_to_bf16x8(q1.z, q1.w);
      } else {
        float v[4][8];
        load_x<DTX>(src, xr, kb, g, live, v);
        quantised_frag<DTX>(v, b);
      }
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        tm_f32x4 p = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          p = tm_mfma16x16x32<TM_DT_BF16>(tm_fp8_to_bf16x8(w[m][j][h].x, w[m][j][h].y), b[2 * h], p);
          p = tm_mfma16x16x32<TM_DT_BF16>(tm_fp8_to_bf16x8(w[m][j][h].z, w[m][j][h].w), b[2 * h + 1], p);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(p[i], sw[m][j] * sx, acc[m][i]);
      }
    }
    }
#pragma unroll
    for (int m = 0; m < NM; ++m) red[wave][m][lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
    __syncthreads();
    if (wave == 0 && live) {
      // lane: row t, columns n0 + 4 g .. + 3
      float v[NM][4] = {};
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const float4 p = red[s][m][lane];
          v[m][0] += p.x; v[m][1] += p.y; v[m][2] += p.z; v[m][3] += p.w;
        }
      const int c = n0 + 4 * g;
      if constexpr (MODE == kUp) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = v[0][i] * __builtin_amdgcn_rcpf(1.f + __expf(-v[0][i])) * v[NM - 1][i];
        const int64_t fr = rows.ids != nullptr ? list[c0 + t] : first + c0 + t;
        store4<TM_DT_F32>(dst.y, fr * dst.ld, f, c, n_out, true);
      } else {
        int64_t at = xr * dst.ld;
        if (rows.ids != nullptr) {
          const int p = list[c0 + t];
          at = (p / rows.top_k) * dst.so_b + (p % rows.top_k) * dst.so_s;
        } else if (rows.offsets != nullptr) {
          at = rows.row_out[first + c0 + t];
        }
        if (dst.add != nullptr)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < n_out) v[0][i] += at_f<DT>(dst.add, xr * dst.ld_add + c + i);
        store4<DT>(dst.y, at, v[0], c, n_out, vec_out);
      }
    }
    __syncthreads();
  }
}

template <int DT, int DTX, int MODE>
int stream_launch(const char *name, const Fp8Src &src, const Fp8Rows &rows, const Fp8Mat &m0, const Fp8Mat &m1,
                  int n_out, int KT, const Fp8Dst &dst, hipStream_t s) {
  const int n_groups = (int)tm_cdiv(n_out, 16);
  const int64_t items = rows.ids != nullptr ? rows.n * rows.top_k : rows.offsets != nullptr ? rows.n_experts : 1;
  TM_REQUIRE(items * n_groups < ((int64_t)1 << 31), TM_EINVAL_SHAPE, "%s: too many rows", name);
  const int64_t esz = Elem<DT>::kBytes;
  const bool vec_out = (reinterpret_cast<uintptr_t>(dst.y) & 15) == 0 && dst.ld * esz % 16 == 0 &&
                       dst.so_b * esz % 16 == 0 && dst.so_s * esz % 16 == 0;
  const dim3 grid((unsigned)(items * n_groups));
  const int ld_w = KT * kFp8Block;
#define TM_STREAM(KPW_)                                                                                            \
  hipLaunchKernelGGL((stream_kernel<DT, DTX, MODE, KPW_>), grid, dim3(64 * (unsigned)waves(KPW_)), 0, s, src, \
                     rows, m0, m1, n_out, ld_w, KT, n_groups, dst, vec_out)
  auto waves = [&](int kpw) { return tm_cdiv(KT, kpw) < kMaxWaves ? tm_cdiv(KT, kpw) : kMaxWaves; };
  if (KT <= 8) TM_STREAM(2);
  else TM_STREAM(4);
#undef TM_STREAM
  TM_LAUNCH_CHECK(name);
  return TM_OK;
}

bool aligned(const void *p, int64_t stride_bytes) { return tm_aligned16(p) && stride_bytes % 16 == 0; }

int64_t round_up(int64_t v, int64_t m) { return tm_cdiv(v, m) * m; }

}  // namespace

// ---------------------------------------------------------------------------
// linear
// ---------------------------------------------------------------------------
extern "C" size_t tm_fp8_linear_workspace_size(int64_t n_rows, int64_t k, int32_t dtype) {
  if (n_rows <= 0 || k <= 0) return 0;
  const int64_t kb = tm_cdiv(k, kFp8Block);
  return (size_t)(round_up(n_rows * kb * kFp8Block, 256) + round_up(n_rows * kb * 4, 256));
}

extern "C" int tm_fp8_linear(int32_t dtype, const void *x, const float *x_scale, int64_t n_rows, int64_t k, int64_t ld_x,
                             int64_t ld_xs, const void *w, const float *w_scale, int64_t n_out, const void *bias,
                             void *out, int64_t ld_out, void *workspace, size_t workspace_bytes, tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F32 || dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE,
             "tm_fp8_linear: unsupported dtype tag %d", (int)dtype);
  const int64_t kb = tm_cdiv(k < 0 ? 0 : k, kFp8Block), kp = kb * kFp8Block;
  TM_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 31) && k >= 1 && k <= 16384 && n_out >= 1 &&
                 n_out < ((int64_t)1 << 24),
             TM_EINVAL_SHAPE, "tm_fp8_linear: bad sizes (%lld rows, %lld columns, %lld outputs)", (long long)n_rows,
             (long long)k, (long long)n_out);
  TM_REQUIRE(ld_x >= (x_scale ? kp : k) && ld_out >= n_out && (!x_scale || ld_xs >= kb), TM_EINVAL_SHAPE,
             "tm_fp8_linear: row strides (%lld, %lld) are shorter than the rows", (long long)ld_x, (long long)ld_out);
  if (n_rows == 0) return TM_OK;
  TM_REQUIRE(x && w && w_scale && out, TM_EINVAL_ARG, "tm_fp8_linear: null pointer");
  TM_REQUIRE(tm_aligned16(w), TM_EINVAL_SHAPE, "tm_fp8_linear: w must be 16-byte aligned");
  hipStream_t s = tm_hip_stream(stream);
  Fp8Src src{x, ld_x, k, x_scale, ld_xs};
  if (x_scale) {
    TM_REQUIRE(aligned(x, ld_x), TM_EINVAL_SHAPE, "tm_fp8_linear: rows of 8-bit x must be 16-byte aligned");
  } else {
    const size_t need = tm_fp8_linear_workspace_size(n_rows, k, dtype);
    TM_REQUIRE(workspace != nullptr && workspace_bytes >= need && tm_aligned16(workspace), TM_EWORKSPACE,
               "tm_fp8_linear: workspace %zu bytes < %zu", workspace_bytes, need);
  }
  if (!x_scale && !aligned(x, ld_x * (dtype == TM_DT_F32 ? 4 : 2))) {
    float *const xs = reinterpret_cast<float *>(static_cast<char *>(workspace) + round_up(n_rows * kp, 256));
    const int st = tm_internal_fp8_rows(dtype, x, n_rows, k, ld_x, workspace, kp, xs, kb, false, s);
    if (st != TM_OK) return st;
    src = Fp8Src{workspace, kp, kp, xs, kb};
  }
  const Fp8Rows rows{n_rows};
  const Fp8Mat m{static_cast<const uint8_t *>(w), w_scale};
  const Fp8Dst dst{out, ld_out, 0, 0, bias, 0};
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    return src.scale ? stream_launch<DT, kE4M3, kOut>("tm_fp8_linear", src, rows, m, m, (int)n_out, (int)kb, dst, s)
                     : stream_launch<DT, DT, kOut>("tm_fp8_linear", src, rows, m, m, (int)n_out, (int)kb, dst, s);
  });
}

// ---------------------------------------------------------------------------
// experts
// ---------------------------------------------------------------------------
namespace {

int check_experts(const char *name, const tm_fp8_experts *ex, int32_t dtype) {
  TM_REQUIRE(ex != nullptr, TM_EINVAL_ARG, "%s: null weights", name);
  TM_REQUIRE(dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE, "%s: dtype must be F16 or BF16", name);
  TM_REQUIRE(ex->n_experts >= 1 && ex->n_experts <= 1024 && ex->hidden > 0 && ex->inter > 0 &&
                 ex->hidden % kFp8Block == 0 && ex->inter % kFp8Block == 0 && ex->hidden <= 16384 && ex->inter <= 16384,
             TM_EINVAL_SHAPE, "%s: hidden and inter must be multiples of %d up to 16384, experts at most 1024", name,
             kFp8Block);
  TM_REQUIRE(ex->w1 && ex->w3 && ex->w2 && ex->s1 && ex->s3 && ex->s2, TM_EINVAL_ARG, "%s: null weights", name);
  TM_REQUIRE(tm_aligned16(ex->w1) && tm_aligned16(ex->w3) && tm_aligned16(ex->w2), TM_EINVAL_SHAPE,
             "%s: weights must be 16-byte aligned", name);
  return TM_OK;
}

struct ExpertsWs {
  size_t f, offsets, row_token, row_out, tiles, group, total;
};

ExpertsWs experts_ws(int64_t n, int32_t top_k, const tm_fp8_experts *ex) {
  ExpertsWs w{};
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)round_up(bytes, 256);
    return here;
  };
  const int64_t rows = n * top_k;
  w.f = take(rows * ex->inter * 4);
  if (rows > kMaxSlots) {
    w.offsets = take(4 * ((int64_t)ex->n_experts + 1));
    w.row_token = take(4 * rows);
    w.row_out = take(8 * rows);
    w.tiles = take(4 * (2 + 2 * tm_group_slots_tiles(rows, ex->n_experts)));
    w.group = take((int64_t)tm_group_slots_workspace_size(n, top_k, ex->n_experts));
  }
  w.total = at;
  return w;
}

template <int DT>
int mlp_launch(const char *name, const tm_fp8_experts *ex, const Fp8Src &x, const Fp8Rows &rows, float *f,
               const Fp8Dst &dst, hipStream_t s) {
  const int h = ex->hidden, inter = ex->inter;
  const Fp8Mat w1{static_cast<const uint8_t *>(ex->w1), ex->s1}, w3{static_cast<const uint8_t *>(ex->w3), ex->s3},
      w2{static_cast<const uint8_t *>(ex->w2), ex->s2};
  const Fp8Dst mid{f, inter, 0, 0, nullptr, 0};
  const int st = stream_launch<DT, DT, kUp>(name, x, rows, w1, w3, inter, h / kFp8Block, mid, s);
  if (st != TM_OK) return st;
  const Fp8Src fs{f, inter, inter, nullptr, 0};
  return stream_launch<DT, TM_DT_F32, kOut>(name, fs, rows, w2, w2, h, inter / kFp8Block, dst, s);
}

}  // namespace

extern "C" size_t tm_fp8_grouped_swiglu_workspace_size(const tm_fp8_experts *experts, int64_t n_tokens,
                                                       int32_t top_k) {
  if (experts == nullptr || n_tokens <= 0 || top_k <= 0) return 0;
  return experts_ws(n_tokens, top_k, experts).total;
}

extern "C" int tm_fp8_grouped_swiglu(const tm_fp8_experts *experts, int32_t dtype, const void *x, int64_t n_tokens,
                                     int64_t ld_x, const int64_t *ids, int32_t top_k, int64_t ld_ids,
                                     const uint8_t *mask, int64_t ms_b, int64_t ms_s, void *out, int64_t so_b,
                                     int64_t so_s, void *workspace, size_t workspace_bytes, tm_stream_t stream) {
  const char *const name = "tm_fp8_grouped_swiglu";
  const int bad = check_experts(name, experts, dtype);
  if (bad != TM_OK) return bad;
  TM_REQUIRE(n_tokens >= 0 && top_k >= 1 && ld_ids >= top_k && n_tokens * top_k < ((int64_t)1 << 31) &&
                 ld_x >= experts->hidden,
             TM_EINVAL_SHAPE, "%s: bad sizes", name);
  if (n_tokens == 0) return TM_OK;
  TM_REQUIRE(x && ids && mask && out, TM_EINVAL_ARG, "%s: null pointer", name);
  TM_REQUIRE(aligned(x, ld_x * 2) && tm_aligned16(out) && so_b % 8 == 0 && so_s % 8 == 0, TM_EINVAL_SHAPE,
             "%s: rows of x and of the output must be 16-byte aligned", name);
  const ExpertsWs ws = experts_ws(n_tokens, top_k, experts);
  TM_REQUIRE(workspace != nullptr && workspace_bytes >= ws.total && tm_aligned16(workspace), TM_EWORKSPACE,
             "%s: workspace %zu bytes < %zu", name, workspace_bytes, ws.total);
  char *const base = static_cast<char *>(workspace);
  hipStream_t s = tm_hip_stream(stream);
  const Fp8Src src{x, ld_x, experts->hidden, nullptr, 0};
  Fp8Rows rows{n_tokens};
  rows.top_k = top_k;
  rows.n_experts = experts->n_experts;
  if (n_tokens * top_k <= kMaxSlots) {
    rows.ids = ids;
    rows.ld_ids = ld_ids;
    rows.mask = mask;
    rows.ms_b = ms_b;
    rows.ms_s = ms_s;
  } else {
    int32_t *const offsets = reinterpret_cast<int32_t *>(base + ws.offsets);
    int32_t *const row_token = reinterpret_cast<int32_t *>(base + ws.row_token);
    int64_t *const row_out = reinterpret_cast<int64_t *>(base + ws.row_out);
    const size_t gb = tm_group_slots_workspace_size(n_tokens, top_k, experts->n_experts);
    const int st = tm_group_slots_ws(ids, n_tokens, top_k, ld_ids, mask, ms_b, ms_s, experts->n_experts, so_b, so_s,
                                     offsets, row_token, row_out, reinterpret_cast<int32_t *>(base + ws.tiles),
                                     base + ws.group, gb, stream);
    if (st != TM_OK) return st;
    rows.offsets = offsets;
    rows.row_token = row_token;
    rows.row_out = row_out;
  }
  float *const f = reinterpret_cast<float *>(base + ws.f);
  const Fp8Dst dst{out, 0, so_b, so_s, nullptr, 0};
  return dtype == TM_DT_F16 ? mlp_launch<TM_DT_F16>(name, experts, src, rows, f, dst, s)
                            : mlp_launch<TM_DT_BF16>(name, experts, src, rows, f, dst, s);
}

extern "C" size_t tm_fp8_expert_swiglu_workspace_size(const tm_fp8_experts *experts, int64_t n_rows) {
  if (experts == nullptr || n_rows <= 0) return 0;
  return (size_t)round_up(n_rows * experts->inter * 4, 256);
}

extern "C" int tm_fp8_expert_swiglu(const tm_fp8_experts *experts, int32_t dtype, const void *x, int64_t n_rows,
                                    int64_t ld_x, const void *addend, int64_t ld_add, void *out, int64_t ld_out,
                                    void *workspace, size_t workspace_bytes, tm_stream_t stream) {
  const char *const name = "tm_fp8_expert_swiglu";
  const int bad = check_experts(name, experts, dtype);
  if (bad != TM_OK) return bad;
  TM_REQUIRE(experts->n_experts == 1, TM_EINVAL_SHAPE, "%s: takes the weights of one expert", name);
  TM_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 31) && ld_x >= experts->hidden && ld_out >= experts->hidden &&
                 (addend == nullptr || ld_add >= experts->hidden),
             TM_EINVAL_SHAPE, "%s: bad sizes", name);
  if (n_rows == 0) return TM_OK;
  TM_REQUIRE(x && out, TM_EINVAL_ARG, "%s: null pointer", name);
  TM_REQUIRE(aligned(x, ld_x * 2) && aligned(out, ld_out * 2) && (addend == nullptr || aligned(addend, ld_add * 2)),
             TM_EINVAL_SHAPE, "%s: rows of x, addend and out must be 16-byte aligned", name);
  const size_t need = tm_fp8_expert_swiglu_workspace_size(experts, n_rows);
  TM_REQUIRE(workspace != nullptr && workspace_bytes >= need && tm_aligned16(workspace), TM_EWORKSPACE,
             "%s: workspace %zu bytes < %zu", name, workspace_bytes, need);
  hipStream_t s = tm_hip_stream(stream);
  const Fp8Src src{x, ld_x, experts->hidden, nullptr, 0};
  const Fp8Rows rows{n_rows};
  const Fp8Dst dst{out, ld_out, 0, 0, addend, ld_add};
  float *const f = static_cast<float *>(workspace);
  return dtype == TM_DT_F16 ? mlp_launch<TM_DT_F16>(name, experts, src, rows, f, dst, s)
                            : mlp_launch<TM_DT_BF16>(name, experts, src, rows, f, dst, s);
}
