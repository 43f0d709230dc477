// Products with 8-bit weights (e4m3, one fp32 scale per 128 x 128 block) and
// activations quantised in blocks of 128 columns of a row: a linear layer and
// the SwiGLU MLP of experts.
//
//   y[r][c] = sum_b sx[r][b] sw[c / 128][b] sum_{k in block b} x[r][k] w[c][k]
//
// The MLP: g = x W1^T, u = x W3^T (fp32), f = silu(g) u (fp32, not rounded),
// f quantised in blocks of 128 columns, y = f W2^T (one rounding).
//
// Arithmetic.  The 8-bit matrix instructions add the products of 8 consecutive
// columns aligned to the largest of them and drop what lies under 2^-13 of its
// exponent (the rest of the sum is fp32): sums over normal data come out 1.5e-5
// to 6e-5 of their size off, where the 16-bit instructions are off by 1e-8.
// e4m3 values are exact as bf16, so products whose result is kept in fp32 or is
// quantised again (g and u: an error of 3e-5 there turns roundings of f over,
// which costs y as much as its rounding to bf16) run on the bf16 instructions,
// and those that are rounded to 16 bits once at the end on the 8-bit ones.
#include "tm_fp8.h"
#include "tm_fp8_dev.h"
#include "tm_dma.h"

namespace {

enum { kUp = 0, kOut = 1 };
constexpr int kE4M3 = TM_DT_E4M3;  // activations that are quantised already

// Rows of a streamed call: every row (dense), or the (token, slot) pairs of a
// small batch, found in the launch itself.
struct Fp8Rows {
  int64_t n;  // dense: rows; slots: tokens
  const int64_t *ids;
  int64_t ld_ids;
  const uint8_t *mask;
  int64_t ms_b, ms_s;
  int32_t top_k, n_experts;
  bool by_expert;  // a workgroup's item is an expert (else a slot)
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
// A workgroup of S waves owns NA blocks of 16 weight rows (up: of W1 and of W3).
// Wave w holds blocks [w KPW, (w + 1) KPW) of their 128-column blocks in
// registers, loaded at once (K of more than S KPW: in passes, loaded again for
// each chunk of rows).  The workgroup quantises its rows, up to 16 at a time,
// into LDS (16 lanes own a block of a row), multiplies them (16-bit outputs on the
// 8-bit instructions, else on the bf16 ones) and adds the waves' sums in wave order
// through LDS.  No launch before it groups the rows or quantises them: a call is
// its two products.
//
// Bound by HBM: 256 slots of 110 experts (2048 x 768) stream 352 MB in 64 us (up,
// 5.5 TB/s) and 176 MB in 35 (down, 5.0); one token's 8 experts take 10 + 6, a
// chain of latencies (slots, rows, weights, sums).  More rows cost a load's latency each
// (a row's pieces are loaded behind the weights, one trip after the other): a dense MLP
// of 2560 x 1536 takes 13 us for one row, 22 for 8, 34 for 16.  Up: quantising in the
// operand's layout, where every lane does 32 columns of its row whether it is
// live or not, 140; 48 KiB of LDS rows 81; three waves per SIMD instead of four
// 70; non-temporal weight loads 75; 32 columns per workgroup on eight waves 94.
// Down: 16 columns 119, 32 columns 38, on the 16-bit instructions 38.
// ---------------------------------------------------------------------------
constexpr int kMaxSlots = 1024;  // (token, slot) pairs of a call that are found in the launch
constexpr int kMaxWaves = 8;
constexpr int kStreamLds = 20480;  // bytes of quantised rows

// Rows of a chunk: what fits, 16 at most.
__host__ __device__ inline int stream_chunk(int KT, int64_t most) {
  const int64_t fit = kStreamLds / (KT * (kFp8Block + 4) + 16);
  const int64_t c = fit < 1 ? 1 : fit < 16 ? fit : 16;
  return (int)(c < most ? c : most);
}

template <int DT, int DTX, int MODE, int NA, int KPW>
__global__ __launch_bounds__(64 * kMaxWaves) __attribute__((amdgpu_waves_per_eu(MODE != kUp ? 1 : KPW > 4 ? 3 : 4)))
void stream_kernel(Fp8Src src, Fp8Rows rows, Fp8Mat m0, Fp8Mat m1, int n_out, int KT, int n_groups, int chunk,
                   Fp8Dst dst, bool vec_out) {
  constexpr int NM = MODE == kUp ? 2 : 1;
  constexpr bool WIDE = MODE == kUp || DT == TM_DT_F32;  // on the 16-bit instructions
  // the waves' sums [S][NM * NA][64], the chunk's rows [chunk][KT * 128 + 16] bytes,
  // their scales [chunk][KT], the expert's slots
  extern __shared__ float4 red[];
  __shared__ int s_count, s_first;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int threads = blockDim.x, S = threads >> 6;
  const int t = lane & 15, g = lane >> 4;
  const int x_row = KT * kFp8Block + 16;  // (16 more: rows start on other banks)
  char *const xb = reinterpret_cast<char *>(red + S * NM * NA * 64);
  float *const xs = reinterpret_cast<float *>(xb + chunk * x_row);
  uint16_t *const list = reinterpret_cast<uint16_t *>(xs + chunk * KT);
  const int n0 = (int)(blockIdx.x % n_groups) * (16 * NA);
  const int64_t item = blockIdx.x / n_groups;
  int e = 0;
  int64_t count = rows.n;
  const bool single = rows.n == 1;
  if (rows.ids != nullptr) {
    // This workgroup's expert: `item` (by_expert), or that of slot `item`, whose
    // first slot's workgroups take all of them; a single token's slots are each by
    // themselves (8 slots: 10 + 6 us; 11 + 6 when they searched for each other).
    const int total = (int)rows.n * rows.top_k;
    auto expert_of = [&](int p) {
      const int b = p / rows.top_k, s = p - b * rows.top_k;
      const int64_t id = rows.ids[b * rows.ld_ids + s];
      const bool live = rows.mask[b * rows.ms_b + s * rows.ms_s] != 0;  // (both loads at once)
      return (live & (id >= 0) & (id < rows.n_experts)) ? (int)id : -1;
    };
    e = rows.by_expert ? (int)item : expert_of((int)item);
    if (e < 0) return;  // uniform
    if (single) {
      count = 1;
    } else {
      if (tid == 0) {
        s_count = 0;
        s_first = total;
      }
      __syncthreads();
      for (int p = tid; p < total; p += threads)
        if (expert_of(p) == e) {
          list[atomicAdd(&s_count, 1)] = (uint16_t)p;  // (a row's result does not depend on its place)
          atomicMin(&s_first, p);
        }
      __syncthreads();
      count = s_count;
      if (count == 0 || (!rows.by_expert && s_first != (int)item)) return;  // uniform
    }
  }
  auto slot_of = [&](int64_t i) { return rows.ids == nullptr ? 0 : single ? (int)item : (int)list[i]; };

  uint4 w[NM][NA][KPW][2];
  float sw[NM][KPW];
  const int nb = (n_out + kFp8Block - 1) / kFp8Block;
  const int64_t ld_w = (int64_t)KT * kFp8Block;
  auto load_w = [&](int kb0) {
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const Fp8Mat &mat = m == 0 ? m0 : m1;
      const float *const ps = mat.s + ((int64_t)e * nb + n0 / kFp8Block) * KT;
#pragma unroll
      for (int j = 0; j < KPW; ++j) {
        const int kb = kb0 + j;
        if (kb < KT) {  // uniform
#pragma unroll
          for (int a = 0; a < NA; ++a) {
            const int r = n0 + 16 * a + t < n_out ? n0 + 16 * a + t : n_out - 1;  // (past n_out: not stored)
            const uint8_t *const p = mat.w + ((int64_t)e * n_out + r) * ld_w + (int64_t)kb * kFp8Block + 16 * g;
            w[m][a][j][0] = *reinterpret_cast<const uint4 *>(p);
            w[m][a][j][1] = *reinterpret_cast<const uint4 *>(p + 64);
          }
          sw[m][j] = ps[kb];
        }
      }
    }
  };
  const bool once = KT <= S * KPW;
  if (once) load_w(wave * KPW);
  for (int64_t c0 = 0; c0 < count; c0 += chunk) {
    const int here = (int)(count - c0 < chunk ? count - c0 : chunk);
    // the chunk's rows to LDS: block b of row r by 16 lanes, 8 columns each
    const bool whole = src.k == (int64_t)KT * kFp8Block;  // no row ends inside a block
    for (int i = tid >> 4; i < here * KT; i += threads >> 4) {
      const int r = i / KT, b = i - r * KT;
      const int p = slot_of(c0 + r);
      const int64_t xr = rows.ids == nullptr ? c0 + r : MODE == kUp ? p / rows.top_k : p;
      const int c = b * kFp8Block + t * 8;
      uint2 q;
      float s;
      if constexpr (DTX == kE4M3) {
        q = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(src.x) + xr * src.ld + c);
        s = src.scale[xr * src.ld_s + b];
      } else {
        float v[8];
        const auto *const px = static_cast<const typename Elem<DTX>::T *>(src.x) + xr * src.ld;
        if (whole || c + 8 <= src.k) {
          tm_load8<DTX>(px + c, v);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = c + k < src.k ? Elem<DTX>::to_f(px[c + k]) : 0.f;
        }
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = tm_fp8_amax(m, v[k]);
        m = tm_row16_max(m);
        float inv;
        s = tm_fp8_scale(m, inv);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = tm_fp8_quot(v[k], inv);
        q = make_uint2(tm_fp8_pack4(v[0], v[1], v[2], v[3]), tm_fp8_pack4(v[4], v[5], v[6], v[7]));
      }
      *reinterpret_cast<uint2 *>(xb + r * x_row + c) = q;
      if (t == 0) xs[r * KT + b] = s;
    }
    __syncthreads();
    const int row = t < here ? t : here - 1;  // (lanes past the chunk: its last row again, not stored)
    tm_f32x4 acc[NM][NA];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int a = 0; a < NA; ++a) acc[m][a] = tm_f32x4{};
    for (int kb0 = wave * KPW; kb0 < KT; kb0 += S * KPW) {
      if (!once) load_w(kb0);
#pragma unroll
      for (int j = 0; j < KPW; ++j) {
        const int kb = kb0 + j;
        if (kb >= KT) continue;  // uniform
        const char *const p = xb + row * x_row + kb * kFp8Block + 16 * g;
        const uint4 q0 = *reinterpret_cast<const uint4 *>(p), q1 = *reinterpret_cast<const uint4 *>(p + 64);
        const float sx = xs[row * KT + kb];
        uint4 b[WIDE ? 4 : 2];
        if constexpr (WIDE) {
          b[0] = tm_fp8_to_bf16x8(q0.x, q0.y);
          b[1] = tm_fp8_to_bf16x8(q0.z, q0.w);
          b[2] = tm_fp8_to_bf16x8(q1.x, q1.y);
          b[3] = tm_fp8_to_bf16x8(q1.z, q1.w);
        } else {
          b[0] = q0;
          b[1] = q1;
        }
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
          for (int a = 0; a < NA; ++a) {
            tm_f32x4 d = {};
            if constexpr (WIDE) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint4 &v = w[m][a][j][h];
                d = tm_mfma16x16x32<TM_DT_BF16>(tm_fp8_to_bf16x8(v.x, v.y), b[2 * h], d);
                d = tm_mfma16x16x32<TM_DT_BF16>(tm_fp8_to_bf16x8(v.z, v.w), b[2 * h + 1], d);
              }
            } else {
              d = tm_mfma16x16x128_fp8(w[m][a][j], b, d);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][a][i] = fmaf(d[i], sw[m][j] * sx, acc[m][a][i]);
          }
      }
    }
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int a = 0; a < NA; ++a)
        red[(wave * (NM * NA) + m * NA + a) * 64 + lane] =
            make_float4(acc[m][a][0], acc[m][a][1], acc[m][a][2], acc[m][a][3]);
    __syncthreads();
    for (int i = tid; i < NA * 64; i += threads) {
      // row t of the chunk, columns n0 + 16 a + 4 g .. + 3
      const int a = i >> 6;
      float v[NM][4] = {};
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const float4 p = red[(s * (NM * NA) + m * NA + a) * 64 + (i & 63)];
          v[m][0] += p.x; v[m][1] += p.y; v[m][2] += p.z; v[m][3] += p.w;
        }
      if (t >= here) continue;
      const int c = n0 + 16 * a + 4 * g;
      const int p = slot_of(c0 + t);
      if constexpr (MODE == kUp) {
        float f[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) f[u] = v[0][u] * __builtin_amdgcn_rcpf(1.f + __expf(-v[0][u])) * v[NM - 1][u];
        store4<TM_DT_F32>(dst.y, (rows.ids != nullptr ? p : c0 + t) * dst.ld, f, c, n_out, true);
      } else {
        const int64_t at = rows.ids != nullptr ? (p / rows.top_k) * dst.so_b + (p % rows.top_k) * dst.so_s
                                               : (c0 + t) * dst.ld;
        if (dst.add != nullptr)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (c + u < n_out) v[0][u] += at_f<DT>(dst.add, (c0 + t) * dst.ld_add + c + u);
        store4<DT>(dst.y, at, v[0], c, n_out, vec_out);
      }
    }
    // (the next chunk's rows go to LDS that every wave has read: it wrote its sums
    // after that; its sums go to red after the next barrier)
  }
}

template <int DT, int DTX, int MODE, int NA, int KPW>
int stream_launch(const char *name, const Fp8Src &src, Fp8Rows rows, const Fp8Mat &m0, const Fp8Mat &m1, int n_out,
                  int KT, const Fp8Dst &dst, hipStream_t s) {
  const int n_groups = (int)tm_cdiv(n_out, 16 * NA);
  const int64_t total = rows.ids != nullptr ? rows.n * rows.top_k : rows.n;
  rows.by_expert = rows.ids != nullptr && rows.n > 1 && total >= rows.n_experts;
  const int64_t items = rows.ids == nullptr ? 1 : rows.by_expert ? rows.n_experts : total;
  TM_REQUIRE(items * n_groups < ((int64_t)1 << 31), TM_EINVAL_SHAPE, "%s: too many rows", name);
  const int64_t esz = Elem<DT>::kBytes;
  const bool vec_out = (reinterpret_cast<uintptr_t>(dst.y) & 15) == 0 && dst.ld * esz % 16 == 0 &&
                       dst.so_b * esz % 16 == 0 && dst.so_s * esz % 16 == 0;
  const int waves = (int)(tm_cdiv(KT, KPW) < kMaxWaves ? tm_cdiv(KT, KPW) : kMaxWaves);
  const int chunk = stream_chunk(KT, total);
  hipLaunchKernelGGL((stream_kernel<DT, DTX, MODE, NA, KPW>), dim3((unsigned)(items * n_groups)), dim3(64 * waves),
                     (size_t)waves * ((MODE == kUp ? 2 : 1) * NA) * 1024 + (size_t)chunk * (KT * (kFp8Block + 4) + 16) +
                         (rows.ids != nullptr ? (size_t)total * 2 : 0),
                     s, src, rows, m0, m1, n_out, KT, n_groups, chunk, dst,
                     vec_out);
  TM_LAUNCH_CHECK(name);
  return TM_OK;
}

// ---------------------------------------------------------------------------
// Many rows: tiles through LDS.
//
// Eight waves: wave w owns 64 weight rows of group w % 4 (up: 32 rows of W1 and
// the same 32 of W3) and NB blocks of 32 activation rows of half w / 4, in
// 32 x 32 products.  A stage is a block of 128 columns, global -> LDS by direct
// loads; LDS holds a ring of three, one barrier per stage: it publishes the
// stage and frees the slot of the one before.  A stage's products start from
// zero and are added to the fp32 accumulators times their scales.
//
// Activations come quantised, e4m3 rows and their scales.  The 8-bit
// instructions take them and the weights as they are; WIDE converts both to bf16
// on the way from LDS (up: the rows' scales, powers of two, with them).  Which
// rows of its 64 a lane's operand takes is chosen so that its results are 32
// (up: 16) consecutive columns; 16-byte chunks of an LDS row are XOR-ed with the
// row bits that differ among 16 lanes, so operand reads are free of bank
// conflicts.
//
// Bound by no unit alone: a stage's LDS reads, conversions, products and sums
// follow each other between its barriers (up: matrix units busy 21 % of the cycles,
// vector units 28 %; direct loads alone would take half of the time).  5280 rows of
// 128 experts (2048 x 768): up 130 us (3.1 TB/s), down 64; 14.7 k rows of 64 experts
// (2560 x 1536): up 318-360 us (0.65-0.73 PFLOP/s), down 130-140; a linear layer,
// 4096 rows, 4096 -> 2048: 47 us (1.46 PFLOP/s).  Output rows stored by the lanes
// that hold them, 8 bytes at a time: 87.  The up product with 128 columns of both
// matrices and its sums kept in units of the block's scale, or the waves' halves a
// phase apart (one reads and converts while the other multiplies): 8 % and 17 % slower.
// ---------------------------------------------------------------------------
constexpr int kTileThreads = 512;
constexpr int kTileBM = 128;    // rows of a tile
constexpr int kTileCols = 256;  // weight rows of a tile (up: 128 of W1 and of W3)
constexpr int kTileRing = 3 * (kTileCols * kFp8Block + kTileBM * (kFp8Block + 4));  // LDS bytes of the stages
constexpr int kMaxExperts = 1024;

// Rows of a tiled call: grouped by expert (what tm_group_slots writes), or
// (offsets null) all of one matrix.
struct Fp8Tiles {
  const int32_t *offsets, *row_token;
  const int64_t *row_out;
  int32_t n_experts, rows;  // rows: dense, their number; grouped, the most
  int32_t bm;               // rows of a tile: kTileBM or (dense) 64
};

// A workgroup barrier that LDS accesses stay on their side of.
__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }

// Stage layout for NB blocks of 32 rows per half.
template <int NB>
struct TileCfg {
  static constexpr int kW = kTileCols * kFp8Block;
  static constexpr int kX = 64 * NB * kFp8Block;
  static constexpr int kS = 64 * NB * 4;
  static constexpr int kStage = kW + kX + kS;
  static constexpr int kDma = 4 + NB + 1;  // loads per wave
  static constexpr int kSlots = kTileRing / kStage;
};

template <int MODE>
__device__ __forceinline__ int w_swz(int row) {
  return ((row >> 1) & 1) | (((row >> (MODE == kUp ? 4 : 5)) & 1) << 1) | (((row >> 2) & 1) << 2);
}
__device__ __forceinline__ int x_swz(int row) { return (row >> 1) & 7; }

// Wait until at most `left` stages of kDma loads are outstanding (and LDS reads
// are done).
template <int kDma, int kMost>
__device__ __forceinline__ void wait_stages(int left) {
  if constexpr (kMost <= 0) {
    tm_wait_vm_lgkm0_mem<0>();
  } else {
    if (left >= kMost) tm_wait_vm_lgkm0_mem<kMost * kDma>();
    else wait_stages<kDma, kMost - 1>(left);
  }
}

// A tile of results, [rows][COLS + 4] in LDS, added to and written as whole lines.
template <int DT, int COLS, int THREADS>
__device__ __forceinline__ void write_tile(const float *tile, int rows, int r0, int n0, int n_out, const Fp8Dst &dst,
                                           const int64_t *row_out, bool vec_out) {
  using T = typename Elem<DT>::T;
  constexpr int kLd = COLS + 4, kLanes = COLS / 8;
  T *const y = static_cast<T *>(dst.y);
  const T *const add = static_cast<const T *>(dst.add);
  const int tid = threadIdx.x;
  if (vec_out) {  // 8 columns a lane
    const int c = (tid % kLanes) * 8, col = n0 + c;
    if (col >= n_out) return;
    for (int tr = tid / kLanes; tr < rows; tr += THREADS / kLanes) {
      const int64_t row = r0 + tr;
      const float4 lo = *reinterpret_cast<const float4 *>(tile + tr * kLd + c);
      const float4 hi = *reinterpret_cast<const float4 *>(tile + tr * kLd + c + 4);
      float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      if (add != nullptr) {
        float b[8];
        tm_load8<DT>(add + row * dst.ld_add + col, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += b[i];
      }
      tm_store8<DT>(y + (row_out != nullptr ? row_out[row] : row * dst.ld) + col, v);
    }
  } else {  // a wave a row, a column a lane: 64 neighbours per store
    for (int tr = tid >> 6; tr < rows; tr += THREADS / 64) {
      const int64_t row = r0 + tr;
      const int64_t at = (row_out != nullptr ? row_out[row] : row * dst.ld) + n0;
#pragma unroll
      for (int j = 0; j < COLS / 64; ++j) {
        const int c = (tid & 63) + 64 * j;
        if (n0 + c >= n_out) break;
        const float b = add != nullptr ? Elem<DT>::to_f(add[row * dst.ld_add + n0 + c]) : 0.f;
        y[at + c] = Elem<DT>::from_f(tile[tr * kLd + c] + b);
      }
    }
  }
}

// Whether write_tile may move 8 columns at a time.
template <int DT>
bool can_write8(const Fp8Dst &dst, int n_out) {
  const int64_t esz = Elem<DT>::kBytes;
  return n_out % 8 == 0 && tm_aligned16(dst.y) && dst.ld * esz % 16 == 0 && dst.so_b * esz % 16 == 0 &&
         dst.so_s * esz % 16 == 0 && tm_aligned16(dst.add) && dst.ld_add * esz % 16 == 0;
}

template <int DT, int MODE, bool WIDE>
__global__ __launch_bounds__(kTileThreads, 2) void tile_kernel(const uint8_t *__restrict__ x, int64_t ld_x,
                                                               const float *__restrict__ xs, int64_t ld_xs, Fp8Mat m0,
                                                               Fp8Mat m1, int n_out, int KT, int n_tiles, Fp8Tiles ts,
                                                               Fp8Dst dst, float *__restrict__ fs, bool vec_out) {
  __shared__ uint4 ring[kTileRing / 16];
  __shared__ int s_off[kMaxExperts + 1], s_part[kMaxExperts + 1];  // each expert's first row and first row tile
  __shared__ uint32_t s_top[MODE == kUp ? kTileBM * 4 : 1];
  __shared__ int s_wave[kTileThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cg = wave & 3, half = wave >> 2, t = lane & 31, h = lane >> 5;
  const uint32_t lds0 = (uint32_t)(uintptr_t)ring;
  const char *const lds = reinterpret_cast<const char *>(ring);
  const int64_t ld_w = (int64_t)KT * kFp8Block;
  const int n_blk = (n_out + kFp8Block - 1) / kFp8Block;

  // Row tiles, counted here: no tile is empty.
  const bool grouped = ts.offsets != nullptr;
  int n_parts = (ts.rows + ts.bm - 1) / ts.bm;
  if (grouped) {
    int o[3], c[2];
#pragma unroll
    for (int u = 0; u < 3; ++u) o[u] = ts.offsets[2 * tid + u < ts.n_experts ? 2 * tid + u : ts.n_experts];
#pragma unroll
    for (int u = 0; u < 2; ++u) c[u] = (o[u + 1] - o[u] + kTileBM - 1) / kTileBM;
    const int upto = (int)tm_wave_incl_scan((uint32_t)(c[0] + c[1]));
    if (lane == 63) s_wave[wave] = upto;
    __syncthreads();
    int before = upto - c[0] - c[1];
    n_parts = 0;
#pragma unroll
    for (int w = 0; w < kTileThreads / 64; ++w) {
      before += w < wave ? s_wave[w] : 0;
      n_parts += s_wave[w];
    }
    s_off[2 * tid] = o[0];
    s_off[2 * tid + 1] = o[1];
    s_part[2 * tid] = before;
    s_part[2 * tid + 1] = before + c[0];
    if (tid == kTileThreads - 1) {
      s_off[kMaxExperts] = o[2];
      s_part[kMaxExperts] = n_parts;
    }
    __syncthreads();
  }
  n_parts = __builtin_amdgcn_readfirstlane(n_parts);

  // Work items: (row tile, column tile), row tile by row tile; XCD x (the
  // dispatcher's round robin) takes the x-th eighth of them, so the column tiles
  // of a row tile and the row tiles of an expert run at the same time on one L2.
  // A workgroup takes every (its XCD's workgroups)-th of its eighth: a launch
  // holds one workgroup per CU, whatever the rows.
  const int64_t total = (int64_t)n_parts * n_tiles;
  const int xcd = (int)(blockIdx.x & 7), on_xcd = ((int)gridDim.x - xcd + 7) / 8;
  const int64_t last = total * (xcd + 1) / 8;
  for (int64_t item = total * xcd / 8 + (blockIdx.x >> 3); item < last; item += on_xcd) {
    const int part = (int)(item / n_tiles);
    const int n0 = (int)(item % n_tiles) * (MODE == kUp ? kTileCols / 2 : kTileCols);
    int e = 0, r0 = part * ts.bm, r_end = ts.rows;
    if (grouped) {
      int n = 0;  // experts whose tiles all come before this one
      for (int i = 0; i < ts.n_experts; i += 64)
        n += __popcll(__ballot(i + lane < ts.n_experts && s_part[i + lane + 1] <= part));
      e = n;
      r0 = __builtin_amdgcn_readfirstlane(s_off[e] + (part - s_part[e]) * kTileBM);
      r_end = __builtin_amdgcn_readfirstlane(s_off[e + 1]);
    }
    const int rows = r_end - r0 < ts.bm ? r_end - r0 : ts.bm;
    r_end = r0 + rows;

    // weight loads: 1 KiB pieces 4 wave + j, 8 rows each (up: waves 0-3 W1, waves 4-7 W3)
    const Fp8Mat &mine = MODE == kUp && wave >= 4 ? m1 : m0;
    constexpr int kWRows = MODE == kUp ? kTileCols / 2 : kTileCols;
    const int w_rows = n_out - n0 < kWRows ? n_out - n0 : kWRows;
    const tm_rsrc_t w_rs = tm_make_rsrc(mine.w + ((int64_t)e * n_out + n0) * ld_w, (uint64_t)w_rows * ld_w);
    uint32_t w_off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int row = ((MODE == kUp ? wave & 3 : wave) * 4 + j) * 8 + (lane >> 3);
      const int chunk = (lane & 7) ^ w_swz<MODE>(row);
      row = row < w_rows ? row : w_rows - 1;  // (results of rows past n_out are dropped)
      w_off[j] = (uint32_t)row * (uint32_t)ld_w + (uint32_t)chunk * 16u;
    }
    // operand row t of block a: weight row
    //   out: 64 cg + 32 (t / 4 % 2) + 16 a + 4 (t / 8) + t % 4
    //   up:  32 cg + 16 (t / 4 % 2) + 4 (t / 8) + t % 4 of matrix a
    // its chunk 2 c + h (c = 0 .. 3), of both operands: the same columns
    uint32_t a_off[4];  // (of block 0)
    {
      const int row = MODE == kUp ? 32 * cg + 16 * ((t >> 2) & 1) + 4 * (t >> 3) + (t & 3)
                                  : 64 * cg + 32 * ((t >> 2) & 1) + 4 * (t >> 3) + (t & 3);
#pragma unroll
      for (int c = 0; c < 4; ++c) a_off[c] = (uint32_t)(row * kFp8Block + ((2 * c + h) ^ w_swz<MODE>(row)) * 16);
    }
    constexpr uint32_t kABlock = (MODE == kUp ? 128 : 16) * kFp8Block;  // block 1 (its swizzle is block 0's)
    // the wave's scales of 64 blocks, one per lane
    const int blk = (MODE == kUp ? n0 : n0 + cg * 64) / kFp8Block;
    const int64_t s_at = ((int64_t)e * n_blk + (blk < n_blk ? blk : n_blk - 1)) * KT;
    float swv[2] = {0.f, 0.f};
    auto load_sw = [&](int kt) {
      const int k = kt + lane < KT ? kt + lane : KT - 1;
      swv[0] = m0.s[s_at + k];
      if constexpr (MODE == kUp) swv[1] = m1.s[s_at + k];
    };
    // The compiler waits for the scales here; at their use, in the loop, its wait
    // would be one for every direct load in flight, which it does not count (that took
    // 149 + 74 us where this takes 132 + 66: 5280 rows of 128 experts).
    auto pin_sw = [&] { asm volatile("" : "+v"(swv[0]), "+v"(swv[1])); };
    load_sw(0);

    tm_f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int q = 0; q < 2; ++q) acc[a][q] = tm_f32x16{};

    auto run = [&](auto nb_c) {
      constexpr int NB = decltype(nb_c)::value;
      using Cfg = TileCfg<NB>;
      constexpr int S = Cfg::kSlots;
      auto row_of = [&](int tr) {  // a row past the tile: its last one again, results dropped
        int gr = r0 + tr;
        gr = gr < r_end ? gr : r_end - 1;
        return MODE == kUp && ts.row_token != nullptr ? (int64_t)ts.row_token[gr] : (int64_t)gr;
      };
      const uint8_t *x_src[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int tr = (wave * NB + j) * 8 + (lane >> 3);
        x_src[j] = x + row_of(tr) * ld_x + ((lane & 7) ^ x_swz(tr)) * 16;
      }
      const float *const s_src = xs + row_of((wave % NB) * 64 + lane) * ld_xs;
      const uint32_t s_dst = (uint32_t)(Cfg::kW + Cfg::kX + (wave % NB) * 256);
      auto issue = [&](int kt, uint32_t slot) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          tm_dma16_buf_so(w_rs, w_off[j], (uint32_t)kt * kFp8Block, lds0 + slot + (uint32_t)(wave * 4 + j) * 1024u);
#pragma unroll
        for (int j = 0; j < NB; ++j)
          tm_dma16_s(x_src[j] + (int64_t)kt * kFp8Block, lds0 + slot + (uint32_t)(Cfg::kW + (wave * NB + j) * 1024));
        tm_dma4_s(s_src + kt, lds0 + slot + s_dst);
      };
      const int tr0 = half * NB * 32 + t;
      uint32_t b_off[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) b_off[c] = (uint32_t)(Cfg::kW + tr0 * kFp8Block + ((2 * c + h) ^ x_swz(tr0)) * 16);
      pin_sw();
      for (int kt = 0; kt < S && kt < KT; ++kt) issue(kt, (uint32_t)(kt * Cfg::kStage));
      uint32_t slot = 0, prev = (S - 1) * Cfg::kStage;
      for (int kt = 0; kt < KT; ++kt) {
        const int left = KT - 1 - kt;
        wait_stages<Cfg::kDma, S - 2>(left < S - 2 ? left : S - 2);
        barrier();  // stage kt landed, in every wave; every wave has read stage kt - 1
        if (kt > 0 && kt - 1 + S < KT) issue(kt - 1 + S, prev);
        const char *const sp = lds + slot;
        const float sw0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(swv[0]), kt & 63));
        const float sw1 = MODE == kUp ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(swv[1]), kt & 63)) : sw0;
        uint4 af[2][WIDE ? 8 : 4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const uint4 r = *reinterpret_cast<const uint4 *>(sp + a_off[c] + a * kABlock);
            if constexpr (WIDE) {
              af[a][2 * c] = tm_fp8_to_bf16x8(r.x, r.y);
              af[a][2 * c + 1] = tm_fp8_to_bf16x8(r.z, r.w);
            } else {
              af[a][c] = r;
            }
          }
#pragma unroll
        for (int q = 0; q < NB; ++q) {
          const float sx = *reinterpret_cast<const float *>(sp + Cfg::kW + Cfg::kX + (tr0 + 32 * q) * 4);
          tm_f32x16 p[2] = {};
          if constexpr (WIDE) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint4 r = *reinterpret_cast<const uint4 *>(sp + b_off[c] + q * 32 * kFp8Block);
              const float s = MODE == kUp ? sx : 1.f;
              const uint4 b[2] = {tm_fp8_to_bf16x8(r.x, r.y, s), tm_fp8_to_bf16x8(r.z, r.w, s)};
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int a = 0; a < 2; ++a) p[a] = tm_mfma32x32x16<TM_DT_BF16>(af[a][2 * c + u], b[u], p[a]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              const uint4 b[2] = {*reinterpret_cast<const uint4 *>(sp + b_off[c] + q * 32 * kFp8Block),
                                  *reinterpret_cast<const uint4 *>(sp + b_off[c + 1] + q * 32 * kFp8Block)};
#pragma unroll
              for (int a = 0; a < 2; ++a) {
                const uint4 w2[2] = {af[a][c], af[a][c + 1]};
                p[a] = tm_mfma32x32x64_fp8(w2, b, p[a]);
              }
            }
          }
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const float s = MODE == kUp ? (a == 1 ? sw1 : sw0) : sw0 * sx;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][q][i] = fmaf(p[a][i], s, acc[a][q][i]);
          }
        }
        if (((kt + 1) & 63) == 0 && kt + 1 < KT) {
          load_sw(kt + 1);
          pin_sw();
        }
        prev = slot;
        slot = slot == (S - 1) * Cfg::kStage ? 0u : slot + Cfg::kStage;
      }
    };
    const int used = rows > 64 ? 2 : 1;  // row blocks per half
    if (used == 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
    const int first = half * used * 32 + t;  // this lane's first row in the tile

    if constexpr (MODE == kUp) {
      // lane: row t of each block, columns n0 + 32 cg + 16 h + i; s_top: [128 rows][4 groups]
      const int c = n0 + cg * 32 + 16 * h;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q >= used) continue;  // uniform
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float gv = acc[0][q][i];
          acc[0][q][i] = gv * __builtin_amdgcn_rcpf(1.f + __expf(-gv)) * acc[1][q][i];
          m = tm_fp8_amax(m, acc[0][q][i]);
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        if (h == 0) s_top[(first + 32 * q) * 4 + cg] = m;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int tr = first + 32 * q;
        if (q >= used || tr >= rows) continue;
        const uint4 m4 = *reinterpret_cast<const uint4 *>(&s_top[tr * 4]);
        float inv;
        const float s = tm_fp8_scale(max(max(m4.x, m4.y), max(m4.z, m4.w)), inv);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = tm_fp8_quot(acc[0][q][i], inv);
        *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(dst.y) + (int64_t)(r0 + tr) * dst.ld + c) =
            make_uint4(tm_fp8_pack4(v[0], v[1], v[2], v[3]), tm_fp8_pack4(v[4], v[5], v[6], v[7]),
                       tm_fp8_pack4(v[8], v[9], v[10], v[11]), tm_fp8_pack4(v[12], v[13], v[14], v[15]));
        if (h == 0 && cg == 0) fs[(int64_t)(r0 + tr) * n_blk + n0 / kFp8Block] = s;
      }
    } else {
      // Through LDS, so that a row's columns are added to and written as whole
      // lines: every lane storing its own row's columns, 8 bytes at a time, took
      // 34 us of a 4096 x 2048 product's 87.
      tm_wait_vm_lgkm0_mem<0>();
      barrier();  // the ring is free
      float *const tile = reinterpret_cast<float *>(ring);  // [128 rows][kTileCols + 4]
      constexpr int kLd = kTileCols + 4;
      static_assert(kTileBM * kLd * 4 <= kTileRing, "output tile");
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q >= used) continue;  // uniform
        float *const p = tile + (first + 32 * q) * kLd + cg * 64 + 32 * h;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<float4 *>(p + 4 * u) =
              make_float4(acc[u >> 2][q][4 * (u & 3)], acc[u >> 2][q][4 * (u & 3) + 1], acc[u >> 2][q][4 * (u & 3) + 2],
                          acc[u >> 2][q][4 * (u & 3) + 3]);
      }
      __syncthreads();
      write_tile<DT, kTileCols, kTileThreads>(tile, rows, r0, n0, n_out, dst, ts.row_out, vec_out);
    }
    __syncthreads();  // the next item's loads come after this one's reads of LDS
  }
}

template <int DT, int MODE, bool WIDE>
int tile_launch(const char *name, const void *x, int64_t ld_x, const float *xs, int64_t ld_xs, const Fp8Mat &m0,
                const Fp8Mat &m1, int n_out, int KT, Fp8Tiles ts, const Fp8Dst &dst, float *fs, hipStream_t s) {
  const int n_tiles = (int)tm_cdiv(n_out, MODE == kUp ? kTileCols / 2 : kTileCols);
  // Tiles of 64 rows where tiles of 128 would leave half of the CUs without one
  // (linear, 700 rows, 2048 -> 2816 in bf16: 20 us, 26 in tiles of 128; 1000 rows,
  // 2560 -> 4096: 26 and 33).
  ts.bm = ts.offsets == nullptr && tm_cdiv(ts.rows, kTileBM) * n_tiles <= 128 ? 64 : kTileBM;
  // one workgroup per CU, or fewer where there cannot be as many tiles
  const int64_t parts = tm_cdiv(ts.rows, ts.bm) + (ts.offsets != nullptr ? ts.n_experts : 0);
  const int64_t grid = parts * n_tiles < 256 ? tm_cdiv(parts * n_tiles, 8) * 8 : 256;
  hipLaunchKernelGGL((tile_kernel<DT, MODE, WIDE>), dim3((unsigned)grid), dim3(kTileThreads), 0, s,
                     static_cast<const uint8_t *>(x), ld_x, xs, ld_xs, m0, m1, n_out, KT, n_tiles, ts, dst, fs,
                     can_write8<DT>(dst, n_out));
  TM_LAUNCH_CHECK(name);
  return TM_OK;
}

// ---------------------------------------------------------------------------
// A linear layer of some rows: 64 x 64 tiles, so that few rows still give many CUs a
// workgroup.  Four waves, one 32 x 32 product each; a stage is two blocks of 128
// columns.  Bound by what a CU's direct loads bring, about 45 bytes/ns at any depth
// of the ring (nine stages of one block: 0.38 us a block as well): 64 rows,
// 4096 -> 2048 take 18 us with the rows' quantisation, in the large tiles 27;
// 333 rows, 1000 -> 1111 in fp32 12 and 20.
// ---------------------------------------------------------------------------
constexpr int kMidThreads = 256, kMidTile = 64;
constexpr int kMidW = kMidTile * kFp8Block, kMidBlock = 2 * kMidW + kMidTile * 4;  // LDS bytes of 128 columns
constexpr int kMidStage = 2 * kMidBlock, kMidSlots = 4, kMidDma = 2 * 5;  // stages in LDS, loads per wave and stage

template <int DT, bool WIDE>
__global__ __launch_bounds__(kMidThreads, 1) void mid_kernel(const uint8_t *__restrict__ x, int64_t ld_x,
                                                             const float *__restrict__ xs, int64_t ld_xs, Fp8Mat mat,
                                                             int n_rows, int n_out, int KT, int n_parts, int total,
                                                             Fp8Dst dst, bool vec_out) {
  __shared__ uint4 ring[kMidSlots * kMidStage / 16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cg = wave & 1, half = wave >> 1, t = lane & 31, h = lane >> 5;
  const uint32_t lds0 = (uint32_t)(uintptr_t)ring;
  const char *const lds = reinterpret_cast<const char *>(ring);
  // XCD x takes the x-th eighth of the tiles, row tiles first: they share weights
  const int xcd = (int)(blockIdx.x & 7);
  const int item = (int)((int64_t)total * xcd / 8) + (int)(blockIdx.x >> 3);
  if (item >= (int)((int64_t)total * (xcd + 1) / 8)) return;
  const int n0 = item / n_parts * kMidTile, r0 = item % n_parts * kMidTile;
  const int rows = n_rows - r0 < kMidTile ? n_rows - r0 : kMidTile;
  const int w_rows = n_out - n0 < kMidTile ? n_out - n0 : kMidTile;

  const int64_t ld_w = (int64_t)KT * kFp8Block;
  const float *const sw_src = mat.s + (int64_t)(n0 / kFp8Block) * KT;
  float swv = 0.f;  // 64 blocks' scales, one per lane
  auto load_sw = [&](int kt) { swv = sw_src[kt + lane < KT ? kt + lane : KT - 1]; };
  auto pin_sw = [&] { asm volatile("" : "+v"(swv)); };  // (waited for here: see tile_kernel)
  load_sw(0);
  pin_sw();
  const tm_rsrc_t w_rs = tm_make_rsrc(mat.w + (int64_t)n0 * ld_w, (uint64_t)w_rows * ld_w);
  uint32_t w_off[2];
  const uint8_t *x_src[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // rows past the end: the last one again, results dropped
    const int row = (wave * 2 + j) * 8 + (lane >> 3);
    w_off[j] = (uint32_t)(row < w_rows ? row : w_rows - 1) * (uint32_t)ld_w + (uint32_t)((lane & 7) ^ w_swz<kUp>(row)) * 16u;
    x_src[j] = x + (int64_t)(r0 + (row < rows ? row : rows - 1)) * ld_x + ((lane & 7) ^ x_swz(row)) * 16;
  }
  const float *const s_src = xs + (int64_t)(r0 + (lane < rows ? lane : rows - 1)) * ld_xs;
  auto issue = [&](int st, uint32_t slot) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int kt = 2 * st + u < KT ? 2 * st + u : KT - 1;  // (a block past the end is not used)
      const uint32_t at = lds0 + slot + (uint32_t)(u * kMidBlock);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        tm_dma16_buf_so(w_rs, w_off[j], (uint32_t)kt * kFp8Block, at + (uint32_t)(wave * 2 + j) * 1024u);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        tm_dma16_s(x_src[j] + (int64_t)kt * kFp8Block, at + (uint32_t)(kMidW + (wave * 2 + j) * 1024));
      tm_dma4_s(s_src + kt, at + (uint32_t)(2 * kMidW));
    }
  };
  // operand rows and columns as in the up product of tile_kernel
  const int a_row = 32 * cg + 16 * ((t >> 2) & 1) + 4 * (t >> 3) + (t & 3), tr = half * 32 + t;
  const uint32_t a_off = (uint32_t)(a_row * kFp8Block + (h ^ w_swz<kUp>(a_row)) * 16);
  const uint32_t b_off = (uint32_t)(kMidW + tr * kFp8Block + (h ^ x_swz(tr)) * 16);
  tm_f32x16 acc = {};
  const int n_st = (KT + 1) / 2;
  for (int st = 0; st < kMidSlots && st < n_st; ++st) issue(st, (uint32_t)(st * kMidStage));
  uint32_t slot = 0, prev = (kMidSlots - 1) * kMidStage;
  for (int st = 0; st < n_st; ++st) {
    const int left = n_st - 1 - st;
    wait_stages<kMidDma, kMidSlots - 2>(left < kMidSlots - 2 ? left : kMidSlots - 2);
    barrier();  // the stage landed, in every wave; every wave has read the one before
    uint4 a[2][4], b[2][4];
    float sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const char *const sp = lds + slot + u * kMidBlock;
      const float sw = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(swv), (2 * st + u) & 63));
      sc[u] = sw * *reinterpret_cast<const float *>(sp + 2 * kMidW + tr * 4);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        a[u][c] = *reinterpret_cast<const uint4 *>(sp + (a_off ^ (c << 5)));
        b[u][c] = *reinterpret_cast<const uint4 *>(sp + (b_off ^ (c << 5)));
      }
    }
    if (st > 0 && st - 1 + kMidSlots < n_st) issue(st - 1 + kMidSlots, prev);
    tm_static_for<2>([&](auto u_c) {
      constexpr int u = decltype(u_c)::value;
      if (u == 1 && 2 * st + 1 >= KT) return;
      tm_f32x16 p = {};
      if constexpr (WIDE) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          p = tm_mfma32x32x16<TM_DT_BF16>(tm_fp8_to_bf16x8(a[u][c].x, a[u][c].y), tm_fp8_to_bf16x8(b[u][c].x, b[u][c].y), p);
          p = tm_mfma32x32x16<TM_DT_BF16>(tm_fp8_to_bf16x8(a[u][c].z, a[u][c].w), tm_fp8_to_bf16x8(b[u][c].z, b[u][c].w), p);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          const uint4 a2[2] = {a[u][c], a[u][c + 1]}, b2[2] = {b[u][c], b[u][c + 1]};
          p = tm_mfma32x32x64_fp8(a2, b2, p);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = fmaf(p[i], sc[u], acc[i]);
    });
    if (((st + 1) & 31) == 0 && st + 1 < n_st) {
      load_sw(2 * st + 2);
      pin_sw();
    }
    prev = slot;
    slot = slot == (kMidSlots - 1) * kMidStage ? 0u : slot + kMidStage;
  }
  tm_wait_vm_lgkm0_mem<0>();
  barrier();  // the ring is free
  constexpr int kLd = kMidTile + 4;
  float *const tile = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int i = 0; i < 16; i += 4)
    *reinterpret_cast<float4 *>(tile + tr * kLd + cg * 32 + 16 * h + i) =
        make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
  __syncthreads();
  write_tile<DT, kMidTile, kMidThreads>(tile, rows, r0, n0, n_out, dst, nullptr, vec_out);
}

template <int DT, bool WIDE>
int mid_launch(const char *name, const void *x, int64_t ld_x, const float *xs, int64_t ld_xs, const Fp8Mat &mat,
               int64_t n_rows, int n_out, int KT, const Fp8Dst &dst, hipStream_t s) {
  const int64_t parts = tm_cdiv(n_rows, kMidTile), total = parts * tm_cdiv(n_out, kMidTile);
  hipLaunchKernelGGL((mid_kernel<DT, WIDE>), dim3((unsigned)(tm_cdiv(total, 8) * 8)), dim3(kMidThreads), 0, s,
                     static_cast<const uint8_t *>(x), ld_x, xs, ld_xs, mat, (int)n_rows, n_out, KT, (int)parts,
                     (int)total, dst, can_write8<DT>(dst, n_out));
  TM_LAUNCH_CHECK(name);
  return TM_OK;
}

bool aligned(const void *p, int64_t stride_bytes) { return tm_aligned16(p) && stride_bytes % 16 == 0; }

int64_t round_up(int64_t v, int64_t m) { return tm_cdiv(v, m) * m; }

}  // namespace

// ---------------------------------------------------------------------------
// linear
// ---------------------------------------------------------------------------
namespace {

// Rows up to which a linear layer streams its weights (stream_kernel), by what the
// row quantisation in every workgroup costs it against tiles, whose own is a launch.
// 2048 -> 4096 in bf16: 8 rows 8.3 us (as 64 x 64 tiles 10.7), 16 rows 13 (10.9);
// 4096 -> 2048: 10.5 (16.6) and 17 (16.6).  K of more than 4096 is read again for
// each chunk of rows: 8192 -> 2048, 4 rows, two chunks: 18 (28), 8 rows 31 (28).
// Where 64 x 64 tiles fill half of the CUs they win earlier: 2048 -> 16384, 4 rows
// 10.3 (11.8), 8 rows 13.8 (11.9); 8192 -> 16384, 2 rows 32 (29).
int64_t linear_stream_rows(int64_t kb, int64_t n_out) {
  const int64_t chunk = stream_chunk((int)kb, 16);
  if (n_out > 128 * kMidTile) return chunk > 2 ? chunk / 2 : 1;
  return kb <= 32 ? 12 : 2 * chunk;
}
// 64 x 64 tiles up to which it takes mid_kernel, one per CU: 512 rows, 4096 -> 2048
// (256 tiles) take 22 us, in the large tiles 31; 2048 -> 4096 (512) 24 and 20.
constexpr int64_t kMidTiles = 256;

}  // namespace

extern "C" size_t tm_fp8_linear_workspace_size(int64_t n_rows, int64_t k, int32_t dtype) {
  if (n_rows <= 0 || k <= 0) return 0;
  const int64_t kb = tm_cdiv(k, kFp8Block);
  return (size_t)(round_up(n_rows * kb * kFp8Block, 256) + round_up(n_rows * kb * 4, 256));
}

extern "C" int tm_fp8_linear(int32_t dtype, const void *x, const float *x_scale, int64_t n_rows, int64_t k, int64_t ld_x,
                             int64_t ld_xs, const void *w, const float *w_scale, int64_t n_out, const void *bias,
                             void *out, int64_t ld_out, void *workspace, size_t workspace_bytes, tm_stream_t stream) {
  const char *const name = "tm_fp8_linear";
  TM_REQUIRE(dtype == TM_DT_F32 || dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE,
             "%s: unsupported dtype tag %d", name, (int)dtype);
  const int64_t kb = tm_cdiv(k < 0 ? 0 : k, kFp8Block), kp = kb * kFp8Block;
  TM_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 31) - 256 && k >= 1 && k <= 16384 && n_out >= 1 &&
                 n_out < ((int64_t)1 << 24),
             TM_EINVAL_SHAPE, "%s: bad sizes (%lld rows, %lld columns, %lld outputs)", name, (long long)n_rows,
             (long long)k, (long long)n_out);
  TM_REQUIRE(ld_x >= (x_scale ? kp : k) && ld_out >= n_out && (!x_scale || ld_xs >= kb), TM_EINVAL_SHAPE,
             "%s: row strides (%lld, %lld) are shorter than the rows", name, (long long)ld_x, (long long)ld_out);
  if (n_rows == 0) return TM_OK;
  TM_REQUIRE(x && w && w_scale && out, TM_EINVAL_ARG, "%s: null pointer", name);
  TM_REQUIRE(tm_aligned16(w), TM_EINVAL_SHAPE, "%s: w must be 16-byte aligned", name);
  TM_REQUIRE(!x_scale || aligned(x, ld_x), TM_EINVAL_SHAPE, "%s: rows of 8-bit x must be 16-byte aligned", name);
  const size_t need = tm_fp8_linear_workspace_size(n_rows, k, dtype);
  TM_REQUIRE(workspace != nullptr && workspace_bytes >= need && tm_aligned16(workspace), TM_EWORKSPACE,
             "%s: workspace %zu bytes < %zu", name, workspace_bytes, need);
  hipStream_t s = tm_hip_stream(stream);
  const bool tiles = n_rows > linear_stream_rows(kb, n_out);
  Fp8Src src{x, ld_x, k, x_scale, ld_xs};
  float *const ws_scale = reinterpret_cast<float *>(static_cast<char *>(workspace) + need - round_up(n_rows * kb * 4, 256));
  if (!x_scale && (tiles || !aligned(x, ld_x * (dtype == TM_DT_F32 ? 4 : 2)))) {
    const int st = tm_internal_fp8_rows(dtype, x, n_rows, k, ld_x, workspace, kp, ws_scale, kb, s);
    if (st != TM_OK) return st;
    src = Fp8Src{workspace, kp, kp, ws_scale, kb};
  }
  const Fp8Rows rows{n_rows};
  const Fp8Mat m{static_cast<const uint8_t *>(w), w_scale};
  const Fp8Dst dst{out, ld_out, 0, 0, bias, 0};
  if (!tiles)
    return TM_DISPATCH_DTYPE(dtype, DT, [&] {
      return src.scale ? stream_launch<DT, kE4M3, kOut, 1, 4>(name, src, rows, m, m, (int)n_out, (int)kb, dst, s)
                       : stream_launch<DT, DT, kOut, 1, 4>(name, src, rows, m, m, (int)n_out, (int)kb, dst, s);
    });
  Fp8Tiles ts{};
  ts.rows = (int32_t)n_rows;
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    if (tm_cdiv(n_rows, kMidTile) * tm_cdiv(n_out, kMidTile) <= kMidTiles)
      return mid_launch<DT, DT == TM_DT_F32>(name, src.x, src.ld, src.scale, src.ld_s, m, n_rows, (int)n_out, (int)kb,
                                             dst, s);
    return tile_launch<DT, kOut, DT == TM_DT_F32>(name, src.x, src.ld, src.scale, src.ld_s, m, m, (int)n_out, (int)kb,
                                                  ts, dst, nullptr, s);
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

// Rows of a call up to which the weights are streamed (stream_kernel; no launch
// groups the rows or quantises them), more go through tiles: about two rows per
// expert, and more where there are few experts to fill the CUs; fewer where K is
// read again for each chunk of rows.  Both, in us: 128 experts (2048 x 768) of 2 rows
// 109 | 127, of 4 rows 145 | 134; 64 (2560 x 1536) of 1.5 rows 153 | 141, of 3 207 |
// 158; 16 (4096 x 1024) of 2 rows 46 | 58, of 4 61 | 59; one (2560 x 1536) of 16 rows
// 31 | 38, of 24 40 | 39; 8 (7168 x 2048) of 2 rows 91 | 100, of 4 143 | 101; one of 8
// rows 57 | 77, of 12 82 | 77.
int64_t stream_rows(const tm_fp8_experts *ex) {
  const int64_t most = 2 * (int64_t)ex->n_experts + (ex->hidden <= 4096 && ex->inter <= 4096 ? 14 : 6);
  return most < kMaxSlots ? most : kMaxSlots;
}

// Workspace: f (stream: fp32 rows; tiles: 8-bit rows and their scales), the
// quantised activations and the row lists of the tiles.
struct ExpertsWs {
  size_t f, fs, x, xs, offsets, row_token, row_out, tiles, group, total;
};

ExpertsWs experts_ws(int64_t n, int32_t top_k, const tm_fp8_experts *ex, bool grouped) {
  ExpertsWs w{};
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)round_up(bytes, 256);
    return here;
  };
  const int64_t rows = n * top_k;
  const bool stream = rows <= stream_rows(ex);
  if (stream) take(rows * ex->inter * 4);  // f, at the start
  const size_t stream_bytes = at;
  at = 0;
  w.f = take(rows * ex->inter);
  w.fs = take(rows * (ex->inter / kFp8Block) * 4);
  w.x = take(n * ex->hidden);
  w.xs = take(n * (ex->hidden / kFp8Block) * 4);
  if (grouped) {
    w.offsets = take(4 * ((int64_t)ex->n_experts + 1));
    w.row_token = take(4 * rows);
    w.row_out = take(8 * rows);
    w.tiles = take(4 * (2 + 2 * tm_group_slots_tiles(rows, ex->n_experts)));
    w.group = take((int64_t)tm_group_slots_workspace_size(n < 8192 ? n : 8192, top_k, ex->n_experts));
  }
  // never less for more rows: the largest call that streams needs this much
  if (!stream) {
    const size_t largest = (size_t)round_up(stream_rows(ex) * ex->inter * 4, 256);
    at = at > largest ? at : largest;
  } else {
    at = at > stream_bytes ? at : stream_bytes;
  }
  w.total = at;
  return w;
}

template <int DT>
int mlp_launch(const char *name, const tm_fp8_experts *ex, const void *x, int64_t ld_x, int64_t n, const Fp8Rows *rows,
               const Fp8Tiles *ts, const ExpertsWs &ws, char *base, const Fp8Dst &dst, hipStream_t s) {
  const int h = ex->hidden, inter = ex->inter;
  const Fp8Mat w1{static_cast<const uint8_t *>(ex->w1), ex->s1}, w3{static_cast<const uint8_t *>(ex->w3), ex->s3},
      w2{static_cast<const uint8_t *>(ex->w2), ex->s2};
  const Fp8Dst mid{base + ws.f, inter, 0, 0, nullptr, 0};
  if (ts == nullptr) {
    // Blocks per wave: what makes whole sets of four waves, one per SIMD.  Up: five
    // where four do not (64 experts of 2560 x 1536, 38 of them with rows: 75 us against 89;
    // not where K takes more than eight waves: 7168, 67 against 59).  Down: two where
    // that does, or three (the same 38: 38 us against 51, 109 of 2048 x 768: 43 against 45;
    // but K of 1024: 14.4 against 13.0).
    const int KT = h / kFp8Block, KT2 = inter / kFp8Block;
    const Fp8Src src{x, ld_x, h, nullptr, 0}, mid_src{base + ws.f, inter, inter, nullptr, 0};
    const int w5 = (KT + 4) / 5;
    const int st = (KT + 3) / 4 % 4 != 0 && w5 % 4 == 0 && w5 <= kMaxWaves
                       ? stream_launch<DT, DT, kUp, 1, 5>(name, src, *rows, w1, w3, inter, KT, mid, s)
                       : stream_launch<DT, DT, kUp, 1, 4>(name, src, *rows, w1, w3, inter, KT, mid, s);
    if (st != TM_OK) return st;
    return (KT2 + 1) / 2 % 4 == 0
               ? stream_launch<DT, TM_DT_F32, kOut, 4, 2>(name, mid_src, *rows, w2, w2, h, KT2, dst, s)
               : stream_launch<DT, TM_DT_F32, kOut, 4, 3>(name, mid_src, *rows, w2, w2, h, KT2, dst, s);
  }
  float *const xs = reinterpret_cast<float *>(base + ws.xs);
  int st = tm_internal_fp8_rows(DT, x, n, h, ld_x, base + ws.x, h, xs, h / kFp8Block, s);
  if (st != TM_OK) return st;
  float *const fs = reinterpret_cast<float *>(base + ws.fs);
  st = tile_launch<DT, kUp, true>(name, base + ws.x, h, xs, h / kFp8Block, w1, w3, inter, h / kFp8Block, *ts, mid, fs,
                                  s);
  if (st != TM_OK) return st;
  return tile_launch<DT, kOut, false>(name, base + ws.f, inter, fs, inter / kFp8Block, w2, w2, h, inter / kFp8Block, *ts,
                                      dst, nullptr, s);
}

}  // namespace

extern "C" size_t tm_fp8_grouped_swiglu_workspace_size(const tm_fp8_experts *experts, int64_t n_tokens,
                                                       int32_t top_k) {
  if (experts == nullptr || n_tokens <= 0 || top_k <= 0) return 0;
  return experts_ws(n_tokens, top_k, experts, true).total;
}

extern "C" int tm_fp8_grouped_swiglu(const tm_fp8_experts *experts, int32_t dtype, const void *x, int64_t n_tokens,
                                     int64_t ld_x, const int64_t *ids, int32_t top_k, int64_t ld_ids,
                                     const uint8_t *mask, int64_t ms_b, int64_t ms_s, void *out, int64_t so_b,
                                     int64_t so_s, void *workspace, size_t workspace_bytes, tm_stream_t stream) {
  const char *const name = "tm_fp8_grouped_swiglu";
  const int bad = check_experts(name, experts, dtype);
  if (bad != TM_OK) return bad;
  TM_REQUIRE(n_tokens >= 0 && top_k >= 1 && ld_ids >= top_k && n_tokens < ((int64_t)1 << 31) / top_k - 256 &&
                 ld_x >= experts->hidden,
             TM_EINVAL_SHAPE, "%s: bad sizes", name);
  if (n_tokens == 0) return TM_OK;
  TM_REQUIRE(x && ids && mask && out, TM_EINVAL_ARG, "%s: null pointer", name);
  TM_REQUIRE(aligned(x, ld_x * 2) && tm_aligned16(out) && so_b % 8 == 0 && so_s % 8 == 0, TM_EINVAL_SHAPE,
             "%s: rows of x and of the output must be 16-byte aligned", name);
  const ExpertsWs ws = experts_ws(n_tokens, top_k, experts, true);
  TM_REQUIRE(workspace != nullptr && workspace_bytes >= ws.total && tm_aligned16(workspace), TM_EWORKSPACE,
             "%s: workspace %zu bytes < %zu", name, workspace_bytes, ws.total);
  char *const base = static_cast<char *>(workspace);
  hipStream_t s = tm_hip_stream(stream);
  const int64_t max_rows = n_tokens * top_k;
  const bool stream_w = max_rows <= stream_rows(experts);
  Fp8Rows rows{n_tokens};
  Fp8Tiles ts{};
  if (stream_w) {
    rows.ids = ids;
    rows.ld_ids = ld_ids;
    rows.mask = mask;
    rows.ms_b = ms_b;
    rows.ms_s = ms_s;
    rows.top_k = top_k;
    rows.n_experts = experts->n_experts;
  } else {
    int32_t *const offsets = reinterpret_cast<int32_t *>(base + ws.offsets);
    int32_t *const row_token = reinterpret_cast<int32_t *>(base + ws.row_token);
    int64_t *const row_out = reinterpret_cast<int64_t *>(base + ws.row_out);
    int32_t *const tiles = reinterpret_cast<int32_t *>(base + ws.tiles);  // (not used here)
    const int st = tm_group_slots_ws(ids, n_tokens, top_k, ld_ids, mask, ms_b, ms_s, experts->n_experts, so_b, so_s,
                                     offsets, row_token, row_out, tiles, base + ws.group,
                                     tm_group_slots_workspace_size(n_tokens, top_k, experts->n_experts), stream);
    if (st != TM_OK) return st;
    ts = Fp8Tiles{offsets, row_token, row_out, experts->n_experts, (int32_t)max_rows, 0};
  }
  const Fp8Dst dst{out, 0, so_b, so_s, nullptr, 0};
  return dtype == TM_DT_F16
             ? mlp_launch<TM_DT_F16>(name, experts, x, ld_x, n_tokens, &rows, stream_w ? nullptr : &ts, ws, base, dst, s)
             : mlp_launch<TM_DT_BF16>(name, experts, x, ld_x, n_tokens, &rows, stream_w ? nullptr : &ts, ws, base, dst, s);
}

extern "C" size_t tm_fp8_expert_swiglu_workspace_size(const tm_fp8_experts *experts, int64_t n_rows) {
  if (experts == nullptr || n_rows <= 0) return 0;
  return experts_ws(n_rows, 1, experts, false).total;
}

extern "C" int tm_fp8_expert_swiglu(const tm_fp8_experts *experts, int32_t dtype, const void *x, int64_t n_rows,
                                    int64_t ld_x, const void *addend, int64_t ld_add, void *out, int64_t ld_out,
                                    void *workspace, size_t workspace_bytes, tm_stream_t stream) {
  const char *const name = "tm_fp8_expert_swiglu";
  const int bad = check_experts(name, experts, dtype);
  if (bad != TM_OK) return bad;
  TM_REQUIRE(experts->n_experts == 1, TM_EINVAL_SHAPE, "%s: takes the weights of one expert", name);
  TM_REQUIRE(n_rows >= 0 && n_rows < ((int64_t)1 << 31) - 256 && ld_x >= experts->hidden && ld_out >= experts->hidden &&
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
  const Fp8Rows rows{n_rows};
  Fp8Tiles ts{};
  ts.rows = (int32_t)n_rows;
  const bool stream_w = n_rows <= stream_rows(experts);
  const Fp8Dst dst{out, ld_out, 0, 0, addend, ld_add};
  const ExpertsWs ws = experts_ws(n_rows, 1, experts, false);
  char *const base = static_cast<char *>(workspace);
  return dtype == TM_DT_F16
             ? mlp_launch<TM_DT_F16>(name, experts, x, ld_x, n_rows, &rows, stream_w ? nullptr : &ts, ws, base, dst, s)
             : mlp_launch<TM_DT_BF16>(name, experts, x, ld_x, n_rows, &rows, stream_w ? nullptr : &ts, ws, base, dst, s);
}
