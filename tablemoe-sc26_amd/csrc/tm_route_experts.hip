// Router of grouped experts with a balancing bias (contract: tm_route_experts
// in tablemoe.h).
//
// 16 lanes own a token, expert e in lane e % 16; a wave holds four tokens.  The
// keys are compared in 64 bits: two experts whose scores differ in the eighth
// digit come out in the order of the definition, not in that of somebody's
// roundings.  Each of the top_k rounds is a lane's best open expert, four DPP
// exchanges of (key, id), and the winner's bit cleared.
#include "tm_common.h"

namespace {

struct RouteArgs {
  int64_t n, ld;
  int n_experts, scoring, n_groups, size, topk_groups, group_rule, top_k, renorm;
  float scale;
  const float *bias;
};

template <int CTRL>
__device__ __forceinline__ float dpp16(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp16(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
template <int CTRL>
__device__ __forceinline__ int dpp16(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
// f(step) with the four exchanges that reduce 16 lanes: quad_perm [1,0,3,2] and
// [2,3,0,1], row_half_mirror, row_mirror; every lane ends with the result.
#define TM_ROW16(F_) F_(0xB1) F_(0x4E) F_(0x141) F_(0x140)

template <typename K>
__device__ __forceinline__ K row16_sum(K v) {
#define F_(C_) v += dpp16<C_>(v);
  TM_ROW16(F_)
#undef F_
  return v;
}
template <typename K>
__device__ __forceinline__ K row16_max(K v) {
#define F_(C_) { const K o = dpp16<C_>(v); v = o > v ? o : v; }
  TM_ROW16(F_)
#undef F_
  return v;
}

template <typename K>
__device__ __forceinline__ K score_of(float l, int scoring, float mx, K sum) {
  if (scoring == TM_ROUTE_SOFTMAX) return exp((K)l - (K)mx) / sum;
  return K(1) / (K(1) + exp(-(K)l));
}

// The top_k winners of a token, winner r in win[r / 16] of lane r % 16.
template <int VPL, typename K>
__device__ __forceinline__ void select(const float (&l)[VPL], uint64_t avail, const RouteArgs &a, int sub, float mx,
                                       K sum, K *vals, K *gval, int (&win)[2]) {
  const K ninf = -(K)__builtin_huge_valf();
  K key[VPL];
  const bool scored = a.bias != nullptr;  // (without a bias the logits order the experts)
  const bool top2 = a.n_groups > 1 && a.group_rule == TM_GROUP_TOP2;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = j * 16 + sub;
    const bool ok = (avail >> j) & 1;
    K v = ninf;
    if (ok && (scored || top2)) {
      v = score_of<K>(l[j], a.scoring, mx, sum);
      if (scored) v += (K)a.bias[e];
    }
    key[j] = !ok ? ninf : scored ? v : (K)l[j];
    if (a.n_groups > 1 && e < a.n_experts) vals[e + e / a.size] = top2 ? v : key[j];
  }
  uint64_t open = 0;
  if (a.n_groups > 1) {
    __syncthreads();
    for (int g = sub; g < a.n_groups; g += 16) {
      const K *const p = vals + g * (a.size + 1);
      K first = ninf, second = ninf;
      for (int i = 0; i < a.size; ++i) {
        const K v = p[i];
        second = v > first ? first : v > second ? v : second;
        first = v > first ? v : first;
      }
      gval[g] = top2 && second > ninf ? first + second : first;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int e = j * 16 + sub;
      if (e >= a.n_experts) continue;
      const int g = e / a.size;
      const K mine = gval[g];
      int ahead = 0;
      for (int o = 0; o < a.n_groups; ++o) ahead += gval[o] > mine || (gval[o] == mine && o < g);
      if (ahead < a.topk_groups) open |= 1ull << j;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (j * 16 + sub < a.n_experts) open |= 1ull << j;
  }
  for (int r = 0; r < a.top_k; ++r) {
    K bv = ninf;
    int bi = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (((open >> j) & 1) && (key[j] > bv || bi == 0x7fffffff)) {
        bv = key[j];
        bi = j * 16 + sub;
      }
#define F_(C_)                                                          \
  {                                                                     \
    const K ov = dpp16<C_>(bv);                                         \
    const int oi = dpp16<C_>(bi);                                       \
    if (oi != 0x7fffffff && (ov > bv || (ov == bv && oi < bi) || bi == 0x7fffffff)) { \
      bv = ov;                                                          \
      bi = oi;                                                          \
    }                                                                   \
  }
    TM_ROW16(F_)
#undef F_
    if ((bi & 15) == sub) open &= ~(1ull << (bi >> 4));
    if ((r & 15) == sub) win[r >> 4] = bi;
  }
}

template <int DT, int VPL>
__global__ __launch_bounds__(64) void route_experts_kernel(const typename Elem<DT>::T *__restrict__ logits, RouteArgs a,
                                                          float *__restrict__ out_w, int64_t *__restrict__ out_ids) {
  extern __shared__ double lds[];
  const int lane = threadIdx.x, sub = lane & 15, tok = lane >> 4;
  const int64_t row = (int64_t)blockIdx.x * 4 + tok;
  const bool valid = row < a.n;  // the others go along with the last row and write nothing
  const typename Elem<DT>::T *const lr = logits + (valid ? row : a.n - 1) * a.ld;
  const float big = 3.402823466e38f;
  float l[VPL];
  uint64_t avail = 0;
  float mx = -big;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = j * 16 + sub;
    l[j] = 0.f;
    if (e < a.n_experts) {
      const float v = Elem<DT>::to_f(lr[e]);
      const float b = a.bias != nullptr ? a.bias[e] : 0.f;
      if (v >= -big && (b >= -big)) {  // (false for NaN)
        l[j] = v > big ? big : v;
        avail |= 1ull << j;
        mx = fmaxf(mx, l[j]);
      }
    }
  }
  mx = row16_max(mx);
  double sum = 0;
  if (a.scoring == TM_ROUTE_SOFTMAX) {
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if ((avail >> j) & 1) sum += exp((double)l[j] - (double)mx);
    sum = row16_sum(sum);
  }
  const int per_tok = a.n_experts + 2 * a.n_groups;  // values, padded by one per group, and the groups' own
  double *const vals = lds + tok * per_tok;
  int win[2] = {0, 0};
  select<VPL, double>(l, avail, a, sub, mx, sum, vals, vals + a.n_experts + a.n_groups, win);
  double w[2], total = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    w[u] = 0;
    if (16 * u + sub < a.top_k) {
      const int e = win[u];
      const float v = Elem<DT>::to_f(lr[e]);
      const float b = a.bias != nullptr ? a.bias[e] : 0.f;
      if (v >= -big && b >= -big) w[u] = score_of<double>(v > big ? big : v, a.scoring, mx, sum);
    }
    total += w[u];
  }
  total = row16_sum(total);
  const double d = a.renorm ? (total > 1e-20 ? total : 1e-20) : 1.0;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (valid && 16 * u + sub < a.top_k) {
      out_w[row * a.top_k + 16 * u + sub] = (float)(w[u] / d * (double)a.scale);
      out_ids[row * a.top_k + 16 * u + sub] = win[u];
    }
}

template <int DT, int VPL>
void launch(const void *logits, const RouteArgs &a, float *out_w, int64_t *out_ids, hipStream_t s) {
  const size_t lds = a.n_groups > 1 ? 4 * (size_t)(a.n_experts + 2 * a.n_groups) * sizeof(double) : 0;
  hipLaunchKernelGGL((route_experts_kernel<DT, VPL>), dim3((unsigned)tm_cdiv(a.n, 4)), dim3(64), lds, s,
                     static_cast<const typename Elem<DT>::T *>(logits), a, out_w, out_ids);
}

}  // namespace

extern "C" int tm_route_experts(int32_t dtype, const void *logits, int64_t n_tokens, int32_t n_experts,
                                int64_t ld_logits, const float *bias, int32_t scoring, int32_t n_groups,
                                int32_t topk_groups, int32_t group_rule, int32_t top_k, int32_t renormalize,
                                float scale, float *out_weights, int64_t *out_ids, tm_stream_t stream) {
  TM_REQUIRE(dtype == TM_DT_F32 || dtype == TM_DT_F16 || dtype == TM_DT_BF16, TM_EINVAL_DTYPE,
             "tm_route_experts: unsupported dtype tag %d", (int)dtype);
  TM_REQUIRE(n_tokens >= 0 && n_tokens < ((int64_t)1 << 32) && n_experts >= 1 && n_experts <= 1024 &&
                 ld_logits >= n_experts,
             TM_EINVAL_SHAPE, "tm_route_experts: bad sizes (experts %d)", n_experts);
  TM_REQUIRE((scoring == TM_ROUTE_SOFTMAX || scoring == TM_ROUTE_SIGMOID) &&
                 (group_rule == TM_GROUP_MAX || group_rule == TM_GROUP_TOP2),
             TM_EINVAL_ARG, "tm_route_experts: bad scoring %d or group rule %d", scoring, group_rule);
  TM_REQUIRE(n_groups >= 1 && n_groups <= 64 && n_experts % n_groups == 0 && topk_groups >= 1 &&
                 topk_groups <= n_groups,
             TM_EINVAL_SHAPE, "tm_route_experts: %d of %d groups of %d experts", topk_groups, n_groups, n_experts);
  TM_REQUIRE(top_k >= 1 && top_k <= 32 && top_k <= topk_groups * (n_experts / n_groups), TM_EINVAL_SHAPE,
             "tm_route_experts: top_k %d out of range", top_k);
  TM_REQUIRE(scale == scale, TM_EINVAL_ARG, "tm_route_experts: scale is NaN");
  if (n_tokens == 0) return TM_OK;
  TM_REQUIRE(logits && out_weights && out_ids, TM_EINVAL_ARG, "tm_route_experts: null pointer");
  const RouteArgs a{n_tokens, ld_logits, n_experts, scoring, n_groups, n_experts / n_groups, topk_groups, group_rule,
                    top_k, renormalize, scale, bias};
  hipStream_t s = tm_hip_stream(stream);
  return TM_DISPATCH_DTYPE(dtype, DT, [&] {
    if (n_experts <= 64) launch<DT, 4>(logits, a, out_weights, out_ids, s);
    else if (n_experts <= 128) launch<DT, 8>(logits, a, out_weights, out_ids, s);
    else if (n_experts <= 256) launch<DT, 16>(logits, a, out_weights, out_ids, s);
    else if (n_experts <= 512) launch<DT, 32>(logits, a, out_weights, out_ids, s);
    else launch<DT, 64>(logits, a, out_weights, out_ids, s);
    TM_LAUNCH_CHECK("tm_route_experts");
    return TM_OK;
  });
}
