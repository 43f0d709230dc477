// Router of grouped experts with a balancing bias (contract: tm_route_experts
// in tablemoe.h).
//
// 16 lanes own a token, expert e in lane e % 16; a wave holds four tokens.  The
// keys that decide are those of the definition, in 64 bits: two experts whose
// scores differ in the eighth digit come out in its order, not in that of their
// roundings.  They are computed in 32 bits first, whose error is
// bounded (kTol); the top_k rounds go on until the next key is far from the
// last, and where two neighbours are near the candidates (a lane each) are put
// in the order of their 64-bit keys, whose scores the weights need anyway.  Where
// a group that stays and one that does not are near, the experts that they can
// be worth are looked at in 64 bits.  Only a run of equal keys past 32 candidates
// makes a wave choose in 64 bits from the start (select64).  Without a bias the
// logits order the experts, exactly.
//
// A softmax's sum has fp32 terms (within two roundings: enough for the weights) until
// a bias meets a choice in 64 bits: there it scales the scores against the bias, so
// the sum is taken again of 64-bit terms (sum64; with the fp32 ones two keys 1e-9
// apart changed places).
//
// Bound by latency: each round is a maximum over the lane's keys, four DPP
// exchanges, the lowest lane that holds it and its key closed, one after the
// other; where at most half of the experts are in the groups that stay, over
// those alone.  8 tokens of 256 experts take 8.1 us, 4099 of 160 8.7 us, 12301 of
// 256 15-17 us (rounds over every key: 9.0, 9.3 and 17.7).  All in 64 bits took 24,
// 20 and 43 (a first pass in 32 bits that chose again in 64 where keys were near:
// 10, 10 and 36).
#include "tm_common.h"

#include <type_traits>

namespace {

struct RouteArgs {
  int64_t n, ld;
  int n_experts, scoring, n_groups, size, topk_groups, group_rule, top_k, renorm;
  float scale;
  const float *bias;
  uint32_t inv;  // ceil(2^20 / size)
};

// e / size: exact for e < 2^10 >= size (e * inv is over e / size * 2^20 by less than e).
__device__ __forceinline__ int group_of(int e, const RouteArgs &a) { return (int)(__umul24((uint32_t)e, a.inv) >> 20); }

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

// 32-bit keys.  A sigmoid takes its argument's product with log2 e, exp2, an
// addition and a reciprocal, a softmax score a difference, the same product,
// exp2, the sum's reciprocal and a product: of a score s = e^-d / sum, 2.5 d + 8
// roundings of 2^-24, at most 5.5e-7 (d e^-d < 0.37); adding the bias, one of
// the key.  Two keys are in the right order if they are further apart than
// twice that.  A sum of two keys has both errors and its own rounding, by the size of
// its terms, which may cancel: kTol / 2 for each term covers them.
constexpr float kTol = 1.5e-6f;

__device__ __forceinline__ double score64(float l, int scoring, float mx, double sum) {
  const double t = exp(scoring == TM_ROUTE_SOFTMAX ? (double)l - (double)mx : -(double)l);
  return scoring == TM_ROUTE_SOFTMAX ? t / sum : 1.0 / (1.0 + t);
}

// Orderable keys of the rounds: 0 closed (chosen, or not in a kept group), 1 not
// available, above that the key's order (tm_orderable(-FLT_MAX) is 2^23).
constexpr uint32_t kClosed = 0, kMasked = 1;

__device__ __forceinline__ bool near(float hi, float lo, float tol) { return hi - lo <= tol * fmaxf(1.f, fabsf(hi)); }

// The groups that stay, from the values in LDS (padded by one per group), as a
// mask in every lane of the token.  UNSURE: also whether a group that stays and
// one that does not are too near to be told from each other in 32 bits, in
// gmin the least value that a group's own is made of and in gerr the bound on its
// error (infinite where the value is out of fp32's range).
template <typename K, bool UNSURE>
__device__ __forceinline__ uint64_t kept_groups(const RouteArgs &a, int sub, const K *vals, K *gval, K *gmin, K *gerr,
                                                bool &unsure) {
  const K ninf = -(K)__builtin_huge_valf();
  const bool top2 = a.group_rule == TM_GROUP_TOP2;
  __syncthreads();  // (one wave)
  // 16 / n_groups lanes read a group, each its share; several groups a lane otherwise
  const int share = a.n_groups <= 2 ? 8 : a.n_groups <= 4 ? 4 : a.n_groups <= 8 ? 2 : 1;
  for (int g = sub / share; g < a.n_groups; g += 16 / share) {
    const K *const p = vals + g * (a.size + 1);
    K first = ninf, second = ninf;
#pragma unroll 4
    for (int i = sub % share; i < a.size; i += share) {
      const K v = p[i];
      second = fmax(second, fmin(first, v));
      first = fmax(first, v);
    }
    for (int o = 1; o < share; o <<= 1) {
      const K f2 = __shfl_xor(first, o, 64), s2 = __shfl_xor(second, o, 64);
      second = fmax(fmax(second, s2), fmin(first, f2));
      first = fmax(first, f2);
    }
    if (sub % share == 0) {
      const bool two = top2 && second > ninf;
      K v = two ? first + second : first;
      if constexpr (UNSURE) {
        constexpr float kBig = 3.402823466e38f;
        gmin[g] = two ? second : first;
        K err = kTol / 2 * (fmaxf(1.f, fabsf(first)) + (two ? fmaxf(1.f, fabsf(second)) : 0.f));
        if (first > ninf && !(fabsf(v) <= kBig)) {  // (an available group stays above the others)
          v = v > 0 ? kBig : -kBig;
          err = -ninf;
        }
        gerr[g] = err;
      }
      gval[g] = v;
    }
  }
  __syncthreads();
  uint64_t kept = 0;
  // the least that one that stays can be worth, the most that another (available) one can
  float low = __builtin_huge_valf(), high = -low;
  for (int g0 = 0; g0 < a.n_groups; g0 += 16) {
    const int g = g0 + sub;
    const bool in = g < a.n_groups;
    const K mine = gval[in ? g : 0];
    int ahead = 0;
    for (int o = 0; o < a.n_groups; ++o) {
      const K v = gval[o];
      ahead += (v > mine) | ((v == mine) & (o < g));
    }
    const bool stays = ahead < a.topk_groups;
    if constexpr (UNSURE) {
      const K err = gerr[in ? g : 0];
      low = (in & stays) ? fminf(low, mine - err) : low;
      high = (in & !stays & (mine > ninf)) ? fmaxf(high, mine + err) : high;
    }
    const uint64_t all = __ballot(in & stays);
    kept |= ((all >> ((threadIdx.x & 63) & ~15)) & 0xffffull) << g0;
  }
  if constexpr (UNSURE) {
    low = -row16_max(-low);
    high = row16_max(high);
    unsure = high > (float)ninf && high >= low;
  }
  return kept;
}

__device__ __forceinline__ bool available(float l, float b) {  // (false for NaN)
  return (l >= -3.402823466e38f) & (b >= -3.402823466e38f);
}

// A softmax's sum of 64-bit terms, for the choices that are made in 64 bits.
template <int DT>
__device__ __forceinline__ double sum64(const typename Elem<DT>::T *lr, const RouteArgs &a, int sub, float mx) {
  double sum = 0;
#pragma unroll 1
  for (int e = sub; e < a.n_experts; e += 16) {
    const float l = Elem<DT>::to_f(lr[e]);
    if (available(l, a.bias != nullptr ? a.bias[e] : 0.f))
      sum += exp((double)fminf(l, 3.402823466e38f) - (double)mx);
  }
  return row16_sum(sum);
}

// The choice in 64 bits: compact, for the few waves that need it.
template <int DT>
__device__ __forceinline__ void select64(const typename Elem<DT>::T *lr, const RouteArgs &a, int sub, float mx,
                                         double sum, double *keys, int (&win)[2]) {
  const double ninf = -__builtin_huge_val();
  const bool scored = a.bias != nullptr, top2 = a.n_groups > 1 && a.group_rule == TM_GROUP_TOP2;
  uint64_t open = 0;
  double *const gval = keys + a.n_experts + a.n_groups;
  auto key_of = [&](int e, bool value) {
    const float l = Elem<DT>::to_f(lr[e]), b = scored ? a.bias[e] : 0.f;
    const float lc = fminf(l, 3.402823466e38f);
    if (!available(l, b)) return ninf;
    return scored || value ? score64(lc, a.scoring, mx, sum) + (double)b : (double)lc;
  };
#pragma unroll 1
  for (int e = sub, j = 0; e < a.n_experts; e += 16, ++j) {
    keys[e + group_of(e, a)] = key_of(e, top2);
    open |= 1ull << j;
  }
  if (a.n_groups > 1) {
    bool none = false;
    const uint64_t kept = kept_groups<double, false>(a, sub, keys, gval, nullptr, nullptr, none);
    open = 0;
#pragma unroll 1
    for (int e = sub, j = 0; e < a.n_experts; e += 16, ++j) {
      if ((kept >> group_of(e, a)) & 1) open |= 1ull << j;
      if (top2 && !scored) keys[e + group_of(e, a)] = key_of(e, false);
    }
  }
#pragma unroll 1
  for (int r = 0; r < a.top_k; ++r) {
    double bv = ninf;
    int bi = 0x7fffffff;
#pragma unroll 1
    for (int e = sub, j = 0; e < a.n_experts; e += 16, ++j) {
      const double k = keys[e + group_of(e, a)];
      if (((open >> j) & 1) && (k > bv || bi == 0x7fffffff)) {
        bv = k;
        bi = e;
      }
    }
#define F_(C_)                                              \
  {                                                         \
    const double ov = dpp16<C_>(bv);                        \
    const int oi = dpp16<C_>(bi);                           \
    const bool take = ov > bv || (ov == bv && oi < bi);     \
    bv = take ? ov : bv;                                    \
    bi = take ? oi : bi;                                    \
  }
    TM_ROW16(F_)
#undef F_
    if ((bi & 15) == sub) open &= ~(1ull << (bi >> 4));
    if ((r & 15) == sub) win[r >> 4] = bi;
  }
}

template <int VPL>
using Mask = std::conditional_t<(VPL > 32), uint64_t, uint32_t>;

template <int DT, int VPL, bool SIGMOID>
__global__ __launch_bounds__(64) void route_experts_kernel(const typename Elem<DT>::T *__restrict__ logits, RouteArgs a,
                                                          float *__restrict__ out_w, int64_t *__restrict__ out_ids) {
  extern __shared__ double lds[];
  const int lane = threadIdx.x, sub = lane & 15, tok = lane >> 4;
  const int64_t row = (int64_t)blockIdx.x * 4 + tok;
  const bool valid = row < a.n;  // the others go along with the last row and write nothing
  const typename Elem<DT>::T *const lr = logits + (valid ? row : a.n - 1) * a.ld;
  const float big = 3.402823466e38f, ninf = -__builtin_huge_valf();
  const bool scored = a.bias != nullptr;  // (without a bias the logits order the experts)
  float l[VPL], v[VPL];                   // logits (NaN: not available), biases and then keys
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = j * 16 + sub, ec = e < a.n_experts ? e : a.n_experts - 1;
    l[j] = Elem<DT>::to_f(lr[ec]);
    v[j] = 0.f;
  }
  if (scored) {  // uniform
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int e = j * 16 + sub;
      v[j] = a.bias[e < a.n_experts ? e : a.n_experts - 1];
    }
  }
  float mx = -big;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const bool ok = (j * 16 + sub < a.n_experts) & available(l[j], v[j]);
    l[j] = ok ? fminf(l[j], big) : __builtin_nanf("");
    mx = fmaxf(mx, l[j]);
  }
  mx = row16_max(mx);
  double sum = 1;
  if constexpr (!SIGMOID) {
    sum = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      // exp of the exact difference l - mx = d + r
      const float d = l[j] - mx, bb = d - l[j], r = (l[j] - (d - bb)) - (mx + bb);
      const float t = expf(d);
      const float term = d > -200.f ? fmaf(t, r, t) : 0.f;  // (NaN: 0)
      sum += (double)term;
    }
    sum = row16_sum(sum);
  }
  const int per_tok = a.n_experts + 2 * a.n_groups;  // values, padded by one per group, and the groups' own
  const bool top2 = a.n_groups > 1 && a.group_rule == TM_GROUP_TOP2;
  float *const vals = reinterpret_cast<float *>(lds) + tok * per_tok;
  bool unsure = false;
  if (scored || top2) {  // uniform
    const float inv_sum = SIGMOID ? 1.f : __builtin_amdgcn_rcpf((float)sum);
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const float s = SIGMOID ? __builtin_amdgcn_rcpf(1.f + __expf(-l[j])) : __expf(l[j] - mx) * inv_sum;
      v[j] += s;
      v[j] = l[j] == l[j] ? v[j] : ninf;
    }
  }
  // The sum for choices in 64 bits: `sum` where it is a common factor of all keys.
  // Weights keep `sum`, so they do not hang on the other tokens of the wave.
  double sum_c = sum;
  bool exact = SIGMOID || !scored;
  auto need_sum64 = [&] {
    if (!exact) sum_c = sum64<DT>(lr, a, sub, mx);
    exact = true;
  };
  uint64_t kept = ~0ull;
  bool compact = false;
  float *const gmin = vals + 4 * per_tok, *const gerr = gmin + a.n_groups;  // (3 n_groups <= per_tok)
  int *const glist = reinterpret_cast<int *>(gerr + a.n_groups);  // the groups that stay, ascending
  if (a.n_groups > 1) {  // uniform
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int e = j * 16 + sub;
      const float k = scored || top2 ? v[j] : l[j] == l[j] ? l[j] : ninf;
      vals[e < a.n_experts ? e + group_of(e, a) : per_tok - 1] = k;  // (the last: a group value, written later)
    }
    float *const gval = vals + a.n_experts + a.n_groups;
    compact = 2 * a.topk_groups * a.size <= 16 * VPL && (scored || !top2);  // (vals holds the keys)
    if (scored || top2) {  // uniform
      kept = kept_groups<float, true>(a, sub, vals, gval, gmin, gerr, unsure);
      if (__ballot(unsure) != 0) {
        // again in 64 bits, of the experts that can be among what a group is worth
        need_sum64();
        Mask<VPL> maybe = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          const int e = j * 16 + sub;
          const float t = gmin[e < a.n_experts ? group_of(e, a) : 0];
          // (not `>=`: the bound of an infinite t is NaN)
          const bool in = (e < a.n_experts) & (v[j] > ninf) & !(v[j] < t - kTol * fmaxf(1.f, fabsf(t)));
          maybe |= (Mask<VPL>)in << j;
        }
        __syncthreads();
        double *const vals64 = lds + tok * per_tok;
        for (int e = sub; e < a.n_experts; e += 16) vals64[e + group_of(e, a)] = (double)ninf;
        while (maybe != 0) {
          const int e = (int)__builtin_ctzll((uint64_t)maybe) * 16 + sub;
          maybe &= maybe - 1;
          const double s64 = score64(fminf(Elem<DT>::to_f(lr[e]), big), SIGMOID ? TM_ROUTE_SIGMOID : TM_ROUTE_SOFTMAX,
                                     mx, sum_c);
          vals64[e + group_of(e, a)] = s64 + (scored ? (double)a.bias[e] : 0.0);
        }
        kept = kept_groups<double, false>(a, sub, vals64, vals64 + a.n_experts + a.n_groups, nullptr, nullptr, unsure);
        unsure = false;
        compact = false;  // (vals is gone)
      }
    } else {
      kept = kept_groups<float, false>(a, sub, vals, gval, nullptr, nullptr, unsure);
    }
    for (int g = sub; g < a.n_groups; g += 16)
      if ((kept >> g) & 1) glist[__popcll(kept & ((1ull << g) - 1))] = g;
    __syncthreads();
  }
  // Winner r goes to lane r % 16.  With 32-bit keys the rounds go on past the last
  // chosen until the next key is far below: the candidates then hold every
  // expert that can be among the chosen.
  const int n_open = a.topk_groups * a.size;
  int cand[2] = {0, 0};
  uint32_t last = 0;
  bool close = false;  // two neighbours of the candidates are near
  int r = 0;
  auto rounds = [&](auto nk_c, auto &key) {
    constexpr int NK = decltype(nk_c)::value;
    for (bool more = true; more; ++r) {
      uint32_t m = key[0];
#pragma unroll
      for (int j = 1; j < NK; ++j) m = max(m, key[j]);
      m = max(m, tm_dpp<0xB1>(m, m));
      m = max(m, tm_dpp<0x4E>(m, m));
      m = max(m, tm_dpp<0x141>(m, m));
      m = max(m, tm_dpp<0x140>(m, m));
      uint32_t at = 0xffffu;  // lowest expert with that key
#pragma unroll
      for (int j = NK - 1; j >= 0; --j) at = key[j] == m ? (uint32_t)j : at;
      uint32_t w = at * 16 + sub;
      w = min(w, tm_dpp<0xB1>(w, w));
      w = min(w, tm_dpp<0x4E>(w, w));
      w = min(w, tm_dpp<0x141>(w, w));
      w = min(w, tm_dpp<0x140>(w, w));
      const uint32_t mine = at * 16 + sub == w ? at : 0xffffu;
#pragma unroll
      for (int j = 0; j < NK; ++j) key[j] = mine == (uint32_t)j ? kClosed : key[j];
      if ((r & 15) == sub) {
        if (r < 16) cand[0] = (int)w;
        else cand[1] = (int)w;
      }
      if (scored) {  // uniform
        const bool touches = (r > 0) & (m > kMasked) & near(tm_from_orderable(last), tm_from_orderable(m), kTol);
        close |= touches;
        last = m;
        more = r + 1 < a.top_k || (r + 1 < n_open && (r + 1 == a.top_k || __ballot(touches) != 0));
        if (more && r + 1 == 32) {  // a long run of equals: past what the candidates hold
          unsure = true;
          more = false;
        }
      } else {
        more = r + 1 < a.top_k;
      }
    }
  };
  auto key_of = [&](float f, bool masked) {
    const uint32_t u = __float_as_uint(f + 0.f);  // (-0 equals 0)
    uint32_t o = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    asm("" : "+v"(o));  // (both sides of the select: no branch for each)
    return masked ? kMasked : o;
  };
  if (compact) {
    // Half of the experts are open at most: a lane takes every 16th of those, in
    // their order, from LDS.
    constexpr int NK = VPL / 2;
    uint32_t key[NK];
    auto expert_at = [&](int p, int pad) {
      const int i = group_of(p, a);
      return glist[i] * (a.size + pad) + p - i * a.size;
    };
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int p = j * 16 + sub;
      const float f = vals[expert_at(p < n_open ? p : 0, 1)];
      const uint32_t o = key_of(f, f == ninf);
      key[j] = p < n_open ? o : kClosed;
    }
    rounds(std::integral_constant<int, NK>{}, key);
#pragma unroll
    for (int u = 0; u < 2; ++u) cand[u] = expert_at(cand[u], 0);
  } else {
    uint32_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int e = j * 16 + sub;
      const uint32_t o = key_of(scored ? v[j] : l[j], l[j] != l[j]);
      const bool open = (kept >> (a.n_groups > 1 ? group_of(e, a) & 63 : 0)) & 1;
      key[j] = (open & (e < a.n_experts)) ? o : kClosed;
    }
    rounds(std::integral_constant<int, VPL>{}, key);
  }
  int n_cand = r;
  if (__ballot(unsure) != 0) {  // uniform
    __syncthreads();
    need_sum64();
    select64<DT>(lr, a, sub, mx, sum_c, lds + tok * per_tok, cand);
    n_cand = a.top_k;
    close = false;
  }
  double w[2], total = 0;
  int place[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    w[u] = 0;
    place[u] = 16 * u + sub;
    if (16 * u >= n_cand) continue;  // uniform
    const float x = Elem<DT>::to_f(lr[cand[u]]);
    if (available(x, scored ? a.bias[cand[u]] : 0.f))
      w[u] = score64(fminf(x, big), SIGMOID ? TM_ROUTE_SIGMOID : TM_ROUTE_SOFTMAX, mx, sum);
  }
  if (__ballot(close) != 0) {  // uniform: the candidates in the order of their 64-bit keys
    need_sum64();
    double k64[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float x = Elem<DT>::to_f(lr[cand[u]]), b = a.bias[cand[u]];
      const double s64 = SIGMOID ? w[u] : score64(fminf(x, big), TM_ROUTE_SOFTMAX, mx, sum_c);
      k64[u] = available(x, b) ? s64 + (double)b : -__builtin_huge_val();
      place[u] = 16 * u + sub < n_cand ? 0 : 32;
    }
    for (int o = 0; o < n_cand; ++o) {
      const int from = (lane & ~15) | (o & 15);
      const double ko = __shfl(o < 16 ? k64[0] : k64[1], from, 64);
      const int eo = __shfl(o < 16 ? cand[0] : cand[1], from, 64);
#pragma unroll
      for (int u = 0; u < 2; ++u) place[u] += (ko > k64[u]) | ((ko == k64[u]) & (eo < cand[u]));
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) total += place[u] < a.top_k ? w[u] : 0.0;
  double d = 1.0;
  if (a.renorm) {  // uniform
    total = row16_sum(total);
    d = total > 1e-20 ? total : 1e-20;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (valid & (place[u] < a.top_k)) {
      out_w[row * a.top_k + place[u]] = (float)(w[u] / d * (double)a.scale);
      out_ids[row * a.top_k + place[u]] = cand[u];
    }
}

template <int DT, int VPL>
void launch(const void *logits, const RouteArgs &a, float *out_w, int64_t *out_ids, hipStream_t s) {
  const size_t lds = 4 * (size_t)(a.n_experts + 2 * a.n_groups) * sizeof(double);
  const dim3 grid((unsigned)tm_cdiv(a.n, 4));
  const auto *const p = static_cast<const typename Elem<DT>::T *>(logits);
  if (a.scoring == TM_ROUTE_SIGMOID)
    hipLaunchKernelGGL((route_experts_kernel<DT, VPL, true>), grid, dim3(64), lds, s, p, a, out_w, out_ids);
  else
    hipLaunchKernelGGL((route_experts_kernel<DT, VPL, false>), grid, dim3(64), lds, s, p, a, out_w, out_ids);
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
  TM_REQUIRE(scale - scale == 0.f, TM_EINVAL_ARG, "tm_route_experts: scale is not finite");  // (0 * inf is NaN)
  if (n_tokens == 0) return TM_OK;
  TM_REQUIRE(logits && out_weights && out_ids, TM_EINVAL_ARG, "tm_route_experts: null pointer");
  const RouteArgs a{n_tokens, ld_logits, n_experts, scoring, n_groups, n_experts / n_groups, topk_groups, group_rule,
                    top_k, renormalize, scale, bias,
                    ((1u << 20) + n_experts / n_groups - 1) / (n_experts / n_groups)};
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
