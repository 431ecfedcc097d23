// Routing to experts: scores, the choice of k experts per token and their weights, the gradient,
// and the expert order of the chosen (token, choice) pairs.
//
//   s = softmax(l) or sigmoid(l);  c = s + bias (what is ranked);  ids = the k largest c among the
//   kept groups, ties to the lowest index;  w = scale * s[ids], over the sum of s[ids] if renormalised.
//
// c is ranked as its 64-bit value: two 32-bit scores may round to one value, or to the wrong order,
// where their logits do not.  Without a bias and with group score "max" c is not formed: s grows
// with l, so the logits rank, exactly.  Otherwise a row is ranked in 32 bits with a bound on their
// error, and again in 64 bits if two candidates that matter are nearer than the bound allows.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "expert_rows.cuh"

namespace cpg {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;       // one lane holds one choice
constexpr int kRouteMaxGroups = 32;  // one lane holds one group
constexpr int kRouteWarps = 4;

enum RouteScoring : int32_t { kRouteSoftmax = 0, kRouteSigmoid = 1 };
enum RouteGroupScore : int32_t { kRouteGroupMax = 0, kRouteGroupTop2 = 1 };

struct RouteParams {
  const void* logits;
  int64_t tokens, ld;
  const float* bias;  // optional [experts]
  int32_t* ids;       // [tokens][k]
  float* weights;     // [tokens][k]
  int32_t experts, k, scoring, groups, kept_groups, group_score, renormalize;
  int32_t vec, vec_bias;  // a lane's run of logits, of biases may be read by vectors
  float scale;
};

__device__ __forceinline__ float route_load(const float* p) { return *p; }
__device__ __forceinline__ float route_load(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
__device__ __forceinline__ void route_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void route_store(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// A lane's run of V consecutive logits: bytes of one vector access to it (at most 16).
template <typename T, int V>
__host__ __device__ constexpr int run_vector_bytes() {
  return V * static_cast<int>(sizeof(T)) < 16 ? V * static_cast<int>(sizeof(T)) : 16;
}

// l[i] = row[e0 + i] for those below `experts`, -inf after them.
template <typename T, int V>
__device__ __forceinline__ void load_run(const T* row, int e0, int experts, bool vec,
                                         float (&l)[V]) {
  constexpr int kBytes = run_vector_bytes<T, V>();
  if (kBytes >= 4 && vec && e0 + V <= experts) {
    constexpr int kWords = V * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kWords > 0 ? kWords : 1];
    if constexpr (kBytes == 16) {
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q) {
        const uint4 v = *reinterpret_cast<const uint4*>(row + e0 + q * (16 / sizeof(T)));
        w[4 * q] = v.x;
        w[4 * q + 1] = v.y;
        w[4 * q + 2] = v.z;
        w[4 * q + 3] = v.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(row + e0);
      w[0] = v.x;
      w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(row + e0);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4)
        l[i] = __uint_as_float(w[i]);
      else
        l[i] = __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) l[i] = e0 + i < experts ? route_load(row + e0 + i) : -INFINITY;
}

// row[e0 + i] = v[i] for those below `experts`.
template <typename T, int V>
__device__ __forceinline__ void store_run(T* row, int e0, int experts, bool vec,
                                          const float (&v)[V]) {
  constexpr int kBytes = run_vector_bytes<T, V>();
  if (kBytes >= 4 && vec && e0 + V <= experts) {
    constexpr int kWords = V * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kWords > 0 ? kWords : 1];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(v[i]);
      else
        w[i] = ptx::pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (kBytes == 16) {
#pragma unroll
      for (int q = 0; q < kWords / 4; ++q)
        *reinterpret_cast<uint4*>(row + e0 + q * (16 / sizeof(T))) =
            make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(row + e0) = make_uint2(w[0], w[1]);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(row + e0) = w[0];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e0 + i < experts) route_store(row + e0 + i, v[i]);
}

__device__ __forceinline__ double neg_inf() { return __longlong_as_double(0xfff0000000000000ll); }
__device__ __forceinline__ float nan_f32() { return __uint_as_float(0x7fc00000u); }

// Reductions and ballots over the L consecutive lanes that share a token (all 32 lanes of the warp
// must call them).
template <int L, typename F>
__device__ __forceinline__ F lanes_sum(F v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ double lanes_max(double v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}
template <int L>
__device__ __forceinline__ uint32_t lanes_min(uint32_t v) {
  return ~lanes_max<L>(~v);
}
// One bit per lane of the token.
template <int L>
__device__ __forceinline__ uint32_t lanes_ballot(bool b) {
  const uint32_t all = __ballot_sync(0xffffffffu, b);
  if constexpr (L == 32) {
    return all;
  } else {
    return (all >> (threadIdx.x & 31u & ~(L - 1u))) & ((1u << L) - 1u);
  }
}

// Unsigned keys that order like the floats (no NaN; -0 just below +0).  Every key of a number above
// -inf exceeds kNoKey, the key of -inf.
constexpr uint32_t kNoKey = 0x007fffffu;
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (L == 32) {
    return key_value(__reduce_max_sync(0xffffffffu, order_key(v)));
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}

// e^x and 1 / x by the hardware's approximations, results below 2^-126 flushed to zero: at most
// 2 + 1.173 |x| ulp (the product with log2 e, then 2 ulp) and 1 ulp off.
__device__ __forceinline__ float fast_exp(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504f));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }
// Within 4.5 ulp: e^-|l| has 2, the sum half of one and the quotient 2.  Nothing overflows, so small
// values keep their size down to the subnormals.
__device__ __forceinline__ float sigmoid32(float l) {
  const float t = expf(-fabsf(l));
  return __fdividef(l >= 0.f ? 1.f : t, 1.f + t);
}

// A logit that cannot be chosen and spoils its row's weights: NaN, and +inf under the softmax.
__device__ __forceinline__ bool route_bad(float l, int32_t scoring) {
  return l != l || (scoring == kRouteSoftmax && l == __uint_as_float(0x7f800000u));
}

// Shares of the chosen experts: lane j holds choice j's logit and (softmax over all experts) its
// probability.  Renormalised softmax shares are the softmax of the chosen logits alone;
// renormalised sigmoid shares of logits all below kSmallLogit likewise: there sigmoid(l) = e^l within
// e^-17 < 2^-24 of it, and scores that underflow still have shares.  Lanes without a choice get 0.
constexpr float kSmallLogit = -17.f;
template <int L>
__device__ __forceinline__ float route_share(int32_t scoring, int32_t renormalize, bool has, float l,
                                             float prob) {
  if (!renormalize) return has ? (scoring == kRouteSoftmax ? prob : sigmoid32(l)) : 0.f;
  const float top = lanes_max<L>(has ? l : -INFINITY);
  float v = 0.f;
  if (has) v = scoring == kRouteSoftmax || top < kSmallLogit ? expf(l - top) : sigmoid32(l);
  const float sum = lanes_sum<L>(v);
  return sum > 0.f ? __fdividef(v, sum) : 0.f;
}

// c of the lane's run of the row (by_logit: l) in 64 bits, -inf where an expert cannot be chosen.
template <typename T, int L, int V>
__device__ __forceinline__ void route_scores64(const RouteParams& p, const T* row, bool by_logit,
                                               double (&c)[V]) {
  const int sub = threadIdx.x % L;
  float l[V];
  load_run<T, V>(row, sub * V, p.experts, p.vec != 0, l);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (route_bad(l[i], p.scoring)) l[i] = -INFINITY;
  const bool softmax = p.scoring == kRouteSoftmax && !by_logit;
  double top = neg_inf(), sum = 0.0;
  if (softmax) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmax(top, static_cast<double>(l[i]));
    top = lanes_max<L>(top);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = 0.0;
    if (by_logit)
      c[i] = static_cast<double>(l[i]);
    else if (l[i] > -INFINITY)
      c[i] = softmax ? exp(static_cast<double>(l[i]) - top) : sigmoid64(static_cast<double>(l[i]));
    sum += c[i];
  }
  if (softmax) sum = lanes_sum<L>(sum);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = sub * V + i;
    if (softmax) c[i] = sum > 0.0 ? c[i] / sum : 0.0;
    if (p.bias != nullptr && e < p.experts) c[i] += static_cast<double>(p.bias[e]);
    if (!(l[i] > -INFINITY) || c[i] != c[i]) c[i] = neg_inf();
  }
}

// The kept groups of a row, one bit each, ranked in 64 bits: lane g scores group g and keeps it if
// fewer than kept_groups are better (a higher score, or the same and a lower index).  c_sh: L * V
// words of the token's own shared memory.
template <typename T, int L, int V>
__device__ __forceinline__ uint32_t route_groups64(const RouteParams& p, const T* row,
                                                double* c_sh) {
  const int sub = threadIdx.x % L;
  double c[V];
  route_scores64<T, L, V>(p, row, false, c);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < V; ++i) c_sh[sub * V + i] = c[i];
  __syncwarp();
  const int per = p.experts / p.groups;
  double a = neg_inf(), b = neg_inf();
  if (sub < p.groups) {
    for (int i = 0; i < per; ++i) {
      const double v = c_sh[sub * per + i];
      b = fmax(b, fmin(a, v));
      a = fmax(a, v);
    }
    if (p.group_score == kRouteGroupTop2 && b > neg_inf()) a += b;
  }
  int better = 0;
  for (int g = 0; g < p.groups; ++g) {
    const double v = __shfl_sync(0xffffffffu, a, g, L);
    better += (v > a || (v == a && g < sub)) ? 1 : 0;
  }
  __syncwarp();
  return lanes_ballot<L>(sub < p.groups && better < p.kept_groups);
}

// Place of this lane's candidate id (-1: none) among those of the token's lanes, c in 64 bits.
template <typename T, int L, int V>
__device__ __forceinline__ int route_place64(const RouteParams& p, const T* row, int32_t id,
                                          bool by_logit) {
  double mine = neg_inf();
  if (id >= 0) mine = static_cast<double>(route_load(row + id));
  if (!by_logit) {
    if (p.scoring == kRouteSoftmax) {
      float l[V];
      load_run<T, V>(row, (threadIdx.x % L) * V, p.experts, p.vec != 0, l);
      double top = neg_inf(), sum = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (route_bad(l[i], p.scoring)) l[i] = -INFINITY;
        top = fmax(top, static_cast<double>(l[i]));
      }
      top = lanes_max<L>(top);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (l[i] > -INFINITY) sum += exp(static_cast<double>(l[i]) - top);
      mine = exp(mine - top) / lanes_sum<L>(sum);
    } else {
      mine = sigmoid64(mine);
    }
    if (id >= 0 && p.bias != nullptr) mine += static_cast<double>(p.bias[id]);
  }
  int place = 0;
  for (int i = 0; i < L; ++i) {
    const double v = __shfl_sync(0xffffffffu, mine, i, L);
    const int32_t other = __shfl_sync(0xffffffffu, id, i, L);
    if (other >= 0) place += (v > mine || (v == mine && other < id)) ? 1 : 0;
  }
  return place;
}

// The k best experts of a row among those whose bit of `open` (one per place of the lane's run) is
// set, c in 64 bits: lane j returns choice j, or -1.
template <typename T, int L, int V>
__device__ __forceinline__ int32_t route_rank64(const RouteParams& p, const T* row, uint32_t open,
                                             bool by_logit) {
  const int sub = threadIdx.x % L;
  double c[V];
  route_scores64<T, L, V>(p, row, by_logit, c);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (((open >> i) & 1u) == 0u) c[i] = neg_inf();
  int32_t my_id = -1;
  for (int j = 0; j < p.k; ++j) {
    double best = neg_inf();
    int at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (c[i] > best) {
        best = c[i];
        at = i;
      }
    }
    const double all = lanes_max<L>(best);
    const bool some = all > neg_inf();
    const int owner = __ffs(lanes_ballot<L>(best == all)) - 1;
    const int id = __shfl_sync(0xffffffffu, sub * V + at, owner, L);
    if (some && sub == j) my_id = id;
    if (some && sub == owner) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i == at) c[i] = neg_inf();
    }
  }
  return my_id;
}

// Sorts a lane's N keys, the largest first (odd-even merge network).
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&a)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2) {
#pragma unroll
    for (int k = p; k >= 1; k /= 2) {
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k) {
#pragma unroll
        for (int i = 0; i < k; ++i) {
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t hi = max(a[i + j], a[i + j + k]);
            a[i + j + k] = min(a[i + j], a[i + j + k]);
            a[i + j] = hi;
          }
        }
      }
    }
  }
}

// L lanes per token (k and groups <= L, experts <= L * V), so that what a warp does per token serves
// 32 / L of them; lane l of them holds experts l * V .. l * V + V - 1.  Each lane sorts the keys of
// its run; the choices are then k maxima over the lanes' first keys, the lane that holds the maximum
// moving up by one.  The low log2 V bits of a key hold the place in the run (lower places
// first), so a key names its expert in the run; what they cost in precision is part of the bound
// below.
//
// Error of the 32-bit scores (u = 2^-23, one ulp of 1):
//   sigmoid: e^-l is off by (2 + 1.173 |l|) u, which s (1 - s) turns into at most 0.63 u of s;
//            the sum 1 + e^-l and the quotient add 2.5: below 4 u = 2^-21 altogether.
//   softmax: p = e^(l - top) inv with inv <= 1 the common factor.  inv is off by at most
//            d = (10.2 + 18.5 + 2) u of itself: the terms' errors weighted by p, whose mean
//            |l - top| is at most ln 1024; V + log2 L <= 37 additions; the quotient.  Two p share
//            it, and since p <= inv it moves their difference by at most d inv.  Beside it each p has
//            its exponential's error, at most 2 u inv, and the product's rounding, at most u / 2
//            inv.  So a difference of two p is off by at most (30.7 + 2 (2 + 0.5)) u inv = 35.7 u inv
//            and one of two sums of two p by twice that; `near` below is 64 u inv = 2^-17 inv.
// c = s + bias adds half an ulp of c, a key's lost bits less than V ulp (`rel`).  Two c nearer than
// the bound are ranked in 64 bits (the choices and what is near the last of them; groups likewise,
// whose scores are not cut to keys), unless logit and bias are the same: such c are equal, and the
// lower index goes first.
template <typename T, int L, int V>
__global__ void __launch_bounds__(32 * kRouteWarps, V <= 8 ? 8 : (V == 16 ? 4 : 2))
    route_kernel(const __grid_constant__ RouteParams p) {
  kernel_begins();
  extern __shared__ double route_smem[];
  __shared__ int32_t chosen[kRouteWarps][kRouteMaxK];
  constexpr uint32_t kPlace = V - 1;  // bits of a key that hold the place in the run
  constexpr int kTokens = 32 / L;  // of a warp
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int sub = lane % L;     // lane of the token
  const int first = lane - sub; // the warp's lane that is the token's first
  double* c_sh = route_smem + warp * (32 * V);
  int32_t* picks = &chosen[warp][first];
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_score == kRouteGroupMax);
  const bool softmax = p.scoring == kRouteSoftmax;
  const int e0 = sub * V;
  const bool off = e0 >= p.experts;  // a lane without experts
  const int per = p.experts / p.groups;  // experts of a group
  const int lanes = per / V;             // lanes of a group, when that is a whole power of two
  const bool whole = lanes * V == per && (lanes & (lanes - 1)) == 0;
  const int group = whole ? sub / lanes : sub;       // the group this lane scores
  const int first_group = e0 / per;                  // group of the run's first expert ...
  const int first_left = per - (e0 - first_group * per);  // ... and how many of it follow
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRouteWarps * kTokens;
  for (int64_t t0 = (blockIdx.x * static_cast<int64_t>(kRouteWarps) + warp) * kTokens;
       t0 < p.tokens; t0 += step) {
    const int64_t t = t0 + lane / L;
    const bool live = t < p.tokens;  // past the last token a lane works on row 0 and stores nothing
    const T* row = static_cast<const T*>(p.logits) + (live ? t : 0) * p.ld;
    float l[V], c[V];
    load_run<T, V>(row, e0, p.experts, p.vec != 0, l);
    bool bad = false;
    // l with what cannot be chosen at -inf.
    auto clean = [&]() {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (route_bad(l[i], p.scoring)) {
          bad = true;
          l[i] = -INFINITY;
        }
        if (off) l[i] = -INFINITY;
      }
    };
    float top = -INFINITY, inv = 1.f;
    // c of the run.  `all` assumes finite logits and biases; otherwise what cannot be chosen
    // becomes -inf.
    auto score = [&](auto all) {
      constexpr bool kAll = decltype(all)::value;
      if (softmax && (!by_logit || !p.renormalize)) {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) top = fmaxf(top, l[i]);
        if (kAll && off) top = -INFINITY;
        top = lanes_max<L>(top);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          c[i] = kAll || l[i] > -INFINITY ? fast_exp(l[i] - top) : 0.f;
          sum += c[i];
        }
        if (kAll && off) sum = 0.f;
        sum = lanes_sum<L>(sum);
        inv = sum > 0.f ? __fdividef(1.f, sum) : 0.f;
      }
      if (by_logit) {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = l[i] + 0.f;  // -0 as +0
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          c[i] = softmax ? c[i] * inv : fast_rcp(1.f + fast_exp(-l[i]));
        if (p.bias != nullptr && !off) {
          float b[V];
          load_run<float, V>(p.bias, e0, p.experts, p.vec_bias != 0, b);
#pragma unroll
          for (int i = 0; i < V; ++i) c[i] += b[i];
        }
      }
      if (!kAll) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (!(l[i] > -INFINITY) || c[i] != c[i]) c[i] = -INFINITY;
      }
    };
    if (off) {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = 0.f;
    }
    score(std::true_type{});
    float finite = 0.f;  // 0 x l is NaN where l is not finite; a bias that is not makes c so
#pragma unroll
    for (int i = 0; i < V; ++i) finite = fmaf(l[i], 0.f, finite);
    if (!by_logit) {
#pragma unroll
      for (int i = 0; i < V; ++i) finite = fmaf(c[i], 0.f, finite);
    }
    if (__any_sync(0xffffffffu, finite != finite)) {
      clean();
      bad = lanes_ballot<L>(bad) != 0u;
      score(std::false_type{});
    }
    // Two c whose difference is at most near + rel (|c1| + |c2|) may be in another order.
    const float near = by_logit ? 0.f : (softmax ? 0x1p-17f * inv : 2.f * 0x1p-21f);
    const float rel = 0x1p-22f + V * 0x1p-23f;
    uint32_t open = ~0u;  // one bit per place of the run: its group is kept
    if (p.groups > 1) {
      float a = -INFINITY, a2 = -INFINITY;  // the group's two best
      if (whole) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a2 = fmaxf(a2, fminf(a, c[i]));
          a = fmaxf(a, c[i]);
        }
        for (int o = 1; o < lanes; o <<= 1) {
          const float u = __shfl_xor_sync(0xffffffffu, a, o);
          const float u2 = __shfl_xor_sync(0xffffffffu, a2, o);
          a2 = fmaxf(fminf(a, u), fmaxf(a2, u2));
          a = fmaxf(a, u);
        }
      } else {
        float* f_sh = reinterpret_cast<float*>(c_sh + first * V);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) f_sh[e0 + i] = c[i];
        __syncwarp();
        if (sub < p.groups) {
          for (int i = 0; i < per; ++i) {
            const float v = f_sh[sub * per + i];
            a2 = fmaxf(a2, fminf(a, v));
            a = fmaxf(a, v);
          }
        }
        __syncwarp();
      }
      const bool real = group < p.groups;
      const bool some = real && a > -INFINITY;
      float slack = 0.5f * near + 0x1p-23f * fabsf(a);
      if (p.group_score == kRouteGroupTop2 && a2 > -INFINITY) {
        slack = near + 0x1p-22f * (fabsf(a) + fabsf(a2));
        a += a2;
      }
      // kept_groups times the best group left, the lowest among equals.
      uint32_t rank_key = real && a > -INFINITY ? order_key(a) : kNoKey;
      bool kept = false;
      for (int i = 0; i < p.kept_groups; ++i) {
        const uint32_t best = lanes_max<L>(rank_key);
        const int owner = __ffs(lanes_ballot<L>(rank_key == best)) - 1;
        if (group == __shfl_sync(0xffffffffu, group, owner, L) && best != kNoKey) {
          kept = true;
          rank_key = kNoKey;
        }
      }
      if (!by_logit) {
        const uint32_t worst_kept =
            lanes_min<L>(kept && some ? order_key(a - slack) : 0xffffffffu);
        const uint32_t best_left =
            lanes_max<L>(!kept && some ? order_key(a + slack) : kNoKey);
        // A sum that overflows (biases of the lowest value as masks) has no 32-bit rank at all.
        const bool lost = some && !(fabsf(a) + slack < INFINITY);
        // Every lane votes, and one token's doubt has all tokens of the warp ranked again: lanes that
        // skipped a vote or a shuffle because of their token would leave the others waiting in it.
        const bool close = best_left >= worst_kept;
        if (__any_sync(0xffffffffu, close | lost))
          kept = (route_groups64<T, L, V>(p, row, c_sh + first * V) >> group) & 1u;
      }
      if (whole) {
        if (!kept) open = 0u;
      } else {
        const uint32_t keep = lanes_ballot<L>(kept);
        int g = first_group, left = first_left;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (g >= p.groups || ((keep >> g) & 1u) == 0u) open &= ~(1u << i);
          if (--left == 0) {
            left = per;
            ++g;
          }
        }
      }
      if (open != ~0u) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (((open >> i) & 1u) == 0u) c[i] = -INFINITY;
      }
    }
    uint32_t key[V];
    const uint32_t value_bits = off ? 0u : ~kPlace;
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = (order_key(c[i]) & value_bits) | (kPlace - i);
    sort_keys(key);
    // The lane's first key stays in a register, the others wait in shared memory.
    uint32_t head = key[0];
    uint32_t* rest = reinterpret_cast<uint32_t*>(c_sh) + lane;
#pragma unroll
    for (int i = 1; i < V; ++i) rest[32 * (i - 1)] = key[i];
    rest[32 * (V - 1)] = 0u;
    // The row's largest key without its place bits (all ones), at most kNoKey if none is left, and
    // the lane that gives it: the lowest among equals.
    auto largest = [&]() { return lanes_max<L>(head | kPlace); };
    auto holds = [&](uint32_t all) {
      const bool equal = (head | kPlace) == all;
      const uint32_t those = lanes_ballot<L>(equal);
      return equal && (those & ((1u << sub) - 1u)) == 0u;
    };
    auto next = [&]() {  // on to the lane's next key
      head = *rest;
      rest += 32;
    };
    uint32_t my_key = kNoKey, last_key = kNoKey;
    int found = 0;
    for (int j = 0; j < p.k; ++j) {
      const uint32_t all = largest();
      const bool some = all > kNoKey;
      if (holds(all) && some) {
        picks[j] = e0 + static_cast<int>(kPlace - (head & kPlace));
        next();
      }
      if (some) {
        if (sub == j) my_key = all;
        last_key = all;
        ++found;
      }
    }
    __syncwarp();
    int32_t my_id = sub < found ? picks[sub] : -1;
    __syncwarp();
    float my_l = my_id >= 0 ? route_load(row + my_id) : 0.f;
    bool near_pair = false;
    int candidates = found;
    // BF16 logits fit in a key whole: ranked by them, the order is exact.
    bool many = false;  // more candidates than lanes
    if (!(by_logit && (sizeof(T) == 2 || V == 1))) {
      auto nearer = [&](uint32_t k1, uint32_t k2) {
        const float c1 = key_value(k1 & ~kPlace), c2 = key_value(k2 & ~kPlace);
        return by_logit ? c1 == c2 : c1 - c2 <= near + rel * (fabsf(c1) + fabsf(c2));
      };
      // Neighbours in the order.
      const float my_b = my_id >= 0 && p.bias != nullptr ? __ldg(p.bias + my_id) : 0.f;
      const uint32_t next_key = __shfl_down_sync(0xffffffffu, my_key, 1, L);
      const float next_l = __shfl_down_sync(0xffffffffu, my_l, 1, L);
      const float next_b = __shfl_down_sync(0xffffffffu, my_b, 1, L);
      near_pair = sub + 1 < found && nearer(my_key, next_key) &&
                  !(my_l == next_l && my_b == next_b);
      // The last choice against the best ones left: those that are near become candidates too.
      const float last_l = __shfl_sync(0xffffffffu, my_l, p.k - 1, L);
      const float last_b = __shfl_sync(0xffffffffu, my_b, p.k - 1, L);
      bool more = found == p.k;
      while (true) {
        const uint32_t all = largest();
        more = more && all > kNoKey && nearer(last_key, all);
        if (more && candidates == L) {
          many = true;
          more = false;
        }
        if (!__any_sync(0xffffffffu, more)) break;
        if (holds(all) && more) {
          const int id = e0 + static_cast<int>(kPlace - (head & kPlace));
          picks[candidates] = id;
          near_pair |= route_load(row + id) != last_l ||
                       (p.bias != nullptr ? __ldg(p.bias + id) : 0.f) != last_b;
          next();
        }
        if (more) ++candidates;
      }
    }
    if (__any_sync(0xffffffffu, near_pair || many)) {
      __syncwarp();
      // For all tokens of the warp alike, again: the 64-bit order is right for every one of them.
      if (__any_sync(0xffffffffu, many)) {
        my_id = route_rank64<T, L, V>(p, row, open, by_logit);
      } else {
        const int32_t id = sub < candidates ? picks[sub] : -1;
        const int place = route_place64<T, L, V>(p, row, id, by_logit);
        __syncwarp();
        if (id >= 0 && place < p.k) picks[place] = id;
        __syncwarp();
        my_id = sub < found ? picks[sub] : -1;
        __syncwarp();
      }
      my_l = my_id >= 0 ? route_load(row + my_id) : 0.f;
    }
    const bool has = my_id >= 0;
    const float prob = has && softmax && !p.renormalize ? expf(my_l - top) * inv : 0.f;
    const float w = route_share<L>(p.scoring, p.renormalize, has, my_l, prob);
    if (live && sub < p.k) {
      p.ids[t * p.k + sub] = my_id;
      p.weights[t * p.k + sub] = bad ? nan_f32() : w * p.scale;
    }
  }
}

struct RouteGradParams {
  const float* dweights;  // [tokens][k]
  const void* logits;
  int64_t tokens, ld;
  const int32_t* ids;  // [tokens][k]
  void* dlogits;
  int64_t ldd;
  int32_t experts, k, scoring, renormalize;
  int32_t vec, vec_out;  // runs of logits and of dlogits may be accessed by vectors
  float scale;
};

// dl of a token, with g = dL/dw of its choices and r their shares (w = scale r):
//   softmax, renormalised:  dl_j = scale r_j (g_j - sum g r)        (0 elsewhere)
//   softmax:                dl_e = scale p_e (g_e - sum g p)        (g_e = 0 where not chosen)
//   sigmoid, renormalised:  dl_j = scale r_j (g_j - sum g r) (1 - s_j)
//   sigmoid:                dl_j = scale g_j s_j (1 - s_j)
// L lanes per token (k <= L, experts <= L * V), so that a warp's sums and exponentials serve 32 / L
// tokens; lane l holds the vectors l, L + l, 2 L + l, ... of the row.  An expert that is chosen
// twice gets both terms.
template <typename T, int L, int V>
__global__ void __launch_bounds__(32 * kRouteWarps) route_grad_kernel(const RouteGradParams p) {
  kernel_begins();
  constexpr int kPer = 16 / static_cast<int>(sizeof(T)) < V ? 16 / static_cast<int>(sizeof(T)) : V;
  constexpr int kVecs = V / kPer;  // vectors of kPer logits a lane holds
  constexpr int kTokens = 32 / L * kRouteWarps;
  const int sub = threadIdx.x % L;
  const bool dense = p.scoring == kRouteSoftmax && !p.renormalize;
  auto sum_of = [](float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto max_of = [](float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  for (int64_t t0 = blockIdx.x * static_cast<int64_t>(kTokens); t0 < p.tokens;
       t0 += static_cast<int64_t>(gridDim.x) * kTokens) {
    const int64_t t = t0 + threadIdx.x / L;
    const bool live = t < p.tokens;
    const T* row = static_cast<const T*>(p.logits) + (live ? t : 0) * p.ld;
    int id = -1;
    float g = 0.f;
    if (live && sub < p.k) {
      id = p.ids[t * p.k + sub];
      g = p.dweights[t * p.k + sub];
    }
    float l[kVecs][kPer];
    float finite = 0.f;  // NaN once a logit is +-inf or NaN
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
      const int e0 = (q * L + sub) * kPer;
      load_run<T, kPer>(row, e0, live ? p.experts : 0, p.vec != 0, l[q]);
    }
    // A masked expert (logit -inf) scores 0 whatever its logit does: it takes no part.
    float lj = -INFINITY;
    if (id >= 0 && id < p.experts) lj = route_load(row + id);
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
#pragma unroll
      for (int i = 0; i < kPer; ++i) finite = fmaf(l[q][i], 0.f, finite);
    bool bad = false;
    if (__any_sync(0xffffffffu, finite != finite)) {
      float spoiled = 0.f;
#pragma unroll
      for (int q = 0; q < kVecs; ++q)
#pragma unroll
        for (int i = 0; i < kPer; ++i) spoiled += route_bad(l[q][i], p.scoring) ? 1.f : 0.f;
      bad = sum_of(spoiled) > 0.f;
    }
    float top = -INFINITY, inv = 0.f;
    float out[kVecs][kPer];
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
#pragma unroll
      for (int i = 0; i < kPer; ++i) out[q][i] = 0.f;
    if (dense) {
#pragma unroll
      for (int q = 0; q < kVecs; ++q)
#pragma unroll
        for (int i = 0; i < kPer; ++i) top = fmaxf(top, l[q][i]);
      top = max_of(top);
      const float from = top > -INFINITY ? top : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < kVecs; ++q)
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          out[q][i] = expf(l[q][i] - from);
          sum += out[q][i];
        }
      sum = sum_of(sum);
      inv = sum > 0.f ? __fdividef(1.f, sum) : 0.f;
    }
    const bool has = lj > -INFINITY && !bad;
    float r = 0.f;  // as route_share
    if (!p.renormalize) {
      if (has) r = dense ? expf(lj - top) * inv : sigmoid32(lj);
    } else {
      const float best = max_of(has ? lj : -INFINITY);
      if (has)
        r = p.scoring == kRouteSoftmax || best < kSmallLogit ? expf(lj - best) : sigmoid32(lj);
      const float sum = sum_of(r);
      r = sum > 0.f ? __fdividef(r, sum) : 0.f;
    }
    float add = 0.f;  // the choice's own term
    float mean = 0.f;
    if (dense || p.renormalize) mean = sum_of(has ? g * r : 0.f);
    if (has) {
      add = p.renormalize ? r * (g - mean) : g * r;
      if (p.scoring == kRouteSigmoid) add *= sigmoid32(-lj);
    }
    // An expert chosen twice: every lane that holds it sums both terms, in the order of j.
    const int at = has ? id : -1;
    float sum_at = 0.f;
    for (int j = 0; j < p.k; ++j) {
      const int ej = __shfl_sync(0xffffffffu, at, j, L);
      const float aj = __shfl_sync(0xffffffffu, add, j, L);
      if (ej == at) sum_at += aj;
    }
    // The row as if nothing were chosen, then the choices over it (ordered by the __syncwarp).
    T* drow = static_cast<T*>(p.dlogits) + (live ? t : 0) * p.ldd;
    const float all_scale = bad ? nan_f32() : dense ? -inv * mean * p.scale : 0.f;
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) out[q][i] *= all_scale;
      store_run<T, kPer>(drow, (q * L + sub) * kPer, live ? p.experts : 0, p.vec_out != 0, out[q]);
    }
    __syncwarp();
    if (has) route_store(drow + id, (sum_at - (dense ? r * mean : 0.f)) * p.scale);
  }
}

// ------------------------------------------------------------------------------- expert order
// offsets[e] = pairs of the experts before e; slot of a pair = offsets[e] + the pairs of e before it
// in (token, choice) order, so the order is the same in every run.  One cluster does it all: every
// warp owns a contiguous run of pairs and counts its experts, the counts are summed over the
// warps and, through distributed shared memory, over the cluster's blocks, and each warp walks its
// run again handing out slots.
constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kOrderMaxCluster = 16;  // 8 where 16 blocks do not fit in one cluster
constexpr int kOrderHold = 16;  // pairs a lane loads at a time

struct OrderParams {
  const int32_t* ids;
  int64_t pairs;
  int32_t experts;
  int32_t* offsets;  // [experts + 1]
  int32_t* slots;    // [pairs]
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// Shared memory: counts[kOrderWarps][experts], then total[experts].
// kBits: bits of an expert's index.
template <int kBits>
__global__ void __launch_bounds__(kOrderThreads, 1) expert_order_kernel(const OrderParams p) {
  kernel_begins();
  extern __shared__ uint32_t order_smem[];
  __shared__ uint32_t warp_sums[kOrderWarps];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int E = p.experts;
  const uint32_t blocks = gridDim.x;  // one cluster
  const uint32_t rank = blockIdx.x;
  uint32_t* total = order_smem + kOrderWarps * E;
  uint32_t* mine = order_smem + warp * E;
  // This warp's run of pairs (a multiple of 32 of them).
  const int64_t warps = static_cast<int64_t>(blocks) * kOrderWarps;
  const int64_t run = (p.pairs + warps * 32 - 1) / (warps * 32) * 32;
  const int64_t first = (static_cast<int64_t>(rank) * kOrderWarps + warp) * run;
  const int64_t last = first + run < p.pairs ? first + run : p.pairs;
  // kOrderHold pairs per lane at a time, all loaded before the first is used; a run of one such
  // chunk keeps them, and their ranks, for the second walk.
  constexpr int kChunk = 32 * kOrderHold;
  const bool hold = run <= kChunk;
  int32_t held[kOrderHold];
  uint32_t rnk[kOrderHold];
  auto load = [&](int64_t i0) {
#pragma unroll
    for (int u = 0; u < kOrderHold; ++u) {
      const int64_t i = i0 + u * 32 + lane;
      held[u] = i < last ? p.ids[i] : -1;
      if (held[u] >= E) held[u] = -1;  // no expert
    }
  };
  // Ranks of the held pairs among the run's pairs of the same expert, counting on in `mine`.  The
  // lanes with the same expert are found by one ballot per bit of it (match.any takes several
  // times as long), and the lowest of them counts them all.
  auto count = [&](int64_t i0) {
#pragma unroll
    for (int u = 0; u < kOrderHold; ++u) {
      if (i0 + u * 32 >= last) break;
      const bool real = held[u] >= 0;
      uint32_t peers = __ballot_sync(0xffffffffu, real);
#pragma unroll
      for (int bit = 0; bit < kBits; ++bit) {
        const uint32_t v = __ballot_sync(0xffffffffu, (held[u] >> bit) & 1);
        peers &= v ^ (((held[u] >> bit) & 1) - 1u);  // those with the same bit
      }
      const uint32_t before = __popc(peers & ((1u << lane) - 1u));
      rnk[u] = real ? mine[held[u]] + before : 0u;
      __syncwarp();
      if (real && before == 0u) mine[held[u]] = rnk[u] + __popc(peers);
      __syncwarp();
    }
  };
  if (hold) load(first);
  for (int i = threadIdx.x; i < kOrderWarps * E; i += kOrderThreads) order_smem[i] = 0u;
  __syncthreads();
  if (hold) {
    count(first);
  } else {
    for (int64_t i0 = first; i0 < last; i0 += kChunk) {
      load(i0);
      count(i0);
    }
  }
  __syncthreads();
  // The block's counts of expert e, thread e.
  const int e = threadIdx.x;
  if (e < E) {
    uint32_t s = 0u;
#pragma unroll 8
    for (int w = 0; w < kOrderWarps; ++w) s += order_smem[w * E + e];
    total[e] = s;
  }
  if (blocks > 1) {
    ptx::cluster_sync();
  } else {
    __syncthreads();
  }
  uint32_t all = 0u, before = 0u;  // of the expert in the cluster, and in the blocks before
  if (e < E) {
    if (blocks > 1) {
      const uint32_t addr = ptx::smem_u32(total + e);
#pragma unroll
      for (uint32_t b = 0; b < kOrderMaxCluster; ++b) {
        if (b >= blocks) break;
        const uint32_t v = ld_cluster_u32(ptx::mapa_shared(addr, b));
        if (b < rank) before += v;
        all += v;
      }
    } else {
      all = total[e];
    }
  }
  // Exclusive scan of the experts' totals over the block's threads.
  uint32_t incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  const uint32_t base = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0u);
  const uint32_t start = base + incl - all;
  if (e < E) {
    if (rank == 0) {
      p.offsets[e] = static_cast<int32_t>(start);
      if (e == E - 1) p.offsets[E] = static_cast<int32_t>(start + all);
    }
    // First slot of every warp's pairs of the expert.
    uint32_t s = start + before;
    for (int w0 = 0; w0 < kOrderWarps; w0 += 8) {
      uint32_t of_warp[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) of_warp[w] = order_smem[(w0 + w) * E + e];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        order_smem[(w0 + w) * E + e] = s;
        s += of_warp[w];
      }
    }
  }
  __syncthreads();
  auto store = [&](int64_t i0, bool add) {
#pragma unroll
    for (int u = 0; u < kOrderHold; ++u) {
      const int64_t i = i0 + u * 32 + lane;
      if (i < last)
        p.slots[i] = held[u] >= 0 ? static_cast<int32_t>(rnk[u] + (add ? mine[held[u]] : 0u)) : -1;
    }
  };
  if (hold) {
    store(first, true);
  } else {
    // Counting on from the first slots gives the slots themselves.
    for (int64_t i0 = first; i0 < last; i0 += kChunk) {
      load(i0);
      count(i0);
      store(i0, false);
    }
  }
  if (blocks > 1) ptx::cluster_sync();  // no block leaves while another may read its totals
}

}  // namespace cpg
