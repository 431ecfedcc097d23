// Routing to experts: scores, the choice of k experts per token and their weights, the gradient,
// and the expert order of the chosen (token, choice) pairs.
//
//   s = softmax(l) or sigmoid(l);  c = s + bias (what is ranked);  ids = the k largest c among the
//   kept groups, ties to the lowest index;  w = scale * s[ids], over the sum of s[ids] if renormalised.
//
// c is ranked in 64 bits: two 32-bit scores may round to one value, or to the wrong order, where
// their logits do not.  Without a bias and with group score "max" c is not formed: s grows with l,
// so the logits rank, exactly.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "ptx.cuh"

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

__device__ __forceinline__ double neg_inf() { return __longlong_as_double(0xfff0000000000000ll); }
__device__ __forceinline__ float nan_f32() { return __uint_as_float(0x7fc00000u); }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }

// A logit that cannot be chosen and spoils its row's weights: NaN, and +inf under the softmax.
__device__ __forceinline__ bool route_bad(float l, int32_t scoring) {
  return l != l || (scoring == kRouteSoftmax && l == __uint_as_float(0x7f800000u));
}

// Weights of the chosen experts: lane j holds choice j's logit and (softmax over all experts) its
// probability.  Renormalised softmax weights are the softmax of the chosen logits alone;
// renormalised sigmoid weights of logits all below -60, where sigmoid(l) = e^l, likewise (the
// sum of the scores would underflow).  Lanes without a choice get 0.
__device__ __forceinline__ double route_part(int32_t scoring, int32_t renormalize, bool has,
                                             double l, double p) {
  if (!renormalize) return has ? (scoring == kRouteSoftmax ? p : sigmoid64(l)) : 0.0;
  const double top = warp_max(has ? l : neg_inf());
  double v;
  if (scoring == kRouteSoftmax || top < -60.0)
    v = has ? exp(l - top) : 0.0;
  else
    v = has ? sigmoid64(l) : 0.0;
  const double sum = warp_sum(v);
  return sum > 0.0 ? v / sum : 0.0;
}

// One warp per token; lane l holds experts l * V .. l * V + V - 1.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteParams p) {
  extern __shared__ double route_smem[];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  double* c_sh = route_smem + warp * (32 * V);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRouteWarps;
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_score == kRouteGroupMax);
  for (int64_t t = blockIdx.x * static_cast<int64_t>(kRouteWarps) + warp; t < p.tokens;
       t += stride) {
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    float l[V];
    bool bad = false;
    double top = neg_inf();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      l[i] = e < p.experts ? route_load(row + e) : -INFINITY;
      if (route_bad(l[i], p.scoring)) {
        bad = true;
        l[i] = -INFINITY;
      }
      top = fmax(top, static_cast<double>(l[i]));
    }
    bad = __any_sync(0xffffffffu, bad);
    top = warp_max(top);
    double s[V], c[V];
    double sum = 0.0;
    const bool scores = !by_logit || (p.scoring == kRouteSoftmax && !p.renormalize);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = 0.0;
      if (scores && l[i] > -INFINITY)
        s[i] = p.scoring == kRouteSoftmax ? exp(static_cast<double>(l[i]) - top)
                                          : sigmoid64(static_cast<double>(l[i]));
      sum += s[i];
    }
    if (scores && p.scoring == kRouteSoftmax) {
      sum = warp_sum(sum);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      if (by_logit) {
        c[i] = static_cast<double>(l[i]);
      } else {
        c[i] = s[i] + (p.bias != nullptr && e < p.experts ? static_cast<double>(p.bias[e]) : 0.0);
        if (!(l[i] > -INFINITY) || c[i] != c[i]) c[i] = neg_inf();
      }
    }
    if (p.groups > 1) {
      // Lane g scores group g, ranks it among the others and keeps it if fewer than kept_groups
      // are better (a higher score, or the same and a lower index).
#pragma unroll
      for (int i = 0; i < V; ++i) c_sh[lane * V + i] = c[i];
      __syncwarp();
      const int per = p.experts / p.groups;
      double a = neg_inf(), b = neg_inf();
      if (lane < p.groups) {
        for (int i = 0; i < per; ++i) {
          const double v = c_sh[lane * per + i];
          if (v > a) {
            b = a;
            a = v;
          } else if (v > b) {
            b = v;
          }
        }
        if (p.group_score == kRouteGroupTop2 && b > neg_inf()) a += b;
      }
      int better = 0;
      for (int g = 0; g < p.groups; ++g) {
        const double v = __shfl_sync(0xffffffffu, a, g);
        better += (v > a || (v == a && g < lane)) ? 1 : 0;
      }
      const uint32_t keep =
          __ballot_sync(0xffffffffu, lane < p.groups && better < p.kept_groups);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int g = (lane * V + i) / per;
        if (g >= p.groups || ((keep >> g) & 1u) == 0u) c[i] = neg_inf();
      }
      __syncwarp();
    }
    // k times: the largest c of the row, the lowest lane (so the lowest index) among equals.
    int my_id = -1;
    float my_l = 0.f;
    double my_s = 0.0;
    for (int j = 0; j < p.k; ++j) {
      double best = neg_inf();
      int at = 0;
      float lb = 0.f;
      double sb = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (c[i] > best) {
          best = c[i];
          at = i;
          lb = l[i];
          sb = s[i];
        }
      }
      const double all = warp_max(best);
      if (!(all > neg_inf())) break;
      const int owner = __ffs(__ballot_sync(0xffffffffu, best == all)) - 1;
      const int id = __shfl_sync(0xffffffffu, lane * V + at, owner);
      const float lw = __shfl_sync(0xffffffffu, lb, owner);
      const double sw = __shfl_sync(0xffffffffu, sb, owner);
      if (lane == j) {
        my_id = id;
        my_l = lw;
        my_s = sw;
      }
      if (lane == owner) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == at) c[i] = neg_inf();
      }
    }
    const double w = route_part(p.scoring, p.renormalize, my_id >= 0, my_l, my_s);
    if (lane < p.k) {
      p.ids[t * p.k + lane] = my_id;
      p.weights[t * p.k + lane] = bad ? nan_f32() : static_cast<float>(w * p.scale);
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
  float scale;
};

// dl of a token, with g = dL/dw of its choices and r their shares (w = scale r):
//   softmax, renormalised:  dl_j = scale r_j (g_j - sum g r)        (0 elsewhere)
//   softmax:                dl_e = scale p_e (g_e - sum g p)        (g_e = 0 where not chosen)
//   sigmoid, renormalised:  dl_j = scale r_j (g_j - sum g r) (1 - s_j)
//   sigmoid:                dl_j = scale g_j s_j (1 - s_j)
// One warp per token; an expert that is chosen twice gets both terms.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kRouteWarps) route_grad_kernel(const RouteGradParams p) {
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRouteWarps;
  for (int64_t t = blockIdx.x * static_cast<int64_t>(kRouteWarps) + warp; t < p.tokens;
       t += stride) {
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    float l[V];
    bool bad = false;
    double top = neg_inf();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      l[i] = e < p.experts ? route_load(row + e) : -INFINITY;
      bad |= route_bad(l[i], p.scoring);
      top = fmax(top, static_cast<double>(l[i]));
    }
    bad = __any_sync(0xffffffffu, bad);
    top = warp_max(top);
    const bool dense = p.scoring == kRouteSoftmax && !p.renormalize;
    double sum = 1.0;
    if (dense) {
      sum = 0.0;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (l[i] > -INFINITY) sum += exp(static_cast<double>(l[i]) - top);
      sum = warp_sum(sum);
    }
    int id = -1;
    double g = 0.0, lj = 0.0;
    if (lane < p.k) {
      id = p.ids[t * p.k + lane];
      if (id < 0 || id >= p.experts) id = -1;
      if (id >= 0) {
        g = static_cast<double>(p.dweights[t * p.k + lane]);
        lj = static_cast<double>(route_load(row + id));
        if (!(lj > neg_inf())) id = -1;  // a masked expert: its score is 0 whatever the logit does
      }
    }
    const bool has = id >= 0 && !bad;
    double pj = 0.0;
    if (dense && has) pj = exp(lj - top) / sum;
    const double r = route_part(p.scoring, p.renormalize, has, lj, pj);
    const double mean = warp_sum(has ? g * r : 0.0);
    double add;  // the choice's own term
    if (dense)
      add = g * r;
    else if (p.renormalize)
      add = r * (g - mean);
    else
      add = g * r;
    if (p.scoring == kRouteSigmoid) add *= sigmoid64(-lj);
    if (!has) add = 0.0;
    double out[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      out[i] = dense && l[i] > -INFINITY
                   ? -exp(static_cast<double>(l[i]) - top) / sum * mean
                   : 0.0;
    for (int j = 0; j < p.k; ++j) {
      const int ej = __shfl_sync(0xffffffffu, has ? id : -1, j);
      const double aj = __shfl_sync(0xffffffffu, add, j);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (ej == lane * V + i) out[i] += aj;
    }
    T* drow = static_cast<T*>(p.dlogits) + t * p.ldd;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      if (e < p.experts)
        route_store(drow + e, bad ? nan_f32() : static_cast<float>(out[i] * p.scale));
    }
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
constexpr int kOrderMaxCluster = 8;

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
__global__ void __launch_bounds__(kOrderThreads, 1) expert_order_kernel(const OrderParams p) {
  extern __shared__ uint32_t order_smem[];
  __shared__ uint32_t warp_sums[kOrderWarps];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int E = p.experts;
  const uint32_t blocks = gridDim.x;  // one cluster
  const uint32_t rank = blockIdx.x;
  uint32_t* total = order_smem + kOrderWarps * E;
  uint32_t* mine = order_smem + warp * E;
  for (int i = threadIdx.x; i < kOrderWarps * E; i += kOrderThreads) order_smem[i] = 0u;
  __syncthreads();
  // This warp's run of pairs (a multiple of 32 of them).
  const int64_t warps = static_cast<int64_t>(blocks) * kOrderWarps;
  const int64_t run = (p.pairs + warps * 32 - 1) / (warps * 32) * 32;
  const int64_t first = (static_cast<int64_t>(rank) * kOrderWarps + warp) * run;
  const int64_t last = first + run < p.pairs ? first + run : p.pairs;
  for (int64_t i = first + lane; i < last; i += 32) {
    const int32_t e = p.ids[i];
    if (e >= 0 && e < E) atomicAdd(mine + e, 1u);  // counts only: any order gives the same sum
  }
  __syncthreads();
  // Exclusive sums over the warps; the block's counts.
  const int e = threadIdx.x;
  if (e < E) {
    uint32_t s = 0u;
    for (int w = 0; w < kOrderWarps; ++w) {
      const uint32_t v = order_smem[w * E + e];
      order_smem[w * E + e] = s;
      s += v;
    }
    total[e] = s;
  }
  __syncthreads();
  if (blocks > 1) ptx::cluster_sync();
  uint32_t all = 0u, before = 0u;
  if (e < E) {
    if (blocks > 1) {
      const uint32_t addr = ptx::smem_u32(total + e);
      for (uint32_t b = 0; b < blocks; ++b) {
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
  uint32_t base = 0u;
  for (int w = 0; w < warp; ++w) base += warp_sums[w];
  const uint32_t start = base + incl - all;
  if (e < E) {
    if (rank == 0) {
      p.offsets[e] = static_cast<int32_t>(start);
      if (e == E - 1) p.offsets[E] = static_cast<int32_t>(start + all);
    }
    for (int w = 0; w < kOrderWarps; ++w) order_smem[w * E + e] += start + before;
  }
  __syncthreads();
  for (int64_t i0 = first; i0 < last; i0 += 32) {
    const int64_t i = i0 + lane;
    int32_t id = i < last ? p.ids[i] : -1;
    if (id >= E) id = -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, id);
    const uint32_t before_me = __popc(peers & ((1u << lane) - 1u));
    uint32_t slot = 0u;
    if (id >= 0) slot = mine[id] + before_me;
    __syncwarp();
    if (id >= 0 && before_me == 0u) mine[id] += __popc(peers);
    __syncwarp();
    if (i < last) p.slots[i] = id >= 0 ? static_cast<int32_t>(slot) : -1;
  }
  if (blocks > 1) ptx::cluster_sync();  // no block leaves while another may read its totals
}

}  // namespace cpg
