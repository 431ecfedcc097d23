// Norm and rotation of query and key heads, and its gradient, one pass over the heads.
//
//   y = R(position) (x * r * w),   r = 1 / sqrt(mean(x^2) + eps)
// where R turns `half` pairs of channels by the angles whose cosines and sines the table holds for
// the token's position; the channels behind them keep their place.  With g = R^T dy, u = g w and
// n = x r:
//   dx = r (u - n mean(u n)),   dw = sum over tokens and heads of g n.
// Bound by HBM: a head is read once (its gradient: x and dy) and written once.  16384 tokens x 32 heads x
// 128, FP32: 87 us, its gradient 133, 0.95 and 0.93 of the copy rate; with BF16 the instructions for twice
// the elements a byte show: 16384 x 40 x 128 68 us (0.75), the gradient of 8191 54 us (0.71).  Narrow
// vectors are bound by instructions: 8192 x 32 x 75 BF16 69 us (0.18), its gradient 177 us (0.10).
//
// A head is split into vectors of V elements, the widest its alignment allows.  A lane takes two
// vectors at a time, those whose channels are turned into one another (channels i and i + half, or
// neighbours), so the rotation needs no exchange between lanes; L lanes share a head and differ
// only in the sum of squares (and of u n), which they add by shuffles.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "row_access.cuh"

namespace cpg {

constexpr int kHeadThreads = 256;

struct HeadPart {
  const void* x;
  const void* dy;  // gradient only
  void* y;         // y, or dx
  const void* w;   // may be null: ones
  int64_t x_token, x_head, dy_token, dy_head, y_token, y_head;
  int32_t heads;
  int32_t w_f32;
  int32_t w_vec;  // it starts on 16 bytes
};

struct HeadParams {
  HeadPart part[2];  // queries, keys
  const float* table;
  int64_t table_rows, table_ld;
  const int32_t* positions;
  int64_t tokens;
  int32_t d, half;
  int32_t interleaved;  // channels 2i and 2i + 1 are turned into one another, else i and i + half
  int32_t table_vec;    // every table row starts on 16 bytes and half is a multiple of 4
  float eps;
  // gradient only
  float* partial;     // [blocks, d]: what each block adds to its part's dw
  int32_t blocks[2];  // blocks of each part
};

// What a lane's pair of vectors is: where they start (-1: none) and how they turn.
struct HeadPair {
  int32_t a, b;    // first channel of each
  int32_t angle;   // first angle of a
  bool turned;     // a and b into one another
  bool inside;     // neighbours within a vector
};

template <int V>
__device__ __forceinline__ HeadPair head_pair(const HeadParams& p, int32_t j) {
  HeadPair r;
  const int32_t nv = p.d / V;
  if (p.interleaved && V > 1) {
    const int32_t far = (nv + 1) / 2;
    r.a = j < far ? j * V : -1;
    r.b = j < far && j + far < nv ? (j + far) * V : -1;
    r.angle = j * V / 2;
    r.turned = false;
    r.inside = true;
    return r;
  }
  const int32_t turned = p.half / V;
  const int32_t rest = nv - 2 * turned;
  const int32_t far = (rest + 1) / 2;
  r.inside = false;
  r.turned = j < turned;
  if (r.turned) {
    r.angle = j * V;
    r.a = p.interleaved ? 2 * j : j * V;
    r.b = p.interleaved ? 2 * j + 1 : (j + turned) * V;
  } else {
    const int32_t i = j - turned;
    r.angle = 0;
    r.a = i < far ? (2 * turned + i) * V : -1;
    r.b = i < far && i + far < rest ? (2 * turned + i + far) * V : -1;
  }
  return r;
}

template <int N>
__device__ __forceinline__ void load_angles(const float* p, bool vec, float* f) {
  if constexpr (N >= 4) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const float4 v = reinterpret_cast<const float4*>(p)[i];
        f[4 * i] = v.x;
        f[4 * i + 1] = v.y;
        f[4 * i + 2] = v.z;
        f[4 * i + 3] = v.w;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = p[i];
}

// Cosines and sines of a lane's pair: of its V angles, or, where neighbours are turned, of a's V / 2,
// then b's.
template <int V>
struct HeadTurn {
  float c[V], s[V];
};

template <int V>
__device__ __forceinline__ void load_turn(const HeadParams& p, const HeadPair& h, int64_t position,
                                          HeadTurn<V>& t) {
  const bool known = position >= 0 && position < p.table_rows;
  const float* cos = p.table + (known ? position : 0) * p.table_ld;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    t.c[i] = 1.f;
    t.s[i] = 0.f;
  }
  if (p.half == 0) return;
  if (!known) {
#pragma unroll
    for (int i = 0; i < V; ++i) t.c[i] = __uint_as_float(0x7fc00000u);
    return;
  }
  if (h.turned) {
    load_angles<V>(cos + h.angle, p.table_vec != 0, t.c);
    load_angles<V>(cos + p.half + h.angle, p.table_vec != 0, t.s);
  } else if (V > 1 && h.inside) {
    constexpr int N = V / 2 > 0 ? V / 2 : 1;
    if (h.a >= 0 && h.a < 2 * p.half) {
      load_angles<N>(cos + h.a / 2, p.table_vec != 0, t.c);
      load_angles<N>(cos + p.half + h.a / 2, p.table_vec != 0, t.s);
    }
    if (h.b >= 0 && h.b < 2 * p.half) {
      load_angles<N>(cos + h.b / 2, p.table_vec != 0, t.c + V / 2);
      load_angles<N>(cos + p.half + h.b / 2, p.table_vec != 0, t.s + V / 2);
    }
  }
}

// Turns the pair by its angles (Back: by their negatives).
template <int V, bool Back>
__device__ __forceinline__ void turn(const HeadParams& p, const HeadPair& h, const HeadTurn<V>& t,
                                     float* a, float* b) {
  if (h.turned) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float s = Back ? -t.s[i] : t.s[i];
      const float x = a[i], y = b[i];
      a[i] = fmaf(x, t.c[i], -y * s);
      b[i] = fmaf(y, t.c[i], x * s);
    }
  } else if (V > 1 && h.inside) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float* f = v == 0 ? a : b;
      const int32_t at = v == 0 ? h.a : h.b;
      if (at < 0 || at >= 2 * p.half) continue;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const int j = v * (V / 2) + i;
        const float s = Back ? -t.s[j] : t.s[j];
        const float x = f[2 * i], y = f[2 * i + 1];
        f[2 * i] = fmaf(x, t.c[j], -y * s);
        f[2 * i + 1] = fmaf(y, t.c[j], x * s);
      }
    }
  }
}

// V elements as they lie.  Not through the read-only path: y may be x.
template <typename T, int V>
__device__ __forceinline__ typename RowAccess<T, V * static_cast<int>(sizeof(T))>::Data load_head(
    const T* head, int32_t at) {
  using A = RowAccess<T, V * static_cast<int>(sizeof(T))>;
  return at >= 0 ? A::template load_all<false>(head + at) : A::zero();
}

template <typename T, int V>
__device__ __forceinline__ void store_head(T* head, int32_t at, int32_t d, const float* f) {
  using A = RowAccess<T, V * static_cast<int>(sizeof(T))>;
  if (at >= 0) A::store(head, at, d, A::pack(f));
}

template <int V>
__device__ __forceinline__ void load_weight(const HeadPart& h, int32_t at, float* f) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = at >= 0 ? 1.f : 0.f;
  if (h.w == nullptr || at < 0) return;
  if constexpr (V >= 4) {
    if (h.w_vec) {  // it starts on 16 bytes, so that every vector does on its size
      if (h.w_f32) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
          RowAccess<float, 16>::unpack(RowAccess<float, 16>::template load_all<false>(
                                           static_cast<const float*>(h.w) + at + 4 * i),
                                       f + 4 * i);
      } else {
        using A = RowAccess<__nv_bfloat16, 2 * V>;
        A::unpack(A::template load_all<false>(static_cast<const __nv_bfloat16*>(h.w) + at), f);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    f[i] = h.w_f32 ? static_cast<const float*>(h.w)[at + i]
                   : __bfloat162float(static_cast<const __nv_bfloat16*>(h.w)[at + i]);
}

template <int L>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A group of L lanes takes HB heads of one part of a token: the angles and the weights are loaded
// once, and all of its heads before the first is used.  (Three blocks an SM although four heads of
// 16-byte vectors then spill 150 bytes: 68 us for 16384 x 40 x 128 in BF16, 73 with two.  Weights
// multiplied into the angles, or two FP32 operations an instruction: 66 and 80 us, their gradients 111
// and 114, not 96, for more registers.)
template <typename T, int V, int L, int NP, int HB>
__global__ void __launch_bounds__(kHeadThreads, 3) head_norm_kernel(const HeadParams p) {
  kernel_begins();
  using A = RowAccess<T, V * static_cast<int>(sizeof(T))>;
  const int32_t sub = threadIdx.x % L;
  const uint32_t parts[2] = {(p.part[0].heads + HB - 1u) / HB, (p.part[1].heads + HB - 1u) / HB};
  const uint32_t per = parts[0] + parts[1];
  const uint32_t unit = blockIdx.x * (kHeadThreads / L) + threadIdx.x / L;
  const uint32_t units = static_cast<uint32_t>(p.tokens) * per;
  const bool has = unit < units;  // the others take part in the shuffles
  const uint32_t token = has ? unit / per : 0u;
  const uint32_t place = has ? unit - token * per : 0u;
  const bool key = place >= parts[0];
  const HeadPart& h = p.part[key ? 1 : 0];
  const int32_t first = static_cast<int32_t>(key ? place - parts[0] : place) * HB;
  const int32_t heads = has ? min(h.heads - first, HB) : 0;
  const T* x = static_cast<const T*>(h.x) + token * h.x_token + first * h.x_head;
  T* y = static_cast<T*>(h.y) + token * h.y_token + first * h.y_head;
  HeadPair at[NP];
  typename A::Data raw[HB][NP][2];
#pragma unroll
  for (int n = 0; n < NP; ++n) at[n] = head_pair<V>(p, sub + n * L);
#pragma unroll
  for (int j = 0; j < HB; ++j)
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      raw[j][n][0] = load_head<T, V>(x + j * h.x_head, j < heads ? at[n].a : -1);
      raw[j][n][1] = load_head<T, V>(x + j * h.x_head, j < heads ? at[n].b : -1);
    }
  const int64_t position = p.positions[token];
  HeadTurn<V> angles[NP];
  float wa[NP][V], wb[NP][V];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    load_turn<V>(p, at[n], position, angles[n]);
    load_weight<V>(h, at[n].a, wa[n]);
    load_weight<V>(h, at[n].b, wb[n]);
  }
  const float inv_d = 1.f / static_cast<float>(p.d);
#pragma unroll
  for (int j = 0; j < HB; ++j) {
    float a[NP][V], b[NP][V];
    float squares = 0.f;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      A::unpack(raw[j][n][0], a[n]);
      A::unpack(raw[j][n][1], b[n]);
#pragma unroll
      for (int i = 0; i < V; ++i)
        squares = fmaf(a[n][i], a[n][i], fmaf(b[n][i], b[n][i], squares));
    }
    const float r = rsqrtf(fmaf(sum_lanes<L>(squares), inv_d, p.eps));
    if (j >= heads) continue;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[n][i] *= r * wa[n][i];
        b[n][i] *= r * wb[n][i];
      }
      turn<V, false>(p, at[n], angles[n], a[n], b[n]);
      store_head<T, V>(y + j * h.y_head, at[n].a, p.d, a[n]);
      store_head<T, V>(y + j * h.y_head, at[n].b, p.d, b[n]);
    }
  }
}

// Gradient.  A block belongs to one part and walks its tokens' heads, HB of a token at a time; each
// lane adds its channels' g n in registers, the block's lanes add theirs in shared memory and
// head_norm_sum_kernel the blocks'.
template <typename T, int V, int L, int NP, int HB>
__global__ void __launch_bounds__(kHeadThreads, 2) head_norm_grad_kernel(const HeadParams p) {
  kernel_begins();
  using A = RowAccess<T, V * static_cast<int>(sizeof(T))>;
  constexpr int kGroups = kHeadThreads / L;
  __shared__ float sums[kHeadThreads * 2 * V * NP];  // [kGroups][d]
  const int32_t sub = threadIdx.x % L;
  const uint32_t group = threadIdx.x / L;
  const bool key = static_cast<int32_t>(blockIdx.x) >= p.blocks[0];
  const HeadPart& h = p.part[key ? 1 : 0];
  const uint32_t block = blockIdx.x - (key ? p.blocks[0] : 0);
  const uint32_t blocks = static_cast<uint32_t>(p.blocks[key ? 1 : 0]);
  const uint32_t per = (static_cast<uint32_t>(h.heads) + HB - 1u) / HB;
  const uint32_t units = static_cast<uint32_t>(p.tokens) * per;
  HeadPair at[NP];
  float wa[NP][V], wb[NP][V], da[NP][V], db[NP][V];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    at[n] = head_pair<V>(p, sub + n * L);
    load_weight<V>(h, at[n].a, wa[n]);
    load_weight<V>(h, at[n].b, wb[n]);
#pragma unroll
    for (int i = 0; i < V; ++i) da[n][i] = db[n][i] = 0.f;
  }
  const float inv_d = 1.f / static_cast<float>(p.d);
  for (uint32_t from = block * kGroups; from < units; from += blocks * kGroups) {
    const uint32_t unit = from + group;
    const bool has = unit < units;
    const uint32_t token = has ? unit / per : 0u;
    const int32_t first = static_cast<int32_t>(has ? unit - token * per : 0u) * HB;
    const int32_t heads = has ? min(h.heads - first, HB) : 0;
    const T* x = static_cast<const T*>(h.x) + token * h.x_token + first * h.x_head;
    const T* dy = static_cast<const T*>(h.dy) + token * h.dy_token + first * h.dy_head;
    T* dx = static_cast<T*>(h.y) + token * h.y_token + first * h.y_head;
    typename A::Data rx[HB][NP][2], rg[HB][NP][2];
#pragma unroll
    for (int j = 0; j < HB; ++j)
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        rx[j][n][0] = load_head<T, V>(x + j * h.x_head, j < heads ? at[n].a : -1);
        rx[j][n][1] = load_head<T, V>(x + j * h.x_head, j < heads ? at[n].b : -1);
        rg[j][n][0] = load_head<T, V>(dy + j * h.dy_head, j < heads ? at[n].a : -1);
        rg[j][n][1] = load_head<T, V>(dy + j * h.dy_head, j < heads ? at[n].b : -1);
      }
    HeadTurn<V> angles[NP];
    const int64_t position = p.positions[token];
#pragma unroll
    for (int n = 0; n < NP; ++n) load_turn<V>(p, at[n], position, angles[n]);
#pragma unroll
    for (int j = 0; j < HB; ++j) {
      float xa[NP][V], xb[NP][V], ga[NP][V], gb[NP][V];
      float squares = 0.f, dot = 0.f;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        A::unpack(rx[j][n][0], xa[n]);
        A::unpack(rx[j][n][1], xb[n]);
        A::unpack(rg[j][n][0], ga[n]);
        A::unpack(rg[j][n][1], gb[n]);
        if (j < heads) turn<V, true>(p, at[n], angles[n], ga[n], gb[n]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          squares = fmaf(xa[n][i], xa[n][i], fmaf(xb[n][i], xb[n][i], squares));
          dot = fmaf(ga[n][i] * wa[n][i], xa[n][i], fmaf(gb[n][i] * wb[n][i], xb[n][i], dot));
        }
      }
      squares = sum_lanes<L>(squares);
      dot = sum_lanes<L>(dot);
      const float r = rsqrtf(fmaf(squares, inv_d, p.eps));
      const float back = dot * inv_d * r * r;  // mean(u n) = r mean(u x), and n = x r
      if (j >= heads) continue;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        float dxa[V], dxb[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          da[n][i] = fmaf(ga[n][i] * r, xa[n][i], da[n][i]);
          db[n][i] = fmaf(gb[n][i] * r, xb[n][i], db[n][i]);
          dxa[i] = r * fmaf(-back, xa[n][i], ga[n][i] * wa[n][i]);
          dxb[i] = r * fmaf(-back, xb[n][i], gb[n][i] * wb[n][i]);
        }
        store_head<T, V>(dx + j * h.y_head, at[n].a, p.d, dxa);
        store_head<T, V>(dx + j * h.y_head, at[n].b, p.d, dxb);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (at[n].a >= 0) sums[group * p.d + at[n].a + i] = da[n][i];
      if (at[n].b >= 0) sums[group * p.d + at[n].b + i] = db[n][i];
    }
  __syncthreads();
  for (int32_t c = threadIdx.x; c < p.d; c += kHeadThreads) {
    float s = 0.f;
    for (int i = 0; i < kGroups; ++i) s += sums[i * p.d + c];
    p.partial[static_cast<int64_t>(blockIdx.x) * p.d + c] = s;
  }
}

// dw of both parts: the sums of their blocks, always in the same order.  A warp per channel.
__global__ void __launch_bounds__(kHeadThreads)
    head_norm_sum_kernel(const float* partial, int32_t blocks_q, int32_t blocks_k, int32_t d,
                         float* dwq, float* dwk) {
  kernel_begins();
  const int32_t warp = static_cast<int32_t>(blockIdx.x * (kHeadThreads / 32) + threadIdx.x / 32);
  const bool key = warp >= d;
  const int32_t first = key ? blocks_q : 0;
  const int32_t count = key ? blocks_k : blocks_q;
  float* out = key ? dwk : dwq;
  const int32_t c = key ? warp - d : warp;
  if (out == nullptr || c >= d) return;
  float s = 0.f;
  for (int32_t i = threadIdx.x % 32; i < count; i += 32)
    s += partial[static_cast<int64_t>(first + i) * d + c];
  s = sum_lanes<32>(s);
  if (threadIdx.x % 32 == 0) out[c] = s;
}

}  // namespace cpg
