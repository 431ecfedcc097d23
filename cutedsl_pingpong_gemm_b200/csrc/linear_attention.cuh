// Linear attention with one decay per head over packed sequences.
//
// One kernel computes, for every sequence and head, in the order of its tokens or against it,
//   S_t = e^g S_{t-1} + b_t c_t^T,    o_t = scale * S_t^T a_t
// and with it both directions of training: the forward pass is (a, b, c) = (q, k, v), and with do
// the gradient of o,
//   dq = pass(do, v, k),   dk = reversed pass(v, do, q),   dv = reversed pass(k, q, do).
// In a reversed pass the state that arrives from behind is the gradient of the state after a token:
// it is used by that token without another decay (forward: the state before it, decayed once).
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "row_access.cuh"

namespace cpg {

struct LinearRows {
  const __nv_bfloat16* p;
  int64_t token, head;  // strides in elements
  int32_t share;        // heads of the decay that read one head of this
};

// A segment of a sequence, in the order of work: whole chunks but for the sequence's end.
struct LinearItem {
  int32_t sequence;
  int32_t first, count;  // tokens
  int32_t index;         // segments of the sequence that come before it
  int32_t last;
};

struct LinearParams {
  LinearRows a, b, c;
  void* o;
  int64_t o_token, o_head;
  int32_t o_f32;
  const float* log_decay;
  const int32_t* offsets;  // null: one sequence of all tokens
  int64_t tokens;
  int32_t sequences, heads;
  int32_t da, dc;          // channels of a and b, of c and o
  float scale;
  const float* state;      // [places, heads, da, dc] (transposed: [.., dc, da]); null: zeros
  const int32_t* state_slots;
  int64_t state_places;
  int32_t state_transposed;
  float state_factor;
  float* final;            // [places, heads, da, dc]; may be state
  const int32_t* final_slots;
  int64_t final_places;
  float final_factor;
  const LinearItem* items;       // null: a unit is a whole sequence
  const int32_t* item_count;
  const int32_t* first_item;     // [sequences + 1]
  // null: sequences stay whole.  [items, heads, da, dc]: what the segment before adds to the state, then
  // the state before each; then [sequences, heads, da, dc]: what the last segment adds, if that is wanted.
  float* segments;
  int32_t most_items;
  int32_t reverse;
};

// Passes over the same sequences and heads, side by side in one launch.
struct LinearBatch {
  LinearParams pass[3];
  int32_t passes;
  int32_t exact;        // states to FP32 accuracy (one is an output)
  int32_t inject;       // test hook: loads that the producer leaves out
  uint64_t timeout_ns;  // limit of a wait within the kernel
};

struct LinearSpan {
  int64_t first;
  int64_t count;
};

// Tokens of sequence s; whatever the offsets hold, they lie within the tensors.
__device__ __forceinline__ LinearSpan linear_span(const int32_t* offsets, int32_t s,
                                                  int64_t tokens) {
  if (offsets == nullptr) return {0, tokens};
  const int64_t a = min(max(static_cast<int64_t>(offsets[s]), int64_t(0)), tokens);
  const int64_t b = min(max(static_cast<int64_t>(offsets[s + 1]), a), tokens);
  return {a, b - a};
}

// Place of sequence s in a pool of states, -1 if it has none.
__device__ __forceinline__ int64_t linear_place(const int32_t* slots, int32_t s, int64_t places) {
  const int64_t at = slots == nullptr ? s : slots[s];
  return at >= 0 && at < places ? at : -1;
}

// The sequences as one item each, the longest first (equal ones in order).  One block.
constexpr int kMostSorted = 2048;

__global__ void __launch_bounds__(1024)
    linear_order_kernel(const int32_t* offsets, int64_t tokens, int32_t sequences,
                        LinearItem* items, int32_t* item_count) {
  kernel_begins();
  __shared__ int32_t counts[kMostSorted];
  for (int32_t s = threadIdx.x; s < sequences; s += 1024)
    counts[s] = static_cast<int32_t>(linear_span(offsets, s, tokens).count);
  __syncthreads();
  for (int32_t s = threadIdx.x; s < sequences; s += 1024) {
    const int32_t mine = counts[s];
    int32_t rank = 0;
    for (int32_t j = 0; j < sequences; ++j)
      rank += counts[j] > mine || (counts[j] == mine && j < s) ? 1 : 0;
    items[rank] = {s, static_cast<int32_t>(linear_span(offsets, s, tokens).first), mine, 0, 1};
  }
  if (threadIdx.x == 0) *item_count = sequences;
}

// The segments of `length` tokens (whole chunks) of every sequence, one after the other in the order of
// work; an empty sequence has one without tokens.  Offsets that decrease could make more than the table
// has room for (`most`): those past it are left out.  One block.
constexpr int kItemThreads = 1024;

__global__ void __launch_bounds__(kItemThreads)
    linear_items_kernel(const int32_t* offsets, int64_t tokens, int32_t sequences, int32_t length,
                        int32_t reverse, int32_t most, LinearItem* items, int32_t* item_count,
                        int32_t* first_item) {
  kernel_begins();
  __shared__ int64_t sums[kItemThreads / 32];
  const int32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int64_t base = 0;
  for (int32_t from = 0; from < sequences; from += kItemThreads) {
    const int32_t s = from + static_cast<int32_t>(threadIdx.x);
    LinearSpan span = {0, 0};
    if (s < sequences) span = linear_span(offsets, s, tokens);
    int32_t n = s < sequences ? static_cast<int32_t>((span.count + length - 1) / length) : 0;
    if (s < sequences && n == 0) n = 1;
    int64_t before = n;  // inclusive sum within the warp
    for (int o = 1; o < 32; o *= 2) {
      const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kItemThreads / 32; ++w) {
      if (w == warp) before += all;
      all += sums[w];
    }
    if (s < sequences) {
      const int32_t at = static_cast<int32_t>(min(base + before - n, static_cast<int64_t>(most)));
      first_item[s] = at;
      for (int32_t k = 0; k < min(n, most - at); ++k) {
        const int64_t first = static_cast<int64_t>(reverse ? n - 1 - k : k) * length;
        const int64_t left = span.count - first;
        items[at + k] = {s, static_cast<int32_t>(span.first + first),
                         static_cast<int32_t>(left < length ? left : length), k,
                         k == n - 1 || at + k == most - 1};
      }
    }
    base += all;
  }
  if (threadIdx.x == 0) {
    const int32_t all = static_cast<int32_t>(min(base, static_cast<int64_t>(most)));
    *item_count = all;
    first_item[sequences] = all;
  }
}

// The state before every segment of a sequence: the state before the previous one, decayed by that
// one's tokens, plus what it adds; after the last one that is the final state.  (The starting states
// are copied: the final ones may take their places.)  Four neighbouring elements a thread; blockIdx.x:
// pass, sequence and head, then the elements.
__global__ void __launch_bounds__(256) linear_segments_kernel(const LinearBatch batch) {
  kernel_begins();
  const int32_t size = batch.pass[0].da * batch.pass[0].dc;
  const int32_t parts = (size + 1023) / 1024;
  const int32_t each = batch.pass[0].sequences * batch.pass[0].heads;
  int32_t pair = static_cast<int32_t>(blockIdx.x) / parts;
  const LinearParams& p = batch.pass[pair / each];
  pair %= each;
  const int32_t s = pair / p.heads, h = pair % p.heads;
  const int32_t e = (blockIdx.x % parts) * 1024 + static_cast<int32_t>(threadIdx.x) * 4;
  const int32_t first = p.first_item[s], last = p.first_item[s + 1] - 1;
  if (e >= size || first > last) return;
  const float g2 = p.log_decay[h] * 1.4426950408889634f;
  const int64_t step = static_cast<int64_t>(p.heads) * size;
  const int64_t own = static_cast<int64_t>(h) * size + e;
  float* x = p.segments + first * step + own;
  float4 state = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.state != nullptr) {
    const int64_t place = linear_place(p.state_slots, s, p.state_places);
    if (place >= 0) {
      const float* from = p.state + (place * p.heads + h) * static_cast<int64_t>(size);
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        f[k] = p.state_factor * (p.state_transposed
                                     ? from[(e + k) % p.dc * p.da + (e + k) / p.dc]
                                     : from[e + k]);
      state = make_float4(f[0], f[1], f[2], f[3]);
    }
    *reinterpret_cast<float4*>(x) = state;
  }
  auto follow = [&](int32_t item, const float* adds) {
    const int32_t n = p.items[item].count;
    const float decay = n == 0 ? 1.f : exp2f(g2 * static_cast<float>(n));
    const float4 v = *reinterpret_cast<const float4*>(adds);
    state.x = fmaf(state.x, decay, v.x);
    state.y = fmaf(state.y, decay, v.y);
    state.z = fmaf(state.z, decay, v.z);
    state.w = fmaf(state.w, decay, v.w);
  };
#pragma unroll 4
  for (int32_t at = first; at < last; ++at) {
    x += step;
    follow(at, x);
    *reinterpret_cast<float4*>(x) = state;
  }
  if (p.final == nullptr) return;
  const int64_t place = linear_place(p.final_slots, s, p.final_places);
  if (place < 0) return;
  follow(last, p.segments + (static_cast<int64_t>(p.most_items) + s) * step + own);
  const float f = p.final_factor;
  *reinterpret_cast<float4*>(p.final + place * step + own) =
      make_float4(f * state.x, f * state.y, f * state.z, f * state.w);
}

// Offsets from the first up to the last pass every row between them on their way; where they also decrease,
// a sequence may lie outside.  Whether they do (asked by a whole block), and whether a row is in one.
__device__ __forceinline__ bool linear_decreases(const int32_t* offsets, int32_t sequences) {
  bool down = false;
  for (int32_t s = threadIdx.x; s < sequences; s += blockDim.x) down |= offsets[s] > offsets[s + 1];
  return __syncthreads_or(down);
}
__device__ __forceinline__ bool linear_inside(const int32_t* offsets, int32_t sequences, int64_t t) {
  for (int32_t s = 0; s < sequences; ++s)
    if (offsets[s] <= t && t < offsets[s + 1]) return true;
  return false;
}

// Rows of up to three [tokens, heads, d] outside the sequences, set to zero, 16 bytes at a time.
struct LinearClearParams {
  char* p[3];
  int64_t token[3], head[3];    // strides in bytes
  int32_t heads[3], pieces[3];  // 16-byte pieces of a head
  const int32_t* offsets;
  int64_t tokens;
  int32_t sequences;
};

__global__ void __launch_bounds__(256) linear_clear_kernel(const LinearClearParams p) {
  kernel_begins();
  const int64_t first = min(max(static_cast<int64_t>(p.offsets[0]), int64_t(0)), p.tokens);
  const int64_t last =
      min(max(static_cast<int64_t>(p.offsets[p.sequences]), first), p.tokens);
  const int64_t rows = first + p.tokens - last;
  if (rows == 0) return;
  const bool down = linear_decreases(p.offsets, p.sequences);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t t = r < first ? r : last + r - first;
    if (down && linear_inside(p.offsets, p.sequences, t)) continue;
#pragma unroll
    for (int n = 0; n < 3; ++n)
      for (int32_t i = threadIdx.x; i < p.heads[n] * p.pieces[n]; i += blockDim.x)
        ptx::st_global_v4(p.p[n] + t * p.token[n] + i / p.pieces[n] * p.head[n] + i % p.pieces[n] * 16,
                          0u, 0u, 0u, 0u);
  }
}

// The gradient of shared heads: the sums over the heads that read one, rounded once.
struct LinearShareParams {
  const float* partial;  // [tokens, heads * share, d]
  __nv_bfloat16* out;
  int64_t token, head;
  int64_t tokens;
  int32_t heads, share, d;
  const int32_t* offsets;
  int32_t sequences;
};

__global__ void __launch_bounds__(256) linear_share_kernel(const LinearShareParams p) {
  kernel_begins();
  int64_t first = 0, last = p.tokens;
  if (p.offsets != nullptr) {
    first = min(max(static_cast<int64_t>(p.offsets[0]), int64_t(0)), p.tokens);
    last = min(max(static_cast<int64_t>(p.offsets[p.sequences]), first), p.tokens);
  }
  const int32_t row = p.heads * p.d / 8;  // eight neighbouring channels a thread
  auto add = [&](int64_t t, int32_t e) {
    const int32_t h = e / p.d, x = e % p.d;
    const float* from = p.partial + (t * p.heads + h) * int64_t(p.share) * p.d + x;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int32_t j = 0; j < p.share; ++j, from += p.d) {
      const float4 u = reinterpret_cast<const float4*>(from)[0];
      const float4 v = reinterpret_cast<const float4*>(from)[1];
      a.x += u.x;
      a.y += u.y;
      a.z += u.z;
      a.w += u.w;
      b.x += v.x;
      b.y += v.y;
      b.z += v.z;
      b.w += v.w;
    }
    ptx::st_global_v4(p.out + t * p.token + h * p.head + x, ptx::pack_bf16x2(a.x, a.y),
                      ptx::pack_bf16x2(a.z, a.w), ptx::pack_bf16x2(b.x, b.y),
                      ptx::pack_bf16x2(b.z, b.w));
  };
  const int64_t n = (last - first) * row;
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += gridDim.x * int64_t(256))
    add(first + i / row, static_cast<int32_t>(i % row) * 8);
  const int64_t rows = first + p.tokens - last;
  if (rows == 0 || !linear_decreases(p.offsets, p.sequences)) return;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t t = r < first ? r : last + r - first;
    if (!linear_inside(p.offsets, p.sequences, t)) continue;
    for (int32_t i = threadIdx.x; i < row; i += 256) add(t, i * 8);
  }
}

// One token of each of many sequences: S <- e^g S + k v^T in place, o = scale * S^T q.
// Bound by HBM: every state is read and written once (256 tokens x 64 heads x 128 x 128: 367 us, 0.90 of
// the copy rate).  A block has one state, a lane four neighbouring columns of every (1024 / dv)-th row,
// whose loads are independent.
struct LinearStepParams {
  LinearRows q, k, v;
  void* o;
  int64_t o_token, o_head;
  int32_t o_f32;
  const float* log_decay;
  float* state;  // [places, heads, dk, dv]
  const int32_t* slots;
  int64_t places;
  int32_t heads, dk, dv;
  float scale;
};

constexpr int kStepThreads = 256;

__global__ void __launch_bounds__(kStepThreads) linear_step_kernel(const LinearStepParams p) {
  kernel_begins();
  __shared__ float4 sums[kStepThreads];
  const int32_t i = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
  const int32_t groups = p.dv / 4;             // lanes across a row
  const int32_t rows = kStepThreads / groups;  // rows at a time
  const int32_t x = threadIdx.x % groups, y = threadIdx.x / groups;
  const int64_t at = linear_place(p.slots, i, p.places);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (at >= 0 && y < rows) {
    const float lambda = expf(p.log_decay[h]);
    float4* s = reinterpret_cast<float4*>(p.state + (at * p.heads + h) * int64_t(p.dk) * p.dv) + x;
    const __nv_bfloat16* q = p.q.p + i * p.q.token + h / p.q.share * p.q.head;
    const __nv_bfloat16* k = p.k.p + i * p.k.token + h / p.k.share * p.k.head;
    const __nv_bfloat16* vp = p.v.p + i * p.v.token + h / p.v.share * p.v.head + 4 * x;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __bfloat162float(vp[j]);
    for (int32_t r = y; r < p.dk; r += rows) {
      float4 f = s[r * groups];
      const float kr = __bfloat162float(k[r]), qr = __bfloat162float(q[r]);
      f.x = fmaf(kr, v[0], lambda * f.x);
      f.y = fmaf(kr, v[1], lambda * f.y);
      f.z = fmaf(kr, v[2], lambda * f.z);
      f.w = fmaf(kr, v[3], lambda * f.w);
      s[r * groups] = f;
      o.x = fmaf(qr, f.x, o.x);
      o.y = fmaf(qr, f.y, o.y);
      o.z = fmaf(qr, f.z, o.z);
      o.w = fmaf(qr, f.w, o.w);
    }
  }
  sums[threadIdx.x] = o;
  __syncthreads();
  if (threadIdx.x >= groups) return;
  o = sums[threadIdx.x];
  for (int32_t r = 1; r < rows; ++r) {
    const float4 f = sums[r * groups + threadIdx.x];
    o.x += f.x;
    o.y += f.y;
    o.z += f.z;
    o.w += f.w;
  }
  const int64_t to = i * p.o_token + h * p.o_head + 4 * x;
  const float f[4] = {p.scale * o.x, p.scale * o.y, p.scale * o.z, p.scale * o.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (p.o_f32)
      static_cast<float*>(p.o)[to + j] = f[j];
    else
      static_cast<__nv_bfloat16*>(p.o)[to + j] = __float2bfloat16_rn(f[j]);
  }
}

}  // namespace cpg
