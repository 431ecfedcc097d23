// C ABI of the operators between a layer's projections: norm and rotation of query and key heads,
// linear attention with a decay per head, and their gradients (include/cpgemm.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <mutex>
#include <type_traits>

#include "capi_common.h"
#include "capi_launch.h"
#include "cpgemm.h"
#include "head_norm.cuh"
#include "linear_attention.cuh"
#include "linear_chunks.cuh"

using cpg::Work;
using cpg_capi::bytes_of;
using cpg_capi::cuda_fail;
using cpg_capi::encode_fn;
using cpg_capi::fail;
using cpg_capi::float_dtype;
using cpg_capi::launch;
using cpg_capi::misaligned;

namespace {

static_assert(cpg::kLinearSkipLoads == CPG_INJECT_SKIP_LOADS &&
                  cpg::kLinearSkipValues == CPG_INJECT_SKIP_VALUES,
              "the flags go to the kernel as they are");

constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1;
constexpr int32_t kMaxLinearHeads = 1 << 20;
constexpr int64_t kMaxStride = int64_t(1) << 38;  // elements; tensor maps take 2^40 bytes

// Heads [tokens, heads, channels] with elements aligned to `bytes`; `written`: no two overlap.
int check_heads(const char* name, const cpg_heads* x, int64_t tokens, int64_t channels, int bytes,
                bool written) {
  if (x == nullptr) return fail(CPG_ERR_NULL, "%s is NULL", name);
  if (!float_dtype(x->dtype)) return fail(CPG_ERR_DTYPE, "%s must be BF16 or FP32", name);
  if (x->heads < 1) return fail(CPG_ERR_INVALID_SHAPE, "%s has %d heads", name, x->heads);
  if (tokens == 0) return CPG_OK;
  if (x->ptr == nullptr) return fail(CPG_ERR_NULL, "%s is NULL", name);
  const int64_t ts = tokens > 1 ? x->token_stride : 0, hs = x->heads > 1 ? x->head_stride : 0;
  if (ts < 0 || hs < 0 || ts > kMaxStride || hs > kMaxStride)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: token stride %lld, head stride %lld", name,
                static_cast<long long>(ts), static_cast<long long>(hs));
  const int eb = bytes_of(x->dtype);
  if (misaligned(x->ptr, bytes) || (ts * eb) % bytes != 0 || (hs * eb) % bytes != 0)
    return fail(CPG_ERR_ALIGNMENT, "%s: address and strides must be multiples of %d bytes", name,
                bytes);
  if (!written) return CPG_OK;
  const bool heads_inside = (x->heads < 2 || hs >= channels) &&
                            (tokens < 2 || ts >= (x->heads - 1) * hs + channels);
  const bool tokens_inside = (tokens < 2 || ts >= channels) &&
                             (x->heads < 2 || hs >= (tokens - 1) * ts + channels);
  if (!heads_inside && !tokens_inside)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: heads overlap (token stride %lld, head stride %lld)",
                name, static_cast<long long>(ts), static_cast<long long>(hs));
  return CPG_OK;
}

// ------------------------------------------------------------------------- norm and rotation
// Blocks of the gradient, of both parts together, at most.  Two an SM are on it at once whatever the
// vectors; with four a second round follows (8191 tokens x 40 heads x 128, BF16: 55 us, 60 with four; 8192
// x 32 x 20 in BF16 23 and 25, x 75 in FP32 110 and 118, in BF16 180 and 174).
constexpr int kGradBlocks = 148 * 2;
constexpr int64_t kManyThreads = int64_t(148) * 2048 * 4;

// Address bits that some head of x has set (of the lowest ones).
uint64_t address_bits(const cpg_heads* x, int64_t tokens) {
  const int eb = bytes_of(x->dtype);
  return reinterpret_cast<uintptr_t>(x->ptr) |
         (tokens > 1 ? static_cast<uint64_t>(x->token_stride * eb) : 0u) |
         (x->heads > 1 ? static_cast<uint64_t>(x->head_stride * eb) : 0u);
}

struct NormRope {
  const cpg_heads *q, *k, *q_out, *k_out, *dq, *dk;  // dq, dk: gradient only
  int64_t tokens;
  int32_t channels;
  const void *wq, *wk;
  int32_t dtype_w;
  float eps;
  const float* table;
  int64_t table_rows, table_ld;
  int32_t rotary;
  const int32_t* positions;
  int32_t interleaved;
};

int check_norm_sizes(int64_t tokens, int64_t heads, int32_t channels) {
  if (tokens < 0 || heads < 1 || heads > kMaxRows || tokens > kMaxRows ||
      tokens * heads > kMaxRows)
    return fail(CPG_ERR_INVALID_SHAPE, "%lld tokens x %lld heads: at most 2^31 - 1 rows",
                static_cast<long long>(tokens), static_cast<long long>(heads));
  if (channels < 2 || channels > CPG_HEAD_MAX_CHANNELS)
    return fail(CPG_ERR_INVALID_SHAPE, "2 <= channels <= %d, got %d", CPG_HEAD_MAX_CHANNELS,
                channels);
  return CPG_OK;
}

int check_norm_rope(const NormRope& n, bool back) {
  if (n.q == nullptr || n.q_out == nullptr || (back && n.dq == nullptr))
    return fail(CPG_ERR_NULL, "q and its outputs must be non-NULL");
  if ((n.k == nullptr) != (n.k_out == nullptr) || (back && (n.k == nullptr) != (n.dk == nullptr)))
    return fail(CPG_ERR_NULL, "k, its outputs and its gradient go together");
  const int64_t heads = int64_t(n.q->heads) + (n.k != nullptr ? n.k->heads : 0);
  int rc = check_norm_sizes(n.tokens, heads, n.channels);
  if (rc != CPG_OK) return rc;
  if (n.rotary < 0 || n.rotary > n.channels || n.rotary % 2 != 0)
    return fail(CPG_ERR_INVALID_SHAPE, "rotary %d of %d channels: even, at most all", n.rotary,
                n.channels);
  if (!float_dtype(n.dtype_w)) return fail(CPG_ERR_DTYPE, "weights must be BF16 or FP32");
  if (!(n.eps >= 0.f) || std::isinf(n.eps))
    return fail(CPG_ERR_INVALID_CONFIG, "eps must be finite and not negative");
  for (int i = 0; i < 2; ++i) {
    const cpg_heads* x = i == 0 ? n.q : n.k;
    const cpg_heads* y = i == 0 ? n.q_out : n.k_out;
    const cpg_heads* dy = i == 0 ? n.dq : n.dk;
    if (x == nullptr) continue;
    if (!float_dtype(x->dtype)) return fail(CPG_ERR_DTYPE, "q and k must be BF16 or FP32");
    const int eb = bytes_of(x->dtype);
    rc = check_heads(i == 0 ? "q" : "k", x, n.tokens, n.channels, eb, false);
    if (rc == CPG_OK)
      rc = check_heads(i == 0 ? "q's output" : "k's output", y, n.tokens, n.channels, eb, true);
    if (rc == CPG_OK && back)
      rc = check_heads(i == 0 ? "dq" : "dk", dy, n.tokens, n.channels, eb, false);
    if (rc != CPG_OK) return rc;
    if (x->dtype != n.q->dtype || y->dtype != n.q->dtype || (back && dy->dtype != n.q->dtype))
      return fail(CPG_ERR_DTYPE, "q, k, their outputs and gradients have one type");
    if (y->heads != x->heads || (back && dy->heads != x->heads))
      return fail(CPG_ERR_INVALID_SHAPE, "%s's output or gradient has another number of heads",
                  i == 0 ? "q" : "k");
  }
  if (n.tokens == 0) return CPG_OK;
  if (n.positions == nullptr || (n.rotary > 0 && n.table == nullptr))
    return fail(CPG_ERR_NULL, "table and positions must be non-NULL");
  if (n.table_rows < 0 || n.table_rows > kMaxRows || n.table_ld < n.rotary ||
      n.table_ld > kMaxStride)
    return fail(CPG_ERR_INVALID_SHAPE, "table: %lld rows of stride %lld",
                static_cast<long long>(n.table_rows), static_cast<long long>(n.table_ld));
  if (misaligned(n.positions, 4) || misaligned(n.table, 4) ||
      misaligned(n.wq, bytes_of(n.dtype_w)) || misaligned(n.wk, bytes_of(n.dtype_w)))
    return fail(CPG_ERR_ALIGNMENT,
                "table, positions and weights must be aligned to their elements");
  return CPG_OK;
}

cpg::HeadParams head_params(const NormRope& n) {
  cpg::HeadParams p = {};
  for (int i = 0; i < 2; ++i) {
    const cpg_heads* x = i == 0 ? n.q : n.k;
    const cpg_heads* y = i == 0 ? n.q_out : n.k_out;
    const cpg_heads* dy = i == 0 ? n.dq : n.dk;
    if (x == nullptr) continue;
    cpg::HeadPart& h = p.part[i];
    h.x = x->ptr;
    h.x_token = x->token_stride;
    h.x_head = x->head_stride;
    h.y = y->ptr;
    h.y_token = y->token_stride;
    h.y_head = y->head_stride;
    if (dy != nullptr) {
      h.dy = dy->ptr;
      h.dy_token = dy->token_stride;
      h.dy_head = dy->head_stride;
    }
    h.w = i == 0 ? n.wq : n.wk;
    h.w_f32 = n.dtype_w == CPG_DTYPE_F32 ? 1 : 0;
    h.w_vec = !misaligned(h.w, 16) ? 1 : 0;
    h.heads = x->heads;
  }
  p.table = n.table;
  p.table_rows = n.table_rows;
  p.table_ld = n.table_ld;
  p.positions = n.positions;
  p.tokens = n.tokens;
  p.d = n.channels;
  p.half = n.rotary / 2;
  p.interleaved = n.interleaved != 0 ? 1 : 0;
  p.table_vec = !misaligned(n.table, 16) && n.table_ld % 4 == 0 && p.half % 4 == 0 ? 1 : 0;
  p.eps = n.eps;
  return p;
}

// Elements of the widest vector that every head starts on and that the turned channels, each half
// of them and the others divide into.
int head_vector(const NormRope& n) {
  uint64_t bits = 16;
  for (const cpg_heads* x : {n.q, n.k, n.q_out, n.k_out, n.dq, n.dk})
    if (x != nullptr) bits |= address_bits(x, n.tokens);
  const int eb = bytes_of(n.q->dtype);
  const int turned = n.interleaved ? n.rotary : n.rotary / 2;
  const uint64_t sizes =
      static_cast<uint64_t>(n.channels * eb) | static_cast<uint64_t>(turned * eb);
  bits |= sizes;
  return static_cast<int>(bits & (~bits + 1)) / eb;
}

// f(type, vector, lanes, pairs a lane, heads at a time) for the sizes at hand: the fewest lanes that hold
// a head, and Many heads at a time where there are more threads than the SMs hold at once (16384 tokens
// x 40 heads x 128, BF16: 68 us, one at a time 90; few threads would leave SMs idle).
template <typename T, int V, int Many, typename F>
int by_lanes(const NormRope& n, F&& f) {
  using std::integral_constant;
  const int vectors = n.channels / V;
  int pairs = (vectors + 1) / 2;
  if (!(n.interleaved && V > 1)) {
    const int turned = n.rotary / 2 / V;
    pairs = turned + (vectors - 2 * turned + 1) / 2;
  }
  const integral_constant<int, V> v;
  const integral_constant<int, 1> one;
  auto heads = [&](auto lanes, auto each) {
    const int64_t rows = n.tokens * (int64_t(n.q->heads) + (n.k != nullptr ? n.k->heads : 0));
    if (rows * decltype(lanes)::value > kManyThreads)
      return f(T{}, v, lanes, each, integral_constant<int, V * sizeof(T) == 16 ? Many : 2>{});
    return f(T{}, v, lanes, each, one);
  };
  if (pairs <= 4) return heads(integral_constant<int, 4>{}, one);
  if (pairs <= 8) return heads(integral_constant<int, 8>{}, one);
  if (pairs <= 16) return heads(integral_constant<int, 16>{}, one);
  const integral_constant<int, 32> warp;
  // At most CPG_HEAD_MAX_CHANNELS / V / 2 pairs: V = 8 has 16, V = 4 32, V = 2 64, V = 1 128.
  if constexpr (V <= 4) {
    if (pairs <= 32) return heads(warp, one);
  }
  if constexpr (V <= 2) {
    if (pairs <= 64) return heads(warp, integral_constant<int, 2>{});
  }
  if constexpr (V == 1) {
    if (pairs <= 128) return heads(warp, integral_constant<int, 4>{});
  }
  return fail(CPG_ERR_UNSUPPORTED, "%d channels", n.channels);
}

template <int Many, typename F>
int by_head(const NormRope& n, F&& f) {
  const int v = head_vector(n);
  if (n.q->dtype == CPG_DTYPE_BF16) {
    using B = __nv_bfloat16;
    if (v == 8) return by_lanes<B, 8, Many>(n, f);
    if (v == 4) return by_lanes<B, 4, Many>(n, f);
    if (v == 2) return by_lanes<B, 2, Many>(n, f);
    return by_lanes<B, 1, Many>(n, f);
  }
  if (v == 4) return by_lanes<float, 4, Many>(n, f);
  if (v == 2) return by_lanes<float, 2, Many>(n, f);
  return by_lanes<float, 1, Many>(n, f);
}

// Blocks of each part in the gradient, in proportion to their heads and at most one per row.
void grad_blocks(int64_t tokens, int32_t q_heads, int32_t k_heads, int32_t* blocks) {
  const int64_t heads = int64_t(q_heads) + k_heads;
  for (int i = 0; i < 2; ++i) {
    const int64_t h = i == 0 ? q_heads : k_heads;
    blocks[i] = h == 0 ? 0
                       : static_cast<int32_t>(std::max<int64_t>(
                             1, std::min<int64_t>(tokens * h, kGradBlocks * h / heads)));
  }
}

// ---------------------------------------------------------------------------- linear attention
int check_linear(const cpg_linear_problem* p) {
  if (p == nullptr) return fail(CPG_ERR_NULL, "the problem is NULL");
  if (p->tokens < 0 || p->tokens > kMaxRows)
    return fail(CPG_ERR_INVALID_SHAPE, "%lld tokens", static_cast<long long>(p->tokens));
  // (Heads: a token's channels of all of them are counted in 32 bits, a workspace's bytes in 64.)
  if (p->sequences < 0 || p->heads < 1 || p->heads > kMaxLinearHeads ||
      int64_t(p->sequences) * p->heads > kMaxRows / 4)
    return fail(CPG_ERR_INVALID_SHAPE, "%d sequences x %d heads", p->sequences, p->heads);
  if (p->dk < 8 || p->dk > CPG_LINEAR_MAX_CHANNELS || p->dk % 8 != 0 || p->dv < 8 ||
      p->dv > CPG_LINEAR_MAX_CHANNELS || p->dv % 8 != 0)
    return fail(CPG_ERR_INVALID_SHAPE,
                "dk = %d, dv = %d must be multiples of 8 from 8 to %d", p->dk, p->dv,
                CPG_LINEAR_MAX_CHANNELS);
  if (!std::isfinite(p->scale) || !std::isfinite(1.f / p->scale))
    return fail(CPG_ERR_INVALID_CONFIG, "scale and 1 / scale must be finite");
  return CPG_OK;
}

int check_operand(const char* name, const cpg_linear_problem* p, const cpg_heads* x, int32_t d,
                  bool written, bool f32_too = false) {
  if (x == nullptr) return fail(CPG_ERR_NULL, "%s is NULL", name);
  if (x->dtype != CPG_DTYPE_BF16 && !(f32_too && x->dtype == CPG_DTYPE_F32))
    return fail(CPG_ERR_DTYPE, "%s must be BF16%s", name, f32_too ? " or FP32" : "");
  const int rc = check_heads(name, x, p->tokens, d, 16, written);
  if (rc != CPG_OK) return rc;
  if (p->heads % x->heads != 0)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: %d heads do not divide %d", name, x->heads, p->heads);
  if ((p->tokens > 1 && x->token_stride == 0) || (x->heads > 1 && x->head_stride == 0))
    return fail(CPG_ERR_UNSUPPORTED, "%s: a stride of 0 (give a shared head once)", name);
  return CPG_OK;
}

int check_states(const char* name, const cpg_linear_problem* p, const cpg_states* s) {
  if (s == nullptr) return CPG_OK;
  if (s->places < 0 || s->places > kMaxRows)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: %lld places", name, static_cast<long long>(s->places));
  if (s->slots == nullptr && s->places < p->sequences)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: %lld places for %d sequences", name,
                static_cast<long long>(s->places), p->sequences);
  if (s->ptr == nullptr && s->places > 0) return fail(CPG_ERR_NULL, "%s is NULL", name);
  if (misaligned(s->ptr, 16) || misaligned(s->slots, 4))
    return fail(CPG_ERR_ALIGNMENT, "%s must start on 16 bytes, its slots on 4", name);
  return CPG_OK;
}

int check_sequences(const cpg_linear_problem* p, const float* log_decay, const int32_t* offsets) {
  if (log_decay == nullptr) return fail(CPG_ERR_NULL, "log_decay is NULL");
  if (offsets == nullptr && p->sequences != 1)
    return fail(CPG_ERR_NULL, "%d sequences need offsets", p->sequences);
  if (misaligned(log_decay, 4) || misaligned(offsets, 4))
    return fail(CPG_ERR_ALIGNMENT, "log_decay and offsets must be aligned to their elements");
  return CPG_OK;
}

cpg::LinearRows linear_rows(const cpg_linear_problem* p, const cpg_heads* x) {
  return {static_cast<const __nv_bfloat16*>(x->ptr), x->token_stride, x->head_stride,
          p->heads / x->heads};
}

cpg::LinearParams linear_params(const cpg_linear_problem* p, const cpg_heads* a,
                                const cpg_heads* b, const cpg_heads* c, int32_t da, int32_t dc,
                                const cpg_heads* o, const float* log_decay,
                                const int32_t* offsets) {
  cpg::LinearParams r = {};
  r.a = linear_rows(p, a);
  r.b = linear_rows(p, b);
  r.c = linear_rows(p, c);
  r.o = o->ptr;
  r.o_token = o->token_stride;
  r.o_head = o->head_stride;
  r.o_f32 = o->dtype == CPG_DTYPE_F32 ? 1 : 0;
  r.log_decay = log_decay;
  r.offsets = offsets;
  r.tokens = p->tokens;
  r.sequences = p->sequences;
  r.heads = p->heads;
  r.da = da;
  r.dc = dc;
  r.scale = p->scale;
  r.state_factor = r.final_factor = 1.f;
  return r;
}

void set_state(cpg::LinearParams* r, const cpg_states* s, bool transposed, float factor) {
  if (s == nullptr) return;
  r->state = s->ptr;
  r->state_slots = s->slots;
  r->state_places = s->places;
  r->state_transposed = transposed ? 1 : 0;
  r->state_factor = factor;
}

void set_final(cpg::LinearParams* r, const cpg_states* s, float factor) {
  if (s == nullptr) return;
  r->final = s->ptr;
  r->final_slots = s->slots;
  r->final_places = s->places;
  r->final_factor = factor;
}

// Tiles of 128 tokens x 64 channels of one head; channels and tokens past the end read as zeros.
int encode_heads(CUtensorMap* m, const cpg::LinearRows& x, int64_t tokens, int32_t heads,
                 int32_t d) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(CPG_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int64_t any = d;  // the stride of a single head or token is not used
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(2 * (heads > 1 ? x.head : any)),
                           static_cast<cuuint64_t>(2 * (tokens > 1 ? x.token : any))};
  cuuint32_t box[3] = {64, 1, cpg::kChunk};
  cuuint32_t steps[3] = {1, 1, 1};
  const CUresult r =
      fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(x.p), dims, strides,
         box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(CPG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): %lld tokens x %d heads x %d",
                static_cast<int>(r), static_cast<long long>(tokens), heads, d);
  return CPG_OK;
}

// Limit of the kernels' waits in ms (0: not yet read from the environment), and the loads that the
// producers leave out.
std::atomic<int32_t> g_timeout_ms{0}, g_inject{0};

uint64_t timeout_ns() {
  int32_t ms = g_timeout_ms.load();
  if (ms == 0) {
    const char* env = std::getenv("CPG_WAIT_TIMEOUT_MS");
    int32_t first = env != nullptr ? std::atoi(env) : 0;
    if (first <= 0) first = 10000;
    if (g_timeout_ms.compare_exchange_strong(ms, first)) ms = first;
  }
  return static_cast<uint64_t>(ms) * 1000000ull;
}

// SMs of the current device; also raises the shared-memory limit of the chunk kernels there, once.
int device_ready(int* sms) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static int known[kDevices];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kDevices) return fail(CPG_ERR_NO_DEVICE, "device %d", dev);
  std::lock_guard<std::mutex> lock(mu);
  if (known[dev] == 0) {
    int n = 0;
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    auto raise = [&](auto kernel, uint32_t bytes) {
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(bytes));
    };
    auto both = [&](auto da, auto dc) {
      constexpr int kDA = decltype(da)::value, kDC = decltype(dc)::value;
      constexpr uint32_t kBytes = cpg::ChunkLayout<kDA, kDC>::kBytes;
      raise(&cpg::linear_chunks_kernel<kDA, kDC, Work::kStates>, kBytes);
      raise(&cpg::linear_chunks_kernel<kDA, kDC, Work::kOutput>, kBytes);
      raise(&cpg::linear_chunks_kernel<kDA, kDC, Work::kFine>, kBytes);
      raise(&cpg::linear_chunks_kernel<kDA, kDC, Work::kExact>, kBytes);
    };
    const std::integral_constant<int, 64> d64;
    const std::integral_constant<int, 128> d128;
    both(d64, d64);
    both(d64, d128);
    both(d128, d64);
    both(d128, d128);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(linear attention)");
    known[dev] = n;
  }
  *sms = known[dev];
  return CPG_OK;
}

// How a pass is cut: the tokens of a segment (0: sequences stay whole) and the most segments there can
// be.  A unit (a sequence or segment of one head) is a chain of chunks of one SM, 2.8 us each alone
// and 3.5 us where all SMs share the bandwidth.  Cutting sequences costs a pass over B and C for the
// segments' states (2 us a chunk) and their joining, but fills the SMs: 65536 tokens x 16 heads of 128
// channels 1470 -> 340 to 400 us.  The lengths are known to the device alone: the mean stands for them.
// Ragged sequences that stay whole are items too, begun in the order of their lengths, where there is
// more than one unit per SM: a long one begun last would run alone.
struct LinearCut {
  int64_t length, items;
};

LinearCut linear_cut(const cpg_linear_problem* p, int passes) {
  constexpr int64_t kSms = 148, kMostCut = 1024;
  if (p->sequences == 0 || p->tokens == 0) return {0, 0};
  const int64_t mean = (p->tokens + p->sequences - 1) / p->sequences;
  const int64_t chunks = (mean + cpg::kChunk - 1) / cpg::kChunk;
  const int64_t units = int64_t(p->sequences) * p->heads * passes;
  const int64_t waves = (units + kSms - 1) / kSms;
  double best = chunks * (units < kSms ? 2.8 : 3.5 * waves);
  int64_t cut = 0;
  const bool sorted = units > kSms && p->sequences > 1 && p->sequences <= cpg::kMostSorted;
  const LinearCut uncut{0, sorted ? p->sequences : 0};
  if (units > kMostCut) return uncut;
  for (int64_t length = 2; length < std::min<int64_t>(chunks, 128); ++length) {
    const int64_t segments = (chunks + length - 1) / length;
    const int64_t turns = (segments * units + kSms - 1) / kSms;
    // The last segment's state is not needed; 30 us: the launches in between.
    const double cost = turns * (length + 1.0) * 3.5 + 30.0 +
                        (((segments - 1) * units + kSms - 1) / kSms) * (length + 1.0) * 2.0;
    if (cost < best) {
      best = cost;
      cut = length;
    }
  }
  if (cut == 0) return uncut;
  return {cut * cpg::kChunk, p->tokens / (cut * cpg::kChunk) + p->sequences};
}

// Workspace of passes that run together: the segments' states of each, then the table of segments or
// sequences in their order and one against it.
struct LinearSpace {
  int64_t states, tables, table;  // bytes of one pass's states, where the tables begin, bytes of one
  int64_t first, count, bytes;    // offsets within a table, all bytes
};
LinearSpace linear_space(const cpg_linear_problem* p, const LinearCut& cut, int passes) {
  if (cut.items == 0) return {};
  LinearSpace r;
  r.states = cut.length == 0 ? 0 : (cut.items + p->sequences) * p->heads * p->dk * p->dv * 4;
  r.tables = r.states * passes;
  r.first = cut.items * static_cast<int64_t>(sizeof(cpg::LinearItem));
  r.count = r.first + (cut.length == 0 ? 0 : (int64_t(p->sequences) + 1) * 4);
  r.table = (r.count + 4 + 15) / 16 * 16;
  r.bytes = r.tables + 2 * r.table;
  return r;
}

template <int DA, int DC, Work W>
int run_chunks(const cpg::LinearBatch& b, int64_t units, int sms, cudaStream_t st) {
  cpg::LinearMaps maps = {};
  for (int j = 0; j < b.passes && b.pass[0].tokens > 0; ++j) {
    const cpg::LinearParams& r = b.pass[j];
    const cpg::LinearRows* x[3] = {&r.a, &r.b, &r.c};
    for (int i = 0; i < 3; ++i) {
      const int rc = encode_heads(&maps.m[j][i], *x[i], r.tokens, r.heads / x[i]->share,
                                  i < 2 ? r.da : r.dc);
      if (rc != CPG_OK) return rc;
    }
  }
  return launch("linear attention kernel", true, &cpg::linear_chunks_kernel<DA, DC, W>,
                static_cast<unsigned>(std::min<int64_t>(units, sms)), cpg::kChunkThreads,
                cpg::ChunkLayout<DA, DC>::kBytes, st, 1, maps, b);
}

template <Work W>
int run_chunks(const cpg::LinearBatch& b, int64_t units, int sms, cudaStream_t st) {
  bool wide_a = false, wide_c = false;
  for (int j = 0; j < b.passes; ++j) {
    wide_a |= b.pass[j].da > 64;
    wide_c |= b.pass[j].dc > 64;
  }
  if (wide_a)
    return wide_c ? run_chunks<128, 128, W>(b, units, sms, st)
                  : run_chunks<128, 64, W>(b, units, sms, st);
  return wide_c ? run_chunks<64, 128, W>(b, units, sms, st)
                : run_chunks<64, 64, W>(b, units, sms, st);
}

// Passes over the same sequences and heads in one launch, in the kernel that is wide enough for all.
int run_passes(const cpg_linear_problem* p, cpg::LinearBatch b, void* space, cudaStream_t st) {
  if (p->sequences == 0) return CPG_OK;
  int sms = 0;
  int rc = device_ready(&sms);
  if (rc != CPG_OK) return rc;
  bool ways[2] = {false, false};
  for (int j = 0; j < b.passes; ++j) {
    if (b.pass[j].final != nullptr) b.exact = 1;
    ways[b.pass[j].reverse] = true;
  }
  b.timeout_ns = timeout_ns();
  b.inject = g_inject.load();
  const LinearCut cut = linear_cut(p, b.passes);
  const int64_t heads = int64_t(p->heads) * b.passes;
  auto run_out = [&](int64_t units) {
    if ((p->tokens / cpg::kChunk + p->sequences) * heads <= sms ||
        p->tokens <= int64_t(4) * p->sequences)  // (why: at the kernel)
      return run_chunks<Work::kFine>(b, units, sms, st);
    return b.exact ? run_chunks<Work::kExact>(b, units, sms, st)
                   : run_chunks<Work::kOutput>(b, units, sms, st);
  };
  if (cut.items == 0) return run_out(p->sequences * heads);
  const LinearSpace at = linear_space(p, cut, b.passes);
  char* const bytes = static_cast<char*>(space);
  const cpg::LinearParams& any = b.pass[0];
  for (int way = 0; way < 2; ++way) {
    // The order of whole sequences is the same either way.
    if (!(cut.length == 0 ? way == 0 : ways[way])) continue;
    char* const table = bytes + at.tables + way * at.table;
    auto* items = reinterpret_cast<cpg::LinearItem*>(table);
    auto* first = reinterpret_cast<int32_t*>(table + at.first);
    auto* count = reinterpret_cast<int32_t*>(table + at.count);
    rc = cut.length == 0
             ? launch("sequence order kernel", true, &cpg::linear_order_kernel, 1, 1024, 0, st, 1,
                      any.offsets, any.tokens, any.sequences, items, count)
             : launch("segment table kernel", true, &cpg::linear_items_kernel, 1,
                      cpg::kItemThreads, 0, st, 1, any.offsets, any.tokens, any.sequences,
                      static_cast<int32_t>(cut.length), way, static_cast<int32_t>(cut.items), items,
                      count, first);
    if (rc != CPG_OK) return rc;
    for (int j = 0; j < b.passes; ++j) {
      if (cut.length != 0 && b.pass[j].reverse != way) continue;
      b.pass[j].items = items;
      b.pass[j].item_count = count;
      b.pass[j].first_item = first;
      if (cut.length == 0) continue;
      b.pass[j].segments = reinterpret_cast<float*>(bytes + j * at.states);
      b.pass[j].most_items = static_cast<int32_t>(cut.items);
    }
  }
  if (cut.length == 0) return run_out(p->sequences * heads);
  rc = run_chunks<Work::kStates>(b, cut.items * heads, sms, st);
  if (rc != CPG_OK) return rc;
  const unsigned parts = static_cast<unsigned>((any.da * any.dc + 1023) / 1024);
  rc = launch("segment state kernel", true, &cpg::linear_segments_kernel,
              static_cast<unsigned>(p->sequences * heads) * parts, 256, 0, st, 1, b);
  if (rc != CPG_OK) return rc;
  // The final states are made: this pass's need no third part and C has both slots (65536 tokens x 16
  // heads of 128 channels with the final states, in a long loop: 470 us, 494 with them made here).
  b.exact = 0;
  return run_out(cut.items * heads);
}

// Whether all three passes of the gradient run together, or dq and dk before dv.  Where dk and dv are not
// both up to 64 or above, together means 128 channels for all, which pays where launches and the last
// blocks' tails count (dk = 64, dv = 128 x 16 heads in a graph: 37 tokens 18 -> 10 us, 2 sequences of 1024
// 57 -> 32, 5 of 820 75 -> 56) and costs where the chunks do (8 of 1024 92 -> 98 us, of 2048 x 32 heads 347 ->
// 379).
bool one_launch(const cpg_linear_problem* p) {
  if ((p->dk > 64) == (p->dv > 64)) return true;
  return p->tokens <= int64_t(8) * cpg::kChunk * p->sequences &&
         int64_t(p->sequences) * p->heads * 3 <= 2 * 148;
}

// Workspace: that of the passes, then FP32 sums of a head each for every gradient of shared heads.
struct BackwardSpace {
  int64_t grads[3], bytes;  // offsets of q's, k's and v's
};
BackwardSpace backward_space(const cpg_linear_problem* p, int32_t q_heads, int32_t k_heads,
                             int32_t v_heads) {
  BackwardSpace r;
  r.bytes = 0;
  for (int passes = 1; passes <= 3; ++passes)
    if (one_launch(p) ? passes == 3 : passes < 3)
      r.bytes = std::max(r.bytes, linear_space(p, linear_cut(p, passes), passes).bytes);
  const int32_t heads[3] = {q_heads, k_heads, v_heads}, channels[3] = {p->dk, p->dk, p->dv};
  for (int i = 0; i < 3; ++i) {
    r.grads[i] = r.bytes;
    if (heads[i] < p->heads) r.bytes += p->tokens * p->heads * channels[i] * 4;
  }
  return r;
}

// Clearing of rows outside the sequences.
void add_cleared(cpg::LinearClearParams* c, int i, const cpg_heads* x, int32_t d) {
  const int eb = bytes_of(x->dtype);
  c->p[i] = static_cast<char*>(x->ptr);
  c->token[i] = x->token_stride * eb;
  c->head[i] = x->head_stride * eb;
  c->heads[i] = x->heads;
  c->pieces[i] = d * eb / 16;
}

int run_clear(cpg::LinearClearParams c, const cpg_linear_problem* p, const int32_t* offsets,
              cudaStream_t st) {
  c.offsets = offsets;
  c.tokens = p->tokens;
  c.sequences = p->sequences;
  return launch("clear kernel", true, &cpg::linear_clear_kernel,
                static_cast<unsigned>(std::min<int64_t>(p->tokens, 148)), 256, 0, st, 1, c);
}

}  // namespace

extern "C" {

int cpg_norm_rope(const cpg_heads* q, const cpg_heads* k, int64_t tokens, int32_t channels,
                  const void* q_weight, const void* k_weight, int32_t dtype_w, float eps,
                  const float* table, int64_t table_rows, int64_t table_ld, int32_t rotary,
                  const int32_t* positions, int32_t interleaved, const cpg_heads* q_out,
                  const cpg_heads* k_out, void* stream) {
  const NormRope n{q,        k,        q_out, k_out, nullptr,    nullptr,  tokens, channels,
                   q_weight, k_weight, dtype_w, eps, table,      table_rows, table_ld, rotary,
                   positions, interleaved};
  const int rc = check_norm_rope(n, false);
  if (rc != CPG_OK || tokens == 0) return rc;
  const cpg::HeadParams p = head_params(n);
  return by_head<4>(n, [&](auto type, auto v, auto lanes, auto pairs, auto heads) {
    constexpr int kHeads = decltype(heads)::value;
    constexpr int kUnits = cpg::kHeadThreads / decltype(lanes)::value;
    const int64_t units = tokens * ((p.part[0].heads + kHeads - 1) / kHeads +
                                    (p.part[1].heads + kHeads - 1) / kHeads);
    return launch("head norm kernel", true,
                  &cpg::head_norm_kernel<decltype(type), decltype(v)::value,
                                         decltype(lanes)::value, decltype(pairs)::value, kHeads>,
                  static_cast<unsigned>((units + kUnits - 1) / kUnits), cpg::kHeadThreads, 0,
                  static_cast<cudaStream_t>(stream), 1, p);
  });
}

int cpg_norm_rope_workspace(int64_t tokens, int32_t q_heads, int32_t k_heads, int32_t channels,
                            int64_t* bytes) {
  if (bytes == nullptr) return fail(CPG_ERR_NULL, "bytes is NULL");
  if (q_heads < 1 || k_heads < 0)
    return fail(CPG_ERR_INVALID_SHAPE, "%d query and %d key heads", q_heads, k_heads);
  const int rc = check_norm_sizes(tokens, int64_t(q_heads) + k_heads, channels);
  if (rc != CPG_OK) return rc;
  int32_t blocks[2];
  grad_blocks(tokens, q_heads, k_heads, blocks);
  *bytes = (int64_t(blocks[0]) + blocks[1]) * channels * 4;
  return CPG_OK;
}

int cpg_norm_rope_backward(const cpg_heads* dq, const cpg_heads* dk, const cpg_heads* q,
                           const cpg_heads* k, int64_t tokens, int32_t channels,
                           const void* q_weight, const void* k_weight, int32_t dtype_w, float eps,
                           const float* table, int64_t table_rows, int64_t table_ld,
                           int32_t rotary, const int32_t* positions, int32_t interleaved,
                           const cpg_heads* dq_in, const cpg_heads* dk_in, float* dq_weight,
                           float* dk_weight, void* workspace, int64_t workspace_bytes,
                           void* stream) {
  const NormRope n{q,        k,        dq_in,   dk_in, dq,    dk,         tokens,   channels,
                   q_weight, k_weight, dtype_w, eps,   table, table_rows, table_ld, rotary,
                   positions, interleaved};
  int rc = check_norm_rope(n, true);
  if (rc != CPG_OK) return rc;
  if (misaligned(dq_weight, 4) || misaligned(dk_weight, 4) || misaligned(workspace, 16))
    return fail(CPG_ERR_ALIGNMENT, "weight gradients must be aligned to 4 bytes, workspace to 16");
  if (dk_weight != nullptr && k == nullptr)
    return fail(CPG_ERR_NULL, "the gradient of k's weight needs k");
  cpg::HeadParams p = head_params(n);
  grad_blocks(tokens, p.part[0].heads, p.part[1].heads, p.blocks);
  int64_t bytes = 0;
  rc = cpg_norm_rope_workspace(tokens, p.part[0].heads, p.part[1].heads, channels, &bytes);
  if (rc != CPG_OK) return rc;
  if (tokens > 0 && (workspace == nullptr || workspace_bytes < bytes))
    return fail(CPG_ERR_NULL, "the workspace must have %lld bytes", static_cast<long long>(bytes));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  p.partial = static_cast<float*>(workspace);
  if (tokens > 0) {
    rc = by_head<2>(n, [&](auto type, auto v, auto lanes, auto pairs, auto heads) {
      return launch("head norm gradient kernel", true,
                    &cpg::head_norm_grad_kernel<decltype(type), decltype(v)::value,
                                                decltype(lanes)::value, decltype(pairs)::value,
                                                decltype(heads)::value>,
                    static_cast<unsigned>(p.blocks[0] + p.blocks[1]), cpg::kHeadThreads, 0, st, 1,
                    p);
    });
    if (rc != CPG_OK) return rc;
  }
  if (dq_weight == nullptr && dk_weight == nullptr) return CPG_OK;
  const unsigned grid = static_cast<unsigned>((2 * channels + 7) / 8);
  return launch("head norm sum kernel", true, &cpg::head_norm_sum_kernel, grid,
                cpg::kHeadThreads, 0, st, 1, static_cast<const float*>(p.partial),
                tokens > 0 ? p.blocks[0] : 0, tokens > 0 ? p.blocks[1] : 0, channels, dq_weight,
                dk_weight);
}

int cpg_linear_attention_workspace(const cpg_linear_problem* p, int32_t q_heads, int32_t k_heads,
                                   int32_t v_heads, int32_t backward, int64_t* bytes) {
  if (bytes == nullptr) return fail(CPG_ERR_NULL, "bytes is NULL");
  const int rc = check_linear(p);
  if (rc != CPG_OK) return rc;
  if (q_heads < 1 || k_heads < 1 || v_heads < 1)
    return fail(CPG_ERR_INVALID_SHAPE, "%d, %d and %d heads", q_heads, k_heads, v_heads);
  *bytes = backward ? backward_space(p, q_heads, k_heads, v_heads).bytes
                    : linear_space(p, linear_cut(p, 1), 1).bytes;
  return CPG_OK;
}

int cpg_linear_attention(const cpg_linear_problem* p, const cpg_heads* q, const cpg_heads* k,
                         const cpg_heads* v, const float* log_decay, const int32_t* offsets,
                         const cpg_states* state, const cpg_states* final, const cpg_heads* out,
                         void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_linear(p);
  if (rc == CPG_OK) rc = check_operand("q", p, q, p->dk, false);
  if (rc == CPG_OK) rc = check_operand("k", p, k, p->dk, false);
  if (rc == CPG_OK) rc = check_operand("v", p, v, p->dv, false);
  if (rc == CPG_OK) rc = check_operand("out", p, out, p->dv, true, true);
  if (rc == CPG_OK) rc = check_sequences(p, log_decay, offsets);
  if (rc == CPG_OK) rc = check_states("state", p, state);
  if (rc == CPG_OK) rc = check_states("final", p, final);
  if (rc != CPG_OK) return rc;
  if (out->heads != p->heads)
    return fail(CPG_ERR_INVALID_SHAPE, "out has %d heads, not %d", out->heads, p->heads);
  int64_t bytes = 0;
  rc = cpg_linear_attention_workspace(p, q->heads, k->heads, v->heads, 0, &bytes);
  if (rc != CPG_OK) return rc;
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes))
    return fail(CPG_ERR_NULL, "the workspace must have %lld bytes", static_cast<long long>(bytes));
  if (misaligned(workspace, 16))
    return fail(CPG_ERR_ALIGNMENT, "the workspace must start on 16 bytes");
  cpg::LinearBatch b = {};
  b.passes = 1;
  b.pass[0] = linear_params(p, q, k, v, p->dk, p->dv, out, log_decay, offsets);
  set_state(&b.pass[0], state, false, 1.f);
  set_final(&b.pass[0], final, 1.f);
  return run_passes(p, b, workspace, static_cast<cudaStream_t>(stream));
}

int cpg_linear_attention_backward(const cpg_linear_problem* p, const cpg_heads* dy,
                                  const cpg_heads* q, const cpg_heads* k, const cpg_heads* v,
                                  const float* log_decay, const int32_t* offsets,
                                  const cpg_states* state, const cpg_states* dfinal,
                                  const cpg_heads* dq, const cpg_heads* dk, const cpg_heads* dv,
                                  const cpg_states* dstate, int32_t clear, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  int rc = check_linear(p);
  if (rc == CPG_OK) rc = check_operand("dy", p, dy, p->dv, false);
  if (rc == CPG_OK) rc = check_operand("q", p, q, p->dk, false);
  if (rc == CPG_OK) rc = check_operand("k", p, k, p->dk, false);
  if (rc == CPG_OK) rc = check_operand("v", p, v, p->dv, false);
  if (rc == CPG_OK) rc = check_operand("dq", p, dq, p->dk, true);
  if (rc == CPG_OK) rc = check_operand("dk", p, dk, p->dk, true);
  if (rc == CPG_OK) rc = check_operand("dv", p, dv, p->dv, true);
  if (rc == CPG_OK) rc = check_sequences(p, log_decay, offsets);
  if (rc == CPG_OK) rc = check_states("state", p, state);
  if (rc == CPG_OK) rc = check_states("dfinal", p, dfinal);
  if (rc == CPG_OK) rc = check_states("dstate", p, dstate);
  if (rc != CPG_OK) return rc;
  if (dy->heads != p->heads || dq->heads != q->heads || dk->heads != k->heads ||
      dv->heads != v->heads)
    return fail(CPG_ERR_INVALID_SHAPE, "dy has %d heads, gradients those of q, k and v", p->heads);
  int64_t bytes = 0;
  rc = cpg_linear_attention_workspace(p, q->heads, k->heads, v->heads, 1, &bytes);
  if (rc != CPG_OK) return rc;
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes))
    return fail(CPG_ERR_NULL, "the workspace must have %lld bytes", static_cast<long long>(bytes));
  if (misaligned(workspace, 16))
    return fail(CPG_ERR_ALIGNMENT, "the workspace must start on 16 bytes");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // dq, dk and dv as passes; the gradient of a head that several read: each one's in FP32 first.
  const BackwardSpace space = backward_space(p, q->heads, k->heads, v->heads);
  const cpg_heads* grads[3] = {dq, dk, dv};
  cpg_heads outs[3];
  for (int i = 0; i < 3; ++i) {
    const int32_t d = i < 2 ? p->dk : p->dv;
    outs[i] = *grads[i];
    if (grads[i]->heads < p->heads)
      outs[i] = {static_cast<char*>(workspace) + space.grads[i], int64_t(p->heads) * d, d, p->heads,
                 CPG_DTYPE_F32};
  }
  cpg::LinearBatch b = {};
  b.pass[0] = linear_params(p, dy, v, k, p->dv, p->dk, &outs[0], log_decay, offsets);
  set_state(&b.pass[0], state, true, 1.f);
  b.pass[1] = linear_params(p, v, dy, q, p->dv, p->dk, &outs[1], log_decay, offsets);
  b.pass[1].reverse = 1;
  set_state(&b.pass[1], dfinal, true, 1.f / p->scale);
  b.pass[2] = linear_params(p, k, q, dy, p->dk, p->dv, &outs[2], log_decay, offsets);
  b.pass[2].reverse = 1;
  set_state(&b.pass[2], dfinal, false, 1.f / p->scale);
  set_final(&b.pass[2], dstate, p->scale);
  b.passes = one_launch(p) ? 3 : 2;
  rc = run_passes(p, b, workspace, st);
  if (rc == CPG_OK && b.passes == 2) {
    b.pass[0] = b.pass[2];
    b.passes = 1;
    rc = run_passes(p, b, workspace, st);
  }
  for (int i = 0; i < 3 && p->tokens > 0; ++i) {
    if (rc != CPG_OK) return rc;
    if (grads[i]->heads == p->heads) continue;
    const int32_t d = i < 2 ? p->dk : p->dv;
    const cpg::LinearShareParams s{static_cast<const float*>(outs[i].ptr),
                                   static_cast<__nv_bfloat16*>(grads[i]->ptr),
                                   grads[i]->token_stride,
                                   grads[i]->head_stride,
                                   p->tokens,
                                   grads[i]->heads,
                                   p->heads / grads[i]->heads,
                                   d,
                                   offsets,
                                   p->sequences};
    const int64_t n = p->tokens * grads[i]->heads * d / 8;
    rc = launch("shared gradient kernel", true, &cpg::linear_share_kernel,
                static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 148 * 8)), 256, 0, st, 1,
                s);
  }
  if (rc != CPG_OK || clear == 0 || offsets == nullptr || p->tokens == 0) return rc;
  cpg::LinearClearParams c = {};
  for (int i = 0; i < 3; ++i) add_cleared(&c, i, grads[i], i < 2 ? p->dk : p->dv);
  return run_clear(c, p, offsets, st);
}

int cpg_linear_attention_clear(const cpg_linear_problem* p, const cpg_heads* out,
                               const int32_t* offsets, void* stream) {
  int rc = check_linear(p);
  if (rc == CPG_OK) rc = check_operand("out", p, out, p->dv, true, true);
  if (rc != CPG_OK) return rc;
  if (offsets == nullptr) return fail(CPG_ERR_NULL, "offsets is NULL");
  if (misaligned(offsets, 4)) return fail(CPG_ERR_ALIGNMENT, "offsets must be aligned to 4 bytes");
  if (p->tokens == 0) return CPG_OK;
  cpg::LinearClearParams c = {};
  add_cleared(&c, 0, out, p->dv);
  return run_clear(c, p, offsets, static_cast<cudaStream_t>(stream));
}

int cpg_attention_status(int32_t* status) {
  if (status == nullptr) return fail(CPG_ERR_NULL, "status is NULL");
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize");
  e = cudaMemcpyFromSymbol(status, cpg::linear_status_word, sizeof(*status));
  return e == cudaSuccess ? CPG_OK : cuda_fail(e, "cudaMemcpyFromSymbol");
}

int cpg_attention_set_timeout_ms(int32_t timeout_ms) {
  if (timeout_ms <= 0) return fail(CPG_ERR_INVALID_SHAPE, "timeout must be positive");
  g_timeout_ms.store(timeout_ms);
  return CPG_OK;
}

int cpg_attention_set_fault_injection(int32_t flags) {
  if ((flags & ~(CPG_INJECT_SKIP_LOADS | CPG_INJECT_SKIP_VALUES)) != 0)
    return fail(CPG_ERR_INVALID_CONFIG, "unknown fault-injection flags %d", flags);
  g_inject.store(flags);
  return CPG_OK;
}

int cpg_linear_attention_step(const cpg_linear_problem* p, const cpg_heads* q, const cpg_heads* k,
                              const cpg_heads* v, const float* log_decay, const cpg_states* state,
                              const cpg_heads* out, void* stream) {
  int rc = check_linear(p);
  if (rc == CPG_OK && p->tokens * p->heads > kMaxRows)
    rc = fail(CPG_ERR_INVALID_SHAPE, "%lld tokens x %d heads", static_cast<long long>(p->tokens),
              p->heads);
  if (rc == CPG_OK) rc = check_operand("q", p, q, p->dk, false);
  if (rc == CPG_OK) rc = check_operand("k", p, k, p->dk, false);
  if (rc == CPG_OK) rc = check_operand("v", p, v, p->dv, false);
  if (rc == CPG_OK) rc = check_operand("out", p, out, p->dv, true, true);
  if (rc != CPG_OK) return rc;
  if (log_decay == nullptr || state == nullptr)
    return fail(CPG_ERR_NULL, "log_decay and state must be non-NULL");
  if (misaligned(log_decay, 4)) return fail(CPG_ERR_ALIGNMENT, "log_decay must be aligned");
  cpg_linear_problem one = *p;
  one.sequences = static_cast<int32_t>(p->tokens);
  rc = check_states("state", &one, state);
  if (rc != CPG_OK) return rc;
  if (out->heads != p->heads)
    return fail(CPG_ERR_INVALID_SHAPE, "out has %d heads, not %d", out->heads, p->heads);
  if (p->tokens == 0) return CPG_OK;
  const cpg::LinearStepParams r{linear_rows(p, q),
                                linear_rows(p, k),
                                linear_rows(p, v),
                                out->ptr,
                                out->token_stride,
                                out->head_stride,
                                out->dtype == CPG_DTYPE_F32 ? 1 : 0,
                                log_decay,
                                state->ptr,
                                state->slots,
                                state->places,
                                p->heads,
                                p->dk,
                                p->dv,
                                p->scale};
  return launch("linear attention step kernel", true, &cpg::linear_step_kernel,
                static_cast<unsigned>(p->tokens * p->heads), cpg::kStepThreads, 0,
                static_cast<cudaStream_t>(stream), 1, r);
}

}  // extern "C"
