// C ABI of the INT8 row quantiser and of the operators around the experts' products: routing,
// expert order, dispatch and combine, and their gradients (include/cpgemm.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <mutex>
#include <type_traits>

#include "capi_common.h"
#include "capi_launch.h"
#include "cpgemm.h"
#include "expert_route.cuh"
#include "expert_rows.cuh"

using cpg_capi::bytes_of;
using cpg_capi::cuda_fail;
using cpg_capi::fail;
using cpg_capi::float_dtype;
using cpg_capi::launch;
using cpg_capi::misaligned;

namespace {

constexpr int64_t kRouteBlocks = 148 * 8;
constexpr int64_t kFewThreads = 148 * 1024;  // half of the threads that fit on the SMs
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1;  // rows and pairs are counted in int32
constexpr int64_t kMaxCols = int64_t(1) << 30;         // the kernels' column arithmetic is 32-bit

unsigned row_grid(int64_t rows) { return static_cast<unsigned>(std::min<int64_t>(rows, kMaxRows)); }

// rows x cols of a row-major matrix with row stride ld: sizes and stride make sense.
int check_matrix(const char* name, int64_t rows, int64_t cols, int64_t ld) {
  if (rows < 0 || rows > kMaxRows || cols < 0 || cols >= kMaxCols)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: %lld x %lld is not within [0, 2^31) x [0, 2^30)", name,
                static_cast<long long>(rows), static_cast<long long>(cols));
  if (ld < cols)
    return fail(CPG_ERR_INVALID_SHAPE, "%s: row stride %lld below the row length %lld", name,
                static_cast<long long>(ld), static_cast<long long>(cols));
  return CPG_OK;
}

int check_pairs(int64_t tokens, int32_t k) {
  if (tokens < 0 || tokens > kMaxRows || k < 1 || k > CPG_ROUTE_MAX_K || tokens * k > kMaxRows)
    return fail(CPG_ERR_INVALID_SHAPE,
                "%lld tokens x %d choices: 1 <= k <= %d and at most 2^31 - 1 pairs",
                static_cast<long long>(tokens), k, CPG_ROUTE_MAX_K);
  return CPG_OK;
}

// A matrix whose rows' alignment selects a kernel.  The stride of a single row is not used.
struct Rows {
  const void* p;
  int64_t ld, rows;
};
// Address bits that some row has set (of the lowest ones).
uint64_t address_bits(const Rows& r, int elem) {
  return reinterpret_cast<uintptr_t>(r.p) |
         (r.rows > 1 ? static_cast<uint64_t>(r.ld * elem) : uint64_t(0));
}

// Rows that start on `bytes` (a power of two).
bool rows_start_on(const Rows& r, int elem, int bytes) {
  return (address_bits(r, elem) & static_cast<uint64_t>(bytes - 1)) == 0;
}

// The widest access (16, 8, 4 or 2 bytes) that every row of these matrices starts on.
// 8192 tokens x 4 choices, BF16, in us with accesses of 16 / 8 / 4 / 2 bytes (2048, 2052, 2050 and
// 2049 columns) and, in brackets, of the kernels of one element an access that these replaced:
// copy 28 / 31 / 34 / 33 (dispatch, with the order kernel's 7: 36 / 39 / 41 / 41 [79]), combine
// 30 / 41 / 50 / 67 [82], its gradient 50 / 57 / 61 / 81 [116].
int row_width(std::initializer_list<Rows> all, int elem) {
  uint64_t bits = 16;
  for (const Rows& r : all) bits |= address_bits(r, elem);
  return static_cast<int>(bits & (~bits + 1));
}

// f(type of the elements, width of the accesses) for the pair at hand.
template <typename F>
int by_width(int32_t dtype, int width, F&& f) {
  using std::integral_constant;
  if (dtype == CPG_DTYPE_BF16) {
    if (width == 16) return f(__nv_bfloat16{}, integral_constant<int, 16>{});
    if (width == 8) return f(__nv_bfloat16{}, integral_constant<int, 8>{});
    if (width == 4) return f(__nv_bfloat16{}, integral_constant<int, 4>{});
    return f(__nv_bfloat16{}, integral_constant<int, 2>{});
  }
  if (width == 16) return f(float{}, integral_constant<int, 16>{});
  if (width == 8) return f(float{}, integral_constant<int, 8>{});
  return f(float{}, integral_constant<int, 4>{});
}

template <typename T, int W, int G, int NV, bool Resident>
int launch_int8_vec(const cpg::RowsParams& p, cudaStream_t st) {
  constexpr int kThreads = cpg::int8_threads<G>();
  constexpr int kRows = kThreads / G;
  return launch("INT8 row kernel", false, &cpg::rows_int8_vec_kernel<T, W, G, NV, Resident>,
                row_grid((p.tokens + kRows - 1) / kRows), kThreads, 0, st, 1, p);
}

template <typename T, int W>
int launch_int8_vec(const cpg::RowsParams& p, cudaStream_t st) {
  // The fewest threads that hold a row (16384 x 4096 BF16: 128 threads 49 us, 256 61 us); more while
  // the tokens leave most of the GPU idle (each then has less of a row to wait for).
  // Measured: FP32 16384 x 8192 102.6 us (1.00 of measured HBM), BF16 75.0 us (0.82), where the
  // conversions bound it: three packed FMAs per two elements after 22 issue slots an element before.
  // BF16 16384 x 4096 takes 49-52 us (0.6): a group waits for its row, the maximum and the
  // conversions in turn and has nothing of its next row in flight.
  constexpr int kVecs = cpg::kInt8Vecs;
  constexpr int64_t kEach = kVecs * 16;
  if (p.cols > 2 * 512 * kEach) return launch_int8_vec<T, W, 512, kVecs, false>(p, st);
  if (p.cols > 512 * kEach) return launch_int8_vec<T, W, 512, 2 * kVecs, true>(p, st);
  int64_t threads = 32;
  while (p.cols > threads * kEach) threads *= 2;
  while (threads < 256 && p.tokens * threads < kFewThreads && p.cols > threads * 16) threads *= 2;
  switch (threads) {
    case 32: return launch_int8_vec<T, W, 32, kVecs, true>(p, st);
    case 64: return launch_int8_vec<T, W, 64, kVecs, true>(p, st);
    case 128: return launch_int8_vec<T, W, 128, kVecs, true>(p, st);
    case 256: return launch_int8_vec<T, W, 256, kVecs, true>(p, st);
    default: return launch_int8_vec<T, W, 512, kVecs, true>(p, st);
  }
}

// Chunks of a row for warps whose lanes make n accesses of W bytes, and blocks of 8 warps.
template <typename T, int W>
int32_t row_chunks(int64_t cols, int n) {
  const int64_t per = int64_t(32) * n * cpg::RowAccess<T, W>::kElems;
  return static_cast<int32_t>((cols + per - 1) / per);
}
unsigned warp_grid(int64_t warps) { return row_grid((warps + 7) / 8); }

// Rows of INT8 that start on 16 bytes (as the GEMM wants them) whatever the alignment of x; others
// one element at a time.  16384 rows in us, by accesses of 16 / 8 / 4 / 2 bytes (4096, 4100, 4098 and
// 4097 columns) and [by elements]: BF16 52 / 64 / 67 / 89 [150]; FP32 57 / 89 / 144 by 16, 8 (4098)
// and 4 (4097) bytes [150].
int launch_int8(const cpg::RowsParams& p, int32_t dtype_x, cudaStream_t st) {
  if (rows_start_on({p.rows, p.ldr, p.num_rows}, 1, 16)) {
    const int width = row_width({{p.x, p.ldx, p.tokens}}, bytes_of(dtype_x));
    return by_width(dtype_x, width, [&](auto type, auto w) {
      return launch_int8_vec<decltype(type), decltype(w)::value>(p, st);
    });
  }
  auto fn = dtype_x == CPG_DTYPE_BF16 ? &cpg::rows_int8_kernel<__nv_bfloat16>
                                      : &cpg::rows_int8_kernel<float>;
  return launch("INT8 row kernel", false, fn, row_grid(p.tokens), 256, 0, st, 1, p);
}

// Blocks the cluster of an expert order kernel (`which`: its place among the variants) may have on
// the current device: 16, which is beyond what every device must offer, if they fit, else 8.  Also
// raises the kernel's shared-memory limit to that of its largest call.  Asked once per device.
int order_cluster(const void* fn, int which, int* most) {
  constexpr int kDevices = 64, kVariants = 4;
  static std::mutex mu;
  static int known[kDevices][kVariants];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kDevices) return fail(CPG_ERR_NO_DEVICE, "device %d", dev);
  std::lock_guard<std::mutex> lock(mu);
  int& k = known[dev][which];
  if (k == 0) {
    const int smem =
        static_cast<int>(sizeof(uint32_t)) * (cpg::kOrderWarps + 1) * CPG_ROUTE_MAX_EXPERTS;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(expert order)");
    int fits = 0;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) ==
        cudaSuccess) {
      cudaLaunchConfig_t lc = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = cpg::kOrderMaxCluster;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      lc.gridDim = dim3(cpg::kOrderMaxCluster, 1, 1);
      lc.blockDim = dim3(cpg::kOrderThreads, 1, 1);
      lc.dynamicSmemBytes = static_cast<size_t>(smem);
      lc.attrs = attr;
      lc.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&fits, fn, &lc) != cudaSuccess) fits = 0;
    }
    (void)cudaGetLastError();  // a refusal of 16 is no error of this call
    k = fits > 0 ? cpg::kOrderMaxCluster : 8;
  }
  *most = k;
  return CPG_OK;
}

int check_route(const cpg_route_config* c, int64_t tokens) {
  if (c == nullptr) return fail(CPG_ERR_NULL, "route config is NULL");
  if (c->experts < 1 || c->experts > CPG_ROUTE_MAX_EXPERTS)
    return fail(CPG_ERR_INVALID_SHAPE, "1 <= experts <= %d, got %d", CPG_ROUTE_MAX_EXPERTS,
                c->experts);
  if (c->k > c->experts)
    return fail(CPG_ERR_INVALID_SHAPE, "k = %d choices of %d experts", c->k, c->experts);
  if (c->scoring != CPG_ROUTE_SOFTMAX && c->scoring != CPG_ROUTE_SIGMOID)
    return fail(CPG_ERR_INVALID_CONFIG, "scoring %d is not one of CPG_ROUTE_*", c->scoring);
  if (c->groups < 1 || c->groups > CPG_ROUTE_MAX_GROUPS || c->experts % c->groups != 0)
    return fail(CPG_ERR_INVALID_CONFIG, "%d groups must divide %d experts and be at most %d",
                c->groups, c->experts, CPG_ROUTE_MAX_GROUPS);
  if (c->kept_groups < 1 || c->kept_groups > c->groups ||
      c->k > c->kept_groups * (c->experts / c->groups))
    return fail(CPG_ERR_INVALID_CONFIG, "%d of %d groups cannot hold %d choices", c->kept_groups,
                c->groups, c->k);
  if (c->group_score != CPG_GROUP_MAX && c->group_score != CPG_GROUP_TOP2)
    return fail(CPG_ERR_INVALID_CONFIG, "group_score %d is not one of CPG_GROUP_*",
                c->group_score);
  return check_pairs(tokens, c->k);
}

// Whether every lane's run of V elements of every row starts on its vectors.
template <int V>
int32_t run_vectors(const Rows& r, int32_t dtype) {
  const int bytes = dtype == CPG_DTYPE_BF16 ? cpg::run_vector_bytes<__nv_bfloat16, V>()
                                            : cpg::run_vector_bytes<float, V>();
  return rows_start_on(r, bytes_of(dtype), bytes) ? 1 : 0;
}

template <int L, int V>
int launch_route(cpg::RouteParams p, int32_t dtype, cudaStream_t st) {
  p.vec = run_vectors<V>({p.logits, p.ld, p.tokens}, dtype);
  p.vec_bias = run_vectors<V>({p.bias, 0, 1}, CPG_DTYPE_F32);
  const size_t smem = sizeof(double) * 32 * V * cpg::kRouteWarps;
  // At most about as many blocks as fit on the SMs at once; each then walks several tokens.
  const int64_t per = 32 / L * cpg::kRouteWarps;
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>((p.tokens + per - 1) / per, kRouteBlocks));
  auto fn = dtype == CPG_DTYPE_BF16 ? &cpg::route_kernel<__nv_bfloat16, L, V>
                                    : &cpg::route_kernel<float, L, V>;
  return launch("route kernel", true, fn, grid, 32 * cpg::kRouteWarps, smem, st, 1, p);
}

template <int L, int V>
int launch_route_grad(cpg::RouteGradParams p, int32_t dtype, cudaStream_t st) {
  const int64_t per = 32 / L * cpg::kRouteWarps;
  const unsigned grid = static_cast<unsigned>((p.tokens + per - 1) / per);
  // Vectors of as many logits as 16 bytes or V hold.
  if (dtype == CPG_DTYPE_BF16) {
    constexpr int kPer = V < 8 ? V : 8;
    p.vec = run_vectors<kPer>({p.logits, p.ld, p.tokens}, dtype);
    p.vec_out = run_vectors<kPer>({p.dlogits, p.ldd, p.tokens}, dtype);
    return launch("route gradient kernel", true, &cpg::route_grad_kernel<__nv_bfloat16, L, V>, grid,
                  32 * cpg::kRouteWarps, 0, st, 1, p);
  } else {
    p.vec = run_vectors<4>({p.logits, p.ld, p.tokens}, dtype);
    p.vec_out = run_vectors<4>({p.dlogits, p.ldd, p.tokens}, dtype);
    return launch("route gradient kernel", true, &cpg::route_grad_kernel<float, L, V>, grid,
                  32 * cpg::kRouteWarps, 0, st, 1, p);
  }
}

static_assert(CPG_ROUTE_MAX_EXPERTS == cpg::kRouteMaxExperts &&
                  CPG_ROUTE_MAX_K == cpg::kRouteMaxK &&
                  CPG_ROUTE_MAX_GROUPS == cpg::kRouteMaxGroups,
              "routing limits");
static_assert(CPG_ROUTE_SOFTMAX == cpg::kRouteSoftmax && CPG_ROUTE_SIGMOID == cpg::kRouteSigmoid &&
                  CPG_GROUP_MAX == cpg::kRouteGroupMax && CPG_GROUP_TOP2 == cpg::kRouteGroupTop2,
              "routing codes");

}  // namespace

extern "C" {

int cpg_quantize_int8(const void* x, int32_t dtype_x, int64_t rows, int64_t cols, int64_t ldx,
                      void* q, int64_t ldq, float* scales, void* stream) {
  if (!float_dtype(dtype_x)) return fail(CPG_ERR_DTYPE, "x must be BF16 or FP32");
  int rc = check_matrix("x", rows, cols, ldx);
  if (rc == CPG_OK) rc = check_matrix("q", rows, cols, ldq);
  if (rc != CPG_OK) return rc;
  if (rows == 0) return CPG_OK;
  if (scales == nullptr || (cols > 0 && (x == nullptr || q == nullptr)))
    return fail(CPG_ERR_NULL, "x, q and scales must be non-NULL");
  if (misaligned(x, bytes_of(dtype_x)) || misaligned(scales, 4))
    return fail(CPG_ERR_ALIGNMENT, "x and scales must be aligned to their elements");
  const cpg::RowsParams p{x, rows, cols, ldx, nullptr, 1, q, rows, ldq, scales};
  return launch_int8(p, dtype_x, static_cast<cudaStream_t>(stream));
}

int cpg_route(const cpg_route_config* c, const void* logits, int32_t dtype, int64_t tokens,
              int64_t ld, const float* bias, int32_t* ids, float* weights, void* stream) {
  int rc = check_route(c, tokens);
  if (rc != CPG_OK) return rc;
  if (!float_dtype(dtype)) return fail(CPG_ERR_DTYPE, "logits must be BF16 or FP32");
  rc = check_matrix("logits", tokens, c->experts, ld);
  if (rc != CPG_OK) return rc;
  if (tokens == 0) return CPG_OK;
  if (logits == nullptr || ids == nullptr || weights == nullptr)
    return fail(CPG_ERR_NULL, "logits, ids and weights must be non-NULL");
  if (misaligned(logits, bytes_of(dtype)) || misaligned(bias, 4) || misaligned(ids, 4) ||
      misaligned(weights, 4))
    return fail(CPG_ERR_ALIGNMENT, "logits, bias, ids and weights must be aligned to their elements");
  cpg::RouteParams p{logits,         tokens,         ld,         bias,      ids,
                     weights,        c->experts,     c->k,       c->scoring, c->groups,
                     c->kept_groups, c->group_score, c->renormalize != 0 ? 1 : 0, 0, 0, c->scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Fewer lanes per token (and more experts a lane) while they hold the choices and the groups, and
  // where scores are ranked one candidate more.  16384 tokens, top 8, ranked by logit / by sigmoid
  // and bias in 8 groups: 64 experts 32 lanes 10.5 / 14.8 us, 8 and 16 lanes 5.3 / 11.0;
  // 128 experts 32 lanes 11.2 / 15.7 us, 16 lanes 9.4 / 14.8; 256 experts 32 lanes 14.4 / 21.8 us,
  // 16 lanes (whose 16 experts a lane leave room for too few warps) 14.8 / 27.5.
  const bool by_logit = bias == nullptr && (c->groups == 1 || c->group_score == CPG_GROUP_MAX);
  const int32_t e = c->experts, need = std::max(by_logit ? c->k : c->k + 1, c->groups);
  if (need <= 8 && e <= 32) return launch_route<8, 4>(p, dtype, st);
  if (need <= 8 && e <= 64) return launch_route<8, 8>(p, dtype, st);
  if (need <= 16 && e <= 64) return launch_route<16, 4>(p, dtype, st);
  if (need <= 16 && e <= 128) return launch_route<16, 8>(p, dtype, st);
  if (e <= 32) return launch_route<32, 1>(p, dtype, st);
  if (e <= 64) return launch_route<32, 2>(p, dtype, st);
  if (e <= 128) return launch_route<32, 4>(p, dtype, st);
  if (e <= 256) return launch_route<32, 8>(p, dtype, st);
  if (e <= 512) return launch_route<32, 16>(p, dtype, st);
  return launch_route<32, 32>(p, dtype, st);
}

int cpg_route_backward(const cpg_route_config* c, const float* dweights, const void* logits,
                       int32_t dtype, int64_t tokens, int64_t ld, const int32_t* ids,
                       void* dlogits, int64_t ldd, void* stream) {
  int rc = check_route(c, tokens);
  if (rc != CPG_OK) return rc;
  if (!float_dtype(dtype)) return fail(CPG_ERR_DTYPE, "logits must be BF16 or FP32");
  rc = check_matrix("logits", tokens, c->experts, ld);
  if (rc == CPG_OK) rc = check_matrix("dlogits", tokens, c->experts, ldd);
  if (rc != CPG_OK) return rc;
  if (tokens == 0) return CPG_OK;
  if (dweights == nullptr || logits == nullptr || ids == nullptr || dlogits == nullptr)
    return fail(CPG_ERR_NULL, "dweights, logits, ids and dlogits must be non-NULL");
  if (misaligned(logits, bytes_of(dtype)) || misaligned(dlogits, bytes_of(dtype)) ||
      misaligned(dweights, 4) || misaligned(ids, 4))
    return fail(CPG_ERR_ALIGNMENT,
                "dweights, logits, ids and dlogits must be aligned to their elements");
  cpg::RouteGradParams p{dweights, logits, tokens,     ld,   ids,
                         dlogits,  ldd,    c->experts, c->k, c->scoring,
                         c->renormalize != 0 ? 1 : 0, 0, 0, c->scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The fewest lanes per token that hold its choices and at most 16 of its logits each.
  const int32_t e = c->experts, k = c->k;
  if (k <= 8 && e <= 32) return launch_route_grad<8, 4>(p, dtype, st);
  if (k <= 8 && e <= 64) return launch_route_grad<8, 8>(p, dtype, st);
  if (k <= 8 && e <= 128) return launch_route_grad<8, 16>(p, dtype, st);
  if (k <= 16 && e <= 64) return launch_route_grad<16, 4>(p, dtype, st);
  if (k <= 16 && e <= 128) return launch_route_grad<16, 8>(p, dtype, st);
  if (k <= 16 && e <= 256) return launch_route_grad<16, 16>(p, dtype, st);
  if (e <= 128) return launch_route_grad<32, 4>(p, dtype, st);
  if (e <= 256) return launch_route_grad<32, 8>(p, dtype, st);
  if (e <= 512) return launch_route_grad<32, 16>(p, dtype, st);
  return launch_route_grad<32, 32>(p, dtype, st);
}

int cpg_expert_order(const int32_t* ids, int64_t tokens, int32_t k, int32_t experts,
                     int32_t* offsets, int32_t* slots, void* stream) {
  int rc = check_pairs(tokens, k);
  if (rc != CPG_OK) return rc;
  if (experts < 1 || experts > CPG_ROUTE_MAX_EXPERTS)
    return fail(CPG_ERR_INVALID_SHAPE, "1 <= experts <= %d, got %d", CPG_ROUTE_MAX_EXPERTS,
                experts);
  const int64_t pairs = tokens * k;
  if (offsets == nullptr || (pairs > 0 && (ids == nullptr || slots == nullptr)))
    return fail(CPG_ERR_NULL, "ids, offsets and slots must be non-NULL");
  if (misaligned(ids, 4) || misaligned(offsets, 4) || misaligned(slots, 4))
    return fail(CPG_ERR_ALIGNMENT, "ids, offsets and slots must be 4-byte aligned");
  const int smem = static_cast<int>(sizeof(uint32_t)) * (cpg::kOrderWarps + 1) * experts;
  auto fn = experts <= 16    ? &cpg::expert_order_kernel<4>
            : experts <= 64  ? &cpg::expert_order_kernel<6>
            : experts <= 256 ? &cpg::expert_order_kernel<8>
                             : &cpg::expert_order_kernel<10>;
  int most = 0;
  rc = order_cluster(reinterpret_cast<const void*>(fn), experts <= 16    ? 0
                                                        : experts <= 64  ? 1
                                                        : experts <= 256 ? 2
                                                                         : 3, &most);
  if (rc != CPG_OK) return rc;
  // One block while its 32 warps have at most 64 pairs each, then the blocks of one cluster.
  // 131072 pairs of 256 experts: 8 blocks 13.9 us, 16 blocks 10.2 us.
  int blocks = 1;
  while (blocks < most && pairs > int64_t(blocks) * cpg::kOrderWarps * 64) blocks *= 2;
  const cpg::OrderParams p{ids, pairs, experts, offsets, slots};
  return launch("expert order kernel", true, fn, static_cast<unsigned>(blocks), cpg::kOrderThreads, smem,
                static_cast<cudaStream_t>(stream), blocks, p);
}

int cpg_dispatch_rows(const void* x, int32_t dtype_x, int64_t tokens, int64_t cols, int64_t ldx,
                      const int32_t* slots, int32_t k, void* rows, int32_t dtype_rows,
                      int64_t num_rows, int64_t ldr, float* scales, void* stream) {
  int rc = check_pairs(tokens, k);
  if (rc != CPG_OK) return rc;
  if (!float_dtype(dtype_x) || (dtype_rows != dtype_x && dtype_rows != CPG_DTYPE_I8))
    return fail(CPG_ERR_DTYPE, "x must be BF16 or FP32 and rows of the same type or INT8");
  rc = check_matrix("x", tokens, cols, ldx);
  if (rc == CPG_OK) rc = check_matrix("rows", num_rows, cols, ldr);
  if (rc != CPG_OK) return rc;
  const bool int8 = dtype_rows == CPG_DTYPE_I8;
  if (tokens == 0 || num_rows == 0 || (cols == 0 && !int8)) return CPG_OK;
  if (slots == nullptr || (int8 && scales == nullptr) ||
      (cols > 0 && (x == nullptr || rows == nullptr)))
    return fail(CPG_ERR_NULL, "x, slots, rows (and scales with INT8) must be non-NULL");
  if (misaligned(x, bytes_of(dtype_x)) || misaligned(rows, bytes_of(dtype_rows)) ||
      misaligned(slots, 4) || misaligned(scales, 4))
    return fail(CPG_ERR_ALIGNMENT, "x, rows, slots and scales must be aligned to their elements");
  const cpg::RowsParams p{x, tokens, cols, ldx, slots, k, rows, num_rows, ldr, scales};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int8) return launch_int8(p, dtype_x, st);
  return by_width(dtype_x, row_width({{x, ldx, tokens}, {rows, ldr, num_rows}}, bytes_of(dtype_x)),
                  [&](auto type, auto width) {
    using T = decltype(type);
    constexpr int W = decltype(width)::value;
    const int32_t chunks = row_chunks<T, W>(cols, cpg::row_accesses<W>(cpg::kCopyVecs));
    return launch("row copy kernel", true, &cpg::rows_copy_kernel<T, W>,
                  warp_grid(tokens * chunks), 256, 0, st, 1, p, chunks);
  });
}

int cpg_combine_rows(const void* rows, int32_t dtype, int64_t num_rows, int64_t cols, int64_t ldr,
                     const int32_t* slots, const float* weights, int64_t tokens, int32_t k,
                     const void* source, int64_t ld_source, void* y, int64_t ldy, void* stream) {
  int rc = check_pairs(tokens, k);
  if (rc != CPG_OK) return rc;
  if (!float_dtype(dtype)) return fail(CPG_ERR_DTYPE, "rows must be BF16 or FP32");
  rc = check_matrix("rows", num_rows, cols, ldr);
  if (rc == CPG_OK) rc = check_matrix("y", tokens, cols, ldy);
  if (rc == CPG_OK && source != nullptr) rc = check_matrix("source", tokens, cols, ld_source);
  if (rc != CPG_OK) return rc;
  if (tokens == 0 || cols == 0) return CPG_OK;
  if ((num_rows > 0 && rows == nullptr) || slots == nullptr || y == nullptr)
    return fail(CPG_ERR_NULL, "rows, slots and y must be non-NULL");
  const int es = bytes_of(dtype);
  if (misaligned(rows, es) || misaligned(source, es) || misaligned(y, es) ||
      misaligned(slots, 4) || misaligned(weights, 4))
    return fail(CPG_ERR_ALIGNMENT, "rows, slots, weights, source and y must be aligned to their elements");
  const cpg::CombineParams p{rows,   num_rows, cols,   ldr,       slots, weights,
                             tokens, k,        source, ld_source, y,     ldy};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Rows src = source != nullptr ? Rows{source, ld_source, tokens} : Rows{y, ldy, tokens};
  const int w = row_width({{rows, ldr, num_rows}, {y, ldy, tokens}, src}, es);
  return by_width(dtype, w, [&](auto type, auto width) {
    using T = decltype(type);
    constexpr int W = decltype(width)::value;
    const int32_t chunks = row_chunks<T, W>(cols, cpg::combine_accesses<T, W>());
    return launch("combine kernel", true, &cpg::combine_kernel<T, W>, warp_grid(tokens * chunks),
                  256, 0, st, 1, p, chunks);
  });
}

int cpg_combine_rows_backward(const void* dy, int32_t dtype, int64_t tokens, int64_t cols,
                              int64_t lddy, const void* rows, int64_t num_rows, int64_t ldr,
                              const int32_t* slots, const float* weights, int32_t k, void* drows,
                              int64_t lddr, float* dweights, void* stream) {
  int rc = check_pairs(tokens, k);
  if (rc != CPG_OK) return rc;
  if (!float_dtype(dtype)) return fail(CPG_ERR_DTYPE, "dy and rows must be BF16 or FP32");
  rc = check_matrix("dy", tokens, cols, lddy);
  if (rc == CPG_OK) rc = check_matrix("rows", num_rows, cols, ldr);
  if (rc == CPG_OK) rc = check_matrix("drows", num_rows, cols, lddr);
  if (rc != CPG_OK) return rc;
  if (tokens == 0) return CPG_OK;
  if (slots == nullptr || weights == nullptr || dweights == nullptr ||
      (cols > 0 && dy == nullptr) ||
      (cols > 0 && num_rows > 0 && (rows == nullptr || drows == nullptr)))
    return fail(CPG_ERR_NULL, "dy, rows, slots, weights, drows and dweights must be non-NULL");
  const int es = bytes_of(dtype);
  if (misaligned(dy, es) || misaligned(rows, es) || misaligned(drows, es) ||
      misaligned(slots, 4) || misaligned(weights, 4) || misaligned(dweights, 4))
    return fail(CPG_ERR_ALIGNMENT, "every argument must be aligned to its elements");
  const cpg::CombineGradParams p{dy,    tokens,  cols, lddy,  rows, num_rows, ldr,
                                 slots, weights, k,    drows, lddr, dweights};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int w =
      row_width({{dy, lddy, tokens}, {rows, ldr, num_rows}, {drows, lddr, num_rows}}, es);
  return by_width(dtype, w, [&](auto type, auto width) {
    return launch("combine gradient kernel", true,
                  &cpg::combine_grad_kernel<decltype(type), decltype(width)::value>,
                  warp_grid(tokens * k), 256, 0, st, 1, p);
  });
}

int cpg_clear_unnamed_rows(void* rows, int32_t dtype, int64_t num_rows, int64_t cols, int64_t ldr,
                           const int32_t* slots, int64_t tokens, int32_t k, void* stream) {
  int rc = check_pairs(tokens, k);
  if (rc != CPG_OK) return rc;
  if (!float_dtype(dtype)) return fail(CPG_ERR_DTYPE, "rows must be BF16 or FP32");
  rc = check_matrix("rows", num_rows, cols, ldr);
  if (rc != CPG_OK) return rc;
  if (num_rows == 0 || cols == 0) return CPG_OK;
  if (rows == nullptr || (tokens > 0 && slots == nullptr))
    return fail(CPG_ERR_NULL, "rows and slots must be non-NULL");
  if (misaligned(rows, bytes_of(dtype)) || misaligned(slots, 4))
    return fail(CPG_ERR_ALIGNMENT, "rows and slots must be aligned to their elements");
  // A block per SM while there are 32 rows for each, and no more rows than its marks hold.
  int64_t per = ((num_rows + 147) / 148 + 31) / 32 * 32;
  per = std::min<int64_t>(per, cpg::kClearMaxRows);
  const cpg::ClearRowsParams p{rows, num_rows, cols, ldr, slots, tokens * k,
                               static_cast<int32_t>(per)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_width(dtype, row_width({{rows, ldr, num_rows}}, bytes_of(dtype)),
                  [&](auto type, auto width) {
    return launch("row clearing kernel", true,
                  &cpg::rows_clear_kernel<decltype(type), decltype(width)::value>,
                  static_cast<unsigned>((num_rows + per - 1) / per), cpg::kClearThreads,
                  static_cast<size_t>(per / 8), st, 1, p);
  });
}

}  // extern "C"
