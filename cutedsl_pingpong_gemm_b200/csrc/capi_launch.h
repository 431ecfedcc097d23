// Launches, small checks and the tensor-map encoder, shared by the translation units.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "capi_common.h"

namespace cpg_capi {

inline bool float_dtype(int32_t dtype) { return dtype == CPG_DTYPE_BF16 || dtype == CPG_DTYPE_F32; }
inline int bytes_of(int32_t dtype) { return dtype == CPG_DTYPE_F32 ? 4 : (dtype == CPG_DTYPE_I8 ? 1 : 2); }

inline bool misaligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(bytes - 1)) != 0;
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
  });
  return fn;
}

// Launches a kernel, `early` as a programmatic dependent of the stream's previous kernel: it may be
// set up while that one finishes and waits for it before its first access (kernel_begins).
// Measured in a captured chain of route, dispatch and combine of 16 tokens: 12.0 us plain, 10.6 us
// early; letting the next kernel in from the start of each as well: 11.2 us, since its blocks wait
// on the SMs the first still needs.  The INT8 row kernels are not launched early but do let the next
// kernel in: quantise + small-M product of 64 x 8192 x 8192 takes 24.8 us with neither, 25.1 us with
// both and 23.2 us so (16 rows: 22.1, 20.1 and 20.4 us).
template <typename... P>
int launch(const char* what, bool early, void (*kernel)(P...), unsigned grid, unsigned threads,
           size_t smem, cudaStream_t st, int cluster, P... args) {
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  lc.gridDim = dim3(grid, 1, 1);
  lc.blockDim = dim3(threads, 1, 1);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&lc, kernel, args...);
  return e == cudaSuccess ? CPG_OK : cuda_fail(e, what);
}

}  // namespace cpg_capi
