// Error reporting shared by the translation units of the C ABI.
#pragma once
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <string>

#include "cpgemm.h"

namespace cpg_capi {

// Detail of the calling thread's last failure (cpg_last_error_message).
inline thread_local std::string g_last_error;

inline int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

inline int cuda_fail(cudaError_t e, const char* what) {
  return fail(CPG_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

}  // namespace cpg_capi
