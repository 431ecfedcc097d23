// Accesses to rows of BF16 or FP32 elements, as wide as their alignment allows, shared by the row
// kernels.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cpg {

// Before the first access of a kernel: the previous kernel's writes are visible after it.  (All but
// the INT8 row kernels are launched as programmatic dependents, so they may be set up while
// that kernel finishes.  For the INT8 kernels it returns at once; they let the next kernel in first.)
__device__ __forceinline__ void kernel_begins() { ptx::griddep_wait(); }

// 16 bytes that bypass L1 (for rows that are read once).
__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// ------------------------------------------------------ accesses as wide as the rows' alignment
// W bytes of a row of T at a time (16, 8, 4, or 2 for BF16): all the rows' addresses are multiples of
// W.  The last access of a row may be partial.
template <typename T, int W>
struct RowAccess {
  static constexpr int kElems = W / static_cast<int>(sizeof(T));
  static constexpr int kWords = W < 4 ? 1 : W / 4;
  struct Data {
    uint32_t w[kWords];
  };
  __device__ __forceinline__ static Data zero() {
    Data d;
#pragma unroll
    for (int i = 0; i < kWords; ++i) d.w[i] = 0u;
    return d;
  }
  __device__ __forceinline__ static uint32_t bits(const T* p) {
    if constexpr (sizeof(T) == 2)
      return *reinterpret_cast<const uint16_t*>(p);
    else
      return *reinterpret_cast<const uint32_t*>(p);
  }
  // kElems elements at p.  `Once`: read by this kernel only and once (16 bytes: past L1; narrower
  // accesses share their sectors with the neighbours' through L1).
  template <bool Once>
  __device__ __forceinline__ static Data load_all(const T* p) {
    Data d;
    if constexpr (W == 16) {
      const uint4 v = Once ? ld_stream_v4(p) : *reinterpret_cast<const uint4*>(p);
      d.w[0] = v.x;
      d.w[1] = v.y;
      d.w[2] = v.z;
      d.w[3] = v.w;
    } else if constexpr (W == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      d.w[0] = v.x;
      d.w[1] = v.y;
    } else if constexpr (W == 4) {
      d.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      d.w[0] = bits(p);
    }
    return d;
  }
  // Elements [c, c + kElems), zeros past the row's end.
  template <bool Once>
  __device__ __forceinline__ static Data load(const T* row, int32_t c, int32_t cols) {
    if (c + kElems <= cols) return load_all<Once>(row + c);
    Data d = zero();
#pragma unroll
    for (int j = 0; j < kElems; ++j) {
      if (c + j < cols) {
        if constexpr (sizeof(T) == 2)
          d.w[j >> 1] |= bits(row + c + j) << (16 * (j & 1));
        else
          d.w[j] = bits(row + c + j);
      }
    }
    return d;
  }
  __device__ __forceinline__ static void store(T* row, int32_t c, int32_t cols, const Data& d) {
    if (c + kElems <= cols) {
      T* p = row + c;
      if constexpr (W == 16)
        ptx::st_global_v4(p, d.w[0], d.w[1], d.w[2], d.w[3]);
      else if constexpr (W == 8)
        *reinterpret_cast<uint2*>(p) = make_uint2(d.w[0], d.w[1]);
      else if constexpr (W == 4)
        *reinterpret_cast<uint32_t*>(p) = d.w[0];
      else
        *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(d.w[0]);
      return;
    }
#pragma unroll
    for (int j = 0; j < kElems; ++j) {
      if (c + j < cols) {
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint16_t*>(row + c + j) =
              static_cast<uint16_t>(d.w[j >> 1] >> (16 * (j & 1)));
        else
          *reinterpret_cast<uint32_t*>(row + c + j) = d.w[j];
      }
    }
  }
  __device__ __forceinline__ static void unpack(const Data& d, float* f) {
#pragma unroll
    for (int j = 0; j < kElems; ++j) {
      if constexpr (sizeof(T) == 2)
        f[j] = __uint_as_float((j & 1) ? d.w[j >> 1] & 0xffff0000u : d.w[j >> 1] << 16);
      else
        f[j] = __uint_as_float(d.w[j]);
    }
  }
  __device__ __forceinline__ static Data pack(const float* f) {
    Data d;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        d.w[i] = ptx::pack_bf16x2(f[2 * i], kElems > 1 ? f[2 * i + (kElems > 1 ? 1 : 0)] : 0.f);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) d.w[i] = __float_as_uint(f[i]);
    }
    return d;
  }
};

}  // namespace cpg
