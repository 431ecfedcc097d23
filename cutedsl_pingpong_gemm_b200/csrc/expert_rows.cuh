// Row kernels around the experts' products: rows quantised to INT8 (a scale per row), rows copied
// into expert order (dispatch), the weighted sums back (combine) and the gradient of those sums.
//
// All of them move whole rows and are bound by HBM; each row of the input is read once.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cpg {

constexpr float kInt8Max = 127.0f;
constexpr float kInt8AmaxFloor = 1e-12f;

// One 16-byte vector of a row: kElems values of T.
template <typename T>
struct RowVec;
template <>
struct RowVec<__nv_bfloat16> {
  static constexpr int kElems = 8;
  __device__ __forceinline__ static void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ static uint4 pack(const float* f) {
    return make_uint4(ptx::pack_bf16x2(f[0], f[1]), ptx::pack_bf16x2(f[2], f[3]),
                      ptx::pack_bf16x2(f[4], f[5]), ptx::pack_bf16x2(f[6], f[7]));
  }
  __device__ __forceinline__ static float load(const __nv_bfloat16* p) {
    return __bfloat162float(*p);
  }
  __device__ __forceinline__ static void store(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
  }
};
template <>
struct RowVec<float> {
  static constexpr int kElems = 4;
  __device__ __forceinline__ static void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  __device__ __forceinline__ static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  __device__ __forceinline__ static float load(const float* p) { return *p; }
  __device__ __forceinline__ static void store(float* p, float v) { *p = v; }
};

// The bit pattern of |v|: non-negative floats order like their bits, infinities and NaN last.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Scale of a row whose largest |x| has these bits: max(amax, floor) / 127, or NaN when the row
// holds an infinity or a NaN (INT8 has neither, so the scale carries it into every product).
__device__ __forceinline__ float int8_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return __fdiv_rn(fmaxf(__uint_as_float(amax), kInt8AmaxFloor), kInt8Max);
}

// rint(RN(x / s)) as an INT8 byte, 0 for a row whose scale is NaN.
__device__ __forceinline__ uint32_t int8_quotient(float x, float s) {
  return s == s ? static_cast<uint32_t>(__float2int_rn(__fdiv_rn(x, s))) & 0xffu : 0u;
}

struct RowsParams {
  const void* x;
  int64_t tokens, cols, ldx;
  const int32_t* slots;  // [tokens][k] row of each copy, negative for none; NULL: row t
  int32_t k;
  void* rows;
  int64_t num_rows, ldr;
  float* scales;  // INT8: [num_rows]
};

// rows[slot] = x[t] for the k slots of every token, one block per token.  OutT is T, or int8_t for
// q = rint(x / s) with s = max|x[t]| / 127 in scales[slot].
template <typename T, typename OutT>
__global__ void __launch_bounds__(256) rows_kernel(const RowsParams p) {
  constexpr bool kQuant = sizeof(OutT) == 1;
  __shared__ uint32_t red[8];
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    float s = 1.f;
    if constexpr (kQuant) {
      uint32_t m = 0u;
      for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x)
        m = max(m, abs_bits(RowVec<T>::load(x + c)));
      m = __reduce_max_sync(0xffffffffu, m);
      if ((threadIdx.x & 31u) == 0u) red[threadIdx.x >> 5] = m;
      __syncthreads();
      for (int w = 0; w < 8; ++w) m = max(m, red[w]);
      __syncthreads();
      s = int8_scale(m);
    }
    for (int32_t j = 0; j < p.k; ++j) {
      const int64_t slot = p.slots != nullptr ? p.slots[t * p.k + j] : t;
      if (slot < 0 || slot >= p.num_rows) continue;
      OutT* out = static_cast<OutT*>(p.rows) + slot * p.ldr;
      for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
        if constexpr (kQuant) {
          out[c] = static_cast<OutT>(int8_quotient(RowVec<T>::load(x + c), s));
        } else {
          out[c] = x[c];
        }
      }
      if (kQuant && threadIdx.x == 0) p.scales[slot] = s;
    }
  }
}

struct CombineParams {
  const void* rows;
  int64_t num_rows, cols, ldr;
  const int32_t* slots;  // [tokens][k]
  const float* weights;  // [tokens][k], NULL: ones
  int64_t tokens;
  int32_t k;
  const void* source;  // optional [tokens][cols]
  int64_t lds;
  void* y;
  int64_t ldy;
};

// y[t] = source[t] + sum_j w[t][j] rows[slot[t][j]], summed in fp32 in the order of j.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
      float acc = p.source != nullptr
                      ? RowVec<T>::load(static_cast<const T*>(p.source) + t * p.lds + c)
                      : 0.f;
      for (int32_t j = 0; j < p.k; ++j) {
        const int64_t slot = p.slots[t * p.k + j];
        if (slot < 0 || slot >= p.num_rows) continue;
        const float w = p.weights != nullptr ? p.weights[t * p.k + j] : 1.f;
        acc = fmaf(w, RowVec<T>::load(static_cast<const T*>(p.rows) + slot * p.ldr + c), acc);
      }
      RowVec<T>::store(static_cast<T*>(p.y) + t * p.ldy + c, acc);
    }
  }
}

struct CombineGradParams {
  const void* dy;
  int64_t tokens, cols, lddy;
  const void* rows;
  int64_t num_rows, ldr;
  const int32_t* slots;
  const float* weights;
  int32_t k;
  void* drows;
  int64_t lddr;
  float* dweights;
};

// drows[slot] = w dy[t] and dw[t][j] = <dy[t], rows[slot]>: one warp per (token, choice).
template <typename T>
__global__ void __launch_bounds__(256) combine_grad_kernel(const CombineGradParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t pairs = p.tokens * p.k;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5);
       i < pairs; i += stride) {
    const int64_t slot = p.slots[i];
    float dot = 0.f;
    if (slot >= 0 && slot < p.num_rows) {
      const float w = p.weights[i];
      const T* dy = static_cast<const T*>(p.dy) + (i / p.k) * p.lddy;
      const T* row = static_cast<const T*>(p.rows) + slot * p.ldr;
      T* out = static_cast<T*>(p.drows) + slot * p.lddr;
      for (int64_t c = lane; c < p.cols; c += 32) {
        const float g = RowVec<T>::load(dy + c);
        dot = fmaf(g, RowVec<T>::load(row + c), dot);
        RowVec<T>::store(out + c, w * g);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    if (lane == 0) p.dweights[i] = dot;
  }
}

}  // namespace cpg
