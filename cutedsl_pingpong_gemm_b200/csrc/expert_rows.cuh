// Row kernels around the experts' products: rows quantised to INT8 (a scale per row), rows copied
// into expert order (dispatch), the weighted sums back (combine) and the gradient of those sums.
//
// All of them move whole rows and are bound by HBM; each row of the input is read once.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cpg {

// The first statement of every kernel here: the previous kernel's writes are visible after it.  (All
// but the INT8 row kernels are launched as programmatic dependents, so they may be set up while
// that kernel finishes; for the others it returns at once.)
__device__ __forceinline__ void kernel_begins() { ptx::griddep_wait(); }

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

// ---------------------------------------------------------------- rows of whole vectors
// The vector kernels need rows that start on 16 bytes (input and output) and fewer than 2^30
// columns; the last vector of a row may be partial.  Loads bypass L1 (every row is read once).
__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// The first n elements (any n) at p as a vector, zeros after them.
template <typename T>
__device__ __forceinline__ uint4 ld_tail_v4(const T* p, int32_t n) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) w[j >> 1] |= static_cast<uint32_t>(__bfloat16_as_ushort(p[j])) << (16 * (j & 1));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) w[j] = __float_as_uint(p[j]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Elements [c, c + kElems) of a row of `cols` elements, zeros past its end.
template <typename T>
__device__ __forceinline__ uint4 ld_row_vec(const T* row, int32_t c, int32_t cols) {
  if (c + RowVec<T>::kElems <= cols) return ld_stream_v4(row + c);
  return ld_tail_v4(row + c, cols - c);
}

template <typename T>
__device__ __forceinline__ void st_row_vec(T* row, int32_t c, int32_t cols, const uint4& v) {
  if (c + RowVec<T>::kElems <= cols) {
    ptx::st_global_v4(row + c, v.x, v.y, v.z, v.w);
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < RowVec<T>::kElems; ++j) {
    if (c + j < cols) {
      if constexpr (sizeof(T) == 2)
        row[c + j] = __ushort_as_bfloat16(static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1))));
      else
        row[c + j] = __uint_as_float(w[j]);
    }
  }
}

// The largest |value| seen, as bits: of FP32 one word, of BF16 one maximum per half word.
template <typename T>
__device__ __forceinline__ uint32_t abs_max_vec(const uint4& v, uint32_t m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = sizeof(T) == 2 ? __vmaxu2(m, w[i] & 0x7fff7fffu) : max(m, w[i] & 0x7fffffffu);
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t abs_max_bits(uint32_t m) {
  return sizeof(T) == 2 ? max(m << 16, m & 0xffff0000u) : m;
}

// Four quotients x / s by IEEE division, rounded to integers, as the bytes of a word.
__device__ __noinline__ uint32_t int8_word_div(float x0, float x1, float x2, float x3, float s) {
  return int8_quotient(x0, s) | (int8_quotient(x1, s) << 8) | (int8_quotient(x2, s) << 16) |
         (int8_quotient(x3, s) << 24);
}

// x y rounded to integers (nearest even, left in the low bytes of r0 and r1) and what the rounding
// took away (d0, d1), two elements per packed FMA.  Adding 1.5 * 2^23 rounds to an integer.
__device__ __forceinline__ void round2(float x0, float x1, float y, uint32_t& r0, uint32_t& r1,
                                       float& d0, float& d1) {
  asm("{\n\t.reg .b64 x, y, k, r, u, d;\n\t"
      "mov.b64 x, {%4, %5};\n\t"
      "mov.b64 y, {%6, %6};\n\t"
      "mov.b64 k, {%7, %7};\n\t"
      "mov.b64 u, {%8, %8};\n\t"
      "fma.rn.f32x2 r, x, y, k;\n\t"   // k + rint(x y)
      "fma.rn.f32x2 u, r, u, k;\n\t"   // -rint(x y), exact
      "fma.rn.f32x2 d, x, y, u;\n\t"
      "mov.b64 {%0, %1}, r;\n\t"
      "mov.b64 {%2, %3}, d;\n\t}"
      : "=r"(r0), "=r"(r1), "=f"(d0), "=f"(d1)
      : "f"(x0), "f"(x1), "f"(y), "f"(12582912.f), "f"(-1.f));
}

// The same without a division per element.  With y = RN(1 / s), x y is within 127 * 2^-24 < 7.6e-6
// of x / s, and the fp32 quotient within half an ulp, 2^-18 < 3.9e-6, of it; so where x y is farther
// than 4e-5 from a half-integer both round to the same integer, and elsewhere (about 1e-4 of the
// elements) the word takes the division.
__device__ __forceinline__ uint32_t int8_word(const float* x, float s, float y) {
  uint32_t b[4];
  float d[4];
  round2(x[0], x[1], y, b[0], b[1], d[0], d[1]);
  round2(x[2], x[3], y, b[2], b[3], d[2], d[3]);
  const float worst = fmaxf(fmaxf(fabsf(d[0]), fabsf(d[1])), fmaxf(fabsf(d[2]), fabsf(d[3])));
  if (worst > 0.5f - 4e-5f) return int8_word_div(x[0], x[1], x[2], x[3], s);
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// Sixteen consecutive elements as INT8 (rows of a NaN scale: zeros).
template <typename T>
__device__ __forceinline__ uint4 int8_vec(const uint4* raw, float s, float y) {
  constexpr int kVecs = 16 / RowVec<T>::kElems;
  float f[16];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) RowVec<T>::unpack(raw[i], f + i * RowVec<T>::kElems);
  if (s != s) return make_uint4(0u, 0u, 0u, 0u);
  return make_uint4(int8_word(f, s, y), int8_word(f + 4, s, y), int8_word(f + 8, s, y),
                    int8_word(f + 12, s, y));
}

__device__ __forceinline__ void st_int8_vec(int8_t* row, int32_t c, int32_t cols, const uint4& v) {
  if (c + 16 <= cols) {
    ptx::st_global_v4(row + c, v.x, v.y, v.z, v.w);
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (c + j < cols) row[c + j] = static_cast<int8_t>(w[j >> 2] >> (8 * (j & 3)));
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
  kernel_begins();
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

// Quantised rows of whole vectors: G threads per token hold the row packed in registers, NV times 16
// elements each, between its maximum and the quantisation, so the row is read once however many
// copies of it are written.  Longer rows (Resident false) are read a second time, from L2.
constexpr int kInt8Vecs = 2;

template <int G>
__host__ __device__ constexpr int int8_threads() {
  return G < 256 ? 256 : G;
}
// Threads per SM the registers are limited for.
template <typename T, int NV>
__host__ __device__ constexpr int int8_sm_threads() {
  return NV == kInt8Vecs ? (sizeof(T) == 2 ? 1536 : 1024) : (sizeof(T) == 2 ? 1024 : 512);
}

template <typename T, int G, int NV, bool Resident>
__global__ void __launch_bounds__(int8_threads<G>(), int8_sm_threads<T, NV>() / int8_threads<G>())
    rows_int8_vec_kernel(const RowsParams p) {
  // The small-M product that reads these rows may be set up, and fetch its first weights, already.
  ptx::griddep_launch_dependents();
  kernel_begins();
  constexpr int kVecs = 16 / RowVec<T>::kElems;
  constexpr int kE = RowVec<T>::kElems;
  constexpr int kRowsPerBlock = int8_threads<G>() / G;
  constexpr int kPass = G * NV * 16;  // elements per pass over a row
  __shared__ uint32_t red[2][int8_threads<G>() / 32];
  const int lane = threadIdx.x & 31;
  const int li = threadIdx.x % G;
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowsPerBlock;
  int parity = 0;
  for (int64_t t = blockIdx.x * static_cast<int64_t>(kRowsPerBlock) + threadIdx.x / G;
       t < p.tokens; t += step) {
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    uint4 raw[NV][kVecs];
    auto load = [&](int32_t c0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int32_t c = c0 + (i * G + li) * 16;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          raw[i][v] = make_uint4(0u, 0u, 0u, 0u);
          if (c + v * kE < cols) raw[i][v] = ld_row_vec(x, c + v * kE, cols);
        }
      }
    };
    uint32_t m = 0u;
    for (int32_t c0 = 0; c0 < cols; c0 += kPass) {
      load(c0);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int v = 0; v < kVecs; ++v) m = abs_max_vec<T>(raw[i][v], m);
      if constexpr (Resident) break;
    }
    // Slots of this token: lane j of every warp holds choice j.
    int32_t my_slot = -1;
    if (lane < p.k) my_slot = p.slots != nullptr ? p.slots[t * p.k + lane] : static_cast<int32_t>(t);
    if (my_slot >= p.num_rows) my_slot = -1;
    m = __reduce_max_sync(0xffffffffu, abs_max_bits<T>(m));
    if constexpr (G > 32) {
      // The parity keeps the next row's writes off the words a slow warp still reads.
      constexpr int kWarps = G / 32;
      const int first = (threadIdx.x / G) * kWarps;
      if (lane == 0) red[parity][threadIdx.x >> 5] = m;
      ptx::named_barrier_sync(1u + threadIdx.x / G, G);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = max(m, red[parity][first + w]);
      parity ^= 1;
    }
    const float s = int8_scale(m);
    const float y = __frcp_rn(s);
    for (int32_t c0 = 0; c0 < cols; c0 += kPass) {
      if constexpr (!Resident) load(c0);
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i][0] = int8_vec<T>(raw[i], s, y);
      for (int32_t j = 0; j < p.k; ++j) {
        const int32_t slot = __shfl_sync(0xffffffffu, my_slot, j);
        if (slot < 0) continue;
        int8_t* out = static_cast<int8_t*>(p.rows) + slot * p.ldr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int32_t c = c0 + (i * G + li) * 16;
          if (c < cols) st_int8_vec(out, c, cols, raw[i][0]);
        }
      }
      if constexpr (Resident) break;
    }
    if (li < p.k && my_slot >= 0) p.scales[my_slot] = s;
  }
}

// Copied rows of whole vectors: a warp takes 32 * kCopyVecs vectors of one token and writes them
// k times.
constexpr int kCopyVecs = 4;

template <typename T>
__global__ void __launch_bounds__(256) rows_copy_vec_kernel(const RowsParams p, int32_t chunks) {
  kernel_begins();
  constexpr int kE = RowVec<T>::kElems;
  const int lane = threadIdx.x & 31;
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int64_t units = p.tokens * chunks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < units; u += step) {
    const int64_t t = u / chunks;
    const int32_t c0 = static_cast<int32_t>((u - t * chunks) * 32 * kCopyVecs + lane) * kE;
    int64_t my_slot = -1;
    if (lane < p.k) my_slot = p.slots[t * p.k + lane];
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    uint4 raw[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i) {
      const int32_t c = c0 + i * 32 * kE;
      if (c < cols) raw[i] = ld_row_vec(x, c, cols);
    }
    for (int32_t j = 0; j < p.k; ++j) {
      const int64_t slot = __shfl_sync(0xffffffffu, my_slot, j);
      if (slot < 0 || slot >= p.num_rows) continue;
      T* out = static_cast<T*>(p.rows) + slot * p.ldr;
#pragma unroll
      for (int i = 0; i < kCopyVecs; ++i) {
        const int32_t c = c0 + i * 32 * kE;
        if (c < cols) st_row_vec(out, c, cols, raw[i]);
      }
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
  kernel_begins();
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

// As combine_kernel for rows of whole vectors: a warp takes 32 * kCombineVecs vectors of one token
// and keeps the loads of four choices in flight.  Every output element sums its choices in the
// same order as combine_kernel.
constexpr int kCombineVecs = 2;

template <typename T>
__global__ void __launch_bounds__(256) combine_vec_kernel(const CombineParams p, int32_t chunks) {
  kernel_begins();
  constexpr int kE = RowVec<T>::kElems;
  constexpr int kBatch = 4;
  const int lane = threadIdx.x & 31;
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int64_t units = p.tokens * chunks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < units; u += step) {
    const int64_t t = u / chunks;
    const int32_t c0 = static_cast<int32_t>((u - t * chunks) * 32 * kCombineVecs + lane) * kE;
    int64_t my_slot = -1;
    float my_w = 1.f;
    if (lane < p.k) {
      my_slot = p.slots[t * p.k + lane];
      if (p.weights != nullptr) my_w = p.weights[t * p.k + lane];
    }
    if (my_slot >= p.num_rows) my_slot = -1;
    float acc[kCombineVecs][kE];
#pragma unroll
    for (int i = 0; i < kCombineVecs; ++i) {
      const int32_t c = c0 + i * 32 * kE;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (p.source != nullptr && c < cols) {
        // The source may be y itself, so it is not a read-only load.
        const T* src = static_cast<const T*>(p.source) + t * p.lds + c;
        v = c + kE <= cols ? *reinterpret_cast<const uint4*>(src)
                             : ld_tail_v4(src, cols - c);
      }
      RowVec<T>::unpack(v, acc[i]);
    }
    for (int32_t j0 = 0; j0 < p.k; j0 += kBatch) {
      uint4 raw[kBatch][kCombineVecs];
      int64_t slot[kBatch];
      float w[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        // Lanes past k hold slot -1.
        slot[b] = __shfl_sync(0xffffffffu, my_slot, (j0 + b) & 31);
        w[b] = __shfl_sync(0xffffffffu, my_w, (j0 + b) & 31);
        const T* row = static_cast<const T*>(p.rows) + slot[b] * p.ldr;
#pragma unroll
        for (int i = 0; i < kCombineVecs; ++i) {
          const int32_t c = c0 + i * 32 * kE;
          if (slot[b] >= 0 && c < cols) raw[b][i] = ld_row_vec(row, c, cols);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (slot[b] < 0) continue;
#pragma unroll
        for (int i = 0; i < kCombineVecs; ++i) {
          float f[kE];
          RowVec<T>::unpack(raw[b][i], f);
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[i][e] = fmaf(w[b], f[e], acc[i][e]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kCombineVecs; ++i) {
      const int32_t c = c0 + i * 32 * kE;
      if (c < cols)
        st_row_vec(static_cast<T*>(p.y) + t * p.ldy, c, cols, RowVec<T>::pack(acc[i]));
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
  kernel_begins();
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

// As combine_grad_kernel for rows of whole vectors, four vectors of dy and of the row in flight.
template <typename T>
__global__ void __launch_bounds__(256) combine_grad_vec_kernel(const CombineGradParams p) {
  kernel_begins();
  constexpr int kE = RowVec<T>::kElems;
  constexpr int kVecs = 4;
  const int lane = threadIdx.x & 31;
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int64_t pairs = p.tokens * p.k;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < pairs; u += step) {
    const int64_t slot = p.slots[u];
    float dot = 0.f;
    if (slot >= 0 && slot < p.num_rows) {
      const float w = p.weights[u];
      const T* dy = static_cast<const T*>(p.dy) + (u / p.k) * p.lddy;
      const T* row = static_cast<const T*>(p.rows) + slot * p.ldr;
      T* out = static_cast<T*>(p.drows) + slot * p.lddr;
      for (int32_t c0 = lane * kE; c0 < cols; c0 += 32 * kE * kVecs) {
        uint4 g[kVecs], r[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int32_t c = c0 + i * 32 * kE;
          g[i] = r[i] = make_uint4(0u, 0u, 0u, 0u);
          if (c < cols) {
            g[i] = ld_row_vec(dy, c, cols);
            r[i] = ld_row_vec(row, c, cols);
          }
        }
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int32_t c = c0 + i * 32 * kE;
          float gf[kE], rf[kE];
          RowVec<T>::unpack(g[i], gf);
          RowVec<T>::unpack(r[i], rf);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            dot = fmaf(gf[e], rf[e], dot);
            gf[e] *= w;
          }
          if (c < cols) st_row_vec(out, c, cols, RowVec<T>::pack(gf));
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    if (lane == 0) p.dweights[u] = dot;
  }
}

}  // namespace cpg
