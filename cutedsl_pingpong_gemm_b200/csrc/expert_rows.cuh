// Row kernels around the experts' products: rows quantised to INT8 (a scale per row), rows copied
// into expert order (dispatch), the weighted sums back (combine) and the gradient of those sums.
//
// All of them move whole rows and are bound by HBM; each row of the input is read once.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace cpg {

// Before the first access of every kernel here: the previous kernel's writes are visible after it.
// (All but the INT8 row kernels are launched as programmatic dependents, so they may be set up while
// that kernel finishes.  For the INT8 kernels it returns at once; they let the next kernel in first.)
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
  __device__ __forceinline__ static float load(const __nv_bfloat16* p) {
    return __bfloat162float(*p);
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
  __device__ __forceinline__ static float load(const float* p) { return *p; }
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
// Rows that start on 16 bytes and have fewer than 2^30 columns; the last vector of a row may be
// partial.  Loads bypass L1 (every row is read once).
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

// Accesses a lane has in flight where 16-byte ones have n: as many bytes, at most 8 of them.
template <int W>
__host__ __device__ constexpr int row_accesses(int n) {
  return n * (16 / W) < 8 ? n * (16 / W) : (n > 8 ? n : 8);
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

// Quantised rows whose INT8 rows do not start on 16 bytes: rows[slot] = q and scales[slot] = s of x[t]
// for the k slots of every token, q = rint(x / s), s = max|x[t]| / 127; one block per token, the row
// read twice.
template <typename T>
__global__ void __launch_bounds__(256) rows_int8_kernel(const RowsParams p) {
  ptx::griddep_launch_dependents();
  kernel_begins();
  __shared__ uint32_t red[8];
  const int lane = threadIdx.x & 31;
  const int32_t cols = static_cast<int32_t>(p.cols);
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    uint32_t m = 0u;
#pragma unroll 4
    for (int32_t c = threadIdx.x; c < cols; c += 256) m = max(m, abs_bits(RowVec<T>::load(x + c)));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < 8; ++w) m = max(m, red[w]);
    __syncthreads();
    const float s = int8_scale(m);
    int32_t my_slot = -1;
    if (lane < p.k) my_slot = p.slots != nullptr ? p.slots[t * p.k + lane] : static_cast<int32_t>(t);
    if (my_slot >= p.num_rows) my_slot = -1;
    const int32_t turns = (cols + 255) / 256;  // the same for every lane: the slots are shuffled
#pragma unroll 2
    for (int32_t i = 0; i < turns; ++i) {
      const int32_t c = i * 256 + static_cast<int32_t>(threadIdx.x);
      int8_t q = 0;
      if (c < cols) q = static_cast<int8_t>(int8_quotient(RowVec<T>::load(x + c), s));
      for (int32_t j = 0; j < p.k; ++j) {
        const int32_t slot = __shfl_sync(0xffffffffu, my_slot, j);
        if (slot >= 0 && c < cols) static_cast<int8_t*>(p.rows)[slot * p.ldr + c] = q;
      }
    }
    if (threadIdx.x < static_cast<unsigned>(p.k) && my_slot >= 0) p.scales[my_slot] = s;
  }
}

// 16 elements of a row from c on as vectors, zeros past its end, read by accesses of W bytes.
// Narrow ones go out without a branch between them; lanes share their sectors through L1.
template <typename T, int W>
__device__ __forceinline__ void ld_16(const T* x, int32_t c, int32_t cols,
                                      uint4 (&raw)[16 / RowVec<T>::kElems]) {
  constexpr int kE = RowVec<T>::kElems;
  constexpr int kVecs = 16 / kE;
  if constexpr (W == 16) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      raw[v] = make_uint4(0u, 0u, 0u, 0u);
      if (c + v * kE < cols) raw[v] = ld_row_vec(x, c + v * kE, cols);
    }
  } else {
    using A = RowAccess<T, W>;
    constexpr int kN = 16 / A::kElems;
    uint32_t w[4 * kVecs];
#pragma unroll
    for (int i = 0; i < 4 * kVecs; ++i) w[i] = 0u;
    auto place = [&](int a, const typename A::Data& d) {
      if constexpr (W == 2) {
        w[a >> 1] |= d.w[0] << (16 * (a & 1));
      } else {
#pragma unroll
        for (int i = 0; i < A::kWords; ++i) w[a * A::kWords + i] = d.w[i];
      }
    };
    if (c + 16 <= cols) {
      typename A::Data d[kN];
#pragma unroll
      for (int a = 0; a < kN; ++a) d[a] = A::template load_all<true>(x + c + a * A::kElems);
#pragma unroll
      for (int a = 0; a < kN; ++a) place(a, d[a]);
    } else if (c < cols) {
#pragma unroll
      for (int a = 0; a < kN; ++a)
        if (c + a * A::kElems < cols) place(a, A::template load<true>(x, c + a * A::kElems, cols));
    }
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
      raw[v] = make_uint4(w[4 * v], w[4 * v + 1], w[4 * v + 2], w[4 * v + 3]);
  }
}

// Quantised rows stored by whole vectors: G threads per token hold the row packed in registers, NV times 16
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

template <typename T, int W, int G, int NV, bool Resident>
__global__ void __launch_bounds__(int8_threads<G>(), int8_sm_threads<T, NV>() / int8_threads<G>())
    rows_int8_vec_kernel(const RowsParams p) {
  // The small-M product that reads these rows may be set up, and fetch its first weights, already.
  ptx::griddep_launch_dependents();
  kernel_begins();
  constexpr int kVecs = 16 / RowVec<T>::kElems;
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
        ld_16<T, W>(x, c0 + (i * G + li) * 16, cols, raw[i]);
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

// Copied rows: a warp takes 32 x row_accesses(kCopyVecs) accesses of one token and writes them k times.
constexpr int kCopyVecs = 4;

template <typename T, int W>
__global__ void __launch_bounds__(256) rows_copy_kernel(const RowsParams p, int32_t chunks) {
  kernel_begins();
  using A = RowAccess<T, W>;
  constexpr int kN = row_accesses<W>(kCopyVecs);
  const int lane = threadIdx.x & 31;
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int64_t units = p.tokens * chunks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < units; u += step) {
    const int64_t t = u / chunks;
    const int32_t c0 = static_cast<int32_t>((u - t * chunks) * 32 * kN + lane) * A::kElems;
    int64_t my_slot = -1;
    if (lane < p.k) my_slot = p.slots[t * p.k + lane];
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    typename A::Data raw[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int32_t c = c0 + i * 32 * A::kElems;
      if (c < cols) raw[i] = A::template load<true>(x, c, cols);
    }
    for (int32_t j = 0; j < p.k; ++j) {
      const int64_t slot = __shfl_sync(0xffffffffu, my_slot, j);
      if (slot < 0 || slot >= p.num_rows) continue;
      T* out = static_cast<T*>(p.rows) + slot * p.ldr;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int32_t c = c0 + i * 32 * A::kElems;
        if (c < cols) A::store(out, c, cols, raw[i]);
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

// y[t] = source[t] + sum_j w[t][j] rows[slot[t][j]], summed in fp32 in the order of j.  A warp takes
// 32 x combine_accesses() accesses of one token and keeps the loads of four choices in flight.
// Three blocks a SM: without that bound BF16 takes 113 registers, and 16-byte rows of 2048 columns
// (8192 tokens, 4 choices) 36.4 us for 29.8.  Accesses of one element come four at a time: 69 us with
// 2049 BF16 columns, 77 with eight; with two elements (2050 columns) eight are the faster, 50 for 58.
constexpr int kCombineVecs = 2;
template <typename T, int W>
__host__ __device__ constexpr int combine_accesses() {
  return W == static_cast<int>(sizeof(T)) ? 4 : row_accesses<W>(kCombineVecs);
}

template <typename T, int W>
__global__ void __launch_bounds__(256, 3) combine_kernel(const CombineParams p, int32_t chunks) {
  kernel_begins();
  using A = RowAccess<T, W>;
  constexpr int kE = A::kElems;
  constexpr int kN = combine_accesses<T, W>();
  constexpr int kBatch = 4;
  const int lane = threadIdx.x & 31;
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int64_t units = p.tokens * chunks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t u = blockIdx.x * 8ll + (threadIdx.x >> 5); u < units; u += step) {
    const int64_t t = u / chunks;
    const int32_t c0 = static_cast<int32_t>((u - t * chunks) * 32 * kN + lane) * kE;
    int64_t my_slot = -1;
    float my_w = 1.f;
    if (lane < p.k) {
      my_slot = p.slots[t * p.k + lane];
      if (p.weights != nullptr) my_w = p.weights[t * p.k + lane];
    }
    if (my_slot >= p.num_rows) my_slot = -1;
    float acc[kN][kE];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int32_t c = c0 + i * 32 * kE;
      typename A::Data v = A::zero();
      // The source may be y itself, so it is not a read-only load.
      if (p.source != nullptr && c < cols)
        v = A::template load<false>(static_cast<const T*>(p.source) + t * p.lds, c, cols);
      A::unpack(v, acc[i]);
    }
    for (int32_t j0 = 0; j0 < p.k; j0 += kBatch) {
      typename A::Data raw[kBatch][kN];
      int64_t slot[kBatch];
      float w[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        // Lanes past k hold slot -1.
        slot[b] = __shfl_sync(0xffffffffu, my_slot, (j0 + b) & 31);
        w[b] = __shfl_sync(0xffffffffu, my_w, (j0 + b) & 31);
        const T* row = static_cast<const T*>(p.rows) + slot[b] * p.ldr;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const int32_t c = c0 + i * 32 * kE;
          if (slot[b] < 0) continue;
          if constexpr (kE == 1)
            // Without a branch, a lane past the end loads the last element: the loads go out
            // together (with it they took 106 us where these take 69).
            raw[b][i] = A::template load_all<true>(row + min(c, cols - 1));
          else if (c < cols)
            raw[b][i] = A::template load<true>(row, c, cols);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (slot[b] < 0) continue;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          float f[kE];
          A::unpack(raw[b][i], f);
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[i][e] = fmaf(w[b], f[e], acc[i][e]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int32_t c = c0 + i * 32 * kE;
      if (c < cols)
        A::store(static_cast<T*>(p.y) + t * p.ldy, c, cols, A::pack(acc[i]));
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

// drows[slot] = w dy[t] and dw[t][j] = <dy[t], rows[slot]>: one warp per (token, choice), with
// row_accesses(kGradVecs) accesses of dy and of the row in flight per lane.
constexpr int kGradVecs = 4;

template <typename T, int W>
__global__ void __launch_bounds__(256) combine_grad_kernel(const CombineGradParams p) {
  kernel_begins();
  using A = RowAccess<T, W>;
  constexpr int kE = A::kElems;
  constexpr int kVecs = row_accesses<W>(kGradVecs);
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
        typename A::Data g[kVecs], r[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int32_t c = c0 + i * 32 * kE;
          g[i] = r[i] = A::zero();
          if (c < cols) {
            g[i] = A::template load<true>(dy, c, cols);
            r[i] = A::template load<true>(row, c, cols);
          }
        }
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const int32_t c = c0 + i * 32 * kE;
          float gf[kE], rf[kE];
          A::unpack(g[i], gf);
          A::unpack(r[i], rf);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            dot = fmaf(gf[e], rf[e], dot);
            gf[e] *= w;
          }
          if (c < cols) A::store(out, c, cols, A::pack(gf));
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    if (lane == 0) p.dweights[u] = dot;
  }
}

struct ClearRowsParams {
  void* rows;
  int64_t num_rows, cols, ldr;
  const int32_t* slots;
  int64_t pairs;
  int32_t per_block;  // rows of a block, a multiple of 32
};

// Zeros in the rows that no slot names.  Every block walks all slots and marks those of its own rows
// in shared memory, so there is no workspace and no order to wait for; the slots stay in L2.  For
// 16382 rows x 4096 BF16, all named, it costs 5 us beside a gradient of 54, clearing them all 35.
constexpr int kClearThreads = 1024;
constexpr int32_t kClearMaxRows = 1 << 18;  // of a block: 32 KB of marks

template <typename T, int W>
__global__ void __launch_bounds__(kClearThreads) rows_clear_kernel(const ClearRowsParams p) {
  kernel_begins();
  using A = RowAccess<T, W>;
  extern __shared__ uint32_t named[];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.per_block;
  const int64_t left = p.num_rows - first;
  const int32_t count = left < p.per_block ? static_cast<int32_t>(left) : p.per_block;
  for (int32_t i = threadIdx.x; i < p.per_block / 32; i += kClearThreads) named[i] = 0u;
  __syncthreads();
  constexpr int kBatch = 8;  // slots a thread loads before it marks the first
  for (int64_t i0 = threadIdx.x; i0 < p.pairs; i0 += kBatch * kClearThreads) {
    int32_t slot[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t i = i0 + u * kClearThreads;
      slot[u] = i < p.pairs ? p.slots[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t r = slot[u] - first;
      if (r >= 0 && r < count) atomicOr(named + (r >> 5), 1u << (r & 31));
    }
  }
  __syncthreads();
  const int32_t cols = static_cast<int32_t>(p.cols);
  const int lane = threadIdx.x & 31;
  for (int32_t r = threadIdx.x >> 5; r < count; r += kClearThreads / 32) {
    if ((named[r >> 5] >> (r & 31)) & 1u) continue;
    T* row = static_cast<T*>(p.rows) + (first + r) * p.ldr;
    for (int32_t c = lane * A::kElems; c < cols; c += 32 * A::kElems)
      A::store(row, c, cols, A::zero());
  }
}

}  // namespace cpg
