// Shared by the operators that move or sum rows picked by index (embedding.cu,
// experts.cu) and by clip.cu: element conversion, vectors of V elements, the
// argument checks of DcopyMatrix, and the row x column split of a grid.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"

namespace dcopy {

// GE DataType values of the element types these operators take.
constexpr int32_t kF32 = 0, kF16 = 1, kI8 = 2, kI32 = 3, kU8 = 4, kI64 = 9, kBF16 = 27;

inline int elem_size(int32_t type) {
  switch (type) {
    case kF32: case kI32: return 4;
    case kF16: case kBF16: return 2;
    case kI64: return 8;
    case kI8: case kU8: return 1;
    default: return 0;
  }
}
inline bool is_float(int32_t type) { return type == kF32 || type == kF16 || type == kBF16; }
inline bool is_index(int32_t type) { return type == kI32 || type == kI64; }

// Widths beyond this are refused: the column split is the grid's y dimension.
constexpr int64_t kMaxWidth = 1 << 24;

// Shape, pitch, type and span of one matrix argument.  `ok` tells whether the
// type is one the operator takes.
inline int check_matrix(const DcopyMatrix *m, const char *name, bool ok) {
  if (!ok)
    return set_error(DCOPY_ERR_DATATYPE_INVALID, "%s: element type %d is not supported", name,
                     m->type);
  if (m->rows < 0 || m->cols < 0 || m->rows > INT32_MAX || m->cols > INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "%s: %lld x %lld elements", name,
                     (long long)m->rows, (long long)m->cols);
  if (m->rows == 0 || m->cols == 0) return DCOPY_OK;
  if (m->rows > 1 && m->pitch < m->cols)
    return set_error(DCOPY_ERR_PARAM_INVALID, "%s: pitch %lld is less than %lld columns", name,
                     (long long)m->pitch, (long long)m->cols);
  const int eb = elem_size(m->type);
  uint64_t span = 0;
  const int rc = block_span((uint64_t)m->rows, (uint64_t)(m->rows > 1 ? m->pitch : 0) * eb,
                            (uint64_t)m->cols * eb, &span, name);
  if (rc) return rc;
  if (reinterpret_cast<uintptr_t>(m->data) % eb)
    return set_error(DCOPY_ERR_PARAM_INVALID, "%s (%p) is not aligned to its %d-byte elements",
                     name, m->data, eb);
  return check_device_span(m->data, span, name);
}

// Bytes from the first to the last element of a matrix that check_matrix passed.
inline uint64_t matrix_span(const DcopyMatrix *m) {
  if (m->rows == 0 || m->cols == 0) return 0;
  return ((uint64_t)(m->rows - 1) * (m->rows > 1 ? m->pitch : 0) + m->cols) * elem_size(m->type);
}

inline int check_apart(const DcopyMatrix *a, const DcopyMatrix *b, const char *what) {
  return check_disjoint(a->data, matrix_span(a), b->data, matrix_span(b), what);
}

// Largest V in {8, 4, 2, 1} of at most 16 bytes for which a row of the matrix is whole
// vectors of V elements that start on the vector's own alignment.
inline int vector_width(const DcopyMatrix *m) {
  const int eb = elem_size(m->type);
  for (int v = 16 / eb; v > 1; v /= 2) {
    if (m->cols % v == 0 && reinterpret_cast<uintptr_t>(m->data) % (v * eb) == 0 &&
        (m->rows <= 1 || (uint64_t)m->pitch * eb % (v * eb) == 0))
      return v;
  }
  return 1;
}

// ---- device ---------------------------------------------------------------------

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float to(uint32_t bits) { return __uint_as_float(bits); }
  static __device__ __forceinline__ uint32_t from(float f) { return __float_as_uint(f); }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float to(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
  static __device__ __forceinline__ uint32_t from(float f) {
    return __half_as_ushort(__float2half_rn(f));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to(uint32_t bits) {
    return __uint_as_float(bits << 16);
  }
  static __device__ __forceinline__ uint32_t from(float f) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  }
};

// N bytes as 32-bit words (one word for 1 and 2 bytes), moved with the widest
// accesses that N allows.  `stream` loads take the non-coherent path.
template <int N>
struct Words {
  static constexpr int kWords = N < 4 ? 1 : N / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const void *p) {
    if constexpr (N >= 16) {
#pragma unroll
      for (int i = 0; i < N / 16; ++i) {
        const uint4 v = ld_stream(reinterpret_cast<const uint4 *>(p) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (N == 8) {
      const uint2 v = ld_stream(reinterpret_cast<const uint2 *>(p));
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (N == 4) {
      w[0] = ld_stream(reinterpret_cast<const uint32_t *>(p));
    } else if constexpr (N == 2) {
      w[0] = ld_stream(reinterpret_cast<const uint16_t *>(p));
    } else {
      w[0] = ld_stream(reinterpret_cast<const uint8_t *>(p));
    }
  }
  // The same through plain loads, for memory that this kernel also writes.
  __device__ __forceinline__ void load_plain(const void *p) {
    if constexpr (N >= 16) {
#pragma unroll
      for (int i = 0; i < N / 16; ++i) {
        const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (N == 8) {
      const uint2 v = *reinterpret_cast<const uint2 *>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (N == 4) {
      w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
      w[0] = *reinterpret_cast<const uint16_t *>(p);
    } else {
      w[0] = *reinterpret_cast<const uint8_t *>(p);
    }
  }
  __device__ __forceinline__ void store(void *p) const {
    if constexpr (N >= 16) {
#pragma unroll
      for (int i = 0; i < N / 16; ++i)
        reinterpret_cast<uint4 *>(p)[i] =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (N == 8) {
      *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (N == 4) {
      *reinterpret_cast<uint32_t *>(p) = w[0];
    } else if constexpr (N == 2) {
      *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0];
    } else {
      *reinterpret_cast<uint8_t *>(p) = (uint8_t)w[0];
    }
  }
  // The same marked as written once and not read soon: L2 evicts it first.
  __device__ __forceinline__ void store_cs(void *p) const {
    if constexpr (N >= 16) {
#pragma unroll
      for (int i = 0; i < N / 16; ++i)
        __stcs(reinterpret_cast<uint4 *>(p) + i,
               make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    } else if constexpr (N == 8) {
      __stcs(reinterpret_cast<uint2 *>(p), make_uint2(w[0], w[1]));
    } else if constexpr (N == 4) {
      __stcs(reinterpret_cast<uint32_t *>(p), w[0]);
    } else if constexpr (N == 2) {
      __stcs(reinterpret_cast<unsigned short *>(p), (unsigned short)w[0]);
    } else {
      __stcs(reinterpret_cast<unsigned char *>(p), (unsigned char)w[0]);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
};

// V elements of type T: words in memory, floats in registers.  get() rounds
// nothing; put() rounds each value once, to nearest even.
template <typename T, int V>
struct Vec : Words<(int)sizeof(T) * V> {
  static constexpr int kSize = V;
  using Words<(int)sizeof(T) * V>::w;
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return Elem<T>::to(w[i]);
    else return Elem<T>::to(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu);
  }
  __device__ __forceinline__ void put(const float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = Elem<T>::from(f[i]);
    } else if constexpr (V == 1) {
      w[0] = Elem<T>::from(f[0]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        w[i] = Elem<T>::from(f[2 * i]) | Elem<T>::from(f[2 * i + 1]) << 16;
    }
  }
};

// ---- the split of rows x vectors over a grid ---------------------------------------
// A block of kRowThreads threads takes (kRowThreads >> lx) rows and, in each, U
// vectors a thread, 1 << lx vectors apart: rows narrower than the block share
// it, wider ones are split over grid.y.

constexpr int kRowThreads = 256;

struct RowSplit {
  int lx;        // log2 of the threads of a row
  dim3 grid;
};

inline RowSplit split_rows(uint64_t rows, uint64_t vectors, int u, int most_rows = kRowThreads) {
  RowSplit s;
  s.lx = 0;
  while (kRowThreads >> s.lx > most_rows) ++s.lx;
  while ((1 << s.lx) < kRowThreads && ((uint64_t)u << s.lx) < vectors) ++s.lx;
  const uint64_t per_block = kRowThreads >> s.lx, step = (uint64_t)u << s.lx;
  s.grid = dim3((unsigned)((rows + per_block - 1) / per_block),
                (unsigned)((vectors + step - 1) / step));
  return s;
}

// Calls f with a value of type std::integral_constant<int, V> for the vector width v
// (as vector_width gives it) of elements of at most kBytes bytes.
template <int kBytes, typename F>
int with_vector(int v, F &&f) {
  if constexpr (kBytes <= 2)
    if (v == 8) return f(std::integral_constant<int, 8>{});
  if (v == 4) return f(std::integral_constant<int, 4>{});
  if (v == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 1>{});
}

// Zeroes `bytes` bytes by the threads `t` of `threads`: 16-byte granules, bytes at the
// ends.
__device__ __forceinline__ void zero_bytes(uint8_t *at, uint64_t bytes, uint32_t t,
                                           uint32_t threads) {
  const uint64_t head = min((uint64_t)(-(uintptr_t)at & 15), bytes);
  const uint64_t units = (bytes - head) / 16, tail = bytes - head - units * 16;
  uint4 *dst = reinterpret_cast<uint4 *>(at + head);
#pragma unroll 4
  for (uint64_t u = t; u < units; u += threads) dst[u] = make_uint4(0, 0, 0, 0);
  if (t < head) at[t] = 0;
  if (t < tail) at[bytes - 1 - t] = 0;
}

template <typename T>
struct TypeTag {
  using type = T;
};
// Calls f with a TypeTag of the float type `type` (checked by the caller).
template <typename F>
int with_float(int32_t type, F &&f) {
  if (type == kF32) return f(TypeTag<float>{});
  if (type == kF16) return f(TypeTag<__half>{});
  return f(TypeTag<__nv_bfloat16>{});
}

}  // namespace dcopy
