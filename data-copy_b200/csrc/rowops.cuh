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
#include "shift.cuh"

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
constexpr int64_t kMaxWidth = 1 << 23;

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

// `count` elements of a type, aligned to it.
inline int check_array(const void *data, uint64_t count, uint64_t elem_bytes, const char *name) {
  if (count && (uintptr_t)data % elem_bytes)
    return set_error(DCOPY_ERR_PARAM_INVALID, "%s (%p) is not aligned to its %d-byte elements",
                     name, data, (int)elem_bytes);
  return check_device_span(data, count * elem_bytes, name);
}

// Whether no byte belongs to rows of both.  Rows of one pitch may interleave, as column
// slices of one buffer do.
inline bool apart(const DcopyMatrix *a, const DcopyMatrix *b) {
  const uintptr_t pa = (uintptr_t)a->data, pb = (uintptr_t)b->data;
  const uint64_t na = matrix_span(a), nb = matrix_span(b);
  if (!na || !nb || pa >= pb + nb || pb >= pa + na) return true;
  const uint64_t ea = elem_size(a->type), eb = elem_size(b->type);
  const uint64_t step_a = a->rows > 1 ? a->pitch * ea : 0, step_b = b->rows > 1 ? b->pitch * eb : 0;
  const uint64_t step = step_a ? step_a : step_b;
  if (!step || (step_b && step_b != step)) return false;
  const uint64_t at = pb >= pa ? (pb - pa) % step : (step - (pa - pb) % step) % step;
  return at >= a->cols * ea && at + b->cols * eb <= step;
}

inline int check_apart(const DcopyMatrix *a, const DcopyMatrix *b, const char *what,
                       const char *name_a, const char *name_b) {
  if (apart(a, b)) return DCOPY_OK;
  return set_error(DCOPY_ERR_PARAM_INVALID, "%s: %s and %s overlap", what, name_a, name_b);
}

// Whether b is a itself.
inline bool same_rows(const DcopyMatrix *a, const DcopyMatrix *b) {
  return a->data == b->data && a->type == b->type && a->rows == b->rows && a->cols == b->cols &&
         (a->rows <= 1 || a->pitch == b->pitch);
}

// An array as a matrix of one row; NULL is empty.
inline DcopyMatrix flat(const void *data, uint64_t count, int32_t type) {
  return DcopyMatrix{const_cast<void *>(data), 1, data ? (int64_t)count : 0, 0, type, 0};
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

// How the rows of an operator's matrices are cut into vectors of V elements.  Where every
// row starts on a vector and is whole vectors, they are accessed as they lie.  Rows for
// which only vectors of few bytes would do are cut at the 16-byte granules of the row that
// is written, and read by pairs of aligned blocks that are shifted together (kShift); the
// operators that gain by it say from which size on.
struct Cut {
  int v;
  bool shift;
};

// full: elements of 16 bytes of the widest type; least: below so many, shift.
template <typename... M>
Cut cut_rows(int full, int least, const M *...m) {
  const int v = std::min({full, vector_width(m)...});
  return v >= least ? Cut{v, false} : Cut{full, true};
}

// Vectors that cover a row: with shifted cuts one more at each end may hold part of it.
inline uint32_t vectors_of(int64_t width, Cut c) {
  return (uint32_t)(c.shift ? (width + 2 * c.v - 2) / c.v : width / c.v);
}

// Calls f(V, kShift) as compile-time constants; kFull and kLeast as in cut_rows.
template <int kV, int kLeast, typename F>
int with_vector(int v, F &&f) {
  if constexpr (kV / 2 >= kLeast && kV > 1)
    if (v < kV) return with_vector<kV / 2, kLeast>(v, f);
  return f(std::integral_constant<int, kV>{}, std::false_type{});
}
template <int kFull, int kLeast, typename F>
int with_cut(Cut c, F &&f) {
  if constexpr (kLeast > 1)
    if (c.shift) return f(std::integral_constant<int, kFull>{}, std::true_type{});
  return with_vector<kFull, kLeast>(c.v, f);
}

// 16 or 8 bytes (N) from address a, those of them that lie in [begin, end); the others
// are unspecified.  A block is only loaded when it holds a byte of the range, so every
// load stays inside the page of a byte that the caller owns.
template <int N>
__device__ __forceinline__ Words<N> load_shifted(uintptr_t a, uintptr_t begin, uintptr_t end) {
  const uint32_t s = (uint32_t)(a & (N - 1));
  const uintptr_t b = a - s;
  const bool first = b < end && b + N > begin, second = s && b + N < end && b + 2 * N > begin;
  Words<N> out;
  if constexpr (N == 16) {
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (first) x = __ldg(reinterpret_cast<const uint4 *>(b));
    if (second) y = __ldg(reinterpret_cast<const uint4 *>(b) + 1);
    x = shift_pair(x, y, s);
    out.w[0] = x.x, out.w[1] = x.y, out.w[2] = x.z, out.w[3] = x.w;
  } else {
    uint2 x = make_uint2(0, 0), y = x;
    if (first) x = __ldg(reinterpret_cast<const uint2 *>(b));
    if (second) y = __ldg(reinterpret_cast<const uint2 *>(b) + 1);
    uint32_t w0 = x.x, w1 = x.y, w2 = y.x;
    if (s & 4) w0 = w1, w1 = w2, w2 = y.y;
    const uint32_t r = (s & 3) * 8;
    out.w[0] = __funnelshift_r(w0, w1, r), out.w[1] = __funnelshift_r(w1, w2, r);
  }
  return out;
}

// V elements of a row from column c on.  With kShift c may be any column from 1 - V on;
// elements outside the row are unspecified.
template <typename T, int V, bool kShift>
__device__ __forceinline__ void load_columns(Vec<T, V> &v, const T *row, int32_t c,
                                             uint32_t width) {
  if constexpr (kShift) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(row);
    static_cast<Words<(int)sizeof(T) * V> &>(v) = load_shifted<(int)sizeof(T) * V>(
        begin + (int64_t)c * (int)sizeof(T), begin, begin + (uint64_t)width * sizeof(T));
  } else {
    v.load(row + c);
  }
}

// Columns by which a row that is written precedes its first granule: vector q of the
// row holds the columns from q * V - lead on.
template <typename T, int V, bool kShift>
__device__ __forceinline__ int32_t row_lead(const T *row) {
  if constexpr (!kShift) return 0;
  return (int32_t)(reinterpret_cast<uintptr_t>(row) % (V * sizeof(T)) / sizeof(T));
}

// Whether all of a vector lies in the row.
template <int V, bool kShift>
__device__ __forceinline__ bool whole(int32_t c, uint32_t width) {
  return !kShift || (c >= 0 && c + V <= (int32_t)width);
}

template <typename T, int V, bool kShift, bool kStream = true>
__device__ __forceinline__ void store_columns(const Vec<T, V> &v, T *row, int32_t c,
                                              uint32_t width) {
  if (whole<V, kShift>(c, width)) {
    if constexpr (kStream) v.store_cs(row + c);
    else v.store(row + c);
  } else if constexpr (kShift) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i >= 0 && c + i < (int32_t)width) {
        Words<(int)sizeof(T)> one;
        one.w[0] = sizeof(T) == 4 ? v.w[i] : v.w[i / 2] >> 16 * (i & 1);
        one.store(row + c + i);
      }
  }
}

// Zeroes `bytes` bytes by the threads `t` of `threads`: 16-byte granules, bytes at the
// ends.
template <bool kStream = false>
__device__ __forceinline__ void zero_bytes(uint8_t *at, uint64_t bytes, uint32_t t,
                                           uint32_t threads) {
  const uint64_t head = min((uint64_t)(-(uintptr_t)at & 15), bytes);
  const uint64_t units = (bytes - head) / 16, tail = bytes - head - units * 16;
  uint4 *dst = reinterpret_cast<uint4 *>(at + head);
#pragma unroll 4
  for (uint64_t u = t; u < units; u += threads) {
    if (kStream) __stcs(dst + u, make_uint4(0, 0, 0, 0));
    else dst[u] = make_uint4(0, 0, 0, 0);
  }
  if (t < head) at[t] = 0;
  if (t < tail) at[bytes - 1 - t] = 0;
}

// For rows that a warp zeroes one after the other.  Rows of up to 512 bytes are many, so
// that instructions count: units of 16 to 1 bytes that all rows start on, no ends.  Wider
// rows go by zero_bytes (0) unless they are whole granules.
__device__ __forceinline__ uint32_t zero_unit(const void *base, uint64_t pitch, uint64_t bytes) {
  const uint32_t all = (uint32_t)(reinterpret_cast<uintptr_t>(base) | pitch | bytes);
  const uint32_t unit = all % 16 == 0 ? 16 : all & -all;
  return unit == 16 || bytes <= 512 ? unit : 0;
}
template <bool kStream = false>
__device__ __forceinline__ void zero_row(uint8_t *row, uint32_t bytes, uint32_t unit,
                                         uint32_t lane) {
  if (unit == 0) return zero_bytes<kStream>(row, bytes, lane, 32);
  for (uint32_t at = lane * unit; at < bytes; at += 32 * unit) {
    if (unit == 16) {
      if (kStream) __stcs(reinterpret_cast<uint4 *>(row + at), make_uint4(0, 0, 0, 0));
      else *reinterpret_cast<uint4 *>(row + at) = make_uint4(0, 0, 0, 0);
    } else if (unit == 8) {
      *reinterpret_cast<uint2 *>(row + at) = make_uint2(0, 0);
    } else if (unit == 4) {
      *reinterpret_cast<uint32_t *>(row + at) = 0;
    } else if (unit == 2) {
      *reinterpret_cast<uint16_t *>(row + at) = 0;
    } else {
      row[at] = 0;
    }
  }
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
