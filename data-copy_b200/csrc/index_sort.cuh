// Stable sort of entries by a small whole-number key (index_sort.cu): the tokens of
// an embedding gradient by id, a router's choices by expert.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace dcopy {

// Where the keys come from: `rows` x `cols` ids, row-major with a pitch.  An entry's
// key is id - first when that lies in [0, keys), else `keys` (it belongs nowhere).
struct KeySource {
  const void *ids;
  int64_t pitch;   // elements between rows
  int64_t first;
  uint32_t keys;
  uint32_t wide;   // ids are 64-bit
  uint32_t n;      // rows * cols
  FastDiv cols;
};

// The e-th id less `first`, modulo 2^64: with first + keys within 2^63, ids that wrap around
// stay outside [0, keys).
__device__ __forceinline__ int64_t read_id(const KeySource &k, uint32_t e) {
  const uint32_t r = k.cols.div(e);
  const int64_t at = (int64_t)r * k.pitch + (e - r * k.cols.d);
  const int64_t id = k.wide ? static_cast<const int64_t *>(k.ids)[at]
                            : (int64_t)static_cast<const int32_t *>(k.ids)[at];
  return (int64_t)((uint64_t)id - (uint64_t)k.first);
}

// Rows [begin, end) to zero beside the sort: its few blocks leave most SMs idle, so
// each of its launches also clears some, the last ones first.  (Vocabularies have their
// frequent ids in front, and rows that tokens have are written again.)
struct Fill {
  uint8_t *dst = nullptr;
  uint64_t pitch = 0, bytes = 0;  // of a row
  uint64_t begin = 0, end = 0;
};

// Workspace bytes of sort_by_key for n entries.
uint64_t sort_by_key_bytes(uint64_t n);
// key_out[p], pos_out[p]: the p-th entry in key order, equal keys in entry order.
// Both arrays (n values each) lie in the workspace.  n is at least 1.  fill becomes
// the rows that are left.
int sort_by_key(const KeySource &src, Fill *fill, void *workspace, const uint32_t **key_out,
                const uint32_t **pos_out, cudaStream_t s);
// Clears alone.
int fill_zero(const Fill &fill, cudaStream_t s);

// The router's form: at most kMaxExperts keys, offsets padded to `align`.
constexpr uint32_t kMaxExperts = 1023;
uint64_t sort_experts_bytes(uint64_t n, uint32_t experts);
int sort_experts(const KeySource &src, uint32_t align, int32_t *dest, int32_t *source,
                 uint32_t rows, int32_t *offsets, void *workspace, cudaStream_t s);

}  // namespace dcopy
