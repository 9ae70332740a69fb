// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// lookup  out[i,:] = round(scale * table[id_i - first,:]), zero where id_i - first
//         is outside the table (padding, or another rank's part of the vocabulary).
// grad    dW[v,:] = round(scale * sum of dout[i,:] over id_i - first == v), the sum in
//         fp32 and in the order of i within a piece of the sorted list, then piece by
//         piece: the same bits on every run.  Both are bound by HBM bytes.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "index_sort.cuh"
#include "launch.cuh"
#include "rowops.cuh"

namespace dcopy {
namespace {

struct Lookup {
  void *out;
  const void *table;
  int64_t out_pitch, table_pitch;
  KeySource ids;
  uint32_t width, vectors;
  int lx;
  float scale;
};

// A thread takes U vectors of a row, a power of two threads a row.  Bound by HBM: 32768
// rows of 4096 bf16 out of 131072 (11900 different ones, 98 MB, 268 MB written) take 62
// to 65 us, 5.6 to 5.9 TB/s.  Streaming stores keep the table's frequent rows in L2 (78
// us without).
template <typename TIn, typename TOut, int V, bool kShift, int U>
__global__ void __launch_bounds__(kRowThreads) lookup_kernel(Lookup p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t row = blockIdx.x * (kRowThreads >> p.lx) + (threadIdx.x >> p.lx);
  if (row >= p.ids.n) return;
  const uint32_t step = 1u << p.lx;
  const uint32_t q = (blockIdx.y * U << p.lx) + (threadIdx.x & (step - 1));
  const int64_t id = read_id(p.ids, row);
  const bool known = id >= 0 && id < (int64_t)p.ids.keys;
  const TIn *src = static_cast<const TIn *>(p.table) + (known ? id * p.table_pitch : 0);
  TOut *dst = static_cast<TOut *>(p.out) + row * p.out_pitch;
  const int32_t lead = row_lead<TOut, V, kShift>(dst);
  Vec<TIn, V> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int32_t c = (int32_t)((q + u * step) * V) - lead;
    if (known && c < (int32_t)p.width) load_columns<TIn, V, kShift>(in[u], src, c, p.width);
    else in[u].zero();
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int32_t c = (int32_t)((q + u * step) * V) - lead;
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = known ? in[u].get(i) * p.scale : 0.0f;
    Vec<TOut, V> out;
    out.put(f);
    if (c < (int32_t)p.width) store_columns<TOut, V, kShift>(out, dst, c, p.width);
  }
}

// ---- gradient -------------------------------------------------------------------

// Sorted entries of a piece: 32 where there are enough pieces for all SMs (16384
// tokens: 197 us against 206 with 16), 16 below (2047 tokens: 30 us against 34 with 32).
constexpr uint32_t kPiece = 32, kSmallPiece = 16, kFewTokens = 4096;
constexpr uint32_t kMaxPieces = 32;  // pieces of a block
// Bytes zeroed beside the joining of runs, and by a block: small blocks spread a small
// fill over the SMs (36 MB: 30 us with 32 KB, 46 with 128 KB), large ones search less
// often for the rows that tokens have (800 MB: 197 us with 128 KB, 232 with 32 KB).
constexpr uint64_t kFillLate = 32ull << 20;
constexpr uint64_t kFillBlockLeast = 32ull << 10, kFillBlockMost = 128ull << 10;
constexpr uint64_t kFillBlocks = 2048;

struct Grad {
  void *grad;
  const void *dout;
  int64_t grad_pitch, dout_pitch;
  const uint32_t *key, *pos;  // in key order
  float *head, *tail;         // [pieces][width] sums of runs that cross piece ends
  uint32_t n, keys, piece, pieces, vectors, width;  // piece: entries of one
  int lx;
  float scale;
  Fill fill;                  // rows to zero where no token has them
  uint32_t piece_blocks, work_blocks, fill_rows;  // a block's pieces x columns, then the fill
};

// Rows [row0, row1) of the gradient, at most kRowThreads, are zeroed by a block, but
// those whose bit is set (some token has them, and the sums are written to them).
__device__ __forceinline__ void zero_but(const Fill &f, uint64_t row0, uint64_t row1,
                                         const uint32_t *touched) {
  uint32_t any = 0;
  for (uint32_t w = 0; w < kRowThreads / 32; ++w) any |= touched[w];
  if (!any && f.pitch == f.bytes)
    return zero_bytes(f.dst + row0 * f.pitch, (row1 - row0) * f.bytes, threadIdx.x, kRowThreads);
  const uint32_t unit = zero_unit(f.dst, f.pitch, f.bytes);
  for (uint32_t k = threadIdx.x / 32; k < (uint32_t)(row1 - row0); k += kRowThreads / 32)
    if (!(touched[k / 32] >> k % 32 & 1))
      zero_row(f.dst + (row0 + k) * f.pitch, (uint32_t)f.bytes, unit, threadIdx.x % 32);
}

__device__ __forceinline__ void touch(uint32_t *touched, uint32_t row) {
  atomicOr(&touched[row / 32], 1u << row % 32);
}

// Blocks behind a kernel's own: fill_rows rows each of the fill.  The place of the first
// in the sorted ids is found by a search that narrows by the block's size a step.
__device__ __forceinline__ void zero_untouched(const Grad &p, uint32_t block) {
  __shared__ uint32_t touched[kRowThreads / 32];
  const uint64_t row0 = p.fill.begin + (uint64_t)block * p.fill_rows;
  const uint64_t row1 = min(row0 + p.fill_rows, p.fill.end);
  if (threadIdx.x < kRowThreads / 32) touched[threadIdx.x] = 0;
  uint32_t lo = 0, length = p.n;  // the first entry not below row0 lies in [lo, lo + length]
  while (length > 0) {
    const uint32_t step = (length + kRowThreads - 1) / kRowThreads;
    const uint32_t i = threadIdx.x * step;
    const uint32_t below = __syncthreads_count(i < length && p.key[lo + i] < row0);
    if (below == 0) break;  // lo itself
    const uint32_t from = (below - 1) * step + 1;  // the entry before it is below row0
    const uint32_t to = min(below * step, length);
    lo += from;
    length = to - from;
  }
  __syncthreads();
  for (uint32_t i0 = lo; i0 < p.n; i0 += kRowThreads) {
    const uint32_t key = i0 + threadIdx.x < p.n ? p.key[i0 + threadIdx.x] : p.keys;
    const bool in = key < row1;
    if (in) touch(touched, key - (uint32_t)row0);
    if (!__syncthreads_and(in)) break;
  }
  __syncthreads();
  zero_but(p.fill, row0, row1, touched);
}

// round(scale * sum), added to what the row held (`old`) with kAdd.
template <typename T, int V, bool kAdd>
__device__ __forceinline__ void write_row(T *row, uint32_t c, const float (&sum)[V], float scale,
                                          const Vec<T, V> &old) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    f[i] = sum[i] * scale;
    if constexpr (kAdd) f[i] += old.get(i);
  }
  Vec<T, V> out;
  out.put(f);
  out.store(row + (uint64_t)c * V);
}

template <typename T, int V, bool kAdd>
__device__ __forceinline__ void load_old(Vec<T, V> &old, const T *row, uint32_t c) {
  if constexpr (kAdd) old.load_plain(row + (uint64_t)c * V);
}

// At most kFew tokens: no sort.  A block takes a token and some columns; where the token
// is the first of its id, the rows of that id are summed in order.  The other blocks
// zero the rows that no token has.  One launch instead of three, which is what so few
// tokens cost (23 tokens, 1551 x 483: 3.8 us instead of 8.4).
constexpr uint32_t kFew = 512;

template <typename TIn, typename TOut, int V, bool kAdd>
__global__ void __launch_bounds__(kRowThreads) few_sum_kernel(Grad p, KeySource ids) {
  __shared__ uint32_t bits[kFew / 32];  // rows with a token; tokens with the block's id
  static_assert(kFew / 32 >= kRowThreads / 32, "one bit for each row of a block");
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < kFew / 32) bits[threadIdx.x] = 0;
  __syncthreads();
  if (blockIdx.x >= p.work_blocks) {
    const uint64_t row0 = p.fill.begin + (uint64_t)(blockIdx.x - p.work_blocks) * p.fill_rows;
    const uint64_t row1 = min(row0 + p.fill_rows, p.fill.end);
    for (uint32_t i = threadIdx.x; i < p.n; i += kRowThreads) {
      const int64_t id = read_id(ids, i);
      if (id >= (int64_t)row0 && id < (int64_t)row1) touch(bits, (uint32_t)(id - row0));
    }
    __syncthreads();
    return zero_but(p.fill, row0, row1, bits);
  }
  const uint32_t by = blockIdx.x / p.n, token = blockIdx.x - by * p.n;
  const int64_t key = read_id(ids, token);
  if (key < 0 || key >= (int64_t)p.keys) return;
  bool earlier = false;
  for (uint32_t i0 = 0; i0 < p.n; i0 += kRowThreads) {
    const uint32_t i = i0 + threadIdx.x;
    const bool same = i < p.n && read_id(ids, i) == key;
    earlier |= same && i < token;
    const uint32_t mask = __ballot_sync(~0u, same);
    if (threadIdx.x % 32 == 0) bits[i / 32] = mask;
  }
  if (__syncthreads_or(earlier)) return;
  const uint32_t c = by * kRowThreads + threadIdx.x;
  if (c >= p.vectors) return;
  const TIn *dout = static_cast<const TIn *>(p.dout) + (uint64_t)c * V;
  float sum[V] = {};
  constexpr int kAhead = 8;
  uint32_t word = token / 32, mask = bits[word];
  for (;;) {
    uint32_t from[kAhead];
    int held = 0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      while (mask == 0 && ++word < (p.n + 31) / 32) mask = bits[word];
      from[j] = word * 32 + __ffs(mask) - 1;
      if (mask) ++held;
      mask &= mask - 1;
    }
    if (held == 0) break;
    Vec<TIn, V> in[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (j < held) in[j].load(dout + from[j] * p.dout_pitch);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (j < held) {
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += in[j].get(v);
      }
  }
  TOut *row = static_cast<TOut *>(p.grad) + key * p.grad_pitch;
  Vec<TOut, V> old;
  load_old<TOut, V, kAdd>(old, row, c);
  write_row<TOut, V, kAdd>(row, c, sum, p.scale, old);
}

// One piece of the sorted list: runs of equal ids that lie inside it are summed and
// written; what a run that crosses an end of the piece has here goes to head (it
// began earlier) or tail (it begins here and goes on).  Rows of kAhead tokens are
// fetched before the first is added.  Sums in fp32, one rounding when a row is written.
// With the zeroing that goes along, bound by HBM: 16384 tokens, 131072 x 4096 bf16 move
// 0.94 GB in 141 us (6.6 TB/s) here and the whole gradient takes 190 us.
template <typename TIn, typename TOut, int V, bool kAdd>
__global__ void __launch_bounds__(kRowThreads) piece_sum_kernel(Grad p) {
  // The ids of the block's pieces, one before and one behind; positions.
  __shared__ uint32_t keys[kMaxPieces * kPiece + 2], places[kMaxPieces * kPiece];
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x >= p.work_blocks) return zero_untouched(p, blockIdx.x - p.work_blocks);
  const uint32_t by = blockIdx.x / p.piece_blocks, bx = blockIdx.x - by * p.piece_blocks;
  const uint32_t block_pieces = kRowThreads >> p.lx;
  const uint32_t first = bx * block_pieces * p.piece;  // entry
  for (uint32_t i = threadIdx.x; i < block_pieces * p.piece + 2; i += kRowThreads) {
    const uint32_t e = first + i;  // entry e - 1
    keys[i] = e >= 1 && e <= p.n ? p.key[e - 1] : p.keys;
    if (i >= 1 && i <= block_pieces * p.piece && e <= p.n) places[i - 1] = p.pos[e - 1];
  }
  __syncthreads();
  const uint32_t local = (threadIdx.x >> p.lx) * p.piece;
  const uint32_t piece = bx * block_pieces + (threadIdx.x >> p.lx);
  const uint32_t c = (by << p.lx) + (threadIdx.x & ((1u << p.lx) - 1));
  if (piece >= p.pieces || c >= p.vectors) return;
  const uint32_t count = min(p.piece, p.n - piece * p.piece);
  const TIn *dout = static_cast<const TIn *>(p.dout) + (uint64_t)c * V;
  TOut *grad = static_cast<TOut *>(p.grad);
  uint32_t key = keys[local + 1];
  bool open = piece > 0 && keys[local] == key;  // the run began in an earlier piece
  float sum[V] = {};
  constexpr int kAhead = 8;
  for (uint32_t i0 = 0; i0 < count && key < p.keys; i0 += kAhead) {
    Vec<TIn, V> in[kAhead];
    // What is added to, fetched for the rows whose run ends here (2047 tokens, 32000 x
    // 4096: 21 us instead of 25, as no run waits for its own load).
    Vec<TOut, V> old[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t id = keys[local + i0 + j + 1];
      if (i0 + j < count && id < p.keys) {
        in[j].load(dout + (int64_t)places[local + i0 + j] * p.dout_pitch);
        if (keys[local + i0 + j + 2] != id)
          load_old<TOut, V, kAdd>(old[j], grad + id * p.grad_pitch, c);
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j >= count || key >= p.keys) break;
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] += in[j].get(v);
      const uint32_t next = keys[local + i0 + j + 2];
      if (next != key || i0 + j + 1 == count) {
        float *part = open ? p.head : next == key ? p.tail : nullptr;
        if (part) {
          Vec<float, V> out;
          out.put(sum);
          out.store(part + (uint64_t)piece * p.width + (uint64_t)c * V);
        } else {
          write_row<TOut, V, kAdd>(grad + key * p.grad_pitch, c, sum, p.scale, old[j]);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] = 0.0f;
        open = false;
        key = next;
      }
    }
  }
}

// The runs that begin in a piece and go on: tail of that piece plus the heads of the
// following ones, in order, kAhead of them fetched before it is known how many count.
// Bound by the latency of the longest run, one thread a column over all its pieces (1024
// columns, an id that 6 % of 65536 tokens have: 27 us, of 262144: 93); the zeroing of a
// large table beside it hides that, nothing does when gradients accumulate.
template <typename TOut, int V, bool kAdd>
__global__ void __launch_bounds__(kRowThreads, 4) piece_join_kernel(Grad p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x >= p.work_blocks) return zero_untouched(p, blockIdx.x - p.work_blocks);
  const uint32_t by = blockIdx.x / p.piece_blocks, bx = blockIdx.x - by * p.piece_blocks;
  const uint32_t piece = bx * (kRowThreads >> p.lx) + (threadIdx.x >> p.lx);
  const uint32_t c = (by << p.lx) + (threadIdx.x & ((1u << p.lx) - 1));
  if (piece + 1 >= p.pieces || c >= p.vectors) return;
  const uint32_t b = piece * p.piece, last = b + p.piece - 1;
  const uint32_t key = p.key[last];
  if (key >= p.keys || p.key[last + 1] != key) return;    // nothing goes on
  if (p.key[b] == key && b > 0 && p.key[b - 1] == key) return;  // it began earlier
  const uint64_t at = (uint64_t)c * V;
  float sum[V];
  Vec<float, V> part;
  part.load(p.tail + (uint64_t)piece * p.width + at);
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = part.get(v);
  // 32 floats a thread at most: with 64, two blocks fit an SM and the zeroing beside the
  // sums is slower for it (194 us instead of 190 for the gradient above).
  constexpr int kAhead = V == 8 ? 4 : 8;
  bool on = true;
  for (uint32_t q = piece + 1; on && q < p.pieces; q += kAhead) {
    Vec<float, V> head[kAhead];
    bool same[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      same[j] = q + j < p.pieces && p.key[(q + j) * p.piece] == key;
      if (q + j < p.pieces) head[j].load(p.head + (uint64_t)(q + j) * p.width + at);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      on = on && same[j];
      if (on) {
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += head[j].get(v);
      }
    }
  }
  TOut *row = static_cast<TOut *>(p.grad) + key * p.grad_pitch;
  Vec<TOut, V> old;
  load_old<TOut, V, kAdd>(old, row, c);
  write_row<TOut, V, kAdd>(row, c, sum, p.scale, old);
}

int id_source(const DcopyMatrix *ids, int64_t first, int64_t keys, KeySource *src) {
  if (int rc = check_matrix(ids, "ids", is_index(ids->type))) return rc;
  const uint64_t n = (uint64_t)ids->rows * (uint64_t)ids->cols;
  if (n > INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "ids: %llu entries", (unsigned long long)n);
  // Beyond this, the subtraction of first would wrap ids from the other end into the table.
  if (keys > 0 && first > INT64_MAX - (keys - 1))
    return set_error(DCOPY_ERR_PARAM_INVALID, "first_id %lld: the table's %lld rows pass 2^63",
                     (long long)first, (long long)keys);
  src->ids = ids->data;
  src->pitch = ids->pitch;
  src->first = first;
  src->keys = (uint32_t)keys;
  src->wide = ids->type == kI64;
  src->n = (uint32_t)n;
  src->cols = FastDiv((uint32_t)std::max<int64_t>(1, ids->cols));
  return DCOPY_OK;
}

uint32_t piece_of(uint64_t n) { return n <= kFewTokens ? kSmallPiece : kPiece; }
uint64_t pieces_of(uint64_t n) { return (n + piece_of(n) - 1) / piece_of(n); }

}  // namespace
}  // namespace dcopy

using namespace dcopy;

extern "C" {

int dcopy_embedding_lookup(const DcopyMatrix *out, const DcopyMatrix *table,
                           const DcopyMatrix *ids, int64_t first_id, float scale,
                           dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!out || !table || !ids)
    return set_error(DCOPY_ERR_PARAM_INVALID, "embedding_lookup: NULL matrix");
  if (int rc = check_matrix(out, "out", is_float(out->type))) return rc;
  if (int rc = check_matrix(table, "table", is_float(table->type))) return rc;
  Lookup p{};
  if (int rc = id_source(ids, first_id, table->rows, &p.ids)) return rc;
  if (out->rows != (int64_t)p.ids.n || out->cols != table->cols)
    return set_error(DCOPY_ERR_SHAPE_INVALID,
                     "embedding_lookup: out is %lld x %lld for %u ids and a table of width %lld",
                     (long long)out->rows, (long long)out->cols, p.ids.n, (long long)table->cols);
  if (out->cols > kMaxWidth)
    return set_error(DCOPY_ERR_UNSUPPORTED, "embedding_lookup: width %lld", (long long)out->cols);
  if (out->rows == 0 || out->cols == 0) return DCOPY_OK;
  if (int rc = check_apart(out, table, "embedding_lookup", "out", "table")) return rc;
  if (int rc = check_apart(out, ids, "embedding_lookup", "out", "ids")) return rc;
  p.out = out->data;
  p.table = table->data;
  p.out_pitch = out->pitch;
  p.table_pitch = table->pitch;
  p.scale = scale;
  return with_float(table->type, [&](auto tin) {
    return with_float(out->type, [&](auto tout) {
      using TIn = typename decltype(tin)::type;
      using TOut = typename decltype(tout)::type;
      // Shifted below 8-byte vectors (24390 rows of 1025 bf16: 25 us against 60 in single
      // elements; of 1025 fp32: 21 against 33).
      constexpr int kBytes = std::max(sizeof(TIn), sizeof(TOut));
      constexpr int kFull = 16 / kBytes, kLeast = 8 / kBytes;
      const Cut cut = cut_rows(kFull, kLeast, out, table);
      p.width = (uint32_t)out->cols;
      p.vectors = vectors_of(out->cols, cut);
      // Four vectors a thread (32 Ki rows of 8 KB: 62 us, 75 with one), one where the
      // grid is small.
      const bool many = (uint64_t)p.ids.n * p.vectors >= (uint64_t)sm_count() * 2048 * 4;
      const RowSplit split = split_rows(p.ids.n, p.vectors, many ? 4 : 1);
      p.lx = split.lx;
      return with_cut<kFull, kLeast>(cut, [&](auto v, auto shift) {
        auto k = many ? lookup_kernel<TIn, TOut, v(), shift(), 4>
                      : lookup_kernel<TIn, TOut, v(), shift(), 1>;
        return launch_grid(k, split.grid, dim3(kRowThreads), 0, stream, "lookup_kernel", p);
      });
    });
  });
  DCOPY_API_END
}

int dcopy_embedding_grad_workspace(int64_t tokens, int64_t vocab, int64_t width,
                                   uint64_t *bytes) {
  DCOPY_API_BEGIN
  if (!bytes || tokens < 0 || vocab < 0 || width < 0 || tokens > INT32_MAX || vocab > INT32_MAX ||
      width > kMaxWidth)
    return set_error(DCOPY_ERR_PARAM_INVALID, "embedding_grad_workspace: %lld tokens, %lld x %lld",
                     (long long)tokens, (long long)vocab, (long long)width);
  const uint64_t sort = (sort_by_key_bytes(tokens) + 15) / 16 * 16;
  const uint64_t row = ((uint64_t)width * sizeof(float) + 15) / 16 * 16;
  *bytes = sort + 2 * pieces_of(tokens) * row + 32;
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_embedding_grad(const DcopyMatrix *grad, const DcopyMatrix *dout, const DcopyMatrix *ids,
                         int64_t first_id, float scale, int32_t accumulate, void *workspace,
                         uint64_t workspace_bytes, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!grad || !dout || !ids)
    return set_error(DCOPY_ERR_PARAM_INVALID, "embedding_grad: NULL matrix");
  if (int rc = check_matrix(grad, "grad", is_float(grad->type))) return rc;
  if (int rc = check_matrix(dout, "dout", is_float(dout->type))) return rc;
  KeySource src{};
  if (int rc = id_source(ids, first_id, grad->rows, &src)) return rc;
  if (dout->rows != (int64_t)src.n || dout->cols != grad->cols)
    return set_error(DCOPY_ERR_SHAPE_INVALID,
                     "embedding_grad: dout is %lld x %lld for %u ids and a table of width %lld",
                     (long long)dout->rows, (long long)dout->cols, src.n, (long long)grad->cols);
  if (grad->cols > kMaxWidth)
    return set_error(DCOPY_ERR_UNSUPPORTED, "embedding_grad: width %lld", (long long)grad->cols);
  uint64_t need = 0;
  if (int rc = dcopy_embedding_grad_workspace(src.n, grad->rows, grad->cols, &need)) return rc;
  if (src.n && workspace_bytes < need)
    return set_error(DCOPY_ERR_PARAM_INVALID, "embedding_grad: workspace of %llu bytes, %llu needed",
                     (unsigned long long)workspace_bytes, (unsigned long long)need);
  if (int rc = check_apart(grad, dout, "embedding_grad", "grad", "dout")) return rc;
  if (int rc = check_apart(grad, ids, "embedding_grad", "grad", "ids")) return rc;
  if (src.n) {
    if (int rc = check_device_span(workspace, need, "workspace")) return rc;
    const DcopyMatrix space = flat(workspace, need, kU8);
    if (int rc = check_apart(grad, &space, "embedding_grad", "grad", "workspace")) return rc;
    if (int rc = check_apart(dout, &space, "embedding_grad", "dout", "workspace")) return rc;
    if (int rc = check_apart(ids, &space, "embedding_grad", "ids", "workspace")) return rc;
  }
  if (grad->rows == 0 || grad->cols == 0) return DCOPY_OK;
  Fill fill;
  if (!accumulate) {
    const uint64_t eb = elem_size(grad->type);
    fill.dst = static_cast<uint8_t *>(grad->data);
    fill.end = grad->rows;
    fill.bytes = grad->cols * eb;
    fill.pitch = grad->pitch * eb;
  }
  if (src.n == 0) return fill_zero(fill, stream);
  uint8_t *ws = reinterpret_cast<uint8_t *>(((uintptr_t)workspace + 15) / 16 * 16);
  const uint64_t sort = (sort_by_key_bytes(src.n) + 15) / 16 * 16;
  Grad p{};
  const bool few = src.n <= kFew;
  if (!few)
    if (int rc = sort_by_key(src, &fill, ws, &p.key, &p.pos, stream)) return rc;
  p.grad = grad->data;
  p.dout = dout->data;
  p.grad_pitch = grad->pitch;
  p.dout_pitch = dout->pitch;
  p.n = src.n;
  p.keys = src.keys;
  p.piece = piece_of(src.n);
  p.pieces = (uint32_t)pieces_of(src.n);
  p.width = (uint32_t)((grad->cols + 3) / 4 * 4);
  p.head = reinterpret_cast<float *>(ws + sort);
  p.tail = p.head + (uint64_t)p.pieces * p.width;
  p.scale = scale;
  return with_float(dout->type, [&](auto tin) {
    return with_float(grad->type, [&](auto tout) {
      using TIn = typename decltype(tin)::type;
      using TOut = typename decltype(tout)::type;
      // Never shifted: 24366 tokens of 1026 bf16 take 83 us in 4-byte vectors, 107 shifted.
      constexpr int kFull = 16 / std::max(sizeof(TIn), sizeof(TOut));
      const Cut cut = cut_rows(kFull, 1, grad, dout);
      p.vectors = vectors_of(grad->cols, cut);
      // Blocks behind the kernel's own zero `rows` rows from the end of what is left.
      auto fill_blocks = [&](uint64_t rows) {
        const uint64_t block = std::clamp<uint64_t>(rows * fill.bytes / kFillBlocks,
                                                    kFillBlockLeast, kFillBlockMost);
        if (rows)
          p.fill_rows = (uint32_t)std::clamp<uint64_t>(block / fill.bytes, 1, kRowThreads);
        p.fill = fill;
        p.fill.begin = fill.end - rows;
        fill.end -= rows;
        return rows ? (uint32_t)((rows + p.fill_rows - 1) / p.fill_rows) : 0;
      };
      const uint64_t left = fill.bytes ? fill.end - fill.begin : 0;
      return with_cut<kFull, 1>(cut, [&](auto v, auto) {
        constexpr int V = v();
        if (few) {
          auto k = accumulate ? few_sum_kernel<TIn, TOut, V, true>
                              : few_sum_kernel<TIn, TOut, V, false>;
          p.work_blocks = p.n * ((p.vectors + kRowThreads - 1) / kRowThreads);
          const uint32_t blocks = p.work_blocks + fill_blocks(left);
          return launch(k, blocks, dim3(kRowThreads), 0, stream, "few_sum_kernel", p, src);
        }
        const RowSplit split = split_rows(p.pieces, p.vectors, 1, kMaxPieces);
        p.lx = split.lx;
        auto sum = accumulate ? piece_sum_kernel<TIn, TOut, V, true>
                              : piece_sum_kernel<TIn, TOut, V, false>;
        auto join = accumulate ? piece_join_kernel<TOut, V, true> : piece_join_kernel<TOut, V, false>;
        // What is left to zero goes along with the two launches: as much with the second
        // as hides the latency of its few long runs, the rest with the first.
        const uint64_t late = std::min<uint64_t>(
            left, p.pieces > 1 && left ? std::max<uint64_t>(1, kFillLate / fill.bytes) : 0);
        auto step = [&](auto kernel, const char *name, uint64_t rows) {
          p.piece_blocks = split.grid.x;
          p.work_blocks = split.grid.x * split.grid.y;
          const uint32_t blocks = p.work_blocks + fill_blocks(rows);
          return launch(kernel, blocks, dim3(kRowThreads), 0, stream, name, p);
        };
        if (int rc = step(sum, "piece_sum_kernel", left - late)) return rc;
        if (p.pieces == 1) return (int)DCOPY_OK;
        return step(join, "piece_join_kernel", late);
      });
    });
  });
  DCOPY_API_END
}

}  // extern "C"
