// Tokens sorted by expert and back, with weights, and the gradient.
//
// sort      the entries (token i, slot j) in expert order, the earlier first:
//           dest[i,j] = row of the entry, source[row] = i * slots + j
// dispatch  out[dest[i,j],:] = (w[i,j] *) x[i,:], rows without an entry are zeroed
// combine   out[i,:] = round(sum over j of (w[i,j] *) y[dest[i,j],:]), in fp32, j ascending
// combine_grad  dy[dest[i,j],:] = round(w[i,j] * dout[i,:]),
//           dw[i,j] = sum over the columns of dout[i,:] * y[dest[i,j],:]
// All are bound by the bytes of the rows: each row is read once and written once.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "index_sort.cuh"
#include "launch.cuh"
#include "rowops.cuh"

namespace dcopy {
namespace {

// The vectors of a group of tokens laid end to end over the threads of grid.y blocks, so
// that few threads are left over whatever the width (24390 x 4 rows of 1028 bf16, 257
// vectors: combined in 42 us, dispatched in 54; with a power of two threads a row in 64
// and 71).  Dispatch gives narrow rows a power of two all the same: a warp that
// writes to two rows at once is slower (260416 x 4 rows of 90 fp32: 80 us, not 58).
struct Flat {
  dim3 grid;
  uint32_t group, items;  // tokens of a group, their vectors
  FastDiv stride;         // threads of a token
};

Flat flat_tokens(uint64_t tokens, uint32_t vectors, bool whole_warps) {
  Flat f;
  uint32_t stride = std::max<uint32_t>(1, vectors);
  if (whole_warps && vectors <= 64)
    for (stride = 1; stride < vectors;) stride *= 2;
  f.stride = FastDiv(stride);
  // The first group from one block's worth on that leaves less than 5 % over.
  const uint32_t least = std::max<uint32_t>(1, kRowThreads / stride);
  double best = 0.0;
  f.group = 1;
  for (uint32_t g = least; g < least + 16 && best < 0.95; ++g) {
    const uint64_t items = (uint64_t)g * stride;
    const uint64_t blocks = (items + kRowThreads - 1) / kRowThreads;
    const double used = (double)items / (double)(blocks * kRowThreads);
    if (used > best + 0.01) best = used, f.group = g;
  }
  f.items = f.group * stride;
  f.grid = dim3((unsigned)((tokens + f.group - 1) / f.group),
                (f.items + kRowThreads - 1) / kRowThreads);
  return f;
}

struct Route {
  void *out;              // dispatch: rows in expert order; combine: tokens
  const void *in;         // dispatch: tokens; combine: rows in expert order
  const void *dout;       // combine_grad: tokens
  float *dweights;
  int64_t out_pitch, in_pitch, dout_pitch, w_pitch, dw_pitch;
  const int32_t *dest, *source;
  const float *weights;
  uint32_t tokens, slots, rows, width, vectors, unused_blocks, unused_rows;
  Flat flat;
  FastDiv by_slots;
  int lx;
};

// Rows of the buffer in expert order that hold no entry are zeroed by the first blocks
// of the grid, a warp unused_rows of them: padding comes in runs of rows, and ahead of
// the others these blocks do not trail the kernel.  More rows a warp take longer over a
// run (655 x 4 entries, experts padded to 128: 4.3 us with 8, 7.1 with 32), fewer cost
// blocks that find nothing (262144 x 2 x 1024: 246 us with 8, 239 with 32), so the rows
// a warp grow with the buffer.  Where an eighth of the rows or more must be empty, a warp
// takes 16 KB of them at most (10176 rows of 20 KB, 2556 in use: 46 us, with 8 rows a
// warp 55).
uint32_t unused_rows_of(uint64_t rows, uint64_t entries, uint64_t row_bytes) {
  if (rows > entries + rows / 8)
    return (uint32_t)std::clamp<uint64_t>((16 << 10) / std::max<uint64_t>(1, row_bytes), 1, 8);
  uint32_t n = 8;
  while (n < 32 && rows > 1024ull * n * (kRowThreads / 32)) n *= 2;
  return n;
}

__device__ __forceinline__ void zero_unused(const Route &p, uint32_t elem_bytes) {
  const uint32_t lane = threadIdx.x % 32;
  const uint32_t r0 = (blockIdx.x * (kRowThreads / 32) + threadIdx.x / 32) * p.unused_rows;
  const bool mine = lane < p.unused_rows && r0 + lane < p.rows && lane % gridDim.y == blockIdx.y;
  uint32_t empty = __ballot_sync(~0u, mine && p.source[r0 + lane] < 0);
  if (!empty) return;
  const uint64_t pitch = p.out_pitch * elem_bytes;
  const uint32_t bytes = p.width * elem_bytes;
  const uint32_t unit = zero_unit(p.out, pitch, bytes);
  uint8_t *rows = static_cast<uint8_t *>(p.out) + r0 * pitch;
  for (; empty; empty &= empty - 1)
    zero_row<true>(rows + (__ffs(empty) - 1) * pitch, bytes, unit, lane);
}

// The thread's token and vector; false when it has none.
__device__ __forceinline__ bool my_vector(const Route &p, uint32_t *token, uint32_t *q) {
  const uint32_t i = blockIdx.y * kRowThreads + threadIdx.x;
  const uint32_t r = p.flat.stride.div(i);
  *token = (blockIdx.x - p.unused_blocks) * p.flat.group + r;
  *q = i - r * p.flat.stride.d;
  return i < p.flat.items && *token < p.tokens && *q < p.vectors;
}

// Rows moved as bytes (widths and pitches in bytes): units of N bytes, read once for
// all slots.  Bound by HBM, almost all of it writes: 16384 tokens x 8 slots of 8 KB go
// out at 6.3 TB/s (192 us), 147328 rows with the padding of 128 experts to 128 rows at
// 6.2 TB/s.  Fetching each row of the buffer from its token instead, so that rows are
// written front to back, reads every token's row 8 times from L2 and took 204 us.
template <int N>
__global__ void __launch_bounds__(kRowThreads) dispatch_kernel(Route p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x < p.unused_blocks) return zero_unused(p, 1);
  uint32_t token, q;
  if (!my_vector(p, &token, &q)) return;
  Words<N> in;
  in.load(static_cast<const uint8_t *>(p.in) + token * p.in_pitch + (uint64_t)q * N);
  const int32_t *dest = p.dest + (uint64_t)token * p.slots;
  for (uint32_t j = 0; j < p.slots; ++j) {
    const int32_t row = dest[j];
    if (row < 0 || (uint32_t)row >= p.rows) continue;
    in.store_cs(static_cast<uint8_t *>(p.out) + row * p.out_pitch + (uint64_t)q * N);
  }
}

// Rows at odd places: each row that is written is cut at its own 16-byte granules, so
// the token's row is read again (from L1) for each slot.
__global__ void __launch_bounds__(kRowThreads) dispatch_shift_kernel(Route p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x < p.unused_blocks) return zero_unused(p, 1);
  uint32_t token, q;
  if (!my_vector(p, &token, &q)) return;
  const uint8_t *src = static_cast<const uint8_t *>(p.in) + token * p.in_pitch;
  const int32_t *dest = p.dest + (uint64_t)token * p.slots;
  for (uint32_t j = 0; j < p.slots; ++j) {
    const int32_t row = dest[j];
    if (row < 0 || (uint32_t)row >= p.rows) continue;
    uint8_t *dst = static_cast<uint8_t *>(p.out) + row * p.out_pitch;
    const int32_t c = (int32_t)(q * 16) - row_lead<uint8_t, 16, true>(dst);
    if (c >= (int32_t)p.width) continue;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(src);
    const Words<16> in = load_shifted<16>(begin + (int64_t)c, begin, begin + p.width);
    if (whole<16, true>(c, p.width))
      in.store_cs(dst + c);
    else
      store_partial(dst + c, make_uint4(in.w[0], in.w[1], in.w[2], in.w[3]), max(0, -c),
                    min(16, (int32_t)p.width - c));
  }
}

// The same with a factor for each entry; pitches in elements, as below.
template <typename T, int V, bool kShift>
__global__ void __launch_bounds__(kRowThreads) dispatch_weighted_kernel(Route p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x < p.unused_blocks) return zero_unused(p, sizeof(T));
  uint32_t token, q;
  if (!my_vector(p, &token, &q)) return;
  const T *src = static_cast<const T *>(p.in) + token * p.in_pitch;
  Vec<T, V> in;
  if (!kShift) load_columns<T, V, kShift>(in, src, (int32_t)(q * V), p.width);
  for (uint32_t j = 0; j < p.slots; ++j) {
    const int32_t row = p.dest[(uint64_t)token * p.slots + j];
    if (row < 0 || (uint32_t)row >= p.rows) continue;
    const float w = p.weights[token * p.w_pitch + j];
    T *dst = static_cast<T *>(p.out) + row * p.out_pitch;
    const int32_t c = (int32_t)(q * V) - row_lead<T, V, kShift>(dst);
    if (c >= (int32_t)p.width) continue;
    if (kShift) load_columns<T, V, kShift>(in, src, c, p.width);
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = in.get(i) * w;
    Vec<T, V> out;
    out.put(f);
    store_columns<T, V, kShift>(out, dst, c, p.width);
  }
}

// A thread sums one vector of a token over its slots, four rows in flight, and writes it
// once.  Bound by HBM: 8191 x 4 x 5120 fp16 (a tenth dropped, 386 MB) take 63 us, 6.1
// TB/s.  Registers decide: at 64 a thread (four blocks an SM) it took 72 us.
template <typename T, int V, bool kShift>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(Route p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  uint32_t token, q;
  if (!my_vector(p, &token, &q)) return;
  T *dst = static_cast<T *>(p.out) + token * p.out_pitch;
  const int32_t c = (int32_t)(q * V) - row_lead<T, V, kShift>(dst);
  if (c >= (int32_t)p.width) return;
  float sum[V] = {};
  constexpr int kAhead = 4;
  for (uint32_t j0 = 0; j0 < p.slots; j0 += kAhead) {
    Vec<T, V> in[kAhead];
    float w[kAhead];
    bool kept[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const bool there = j0 + j < p.slots;
      const int32_t row = there ? p.dest[(uint64_t)token * p.slots + j0 + j] : -1;
      kept[j] = row >= 0 && (uint32_t)row < p.rows;
      w[j] = 1.0f;
      if (kept[j]) {
        load_columns<T, V, kShift>(in[j], static_cast<const T *>(p.in) + row * p.in_pitch, c,
                                   p.width);
        if (p.weights) w[j] = p.weights[token * p.w_pitch + j0 + j];
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (kept[j]) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = fmaf(w[j], in[j].get(i), sum[i]);
      }
  }
  Vec<T, V> out;
  out.put(sum);
  store_columns<T, V, kShift>(out, dst, c, p.width);
}

// (1 << lx) lanes take an entry, a warp at most or, where entries are few, a block: the
// token's row of dout meets the entry's row of y.  The entries of a token are neighbours, so that its row comes from
// L2 after the first.  Bound by HBM: 16384 x 8 x 2048 bf16 (1.14 GB) take 187 us, 6.1
// TB/s.  (A block a token, slot after slot, with block-wide sums: 210 us
// instead of 187 for 16384 tokens x 8 slots x 2048 bf16.)  The bound on blocks lets the
// compiler keep all loads of a step in flight (1501 x 2 x 1002 fp32: 9.7 us, 12.4 without).
template <typename T, int V>
__global__ void __launch_bounds__(kRowThreads, 4) combine_grad_kernel(Route p) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x < p.unused_blocks)
    return zero_unused(p, sizeof(T));
  const uint32_t entry =
      (blockIdx.x - p.unused_blocks) * (kRowThreads >> p.lx) + (threadIdx.x >> p.lx);
  const uint32_t lanes = 1u << p.lx, lane = threadIdx.x & (lanes - 1);
  const uint32_t token = p.by_slots.div(entry), slot = entry - token * p.slots;
  const bool there = token < p.tokens;
  const int32_t row = there ? p.dest[entry] : -1;
  float dot = 0.0f;
  if (row >= 0 && (uint32_t)row < p.rows) {
    const float w = p.weights[token * p.w_pitch + slot];
    constexpr int N = V * (int)sizeof(T), U = 4;
    const auto *dout = reinterpret_cast<const uint8_t *>(static_cast<const T *>(p.dout) +
                                                         token * p.dout_pitch);
    const auto *y = reinterpret_cast<const uint8_t *>(static_cast<const T *>(p.in) +
                                                      row * p.in_pitch);
    auto *dy = reinterpret_cast<uint8_t *>(static_cast<T *>(p.out) + row * p.out_pitch);
    for (uint32_t q = lane; q < p.vectors; q += U * lanes) {
      Vec<T, V> g[U], in[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u * lanes < p.vectors) {
          in[u].load(y + (uint64_t)(q + u * lanes) * N);
          g[u].load(dout + (uint64_t)(q + u * lanes) * N);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u * lanes < p.vectors) {
          float f[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float d = g[u].get(i);
            dot = fmaf(d, in[u].get(i), dot);
            f[i] = d * w;
          }
          Vec<T, V> out;
          out.put(f);
          out.store_cs(dy + (uint64_t)(q + u * lanes) * N);
        }
    }
  }
  for (uint32_t o = min(lanes, 32u) / 2; o; o /= 2) dot += __shfl_xor_sync(~0u, dot, o);
  if (lanes > 32) {  // the whole block's
    __shared__ float part[kRowThreads / 32];
    if (lane % 32 == 0) part[lane / 32] = dot;
    __syncthreads();
    dot = 0.0f;
    for (uint32_t w = 0; w < kRowThreads / 32; ++w) dot += part[w];
  }
  if (lane == 0 && there) p.dweights[token * p.dw_pitch + slot] = dot;
}

int check_route(const int32_t *dest, int64_t tokens, int64_t slots, const int32_t *source,
                int64_t rows, const DcopyMatrix *weights, const char *what) {
  if (slots < 0 || slots > INT32_MAX ||
      (unsigned __int128)tokens * (uint64_t)slots > (uint64_t)INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "%s: %lld tokens x %lld slots", what,
                     (long long)tokens, (long long)slots);
  const uint64_t n = (uint64_t)tokens * slots;
  if (int rc = check_array(dest, n, 4, "dest")) return rc;
  if (source)
    if (int rc = check_array(source, (uint64_t)rows, 4, "source")) return rc;
  if (weights) {
    if (int rc = check_matrix(weights, "weights", weights->type == kF32)) return rc;
    if (weights->rows != tokens || weights->cols != slots)
      return set_error(DCOPY_ERR_SHAPE_INVALID, "%s: weights are %lld x %lld, not %lld x %lld",
                       what, (long long)weights->rows, (long long)weights->cols,
                       (long long)tokens, (long long)slots);
  }
  return DCOPY_OK;
}

// What a call writes (`out`) lies apart from its routing.
int check_off_route(const DcopyMatrix *out, const char *name, const int32_t *dest, uint64_t entries,
                    const int32_t *source, uint64_t rows, const DcopyMatrix *weights,
                    const char *what) {
  const DcopyMatrix d = flat(dest, entries, kI32), s = flat(source, rows, kI32);
  if (int rc = check_apart(out, &d, what, name, "dest")) return rc;
  if (int rc = check_apart(out, &s, what, name, "source")) return rc;
  return weights ? check_apart(out, weights, what, name, "weights") : (int)DCOPY_OK;
}

int check_width(const DcopyMatrix *a, const DcopyMatrix *b, const char *what) {
  if (a->type != b->type)
    return set_error(DCOPY_ERR_DATATYPE_INVALID, "%s: element types %d and %d differ", what,
                     a->type, b->type);
  if (a->cols != b->cols)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "%s: widths %lld and %lld differ", what,
                     (long long)a->cols, (long long)b->cols);
  if (a->cols > kMaxWidth)
    return set_error(DCOPY_ERR_UNSUPPORTED, "%s: width %lld", what, (long long)a->cols);
  return DCOPY_OK;
}

// Blocks ahead of the others that zero the rows without an entry.
void plan_unused(Route &p, const int32_t *source, int elem_bytes) {
  p.unused_rows = unused_rows_of(p.rows, (uint64_t)p.tokens * p.slots, (uint64_t)p.width * elem_bytes);
  const uint32_t block = p.unused_rows * (kRowThreads / 32);
  p.unused_blocks = source ? (p.rows + block - 1) / block : 0;
}

// The grid of the kernels whose threads take a vector of a token's row.
dim3 token_grid(Route &p, const int32_t *source, int elem_bytes, bool whole_warps) {
  p.flat = flat_tokens(p.tokens, p.vectors, whole_warps);
  plan_unused(p, source, elem_bytes);
  return dim3(p.flat.grid.x + p.unused_blocks, std::max(1u, p.flat.grid.y));
}

}  // namespace
}  // namespace dcopy

using namespace dcopy;

extern "C" {

int dcopy_expert_rows(int64_t entries, int32_t experts, int32_t align, int64_t *rows) {
  DCOPY_API_BEGIN
  if (!rows || entries < 0 || experts < 1 || align < 1)
    return set_error(DCOPY_ERR_PARAM_INVALID, "expert_rows: %lld entries, %d experts, align %d",
                     (long long)entries, experts, align);
  if (entries > INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "expert_rows: %lld entries", (long long)entries);
  const int64_t r = entries + std::min<int64_t>(experts, entries) * (align - 1);
  if (r > INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "expert_rows: %lld rows", (long long)r);
  *rows = r;
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_expert_sort_workspace(int64_t entries, int32_t experts, uint64_t *bytes) {
  DCOPY_API_BEGIN
  if (experts > (int32_t)kMaxExperts)
    return set_error(DCOPY_ERR_UNSUPPORTED, "expert_sort_workspace: %d experts (at most %u)",
                     experts, kMaxExperts);
  if (!bytes || entries < 0 || entries > INT32_MAX || experts < 1)
    return set_error(DCOPY_ERR_PARAM_INVALID, "expert_sort_workspace: %lld entries, %d experts",
                     (long long)entries, experts);
  *bytes = sort_experts_bytes(entries, experts) + 16;
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_expert_sort(int32_t *dest, int32_t *source, int64_t rows, int32_t *offsets,
                      const DcopyMatrix *expert_ids, int32_t experts, int32_t align,
                      void *workspace, uint64_t workspace_bytes, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!expert_ids) return set_error(DCOPY_ERR_PARAM_INVALID, "expert_sort: NULL matrix");
  if (experts < 1 || align < 1)
    return set_error(DCOPY_ERR_PARAM_INVALID, "expert_sort: %d experts, align %d", experts, align);
  if (experts > (int32_t)kMaxExperts)
    return set_error(DCOPY_ERR_UNSUPPORTED, "expert_sort: %d experts (at most %u)", experts,
                     kMaxExperts);
  if (int rc = check_matrix(expert_ids, "expert_ids", is_index(expert_ids->type))) return rc;
  const uint64_t n = (uint64_t)expert_ids->rows * (uint64_t)expert_ids->cols;
  if (n > INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "expert_sort: %llu entries", (unsigned long long)n);
  int64_t least = 0;
  if (int rc = dcopy_expert_rows((int64_t)n, experts, align, &least)) return rc;
  if (rows < least || rows > INT32_MAX)
    return set_error(DCOPY_ERR_SHAPE_INVALID, "expert_sort: source has %lld rows, %lld needed",
                     (long long)rows, (long long)least);
  const uint64_t need = sort_experts_bytes(n, (uint32_t)experts);
  if (need && workspace_bytes < need + 16)
    return set_error(DCOPY_ERR_PARAM_INVALID, "expert_sort: workspace of %llu bytes, %llu needed",
                     (unsigned long long)workspace_bytes, (unsigned long long)need + 16);
  if (int rc = check_array(dest, n, 4, "dest")) return rc;
  if (int rc = check_array(source, (uint64_t)rows, 4, "source")) return rc;
  if (int rc = check_array(offsets, (uint64_t)experts + 1, 4, "offsets")) return rc;
  if (need)
    if (int rc = check_device_span(workspace, need + 16, "workspace")) return rc;
  // dest may be the ids themselves: an entry's id is read before its row is written, by
  // the same block.
  const DcopyMatrix out[] = {flat(dest, n, kI32), flat(source, (uint64_t)rows, kI32),
                             flat(offsets, (uint64_t)experts + 1, kI32),
                             flat(workspace, need ? need + 16 : 0, kU8)};
  const char *const name[] = {"dest", "source", "offsets", "workspace"};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < i; ++j)
      if (int rc = check_apart(&out[j], &out[i], "expert_sort", name[j], name[i])) return rc;
    const bool in_place = i == 0 && expert_ids->data == dest && expert_ids->type == kI32 &&
                          (expert_ids->rows <= 1 || expert_ids->pitch == expert_ids->cols);
    if (!in_place)
      if (int rc = check_apart(&out[i], expert_ids, "expert_sort", name[i], "expert_ids")) return rc;
  }
  KeySource src{};
  src.ids = expert_ids->data;
  src.pitch = expert_ids->pitch;
  src.keys = (uint32_t)experts;
  src.wide = expert_ids->type == kI64;
  src.n = (uint32_t)n;
  src.cols = FastDiv((uint32_t)std::max<int64_t>(1, expert_ids->cols));
  void *ws = reinterpret_cast<void *>(((uintptr_t)workspace + 15) / 16 * 16);
  return sort_experts(src, (uint32_t)align, dest, source, (uint32_t)rows, offsets, ws, stream);
  DCOPY_API_END
}

int dcopy_expert_dispatch(const DcopyMatrix *out, const DcopyMatrix *x, const int32_t *dest,
                          int64_t slots, const int32_t *source, const DcopyMatrix *weights,
                          dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!out || !x) return set_error(DCOPY_ERR_PARAM_INVALID, "expert_dispatch: NULL matrix");
  if (int rc = check_matrix(out, "out", weights ? is_float(out->type) : elem_size(out->type) > 0))
    return rc;
  if (int rc = check_matrix(x, "x", weights ? is_float(x->type) : elem_size(x->type) > 0))
    return rc;
  if (int rc = check_width(out, x, "expert_dispatch")) return rc;
  if (int rc = check_route(dest, x->rows, slots, source, out->rows, weights, "expert_dispatch"))
    return rc;
  if (int rc = check_apart(out, x, "expert_dispatch", "out", "x")) return rc;
  if (int rc = check_off_route(out, "out", dest, (uint64_t)x->rows * slots, source, out->rows,
                               weights, "expert_dispatch"))
    return rc;
  if (out->rows == 0 || out->cols == 0) return DCOPY_OK;
  Route p{};
  p.out = out->data;
  p.in = x->data;
  p.dest = dest;
  p.source = source;
  p.tokens = (uint32_t)x->rows;
  p.slots = (uint32_t)slots;
  p.rows = (uint32_t)out->rows;
  if (weights) {
    p.weights = static_cast<const float *>(weights->data);
    p.w_pitch = weights->pitch;
    p.out_pitch = out->pitch;
    p.in_pitch = x->pitch;
    p.width = (uint32_t)out->cols;
    return with_float(out->type, [&](auto t) {
      using T = typename decltype(t)::type;
      constexpr int kFull = 16 / sizeof(T), kLeast = 8 / sizeof(T);
      const Cut cut = cut_rows(kFull, kLeast, out, x);
      p.vectors = vectors_of(out->cols, cut);
      const dim3 grid = token_grid(p, source, sizeof(T), true);
      if (grid.x == 0) return (int)DCOPY_OK;
      return with_cut<kFull, kLeast>(cut, [&](auto v, auto shift) {
        return launch_grid(dispatch_weighted_kernel<T, v(), shift()>, grid, dim3(kRowThreads), 0,
                           stream, "dispatch_weighted_kernel", p);
      });
    });
  }
  const int eb = elem_size(out->type);
  p.out_pitch = out->pitch * eb;
  p.in_pitch = x->pitch * eb;
  p.width = (uint32_t)out->cols * eb;
  const uint64_t all = (uintptr_t)out->data | (uintptr_t)x->data | p.width |
                       (out->rows > 1 ? p.out_pitch : 0) | (x->rows > 1 ? p.in_pitch : 0);
  // Shifted below 8-byte units (24390 x 4 rows of 1025 bf16: 60 us against 145 in single
  // elements; of 1026: 58 against 101 in 4-byte units; of 1028 in 8-byte units 54 against 56
  // shifted).
  const Cut cut = all % 16 == 0 ? Cut{16, false} : all % 8 == 0 ? Cut{8, false} : Cut{16, true};
  p.vectors = vectors_of(p.width, cut);
  const dim3 grid = token_grid(p, source, 1, true);
  if (grid.x == 0) return DCOPY_OK;
  auto k = cut.shift ? dispatch_shift_kernel : cut.v == 16 ? dispatch_kernel<16> : dispatch_kernel<8>;
  return launch_grid(k, grid, dim3(kRowThreads), 0, stream, "dispatch_kernel", p);
  DCOPY_API_END
}

int dcopy_expert_combine(const DcopyMatrix *out, const DcopyMatrix *y, const int32_t *dest,
                         int64_t slots, const DcopyMatrix *weights, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!out || !y) return set_error(DCOPY_ERR_PARAM_INVALID, "expert_combine: NULL matrix");
  if (int rc = check_matrix(out, "out", is_float(out->type))) return rc;
  if (int rc = check_matrix(y, "y", is_float(y->type))) return rc;
  if (int rc = check_width(out, y, "expert_combine")) return rc;
  if (int rc = check_route(dest, out->rows, slots, nullptr, 0, weights, "expert_combine")) return rc;
  if (int rc = check_apart(out, y, "expert_combine", "out", "y")) return rc;
  if (int rc = check_off_route(out, "out", dest, (uint64_t)out->rows * slots, nullptr, 0, weights,
                               "expert_combine"))
    return rc;
  if (out->rows == 0 || out->cols == 0) return DCOPY_OK;
  Route p{};
  p.out = out->data;
  p.in = y->data;
  p.out_pitch = out->pitch;
  p.in_pitch = y->pitch;
  p.dest = dest;
  if (weights) {
    p.weights = static_cast<const float *>(weights->data);
    p.w_pitch = weights->pitch;
  }
  p.tokens = (uint32_t)out->rows;
  p.slots = (uint32_t)slots;
  p.rows = (uint32_t)y->rows;
  p.width = (uint32_t)out->cols;
  return with_float(out->type, [&](auto t) {
    using T = typename decltype(t)::type;
    // Shifted where single 2-byte elements would be read (24390 x 4 choices of 1025 bf16: 84
    // us against 132); 4-byte vectors do as they are (1026: 70 us against 86 shifted).
    constexpr int kFull = 16 / sizeof(T), kLeast = 4 / sizeof(T);
    const Cut cut = cut_rows(kFull, kLeast, out, y);
    p.vectors = vectors_of(out->cols, cut);
    const dim3 grid = token_grid(p, nullptr, sizeof(T), false);
    return with_cut<kFull, kLeast>(cut, [&](auto v, auto shift) {
      return launch_grid(combine_kernel<T, v(), shift()>, grid, dim3(kRowThreads), 0, stream,
                         "combine_kernel", p);
    });
  });
  DCOPY_API_END
}

int dcopy_expert_combine_grad(const DcopyMatrix *dy, const DcopyMatrix *dweights,
                              const DcopyMatrix *dout, const DcopyMatrix *y, const int32_t *dest,
                              int64_t slots, const int32_t *source, const DcopyMatrix *weights,
                              dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!dy || !dweights || !dout || !y || !weights)
    return set_error(DCOPY_ERR_PARAM_INVALID, "expert_combine_grad: NULL matrix");
  if (int rc = check_matrix(dy, "dy", is_float(dy->type))) return rc;
  if (int rc = check_matrix(dout, "dout", is_float(dout->type))) return rc;
  if (int rc = check_matrix(y, "y", is_float(y->type))) return rc;
  if (int rc = check_matrix(dweights, "dweights", dweights->type == kF32)) return rc;
  if (int rc = check_width(dy, dout, "expert_combine_grad")) return rc;
  if (int rc = check_width(dy, y, "expert_combine_grad")) return rc;
  if (int rc = check_route(dest, dout->rows, slots, source, dy->rows, weights,
                           "expert_combine_grad"))
    return rc;
  if (dy->rows != y->rows || dweights->rows != dout->rows || dweights->cols != slots)
    return set_error(DCOPY_ERR_SHAPE_INVALID,
                     "expert_combine_grad: dy has %lld rows for %lld of y, dweights is %lld x %lld",
                     (long long)dy->rows, (long long)y->rows, (long long)dweights->rows,
                     (long long)dweights->cols);
  // dweights may be the weights themselves: an entry's weight is read before its gradient
  // is written, by the same warp or behind a barrier.
  const char *what = "expert_combine_grad";
  const uint64_t all = (uint64_t)dout->rows * slots;
  const DcopyMatrix *other = same_rows(dweights, weights) ? nullptr : weights;
  if (int rc = check_apart(dy, y, what, "dy", "y")) return rc;
  if (int rc = check_apart(dy, dout, what, "dy", "dout")) return rc;
  if (int rc = check_apart(dy, dweights, what, "dy", "dweights")) return rc;
  if (int rc = check_apart(dweights, y, what, "dweights", "y")) return rc;
  if (int rc = check_apart(dweights, dout, what, "dweights", "dout")) return rc;
  if (int rc = check_off_route(dy, "dy", dest, all, source, dy->rows, weights, what)) return rc;
  if (int rc = check_off_route(dweights, "dweights", dest, all, source, dy->rows, other, what))
    return rc;
  Route p{};
  p.out = dy->data;
  p.in = y->data;
  p.dout = dout->data;
  p.dweights = static_cast<float *>(dweights->data);
  p.out_pitch = dy->pitch;
  p.in_pitch = y->pitch;
  p.dout_pitch = dout->pitch;
  p.w_pitch = weights->pitch;
  p.dw_pitch = dweights->pitch;
  p.dest = dest;
  p.source = source;
  p.weights = static_cast<const float *>(weights->data);
  p.tokens = (uint32_t)dout->rows;
  p.slots = (uint32_t)slots;
  p.rows = (uint32_t)dy->rows;
  p.width = (uint32_t)dy->cols;
  plan_unused(p, source, elem_size(dy->type));
  p.by_slots = FastDiv((uint32_t)std::max<int64_t>(1, slots));
  const uint64_t entries = (uint64_t)p.tokens * p.slots;
  return with_float(dy->type, [&](auto t) {
    using T = typename decltype(t)::type;
    // Never shifted: 24390 x 4 entries of 1025 bf16 take 138 us in single elements, 182
    // shifted.
    constexpr int kFull = 16 / sizeof(T);
    const Cut cut = cut_rows(kFull, 1, dy, dout, y);
    p.vectors = vectors_of(dy->cols, cut);
    p.lx = 0;
    while (p.lx < 5 && (1u << p.lx) < p.vectors) ++p.lx;
    // A block an entry where entries are too few for warps alone to fill the SMs.  A wide row
    // keeps a block's threads at work, so the entries an SM grow with it.  Us with a block
    // against a warp, on the block's side of the limit, then on the warp's: 1024 bf16, 300
    // entries 2.1 : 2.3, 600 entries 2.9 : 2.4; 2048 bf16, 800 entries 3.5 : 3.9, 1900 entries
    // 6.5 : 5.1; 4096 bf16, 1600 entries 7.9 : 9.5, 2200 entries 10.4 : 10.0.  Widest rows gain
    // least at the limit: 8192 fp32, 80 entries 3.7 : 8.9, 2200 entries 28.5 : 31.7, 8000
    // entries 97 : 103.
    if (p.vectors >= 128 && entries <= std::min(p.vectors / 40, 16u) * (uint64_t)sm_count())
      p.lx = 8;
    const uint64_t per_block = kRowThreads >> p.lx;
    const uint64_t blocks = p.unused_blocks + (entries + per_block - 1) / per_block;
    if (blocks == 0) return (int)DCOPY_OK;
    return with_cut<kFull, 1>(cut, [&](auto v, auto) {
      return launch(combine_grad_kernel<T, v()>, (unsigned)blocks, dim3(kRowThreads), 0, stream,
                    "combine_grad_kernel", p);
    });
  });
  DCOPY_API_END
}

}  // extern "C"
