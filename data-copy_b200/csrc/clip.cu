// The global gradient norm over many tensors, and clipping.
//
// total = sum over all tensors of g^2; norm = sqrt(total);
// c = min(1, max_norm / (norm + eps)); out = round(c * g).
// A thread sums the squares of a chunk in fp32, the chunks and blocks in fp64, in an
// order that the tensor sizes fix: the same bits on every run.  Two passes over the
// gradients; bound by HBM bytes, launches where the tensors are small.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cstring>
#include <string>
#include <vector>

#include "common.cuh"
#include "launch.cuh"
#include "rowops.cuh"

namespace dcopy {
namespace {

constexpr int kThreads = 256;
// Bytes that a thread has in flight: 537 M bf16 elements take 487 us with 128, 521 with
// 64.
constexpr int kAhead = 128;

// Elements of a chunk: 32 squares a thread in fp32, 0.2 % of the bytes for the table;
// half of that in lists with fewer chunks than blocks at work (1.5 M fp32: 7.1 us with
// 4096, 8.2 with 8192; 537 M bf16: 634 us with 4096, 495 with 8192).
constexpr uint32_t kChunk = 8192, kSmallChunk = 4096;
constexpr uint64_t kSmallList = 512 * kChunk;

// A piece of one tensor.  `head` elements come before the first that starts a 16-byte
// granule of src and a whole vector of dst; with head == count there is none.
struct alignas(16) Chunk {
  const void *src;
  void *dst;
  uint32_t count, head;
  uint64_t pad;
};
static_assert(sizeof(Chunk) == 32, "Chunk is 32 bytes");

// The caller's buffer: one partial sum for each block of the first pass, the chunks,
// those of one pair of types after the other (a kernel for each pair that occurs: one
// kernel for all of them took 193 registers instead of 40).
constexpr uint32_t kMaxBlocks = 2048;  // of one source type
constexpr uint64_t kPartBytes = 3 * kMaxBlocks * sizeof(double);
constexpr int kPairs = 9;
constexpr int32_t kTypes[3] = {kF32, kF16, kBF16};

int type_index(int32_t type) { return type == kF32 ? 0 : type == kF16 ? 1 : 2; }

struct List {
  const Chunk *chunk;
  double *part;
  uint32_t chunks;
};

__device__ __forceinline__ Chunk load_chunk(const Chunk *c) {
  union {
    Chunk chunk;
    uint4 word[2];
  } u;
  u.word[0] = __ldg(reinterpret_cast<const uint4 *>(c));
  u.word[1] = __ldg(reinterpret_cast<const uint4 *>(c) + 1);
  return u.chunk;
}

// Calls f(vector, first element) on this thread's share of a chunk: vectors of V
// elements, U loads ahead, and single elements at the ends.  The share does not depend
// on U.
template <typename T, int V, int U, typename F>
__device__ __forceinline__ void each_vector(const Chunk &c, F &&f) {
  const T *src = static_cast<const T *>(c.src);
  const uint32_t vectors = (c.count - c.head) / V, tail = c.head + vectors * V;
#pragma unroll 1
  for (uint32_t i0 = threadIdx.x; i0 < vectors; i0 += kThreads * U) {
    Vec<T, V> in[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kThreads < vectors) in[u].load_plain(src + c.head + (i0 + u * kThreads) * V);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kThreads < vectors) f(in[u], c.head + (i0 + u * kThreads) * V);
  }
  const uint32_t ends = c.head + c.count - tail;  // head and tail in one loop
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < ends; i += kThreads) {
    const uint32_t e = i < c.head ? i : tail + i - c.head;
    Vec<T, 1> in;
    in.load_plain(src + e);
    f(in, e);
  }
}

__device__ __forceinline__ double block_sum(double v, double *warp_sum) {
#pragma unroll
  for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) all += warp_sum[w];
  return all;
}

// This thread's sum of squares over one chunk in fp32, unless they leave its range
// (above 2^127, or so small that what underflows could count): then again in fp64.
template <typename T>
__device__ __forceinline__ double chunk_squares(const Chunk &c) {
  constexpr int V = 16 / sizeof(T);
  float sum = 0.0f;
  uint32_t bits = 0;
  each_vector<T, V, kAhead / 16>(c, [&](const auto &v, uint32_t) {
#pragma unroll
    for (int i = 0; i < v.kSize; ++i) sum = fmaf(v.get(i), v.get(i), sum);
#pragma unroll
    for (int i = 0; i < v.kWords; ++i) bits |= v.w[i];
  });
  if (bits == 0 || (sum >= 0x1p-90f && sum < 0x1p+127f)) return sum;
  double wide = 0.0;
  each_vector<T, V, 1>(c, [&](const auto &v, uint32_t) {
#pragma unroll
    for (int i = 0; i < v.kSize; ++i) wide = fma((double)v.get(i), (double)v.get(i), wide);
  });
  return wide;
}

// Bound by HBM reads: 537 M bf16 elements (1.07 GB) at 6.6 to 7.0 TB/s (152 us).
template <typename T>
__global__ void __launch_bounds__(kThreads) sum_squares_kernel(List l) {
  __shared__ double warp_sum[kThreads / 32];
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  double sum = 0.0;
  Chunk next = load_chunk(l.chunk + blockIdx.x);
  for (uint32_t k = blockIdx.x; k < l.chunks; k += gridDim.x) {
    const Chunk c = next;
    if (k + gridDim.x < l.chunks) next = load_chunk(l.chunk + k + gridDim.x);
    sum += chunk_squares<T>(c);
  }
  sum = block_sum(sum, warp_sum);
  if (threadIdx.x == 0) l.part[blockIdx.x] = sum;
}

// The sum of the first pass's partial sums, the same in every block.
__device__ __forceinline__ double sum_parts(const double *part, uint32_t parts) {
  __shared__ double warp_sum[kThreads / 32];
  double v = 0.0;
  for (uint32_t b = threadIdx.x; b < parts; b += kThreads) v += part[b];
  return block_sum(v, warp_sum);
}

__global__ void __launch_bounds__(kThreads) total_kernel(List l, uint32_t parts, double *total) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  const double all = sum_parts(l.part, parts);
  if (threadIdx.x == 0) *total = all;
}

// total NULL: the partial sums of the pass before are added up here, by every block.
// Bound by HBM: 1.07 GB in and out at 6.3 to 6.7 TB/s (319 us alone, 495 us with the
// first pass).  Nothing on the chip holds such a list between the passes; hints to keep
// the end of it in L2 changed nothing (503 us).
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) clip_kernel(List l, uint32_t parts, const double *total,
                                                        float max_norm, float eps, float *norm_out) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  const float norm = (float)sqrt(total ? *total : sum_parts(l.part, parts));
  const float ratio = max_norm / (norm + eps);
  const float f = ratio < 1.0f || ratio != ratio ? ratio : 1.0f;  // NaN goes on
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  if (blockIdx.x >= l.chunks) return;
  // Last chunk first: what the first pass read last is still in L2.
  Chunk next = load_chunk(l.chunk + (l.chunks - 1 - blockIdx.x));
  for (uint32_t k = blockIdx.x; k < l.chunks; k += gridDim.x) {
    const Chunk c = next;
    if (k + gridDim.x < l.chunks) next = load_chunk(l.chunk + (l.chunks - 1 - k - gridDim.x));
    if (f == 1.0f && c.src == c.dst) continue;  // in place: nothing changes
    O *dst = static_cast<O *>(c.dst);
    constexpr int V = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
    each_vector<T, V, kAhead / (V * sizeof(T))>(c, [&](const auto &v, uint32_t e) {
      constexpr int kSize = std::decay_t<decltype(v)>::kSize;
      float g[kSize];
#pragma unroll
      for (int i = 0; i < kSize; ++i) g[i] = v.get(i) * f;
      Vec<O, kSize> out;
      out.put(g);
      out.store(dst + e);
    });
  }
}

// Elements before the first at which src starts a 16-byte granule and dst a vector of
// as many elements; count when there is none.
uint64_t head_of(const DcopyGrad &g) {
  const int sb = elem_size(g.src_type), db = elem_size(g.dst_type), v = 16 / sb;
  const uintptr_t s = (uintptr_t)g.src, d = (uintptr_t)g.dst;
  for (uint64_t head = 0; head < (uint64_t)v && head < g.count; ++head)
    if ((s + head * sb) % 16 == 0 && (d + head * db) % std::min(16, v * db) == 0) return head;
  return g.count;
}

// Chunks that grads can have at most, whatever their alignment: one more each than
// their elements need, as heads shift the chunk ends.
uint64_t most_chunks(const DcopyGrad *grads, uint32_t n, uint32_t size) {
  uint64_t chunks = 0;
  for (uint32_t i = 0; i < n; ++i) chunks += (grads[i].count + size - 1) / size + 1;
  return chunks;
}

uint32_t chunk_size(const DcopyGrad *grads, uint32_t n) {
  uint64_t all = 0;
  for (uint32_t i = 0; i < n; ++i) all += grads[i].count;
  return all < kSmallList ? kSmallChunk : kChunk;
}

uint64_t list_bytes(uint64_t chunks) { return kPartBytes + chunks * sizeof(Chunk); }

int check_grads(const DcopyGrad *grads, uint32_t n, const char *what) {
  if (!grads && n) return set_error(DCOPY_ERR_PARAM_INVALID, "%s: NULL gradients", what);
  if (n > (1u << 24)) return set_error(DCOPY_ERR_UNSUPPORTED, "%s: %u tensors", what, n);
  for (uint32_t i = 0; i < n; ++i)
    if (grads[i].count >> 40)
      return set_error(DCOPY_ERR_SHAPE_INVALID, "%s: gradient %u has %llu elements", what, i,
                       (unsigned long long)grads[i].count);
  if (most_chunks(grads, n, kSmallChunk) >> 31)
    return set_error(DCOPY_ERR_UNSUPPORTED, "%s: too many elements", what);
  return DCOPY_OK;
}

// Memory that a list reads or writes, and the gradient it belongs to.
struct Span {
  uintptr_t begin, end;
  uint32_t gradient;
  bool written;
};
constexpr uint32_t kSpanOfWorkspace = UINT32_MAX;

std::string name_of(const Span &s) {
  if (s.gradient == kSpanOfWorkspace) return "the workspace";
  return (s.written ? "the output of gradient " : "gradient ") + std::to_string(s.gradient);
}

// What is written meets nothing else: the chunks of a list run in any order.
int check_spans(std::vector<Span> &spans) {
  std::sort(spans.begin(), spans.end(),
            [](const Span &a, const Span &b) { return a.begin < b.begin; });
  const Span *furthest = nullptr, *written = nullptr;  // of those before, by their ends
  for (const Span &s : spans) {
    const Span *other = s.written ? furthest : written;
    if (other && s.begin < other->end)
      return set_error(DCOPY_ERR_PARAM_INVALID, "%s overlaps %s", name_of(s).c_str(),
                       name_of(*other).c_str());
    if (!furthest || s.end > furthest->end) furthest = &s;
    if (s.written && (!written || s.end > written->end)) written = &s;
  }
  return DCOPY_OK;
}

int open_list(const DcopyGradList *list) {
  if (!list || !list->workspace)
    return set_error(DCOPY_ERR_PARAM_INVALID, "gradient list: not built");
  return check_device_span(list->workspace, list_bytes(list->first[kPairs]), "workspace");
}

// A number that a call on a list reads or writes lies apart from the list's workspace.
int check_number(const DcopyGradList *list, const void *at, uint64_t bytes, const char *name) {
  if (int rc = check_array(at, 1, bytes, name)) return rc;
  return check_disjoint(list->workspace, list_bytes(list->first[kPairs]), at, bytes, name);
}

// The chunks [begin, end) of a list.
List part_of(const DcopyGradList *list, uint32_t begin, uint32_t end) {
  uint8_t *w = static_cast<uint8_t *>(list->workspace);
  return List{reinterpret_cast<const Chunk *>(w + kPartBytes) + begin,
              reinterpret_cast<double *>(w), end - begin};
}

// Blocks of a pass: as many as fit at once, five and four an SM.  Fixed numbers, since
// the order of the sums hangs on them.
uint32_t list_grid(uint32_t chunks, uint32_t per_sm) {
  return std::min({chunks, per_sm * (uint32_t)sm_count(), kMaxBlocks});
}

// The first pass: a launch for each source type; *parts partial sums.
int run_sum(const DcopyGradList *list, uint32_t *parts, cudaStream_t s) {
  *parts = 0;
  for (int t = 0; t < 3; ++t) {
    const uint32_t begin = list->first[3 * t], end = list->first[3 * t + 3];
    if (begin == end) continue;
    List l = part_of(list, begin, end);
    l.part += *parts;
    const int rc = with_float(kTypes[t], [&](auto tag) {
      auto k = sum_squares_kernel<typename decltype(tag)::type>;
      const uint32_t grid = list_grid(l.chunks, 5);
      *parts += grid;
      return launch(k, grid, dim3(kThreads), 0, s, "sum_squares_kernel", l);
    });
    if (rc) return rc;
  }
  return DCOPY_OK;
}

// The second: a launch for each pair of types, the last one first.  An empty list
// still has a norm.
int run_clip(const DcopyGradList *list, uint32_t parts, const double *total, float max_norm,
             float eps, float *norm, cudaStream_t s) {
  bool any = false;
  for (int q = kPairs - 1; q >= 0; --q) {
    const uint32_t begin = list->first[q], end = list->first[q + 1];
    if (begin == end && (q > 0 || any)) continue;
    any = true;
    List l = part_of(list, begin, end);
    l.part = part_of(list, 0, 0).part;
    const int rc = with_float(kTypes[q / 3], [&](auto tin) {
      return with_float(kTypes[q % 3], [&](auto tout) {
        auto k = clip_kernel<typename decltype(tin)::type, typename decltype(tout)::type>;
        return launch(k, std::max(1u, list_grid(l.chunks, 4)), dim3(kThreads), 0, s, "clip_kernel",
                      l, parts, total, max_norm, eps, norm);
      });
    });
    if (rc) return rc;
  }
  return DCOPY_OK;
}

int check_bound(float max_norm, float eps, const char *what) {
  if (!(max_norm >= 0.0f) || !(eps >= 0.0f))
    return set_error(DCOPY_ERR_PARAM_INVALID, "%s: max_norm %g, eps %g", what, max_norm, eps);
  return DCOPY_OK;
}

}  // namespace
}  // namespace dcopy

using namespace dcopy;

extern "C" {

int dcopy_grad_list_workspace(const DcopyGrad *grads, uint32_t n, uint64_t *bytes) {
  DCOPY_API_BEGIN
  if (!bytes) return set_error(DCOPY_ERR_PARAM_INVALID, "grad_list_workspace: NULL");
  if (int rc = check_grads(grads, n, "grad_list_workspace")) return rc;
  *bytes = list_bytes(most_chunks(grads, n, chunk_size(grads, n)));
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_grad_list_build(DcopyGradList *list, const DcopyGrad *grads, uint32_t n,
                          void *workspace, uint64_t workspace_bytes, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!list) return set_error(DCOPY_ERR_PARAM_INVALID, "grad_list_build: NULL list");
  if (int rc = check_grads(grads, n, "grad_list_build")) return rc;
  const uint32_t size = chunk_size(grads, n);
  const uint64_t need = list_bytes(most_chunks(grads, n, size));
  if (workspace_bytes < need || (uintptr_t)workspace % 16)
    return set_error(DCOPY_ERR_PARAM_INVALID,
                     "grad_list_build: workspace of %llu bytes at %p, %llu needed, 16-byte aligned",
                     (unsigned long long)workspace_bytes, workspace, (unsigned long long)need);
  if (int rc = check_device_span(workspace, need, "workspace")) return rc;
  std::vector<Chunk> chunks[kPairs];
  std::vector<Span> spans{{(uintptr_t)workspace, (uintptr_t)workspace + need, kSpanOfWorkspace, true}};
  for (uint32_t i = 0; i < n; ++i) {
    const DcopyGrad &g = grads[i];
    if (!is_float(g.src_type) || !is_float(g.dst_type))
      return set_error(DCOPY_ERR_DATATYPE_INVALID, "gradient %u: element types %d and %d", i,
                       g.src_type, g.dst_type);
    if (g.count == 0) continue;
    const uint64_t sb = elem_size(g.src_type), db = elem_size(g.dst_type);
    if ((uintptr_t)g.src % sb || (uintptr_t)g.dst % db)
      return set_error(DCOPY_ERR_PARAM_INVALID, "gradient %u is not aligned to its elements", i);
    if (int rc = check_device_span(g.src, g.count * sb, "gradient")) return rc;
    if (int rc = check_device_span(g.dst, g.count * db, "clipped gradient")) return rc;
    if (g.src != g.dst || g.src_type != g.dst_type)  // else in place
      spans.push_back({(uintptr_t)g.src, (uintptr_t)g.src + g.count * sb, i, false});
    spans.push_back({(uintptr_t)g.dst, (uintptr_t)g.dst + g.count * db, i, true});
    // The first chunk takes the head too; the others start on a vector.
    std::vector<Chunk> &mine = chunks[3 * type_index(g.src_type) + type_index(g.dst_type)];
    const uint64_t head = head_of(g);
    const bool scalar = head == g.count;
    for (uint64_t at = 0; at < g.count;) {
      const uint64_t most = at == 0 && !scalar ? head + size : size;
      Chunk c{};
      c.src = static_cast<const uint8_t *>(g.src) + at * sb;
      c.dst = static_cast<uint8_t *>(g.dst) + at * db;
      c.count = (uint32_t)std::min<uint64_t>(most, g.count - at);
      c.head = scalar ? c.count : at == 0 ? (uint32_t)head : 0;
      mine.push_back(c);
      at += c.count;
    }
  }
  if (int rc = check_spans(spans)) return rc;
  list->workspace = workspace;
  list->first[0] = 0;
  for (int q = 0; q < kPairs; ++q) {
    const uint32_t begin = list->first[q];
    list->first[q + 1] = begin + (uint32_t)chunks[q].size();
    if (!chunks[q].empty())
      DCOPY_CUDA_TRY(cudaMemcpyAsync(const_cast<Chunk *>(part_of(list, begin, begin).chunk),
                                     chunks[q].data(), chunks[q].size() * sizeof(Chunk),
                                     cudaMemcpyHostToDevice, stream));
  }
  DCOPY_CUDA_TRY(cudaStreamSynchronize(stream));
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_grad_sum_squares(const DcopyGradList *list, double *total, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (int rc = open_list(list)) return rc;
  if (int rc = check_number(list, total, sizeof(double), "total")) return rc;
  uint32_t parts = 0;
  if (int rc = run_sum(list, &parts, stream)) return rc;
  return launch(total_kernel, 1, dim3(kThreads), 0, stream, "total_kernel", part_of(list, 0, 0),
                parts, total);
  DCOPY_API_END
}

int dcopy_grad_clip(const DcopyGradList *list, const double *total, float max_norm, float eps,
                    float *norm, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (int rc = check_bound(max_norm, eps, "grad_clip")) return rc;
  if (int rc = open_list(list)) return rc;
  if (int rc = check_number(list, total, sizeof(double), "total")) return rc;
  if (norm)
    if (int rc = check_number(list, norm, sizeof(float), "norm")) return rc;
  if (int rc = check_disjoint(total, sizeof(double), norm, norm ? sizeof(float) : 0, "total, norm"))
    return rc;
  return run_clip(list, 0, total, max_norm, eps, norm, stream);
  DCOPY_API_END
}

int dcopy_clip_grad_norm(const DcopyGradList *list, float max_norm, float eps, float *norm,
                         dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (int rc = check_bound(max_norm, eps, "clip_grad_norm")) return rc;
  if (int rc = open_list(list)) return rc;
  if (norm)
    if (int rc = check_number(list, norm, sizeof(float), "norm")) return rc;
  uint32_t parts = 0;
  if (int rc = run_sum(list, &parts, stream)) return rc;
  return run_clip(list, parts, nullptr, max_norm, eps, norm, stream);
  DCOPY_API_END
}

}  // extern "C"
