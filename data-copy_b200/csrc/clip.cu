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
#include <vector>

#include "common.cuh"
#include "launch.cuh"
#include "rowops.cuh"

namespace dcopy {
namespace {

constexpr int kThreads = 512;
constexpr int kV = 8;                         // elements a thread takes at once
constexpr int kUnroll = 4;
constexpr uint32_t kChunk = kThreads * kV * kUnroll;  // elements of one step of a block

// One tensor of the list as the kernels read it.
struct Entry {
  const void *src;
  void *dst;
  uint64_t count;
  uint32_t first_chunk;  // chunks of the tensors before it
  uint8_t src_type, dst_type, vector, pad;
};
static_assert(sizeof(Entry) == 32, "Entry is 32 bytes");

// The caller's buffer: a header, the entries, one partial sum a block.
struct Header {
  double total;
  uint32_t done;   // blocks that have written their partial sum
  uint32_t pad[13];
};
static_assert(sizeof(Header) == 64, "Header is 64 bytes");
constexpr uint32_t kMaxBlocks = 4096;

struct List {
  Header *header;
  const Entry *entry;
  double *part;
  uint32_t count, chunks;
};

// The entry that holds a chunk: the last whose first_chunk is not above it.
__device__ __forceinline__ uint32_t find_entry(const List &l, uint32_t chunk) {
  uint32_t lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (l.entry[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Calls f(vector, index of its first element) on this thread's vectors of one chunk,
// kUnroll loads in flight.
template <typename T, int V, typename F>
__device__ __forceinline__ void each_vector(const T *src, uint64_t begin, uint64_t end, F &&f) {
  constexpr int kSteps = kV / V * kUnroll;
#pragma unroll
  for (int u0 = 0; u0 < kSteps; u0 += kUnroll) {
    Vec<T, V> in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t e = begin + ((uint64_t)(u0 + u) * kThreads + threadIdx.x) * V;
      if (e < end) in[u].load_plain(src + e);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t e = begin + ((uint64_t)(u0 + u) * kThreads + threadIdx.x) * V;
      if (e < end) f(in[u], e);
    }
  }
}

template <typename F>
__device__ __forceinline__ void by_type(int type, F &&f) {
  if (type == kF32) f(TypeTag<float>{});
  else if (type == kF16) f(TypeTag<__half>{});
  else f(TypeTag<__nv_bfloat16>{});
}

__device__ __forceinline__ double block_sum(double v, double *warp_sum) {
#pragma unroll
  for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) all += warp_sum[w];
  return all;
}

// This thread's sum of squares over one chunk: at most 32 of them, in fp32, unless
// they leave fp32's range (above 2^128, or so small that what underflows could count):
// then once more in fp64.
template <typename T, int V>
__device__ __forceinline__ double chunk_squares(const T *src, uint64_t begin, uint64_t end) {
  float sum = 0.0f;
  uint32_t bits = 0;
  each_vector<T, V>(src, begin, end, [&](const Vec<T, V> &v, uint64_t) {
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fmaf(v.get(i), v.get(i), sum);
#pragma unroll
    for (int i = 0; i < Vec<T, V>::kWords; ++i) bits |= v.w[i];
  });
  if (bits == 0 || (sum >= 0x1p-90f && sum < 0x1p+127f)) return sum;
  double wide = 0.0;
  each_vector<T, V>(src, begin, end, [&](const Vec<T, V> &v, uint64_t) {
#pragma unroll
    for (int i = 0; i < V; ++i) wide = fma((double)v.get(i), (double)v.get(i), wide);
  });
  return wide;
}

__global__ void __launch_bounds__(kThreads) sum_squares_kernel(List l) {
  __shared__ double warp_sum[kThreads / 32];
  __shared__ bool last;
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  double wide = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < l.chunks; chunk += gridDim.x) {
    const Entry t = l.entry[find_entry(l, chunk)];
    const uint64_t begin = (uint64_t)(chunk - t.first_chunk) * kChunk;
    const uint64_t end = min(begin + kChunk, t.count);
    by_type(t.src_type, [&](auto tag) {
      using T = typename decltype(tag)::type;
      const T *src = static_cast<const T *>(t.src);
      wide += t.vector ? chunk_squares<T, kV>(src, begin, end)
                       : chunk_squares<T, 1>(src, begin, end);
    });
  }
  const double all = block_sum(wide, warp_sum);
  if (threadIdx.x == 0) {
    l.part[blockIdx.x] = all;
    __threadfence();
    last = atomicAdd(&l.header->done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (uint32_t b = threadIdx.x; b < gridDim.x; b += kThreads) v += __ldcg(&l.part[b]);
  v = block_sum(v, warp_sum);
  if (threadIdx.x == 0) {
    l.header->total = v;
    l.header->done = 0;
  }
}

__global__ void __launch_bounds__(kThreads) clip_kernel(List l, const double *total, float max_norm,
                                                        float eps, float *norm_out) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  const float norm = (float)sqrt(*total);
  const float ratio = max_norm / (norm + eps);
  const float c = ratio < 1.0f || ratio != ratio ? ratio : 1.0f;  // NaN goes on
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  for (uint32_t k = blockIdx.x; k < l.chunks; k += gridDim.x) {
    const uint32_t chunk = l.chunks - 1 - k;  // what the first pass read last is still in L2
    const Entry t = l.entry[find_entry(l, chunk)];
    if (c == 1.0f && t.src == t.dst && t.src_type == t.dst_type) continue;  // nothing changes
    const uint64_t begin = (uint64_t)(chunk - t.first_chunk) * kChunk;
    const uint64_t end = min(begin + kChunk, t.count);
    by_type(t.src_type, [&](auto tin) {
      by_type(t.dst_type, [&](auto tout) {
        using T = typename decltype(tin)::type;
        using O = typename decltype(tout)::type;
        const T *src = static_cast<const T *>(t.src);
        O *dst = static_cast<O *>(t.dst);
        auto write = [&](const auto &v, uint64_t e, auto width) {
          constexpr int V = decltype(width)::value;
          float f[V];
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] = v.get(i) * c;
          Vec<O, V> out;
          out.put(f);
          out.store(dst + e);
        };
        if (t.vector)
          each_vector<T, kV>(src, begin, end, [&](const Vec<T, kV> &v, uint64_t e) {
            write(v, e, std::integral_constant<int, kV>{});
          });
        else
          each_vector<T, 1>(src, begin, end, [&](const Vec<T, 1> &v, uint64_t e) {
            write(v, e, std::integral_constant<int, 1>{});
          });
      });
    });
  }
}

// A tensor's elements that whole vectors cover, its two ends in a scalar entry each.
struct Part {
  uint64_t begin, count;
  bool vector;
};

int split_tensor(const DcopyGrad &g, Part (&part)[3]) {
  const int sb = elem_size(g.src_type), db = elem_size(g.dst_type);
  const uintptr_t s = (uintptr_t)g.src, d = (uintptr_t)g.dst;
  // The first element at which both sides start a 16-byte granule, if there is one.
  for (uint64_t head = 0; head < 8; ++head) {
    if ((s + head * sb) % 16 || (d + head * db) % 16) continue;
    if (g.count < head + kV) break;
    const uint64_t body = (g.count - head) / kV * kV;
    int n = 0;
    if (head) part[n++] = {0, head, false};
    part[n++] = {head, body, true};
    if (head + body < g.count) part[n++] = {head + body, g.count - head - body, false};
    return n;
  }
  part[0] = {0, g.count, false};
  return g.count ? 1 : 0;
}

uint64_t list_bytes(uint64_t n) {
  return sizeof(Header) + kMaxBlocks * sizeof(double) + 3 * n * sizeof(Entry);
}

int open_list(const DcopyGradList *list, List *l) {
  if (!list || !list->workspace)
    return set_error(DCOPY_ERR_PARAM_INVALID, "gradient list: not built");
  uint8_t *w = static_cast<uint8_t *>(list->workspace);
  l->header = reinterpret_cast<Header *>(w);
  l->part = reinterpret_cast<double *>(w + sizeof(Header));
  l->entry = reinterpret_cast<const Entry *>(w + sizeof(Header) + kMaxBlocks * sizeof(double));
  l->count = list->entries;
  l->chunks = list->chunks;
  return check_device_span(w, sizeof(Header) + kMaxBlocks * sizeof(double) +
                                  (uint64_t)list->entries * sizeof(Entry), "workspace");
}

template <typename K>
unsigned list_grid(K kernel, const List &l) {
  return std::max(1u, std::min({l.chunks, resident_ctas(kernel, kThreads, 0), kMaxBlocks}));
}

int run_sum(const List &l, cudaStream_t s) {
  return launch(sum_squares_kernel, list_grid(sum_squares_kernel, l), dim3(kThreads), 0, s,
                "sum_squares_kernel", l);
}

int run_clip(const List &l, const double *total, float max_norm, float eps, float *norm,
             cudaStream_t s) {
  return launch(clip_kernel, list_grid(clip_kernel, l), dim3(kThreads), 0, s, "clip_kernel", l,
                total, max_norm, eps, norm);
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

int dcopy_grad_list_workspace(uint32_t n, uint64_t *bytes) {
  DCOPY_API_BEGIN
  if (!bytes) return set_error(DCOPY_ERR_PARAM_INVALID, "grad_list_workspace: NULL");
  *bytes = list_bytes(n);
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_grad_list_build(DcopyGradList *list, const DcopyGrad *grads, uint32_t n,
                          void *workspace, uint64_t workspace_bytes, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (!list || (!grads && n))
    return set_error(DCOPY_ERR_PARAM_INVALID, "grad_list_build: NULL argument");
  if (n > (1u << 24))
    return set_error(DCOPY_ERR_UNSUPPORTED, "grad_list_build: %u tensors", n);
  if (workspace_bytes < list_bytes(n) || (uintptr_t)workspace % 16)
    return set_error(DCOPY_ERR_PARAM_INVALID,
                     "grad_list_build: workspace of %llu bytes at %p, %llu needed, 16-byte aligned",
                     (unsigned long long)workspace_bytes, workspace,
                     (unsigned long long)list_bytes(n));
  if (int rc = check_device_span(workspace, list_bytes(n), "workspace")) return rc;
  std::vector<uint8_t> image(list_bytes(n));
  Entry *entry = reinterpret_cast<Entry *>(image.data() + sizeof(Header) +
                                           kMaxBlocks * sizeof(double));
  uint32_t entries = 0;
  uint64_t chunks = 0;
  for (uint32_t i = 0; i < n; ++i) {
    const DcopyGrad &g = grads[i];
    if (!is_float(g.src_type) || !is_float(g.dst_type))
      return set_error(DCOPY_ERR_DATATYPE_INVALID, "gradient %u: element types %d and %d", i,
                       g.src_type, g.dst_type);
    if (g.count == 0) continue;
    if (g.count >> 40)
      return set_error(DCOPY_ERR_SHAPE_INVALID, "gradient %u: %llu elements", i,
                       (unsigned long long)g.count);
    const uint64_t sb = elem_size(g.src_type), db = elem_size(g.dst_type);
    if ((uintptr_t)g.src % sb || (uintptr_t)g.dst % db)
      return set_error(DCOPY_ERR_PARAM_INVALID, "gradient %u is not aligned to its elements", i);
    if (int rc = check_device_span(g.src, g.count * sb, "gradient")) return rc;
    if (int rc = check_device_span(g.dst, g.count * db, "clipped gradient")) return rc;
    if (g.src != g.dst || sb != db)  // in place, or apart
      if (int rc = check_disjoint(g.src, g.count * sb, g.dst, g.count * db, "gradient")) return rc;
    Part part[3];
    const int parts = split_tensor(g, part);
    for (int k = 0; k < parts; ++k) {
      Entry &e = entry[entries++];
      e.src = static_cast<const uint8_t *>(g.src) + part[k].begin * sb;
      e.dst = static_cast<uint8_t *>(g.dst) + part[k].begin * db;
      e.count = part[k].count;
      e.first_chunk = (uint32_t)chunks;
      e.src_type = (uint8_t)g.src_type;
      e.dst_type = (uint8_t)g.dst_type;
      e.vector = part[k].vector;
      chunks += (part[k].count + kChunk - 1) / kChunk;
      if (chunks >> 31)
        return set_error(DCOPY_ERR_UNSUPPORTED, "grad_list_build: too many elements");
    }
  }
  DCOPY_CUDA_TRY(cudaMemcpyAsync(workspace, image.data(), image.size(), cudaMemcpyHostToDevice,
                                 stream));
  DCOPY_CUDA_TRY(cudaStreamSynchronize(stream));
  list->workspace = workspace;
  list->entries = entries;
  list->chunks = (uint32_t)chunks;
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_grad_sum_squares(const DcopyGradList *list, double *total, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  List l{};
  if (int rc = open_list(list, &l)) return rc;
  if (int rc = check_device_span(total, sizeof(double), "total")) return rc;
  if (int rc = run_sum(l, stream)) return rc;
  DCOPY_CUDA_TRY(cudaMemcpyAsync(total, &l.header->total, sizeof(double), cudaMemcpyDeviceToDevice,
                                 stream));
  return DCOPY_OK;
  DCOPY_API_END
}

int dcopy_grad_clip(const DcopyGradList *list, const double *total, float max_norm, float eps,
                    float *norm, dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (int rc = check_bound(max_norm, eps, "grad_clip")) return rc;
  List l{};
  if (int rc = open_list(list, &l)) return rc;
  if (int rc = check_device_span(total, sizeof(double), "total")) return rc;
  if (norm)
    if (int rc = check_device_span(norm, sizeof(float), "norm")) return rc;
  return run_clip(l, total, max_norm, eps, norm, stream);
  DCOPY_API_END
}

int dcopy_clip_grad_norm(const DcopyGradList *list, float max_norm, float eps, float *norm,
                         dcopy_stream_t stream) {
  DCOPY_API_BEGIN
  if (int rc = check_bound(max_norm, eps, "clip_grad_norm")) return rc;
  List l{};
  if (int rc = open_list(list, &l)) return rc;
  if (norm)
    if (int rc = check_device_span(norm, sizeof(float), "norm")) return rc;
  if (int rc = run_sum(l, stream)) return rc;
  return run_clip(l, &l.header->total, max_norm, eps, norm, stream);
  DCOPY_API_END
}

}  // extern "C"
