// Stable sort by a small whole-number key.
//
// Counting sort over digits of up to 10 bits, lowest first.  One pass: every
// tile of kTile entries counts its digits (tile_count_kernel); then each tile
// ranks its entries again and writes them behind the digits below its own, the
// same digit's entries of earlier tiles, of earlier warps of the tile, and of
// earlier entries of the warp (tile_place_kernel).  Nothing depends on the order
// in which tiles or atomics run, so the result is the same every time.
// Experts fit one digit; token ids take two up to 2^20 and three beyond.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "index_sort.cuh"
#include "launch.cuh"

namespace dcopy {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kItems = 8;
constexpr uint32_t kTile = kThreads * kItems;
constexpr uint32_t kMaxBins = 1024;

__device__ __forceinline__ uint32_t entry_key(const KeySource &k, uint32_t e) {
  const uint32_t r = k.cols.div(e);
  const int64_t at = (int64_t)r * k.pitch + (e - r * k.cols.d);
  const int64_t id = (k.wide ? static_cast<const int64_t *>(k.ids)[at]
                             : (int64_t)static_cast<const int32_t *>(k.ids)[at]) -
                     k.first;
  return id >= 0 && id < (int64_t)k.keys ? (uint32_t)id : k.keys;
}

struct Pass {
  KeySource src;            // the first pass reads ids ...
  const uint32_t *key_in;   // ... later ones the pairs of the pass before
  const uint32_t *pos_in;
  uint32_t *key_out, *pos_out;
  uint32_t *counts;         // [tiles][bins]
  uint32_t n, tiles, bins, shift;
};

struct ExpertOut {
  int32_t *dest, *source, *offsets;
  uint32_t align, rows;
};

__device__ __forceinline__ uint32_t load_key(const Pass &p, uint32_t e) {
  return p.key_in ? p.key_in[e] : entry_key(p.src, e);
}

__global__ void __launch_bounds__(kThreads) tile_count_kernel(Pass p) {
  __shared__ uint32_t count[kMaxBins];
  pdl_trigger_at_entry();
  for (uint32_t d = threadIdx.x; d < p.bins; d += kThreads) count[d] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t e0 = blockIdx.x * kTile + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = e0 + i * kThreads;
    if (e < p.n) atomicAdd(&count[(load_key(p, e) >> p.shift) & (kMaxBins - 1)], 1u);
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < p.bins; d += kThreads)
    p.counts[blockIdx.x * p.bins + d] = count[d];
}

// Exclusive sum over the block of one value a thread; *total gets the sum.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t *warp_sum,
                                                    uint32_t *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t s = warp_sum[w];
    if (w < warp) before += s;
    all += s;
  }
  *total = all;
  return before + x - v;
}

template <bool kExperts>
__global__ void __launch_bounds__(kThreads) tile_place_kernel(Pass p, ExpertOut o) {
  __shared__ uint16_t seen[kWarps][kMaxBins];  // at most 32 * kItems a warp
  __shared__ uint32_t base[kMaxBins];
  __shared__ uint32_t warp_sum[kWarps];
  pdl_trigger_at_entry();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t d = lane; d < p.bins; d += 32) seen[warp][d] = 0;
  __syncwarp();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t e0 = blockIdx.x * kTile + warp * 32 * kItems + lane;
  uint32_t key[kItems], rank[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = e0 + i * 32;
    key[i] = e < p.n ? load_key(p, e) : 0;
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const bool in = e0 + i * 32 < p.n;
    const uint32_t lanes = __ballot_sync(~0u, in);
    if (in) {
      const uint32_t d = (key[i] >> p.shift) & (kMaxBins - 1);
      const uint32_t same = __match_any_sync(lanes, d);
      const uint32_t before = seen[warp][d];
      __syncwarp(lanes);
      rank[i] = before + __popc(same & ((1u << lane) - 1));
      if ((same >> lane) == 1) seen[warp][d] = (uint16_t)(before + __popc(same));
      __syncwarp(lanes);
    }
  }
  __syncthreads();
  // A thread takes the digits d = threadIdx.x and threadIdx.x + kThreads in turn.
  uint32_t carry = 0;
  for (uint32_t d0 = 0; d0 < p.bins; d0 += kThreads) {
    const uint32_t d = d0 + threadIdx.x;
    uint32_t all = 0, earlier = 0;
    if (d < p.bins) {
      uint32_t run = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t c = seen[w][d];
        seen[w][d] = (uint16_t)run;
        run += c;
      }
      if (p.tiles == 1) {
        all = run;
      } else {
        for (uint32_t t = 0; t < p.tiles; ++t) {
          const uint32_t c = p.counts[t * p.bins + d];
          if (t < blockIdx.x) earlier += c;
          all += c;
        }
      }
    }
    uint32_t room = all, total;
    if (kExperts) {  // the last digit holds the entries without an expert
      room = d + 1 < p.bins ? (all + o.align - 1) / o.align * o.align : 0;
    }
    const uint32_t at = carry + block_exclusive(room, warp_sum, &total);
    carry += total;
    if (d < p.bins) {
      base[d] = at + earlier;
      if (kExperts) {
        if (blockIdx.x == 0) o.offsets[d] = (int32_t)at;  // the last one: all rows in use
        if (d + 1 < p.bins)
          for (uint32_t r = at + all + blockIdx.x; r < at + room; r += gridDim.x) o.source[r] = -1;
      }
    }
  }
  if (kExperts)
    for (uint32_t r = carry + blockIdx.x * kThreads + threadIdx.x; r < o.rows;
         r += gridDim.x * kThreads)
      o.source[r] = -1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = e0 + i * 32;
    if (e >= p.n) continue;
    const uint32_t d = (key[i] >> p.shift) & (kMaxBins - 1);
    const uint32_t to = base[d] + seen[warp][d] + rank[i];
    if (kExperts) {
      const bool kept = d + 1 < p.bins;
      o.dest[e] = kept ? (int32_t)to : -1;
      if (kept) o.source[to] = (int32_t)e;
    } else {
      p.key_out[to] = key[i];
      p.pos_out[to] = p.pos_in ? p.pos_in[e] : e;
    }
  }
}

uint32_t tiles_of(uint64_t n) { return (uint32_t)((n + kTile - 1) / kTile); }

}  // namespace

uint64_t sort_by_key_bytes(uint64_t n, uint64_t keys) {
  (void)keys;
  return 4 * n * sizeof(uint32_t) + (uint64_t)tiles_of(n) * kMaxBins * sizeof(uint32_t);
}

int sort_by_key(const KeySource &src, void *workspace, const uint32_t **key_out,
                const uint32_t **pos_out, cudaStream_t s) {
  uint32_t *w = static_cast<uint32_t *>(workspace);
  uint32_t *key[2] = {w, w + 2ull * src.n}, *pos[2] = {w + src.n, w + 3ull * src.n};
  Pass p{};
  p.src = src;
  p.counts = w + 4ull * src.n;
  p.n = src.n;
  p.tiles = tiles_of(src.n);
  int to = 0;
  for (uint32_t shift = 0; shift == 0 || (shift < 32 && src.keys >> shift != 0); shift += 10) {
    p.shift = shift;
    p.bins = std::min<uint32_t>(kMaxBins, (src.keys >> shift) + 1);
    p.key_out = key[to];
    p.pos_out = pos[to];
    if (p.tiles > 1)
      if (int rc = launch(tile_count_kernel, p.tiles, dim3(kThreads), 0, s, "tile_count_kernel", p))
        return rc;
    if (int rc = launch(tile_place_kernel<false>, p.tiles, dim3(kThreads), 0, s,
                        "tile_place_kernel", p, ExpertOut{}))
      return rc;
    p.key_in = key[to];
    p.pos_in = pos[to];
    to ^= 1;
  }
  *key_out = p.key_in;
  *pos_out = p.pos_in;
  return DCOPY_OK;
}

uint64_t sort_experts_bytes(uint64_t n, uint32_t experts) {
  const uint32_t tiles = tiles_of(n);
  return tiles > 1 ? (uint64_t)tiles * (experts + 1) * sizeof(uint32_t) : 0;
}

int sort_experts(const KeySource &src, uint32_t align, int32_t *dest, int32_t *source,
                 uint32_t rows, int32_t *offsets, void *workspace, cudaStream_t s) {
  Pass p{};
  p.src = src;
  p.counts = static_cast<uint32_t *>(workspace);
  p.n = src.n;
  p.tiles = std::max<uint32_t>(1, tiles_of(src.n));
  p.bins = src.keys + 1;
  if (p.tiles > 1)
    if (int rc = launch(tile_count_kernel, p.tiles, dim3(kThreads), 0, s, "tile_count_kernel", p))
      return rc;
  return launch(tile_place_kernel<true>, p.tiles, dim3(kThreads), 0, s, "tile_place_kernel", p,
                ExpertOut{dest, source, offsets, align, rows});
}

}  // namespace dcopy
