// Stable sort by a small whole-number key.
//
// Counting sort by digits, lowest first.  One pass: every tile
// of entries counts its digits (tile_count_kernel); then each tile ranks its entries
// again and writes them behind the digits below its own, the same digit's entries of
// earlier tiles, of earlier warps of the tile, and of earlier entries of the warp
// (tile_place_kernel).  Nothing depends on the order in which tiles or atomics run,
// so the result is the same every time.  Experts fit one digit of up to 10 bits; token
// ids take two of up to 9 bits below 2^18 and three below 2^27.  What fits one tile
// takes one launch for all digits.
//
// Bound by latency, not bytes: a launch of a pass takes 4 to 5 us (counts) and 10 us
// (places) for 131072 choices, 2.1 MB.  Most of the placing is adding up the tiles'
// counts, 8 loads ahead (one digit a warp and four ahead: 23 us for 512 digits).
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "index_sort.cuh"
#include "launch.cuh"
#include "rowops.cuh"

namespace dcopy {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kExpertBits = 10, kTokenBits = 9;  // digits of the two sorts, at most
constexpr uint32_t kMaxBins = 1 << kExpertBits;
constexpr uint32_t kOneTile = 8 * kThreads;

__device__ __forceinline__ uint32_t entry_key(const KeySource &k, uint32_t e) {
  const int64_t id = read_id(k, e);
  return id >= 0 && id < (int64_t)k.keys ? (uint32_t)id : k.keys;
}

struct Pass {
  KeySource src;            // the first pass reads ids ...
  const uint32_t *key_in;   // ... later ones the pairs of the pass before
  const uint32_t *pos_in;
  uint32_t *key_out, *pos_out;
  uint32_t *counts;         // [tiles][bins]
  uint32_t n, tiles, bins, shift;
  uint32_t passes, bits;    // of the sort in one tile
  Fill fill;
};

struct ExpertOut {
  int32_t *dest, *source, *offsets;
  uint32_t align, rows;
};

__device__ __forceinline__ uint32_t load_key(const Pass &p, uint32_t e) {
  return p.key_in ? p.key_in[e] : entry_key(p.src, e);
}

// The rows of a fill: a block takes a row in turn, or 16 KB where rows adjoin (with
// 64 KB some blocks get a second part when others are done: 199 us instead of 194 for
// 16384 tokens, 131072 x 4096 bf16).
__device__ __forceinline__ void zero_rows(const Fill &f, uint32_t block, uint32_t blocks) {
  if (f.pitch == f.bytes) {
    constexpr uint64_t kPart = 16 << 10;
    const uint64_t bytes = (f.end - f.begin) * f.bytes;
    for (uint64_t b = block * kPart; b < bytes; b += blocks * kPart)
      zero_bytes(f.dst + f.begin * f.bytes + b, min(kPart, bytes - b), threadIdx.x, kThreads);
  } else {
    for (uint64_t r = f.begin + block; r < f.end; r += blocks)
      zero_bytes(f.dst + r * f.pitch, f.bytes, threadIdx.x, kThreads);
  }
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

// Entries of each digit that a warp of the tile holds, then that earlier warps hold.
template <uint32_t kBins>
struct Seen {
  uint16_t of[kWarps][kBins];
};

template <uint32_t kBins>
__device__ __forceinline__ void clear_seen(Seen<kBins> &seen, uint32_t bins) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (uint32_t d = 2 * lane; d < bins; d += 64)
    *reinterpret_cast<uint32_t *>(&seen.of[warp][d]) = 0;
}

// rank[i]: entries of the same digit that precede the thread's i-th entry in its
// warp.  Warp w holds entries [w * 32 * kItems, ...) of the tile, lane by lane.
template <int kItems, uint32_t kBins>
__device__ __forceinline__ void rank_in_warp(Seen<kBins> &seen, const uint32_t (&digit)[kItems],
                                             uint32_t first, uint32_t n,
                                             uint32_t (&rank)[kItems]) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const bool in = first + i * 32 < n;
    const uint32_t lanes = __ballot_sync(~0u, in);
    rank[i] = 0;
    if (in) {
      const uint32_t same = __match_any_sync(lanes, digit[i]);
      const uint32_t before = seen.of[warp][digit[i]];
      __syncwarp(lanes);
      rank[i] = before + __popc(same & ((1u << lane) - 1));
      if ((same >> lane) == 1) seen.of[warp][digit[i]] = (uint16_t)(before + __popc(same));
      __syncwarp(lanes);
    }
  }
}

// seen becomes the entries of earlier warps; returns those of the tile.
template <uint32_t kBins>
__device__ __forceinline__ uint32_t sum_over_warps(Seen<kBins> &seen, uint32_t d) {
  uint32_t run = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t c = seen.of[w][d];
    seen.of[w][d] = (uint16_t)run;
    run += c;
  }
  return run;
}

template <int kItems>
__global__ void __launch_bounds__(kThreads) tile_count_kernel(Pass p) {
  __shared__ uint32_t count[kMaxBins];
  pdl_trigger_at_entry();
  if (blockIdx.x >= p.tiles) {
    pdl_wait();
    pdl_launch_dependents();
    return zero_rows(p.fill, blockIdx.x - p.tiles, gridDim.x - p.tiles);
  }
  for (uint32_t d = threadIdx.x; d < p.bins; d += kThreads) count[d] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t e0 = blockIdx.x * kThreads * kItems + threadIdx.x;
  uint32_t key[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (e0 + i * kThreads < p.n) key[i] = load_key(p, e0 + i * kThreads);
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (e0 + i * kThreads < p.n) atomicAdd(&count[(key[i] >> p.shift) & ((1u << p.bits) - 1)], 1u);
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < p.bins; d += kThreads)
    p.counts[(uint64_t)blockIdx.x * p.bins + d] = count[d];
}

template <int kItems, bool kExperts>
__global__ void __launch_bounds__(kThreads) tile_place_kernel(Pass p, ExpertOut o) {
  constexpr uint32_t kBins = 1 << (kExperts ? kExpertBits : kTokenBits);
  __shared__ Seen<kBins> seen;
  __shared__ uint32_t base[kBins], all[kBins];
  __shared__ uint32_t warp_sum[kWarps];
  pdl_trigger_at_entry();
  if (blockIdx.x >= p.tiles) {
    pdl_wait();
    pdl_launch_dependents();
    return zero_rows(p.fill, blockIdx.x - p.tiles, gridDim.x - p.tiles);
  }
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  clear_seen(seen, p.bins);
  __syncwarp();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t e0 = (blockIdx.x * kThreads + warp * 32) * kItems + lane;
  if (kExperts && p.tiles == 1)  // padding: what is not written below, behind a barrier
    for (uint32_t r = threadIdx.x; r < o.rows; r += kThreads) o.source[r] = -1;
  uint32_t key[kItems], digit[kItems], rank[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    key[i] = e0 + i * 32 < p.n ? load_key(p, e0 + i * 32) : 0;
    digit[i] = (key[i] >> p.shift) & ((1u << p.bits) - 1);
  }
  rank_in_warp(seen, digit, e0, p.n, rank);
  if (p.tiles > 1) {
    // The entries of each digit in all tiles and in earlier ones.  Where the block has
    // threads for it, several share a digit and take every groups-th tile.
    for (uint32_t d = threadIdx.x; d < p.bins; d += kThreads) all[d] = base[d] = 0;
    __syncthreads();
    const uint32_t groups = max(1u, kThreads / p.bins);
    const uint32_t group = p.bins < kThreads ? threadIdx.x / p.bins : 0;
    for (uint32_t d = threadIdx.x - group * p.bins; d < p.bins && group < groups; d += kThreads) {
      uint32_t sum = 0, earlier = 0;
      constexpr uint32_t kLoads = 8;
      for (uint32_t t0 = group; t0 < p.tiles; t0 += kLoads * groups) {
        uint32_t c[kLoads];
#pragma unroll
        for (uint32_t j = 0; j < kLoads; ++j) {
          const uint32_t t = t0 + j * groups;
          c[j] = t < p.tiles ? p.counts[(uint64_t)t * p.bins + d] : 0;
        }
#pragma unroll
        for (uint32_t j = 0; j < kLoads; ++j) {
          sum += c[j];
          if (t0 + j * groups < blockIdx.x) earlier += c[j];
        }
      }
      atomicAdd(&all[d], sum);
      atomicAdd(&base[d], earlier);
    }
  }
  __syncthreads();
  uint32_t carry = 0;
  for (uint32_t d0 = 0; d0 < p.bins; d0 += kThreads) {
    const uint32_t d = d0 + threadIdx.x;
    uint32_t mine = 0, earlier = 0, room = 0, total;
    if (d < p.bins) {
      mine = sum_over_warps(seen, d);
      if (p.tiles > 1) mine = all[d], earlier = base[d];
      room = mine;
      if (kExperts)  // the last digit holds the entries without an expert
        room = d + 1 < p.bins ? (mine + o.align - 1) / o.align * o.align : 0;
    }
    const uint32_t at = carry + block_exclusive(room, warp_sum, &total);
    carry += total;
    if (d < p.bins) {
      base[d] = at + earlier;
      if (kExperts) {
        if (blockIdx.x == 0) o.offsets[d] = (int32_t)at;  // the last one: all rows in use
        if (d + 1 < p.bins && p.tiles > 1)
          for (uint32_t r = at + mine + blockIdx.x; r < at + room; r += p.tiles) o.source[r] = -1;
      }
    }
  }
  if (kExperts && p.tiles > 1)
    for (uint32_t r = carry + blockIdx.x * kThreads + threadIdx.x; r < o.rows;
         r += p.tiles * kThreads)
      o.source[r] = -1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = e0 + i * 32, d = digit[i];
    if (e >= p.n) continue;
    const uint32_t to = base[d] + seen.of[warp][d] + rank[i];
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

// All digits of at most kItems * kThreads entries in one block.
template <int kItems>
__global__ void __launch_bounds__(kThreads) one_tile_kernel(Pass p) {
  constexpr uint32_t kRoom = kItems * kThreads, kBins = 1 << kTokenBits;
  __shared__ Seen<kBins> seen;
  __shared__ uint32_t keys[kRoom], base[kBins], warp_sum[kWarps];
  __shared__ uint16_t places[kRoom];
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  if (blockIdx.x >= 1) return zero_rows(p.fill, blockIdx.x - 1, gridDim.x - 1);
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t e0 = warp * 32 * kItems + lane, bins = 1u << p.bits;
  uint32_t key[kItems], place[kItems], digit[kItems], rank[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    place[i] = e0 + i * 32;
    key[i] = place[i] < p.n ? entry_key(p.src, place[i]) : 0;
  }
  for (uint32_t pass = 0; pass < p.passes; ++pass) {
    clear_seen(seen, bins);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kItems; ++i) digit[i] = (key[i] >> (pass * p.bits)) & (bins - 1);
    rank_in_warp(seen, digit, e0, p.n, rank);
    __syncthreads();
    uint32_t carry = 0;
    for (uint32_t d0 = 0; d0 < bins; d0 += kThreads) {
      const uint32_t d = d0 + threadIdx.x;
      const uint32_t mine = d < bins ? sum_over_warps(seen, d) : 0;
      uint32_t total;
      const uint32_t at = carry + block_exclusive(mine, warp_sum, &total);
      carry += total;
      if (d < bins) base[d] = at;
    }
    __syncthreads();
    const bool last = pass + 1 == p.passes;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (e0 + i * 32 >= p.n) continue;
      const uint32_t to = base[digit[i]] + seen.of[warp][digit[i]] + rank[i];
      if (last) p.key_out[to] = key[i], p.pos_out[to] = place[i];
      else keys[to] = key[i], places[to] = (uint16_t)place[i];
    }
    if (last) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (e0 + i * 32 < p.n) key[i] = keys[e0 + i * 32], place[i] = places[e0 + i * 32];
  }
}

// Entries a thread ranks.  Few keep many tiles (SMs) at work, many keep the tiles'
// counts, which every tile reads, below the entries: 131072 choices are placed in 10 us
// with 2 and 15 us with 8.
int items_of(uint64_t n) { return n <= 128 * 2 * kThreads ? 2 : n <= 1024 * 8 * kThreads ? 8 : 32; }
uint32_t tiles_of(uint64_t n) {
  const uint64_t tile = (uint64_t)items_of(n) * kThreads;
  return (uint32_t)((n + tile - 1) / tile);
}

template <typename F>
int with_items(int items, F &&f) {
  if (items == 2) return f(std::integral_constant<int, 2>{});
  if (items == 8) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 32>{});
}

// Bytes that a launch of the sort clears beside its own work, which takes 5 to 10 us.
// (16384 tokens, 131072 x 4096 bf16: 199 us with 48 MB, 199 with 24, 201 with 96.)
constexpr uint64_t kFillBeside = 48ull << 20, kFillOneTile = 64ull << 20;

// The rows that the next launch clears, taken from the end of fill.
Fill next_fill(Fill *fill, uint64_t bytes, uint32_t *blocks) {
  Fill f = *fill;
  const uint64_t rows = f.bytes ? std::max<uint64_t>(1, bytes / f.bytes) : 0;
  f.begin = f.end - std::min<uint64_t>(rows, f.end - f.begin);
  fill->end = f.begin;
  *blocks = (uint32_t)std::min<uint64_t>(f.end - f.begin, 4ull * sm_count());
  return f;
}

__global__ void __launch_bounds__(kThreads) zero_kernel(Fill f) {
  pdl_trigger_at_entry();
  pdl_wait();
  pdl_launch_dependents();
  zero_rows(f, blockIdx.x, gridDim.x);
}

}  // namespace

int fill_zero(const Fill &fill, cudaStream_t s) {
  const uint64_t rows = fill.bytes ? fill.end - fill.begin : 0;
  if (rows == 0) return DCOPY_OK;
  return launch(zero_kernel, (unsigned)std::min<uint64_t>(rows, 4ull * sm_count()), dim3(kThreads),
                0, s, "zero_kernel", fill);
}

uint64_t sort_by_key_bytes(uint64_t n) {
  return (4 * n + ((uint64_t)tiles_of(n) << kTokenBits)) * sizeof(uint32_t);
}

int sort_by_key(const KeySource &src, Fill *fill, void *workspace, const uint32_t **key_out,
                const uint32_t **pos_out, cudaStream_t s) {
  uint32_t *w = static_cast<uint32_t *>(workspace);
  uint32_t *key[2] = {w, w + 2ull * src.n}, *pos[2] = {w + src.n, w + 3ull * src.n};
  Pass p{};
  p.src = src;
  p.counts = w + 4ull * src.n;
  p.n = src.n;
  uint32_t key_bits = 1;  // keys themselves occur, as the key of what belongs nowhere
  while (key_bits < 32 && src.keys >> key_bits) ++key_bits;
  p.passes = (key_bits + kTokenBits - 1) / kTokenBits;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  uint32_t fills = 0;
  if (src.n <= kOneTile) {
    p.fill = next_fill(fill, kFillOneTile, &fills);
    p.key_out = key[0];
    p.pos_out = pos[0];
    *key_out = key[0];
    *pos_out = pos[0];
    auto k = src.n <= 2 * kThreads ? one_tile_kernel<2> : src.n <= 4 * kThreads ? one_tile_kernel<4> : one_tile_kernel<8>;
    return launch(k, 1 + fills, dim3(kThreads), 0, s, "one_tile_kernel", p);
  }
  p.tiles = tiles_of(src.n);
  for (uint32_t pass = 0; pass < p.passes; ++pass) {
    p.shift = pass * p.bits;
    p.bins = std::min<uint32_t>(1u << p.bits, (src.keys >> p.shift) + 1);
    p.key_out = key[pass & 1];
    p.pos_out = pos[pass & 1];
    const int rc = with_items(items_of(src.n), [&](auto items) {
      constexpr int kItems = decltype(items)::value;
      p.fill = next_fill(fill, kFillBeside, &fills);
      if (int rc = launch(tile_count_kernel<kItems>, p.tiles + fills, dim3(kThreads), 0, s,
                          "tile_count_kernel", p))
        return rc;
      p.fill = next_fill(fill, kFillBeside, &fills);
      return launch(tile_place_kernel<kItems, false>, p.tiles + fills, dim3(kThreads), 0, s,
                    "tile_place_kernel", p, ExpertOut{});
    });
    if (rc) return rc;
    p.key_in = p.key_out;
    p.pos_in = p.pos_out;
  }
  *key_out = p.key_in;
  *pos_out = p.pos_in;
  return DCOPY_OK;
}

uint64_t sort_experts_bytes(uint64_t n, uint32_t experts) {
  return n <= kOneTile ? 0 : (uint64_t)tiles_of(n) * (experts + 1) * sizeof(uint32_t);
}

int sort_experts(const KeySource &src, uint32_t align, int32_t *dest, int32_t *source,
                 uint32_t rows, int32_t *offsets, void *workspace, cudaStream_t s) {
  Pass p{};
  p.src = src;
  p.counts = static_cast<uint32_t *>(workspace);
  p.n = src.n;
  p.bins = src.keys + 1;
  p.bits = kExpertBits;
  const bool one = src.n <= kOneTile;
  const int most = one ? (src.n <= 2 * kThreads ? 2 : 8) : items_of(src.n);
  p.tiles = one ? 1 : tiles_of(src.n);
  return with_items(most, [&](auto items) {
    constexpr int kItems = decltype(items)::value;
    if (!one)
      if (int rc = launch(tile_count_kernel<kItems>, p.tiles, dim3(kThreads), 0, s,
                          "tile_count_kernel", p))
        return rc;
    return launch(tile_place_kernel<kItems, true>, p.tiles, dim3(kThreads), 0, s,
                  "tile_place_kernel", p, ExpertOut{dest, source, offsets, align, rows});
  });
}

}  // namespace dcopy
