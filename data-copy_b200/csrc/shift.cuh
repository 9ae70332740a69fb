// Bytes at odd places: 16 bytes out of two aligned blocks, and a part of an aligned vector.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dcopy {

// The 16 bytes at byte offset `s` (0..15) of the 32 bytes a || b.
__device__ __forceinline__ uint4 shift_pair(uint4 a, uint4 b, uint32_t s) {
  uint32_t w0 = a.x, w1 = a.y, w2 = a.z, w3 = a.w, w4 = b.x, w5 = b.y, w6 = b.z, w7 = b.w;
  if (s & 8) {
    w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = w7;
  }
  if (s & 4) {
    w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5;
  }
  const uint32_t r = (s & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, r), __funnelshift_r(w1, w2, r),
                    __funnelshift_r(w2, w3, r), __funnelshift_r(w3, w4, r));
}

// Bytes [lo, hi) of the aligned 16-byte vector at v, in naturally aligned
// pieces: the span is cut at the 1-, 2-, 4- and 8-byte boundaries from both
// ends, so a partial vector takes at most 4 + 4 stores instead of 15.
__device__ __forceinline__ void store_partial(uint8_t *v, uint4 x, uint32_t lo, uint32_t hi) {
  const uint64_t q0 = ((uint64_t)x.y << 32) | x.x, q1 = ((uint64_t)x.w << 32) | x.z;
  auto piece = [&](uint32_t at, uint32_t bytes) {  // at % bytes == 0, at + bytes <= 16
    const uint64_t q = at < 8 ? q0 : q1;
    const uint64_t bits = q >> ((at & 7) * 8);
    if (bytes == 8) *reinterpret_cast<uint64_t *>(v + at) = bits;
    else if (bytes == 4) *reinterpret_cast<uint32_t *>(v + at) = (uint32_t)bits;
    else if (bytes == 2) *reinterpret_cast<uint16_t *>(v + at) = (uint16_t)bits;
    else v[at] = (uint8_t)bits;
  };
  uint32_t a = lo, b = hi;
#pragma unroll
  for (uint32_t w = 1; w <= 8; w <<= 1)  // grow from the left edge to alignment w*2
    if ((a & w) && a + w <= b) {
      piece(a, w);
      a += w;
    }
#pragma unroll
  for (uint32_t w = 8; w >= 1; w >>= 1)  // then whole aligned pieces, largest first
    if (a + w <= b && (a & (w - 1)) == 0 && (b - a) >= w) {
      piece(a, w);
      a += w;
    }
#pragma unroll
  for (uint32_t w = 4; w >= 1; w >>= 1)  // what remains on the right
    if (a + w <= b) {
      piece(a, w);
      a += w;
    }
}

}  // namespace dcopy
