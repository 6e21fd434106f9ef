// Per-row page lists held by one warp: four entries a lane, entry 32 r + lane in v[r].
#pragma once

#include <cstdint>

namespace ls {

constexpr int32_t kPageSentinel = 0x7FFFFFFF;

// Sorts 128 keys held as v[r] at position 32*r + lane, ascending.
__device__ __forceinline__ void warp_bitonic_sort128(int32_t (&v)[4], int lane) {
#pragma unroll
  for (int k = 2; k <= 128; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= 32) {
        const int rj = j >> 5;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if ((r & rj) == 0) {
            const int pos = 32 * r + lane;
            const bool up = (pos & k) == 0;
            const int32_t a = v[r], b = v[r | rj];
            const bool swap = up ? (a > b) : (a < b);
            v[r] = swap ? b : a;
            v[r | rj] = swap ? a : b;
          }
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int pos = 32 * r + lane;
          const int32_t other = __shfl_xor_sync(0xffffffffu, v[r], j);
          const bool up = (pos & k) == 0;
          const bool lower = (lane & j) == 0;
          const int32_t lo = min(v[r], other), hi = max(v[r], other);
          v[r] = (lower == up) ? lo : hi;
        }
      }
    }
  }
}

// Sorts v ascending, drops sentinels and repeats, writes what is left to
// pages[0 ..) in shared memory and returns how many there are.  Strictly
// ascending entries followed by sentinels (the lists the selection kernels
// write) need no sort.
__device__ __forceinline__ int warp_compact_pages(int32_t (&v)[4], int32_t* pages, int lane) {
  bool ordered = true;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    int32_t next = __shfl_down_sync(0xffffffffu, v[r], 1);
    const int32_t next_row = __shfl_sync(0xffffffffu, v[r < 3 ? r + 1 : r], 0);
    if (lane == 31) next = r < 3 ? next_row : kPageSentinel;
    ordered = ordered && (v[r] < next || next == kPageSentinel);
  }
  if (!__all_sync(0xffffffffu, ordered)) warp_bitonic_sort128(v, lane);
  int base = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    int32_t prev = __shfl_up_sync(0xffffffffu, v[r], 1);
    const int32_t prev_reg = r > 0 ? __shfl_sync(0xffffffffu, v[r - 1], 31) : -1;
    if (lane == 0) prev = prev_reg;
    const bool keep = v[r] != kPageSentinel && v[r] != prev;
    const uint32_t mask = __ballot_sync(0xffffffffu, keep);
    if (keep) pages[base + __popc(mask & ((1u << lane) - 1))] = v[r];
    base += __popc(mask);
  }
  return base;
}

}  // namespace ls
