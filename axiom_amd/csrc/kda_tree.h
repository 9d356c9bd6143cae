// Trees of drafted tokens (include/tree_mi355x.h) on the device.
#pragma once

#include "kda_common.h"

namespace kda {

typedef unsigned long long u64;
constexpr int kTreePlaces = 64;   // a lane of a wave each

// The path of place `lane` as bits (itself and its ancestors), 0 where it holds no
// draft; parent: its entry of `parents` (anything past N).  Every lane's bits
// run up to the place `up`, and double in length a round: six for the longest
// path, two or three for a bushy tree.
__device__ __forceinline__ u64 tree_paths(int parent, int N) {
  const int lane = __lane_id();
  int up = lane >= N ? -2 : parent == -1 ? -1 : parent >= 0 && parent < lane ? parent : -2;
  unsigned lo = lane < 32 ? 1u << lane : 0, hi = lane < 32 ? 0 : 1u << (lane - 32);
  while (__any(up >= 0)) {
    const int at = max(up, 0);
    const unsigned l = __shfl(static_cast<int>(lo), at, 64), h = __shfl(static_cast<int>(hi), at, 64);
    const int next = __shfl(up, at, 64);
    if (up >= 0) {
      lo |= l;
      hi |= h;
      up = next;
    }
  }
  return up == -1 ? static_cast<u64>(hi) << 32 | lo : 0;
}
__device__ __forceinline__ u64 shfl_u64(u64 x, int lane) {
  return static_cast<u64>(static_cast<unsigned>(__shfl(static_cast<int>(x >> 32), lane, 64))) << 32 |
         static_cast<unsigned>(__shfl(static_cast<int>(x), lane, 64));
}
// in scalar registers
__device__ __forceinline__ u64 uniform_u64(u64 x) {
  return static_cast<u64>(static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32)))) << 32 |
         static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}

}  // namespace kda
