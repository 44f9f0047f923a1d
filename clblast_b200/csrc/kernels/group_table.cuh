// Table of the ragged groups of a call, built in shared memory by one warp from the offsets in device memory.
//
// start[g] (g = 0 .. problems) is offset g, clamped to [0, bound] and made monotone: offsets that leave the range or
// descend lose rows instead of leading out of the buffers. tiles[g] is the number of tiles of `bn` vectors of the groups
// before g, so a running tile number finds its group by bisection.
#pragma once

namespace b200 {

__device__ __forceinline__ void build_table(const long long* offsets, int problems, int bound, int bn, int* start,
                                            int* tiles) {
  const int lane = threadIdx.x & 31;
  int carry_start = 0, carry_tiles = 0;
  for (int base = 0; base <= problems; base += 32) {
    const int g = base + lane;
    int s = 0;
    if (g <= problems) {
      const long long o = offsets[g];
      s = static_cast<int>(o < 0 ? 0 : (o > bound ? bound : o));
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d && t > s) s = t;
    }
    if (carry_start > s) s = carry_start;
    // tiles of group g - 1, which ends where group g starts
    int before = __shfl_up_sync(0xFFFFFFFFu, s, 1);
    if (lane == 0) before = carry_start;
    int count = (g >= 1 && g <= problems) ? (s - before + bn - 1) / bn : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, count, d);
      if (lane >= d) count += t;
    }
    count += carry_tiles;
    if (g <= problems) {
      start[g] = s;
      tiles[g] = count;
    }
    carry_start = __shfl_sync(0xFFFFFFFFu, s, 31);
    carry_tiles = __shfl_sync(0xFFFFFFFFu, count, 31);
  }
}

}  // namespace b200
