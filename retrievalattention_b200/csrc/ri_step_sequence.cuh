// Splitting work over a cache evenly: the cache's steps of Args::kStep rows, all groups (request, KV head) behind one another,
// are cut into one contiguous range per CTA.  Groups without rows take no steps.  The requests' lengths are read on the device.
// `Args` has batch, hk (KV heads) and a function int rows_of(const Args&, int b).
#pragma once

#include <stdint.h>

namespace ri_seq {

template <int STEP>
__device__ __forceinline__ int steps_of(int rows) { return (int)((unsigned)(rows + STEP - 1) / STEP); }

// All steps of the cache (whole warps).
template <class Args>
__device__ __forceinline__ int count_steps(const Args& a) {
  int sum = 0;
  for (int b = threadIdx.x & 31; b < a.batch; b += 32) sum += steps_of<Args::kStep>(rows_of(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum * a.hk;
}
// How many CTAs share `total` steps: at least a step per warp, at most max_ctas.
template <int WARPS>
__device__ __forceinline__ int used_ctas(int total, int max_ctas) {
  return min(max_ctas, max(1, (total + WARPS - 1) / WARPS));
}
__device__ __forceinline__ int cta_start(int c, int total, int n) { return (int)((int64_t)c * total / n); }

// A place in the sequence of steps: group g, its first step in the sequence, its rows.
struct Place {
  int g, first, rows;
};
// The group that holds step s (whole warps; s < total).
template <class Args>
__device__ __forceinline__ Place find_place(const Args& a, int s) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const int rows = b < a.batch ? rows_of(a, b) : 0, n = steps_of<Args::kStep>(rows) * a.hk;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, s < before + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int r = __shfl_sync(0xffffffffu, rows, src), start = before + __shfl_sync(0xffffffffu, incl - n, src);
      const int per = steps_of<Args::kStep>(r), h = (s - start) / per;
      return {(b0 + src) * a.hk + h, start + h * per, r};
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return {0, 0, 0};
}
// The next group with rows (there is one: the caller has steps left).
template <class Args>
__device__ __forceinline__ void next_place(const Args& a, Place& p) {
  p.first += steps_of<Args::kStep>(p.rows);
  ++p.g;
  if (p.g % a.hk == 0) {
    int b = p.g / a.hk;
    while ((p.rows = rows_of(a, b)) == 0 && b + 1 < a.batch) ++b;
    p.g = b * a.hk;
  }
}

// The group with rows in front of it (there is one).
template <class Args>
__device__ __forceinline__ void previous_place(const Args& a, Place& p) {
  if (p.g % a.hk == 0) {
    int b = p.g / a.hk - 1;
    while ((p.rows = rows_of(a, b)) == 0 && b > 0) --b;
    p.g = (b + 1) * a.hk;
  }
  --p.g;
  p.first -= steps_of<Args::kStep>(p.rows);
}

}  // namespace ri_seq
