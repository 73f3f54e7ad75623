// What requests of a group have in common, between the kernel that attends it for all of them (ri_paged_attend.cu) and those that
// attend each request's own slots and join the two (ri_paged_decode.cu).
#pragma once

#include "ri_paged.cuh"

namespace ri_shared {

// The partial results over what groups have in common.  An item is up to `pair` neighbouring requests of a group and a KV head; it falls
// to CTAs ctas[2 i] .. ctas[2 i + 1], i = head * batch + its first request, and the part of CTA c has its rows (request, query head)
// behind c * part_rows + i * gs rows of 128 floats, in the order [channels / 8][rows][8].
struct Parts {
  const int32_t* starts;       // [groups + 1] requests
  const int32_t* shared;       // [groups] slots
  int* ctas;
  float* o;
  float2* ml;                  // (reference in the log2 domain, sum)
  int groups, pair, part_rows, max_ctas;
};

__device__ __forceinline__ int clamped(int x, int most) { return min(max(x, 0), most); }
// The group that request b is in, or -1.
__device__ __forceinline__ int group_of(const int32_t* starts, int groups, int b) {
  int lo = 0, hi = groups;               // starts[lo] <= b < starts[hi], if it is in one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (starts[mid] <= b ? lo : hi) = mid;
  }
  return starts[lo] <= b && b < starts[lo + 1] ? lo : -1;
}

// What requests of group g have in common: as far as the first one's slots go.
template <class Args>
__device__ __forceinline__ int in_common(const Args& a, const int32_t* starts, const int32_t* shared, int g) {
  const int b = clamped(starts[g], a.batch);
  return b < a.batch ? clamped(shared[g], ri_page::rows_of(a, b)) : 0;
}
// Slots that request b has in common with its group.
__device__ __forceinline__ int common_of(const ri_page::Pages& a, const Parts& x, int b) {
  const int g = group_of(x.starts, x.groups, b);
  return g >= 0 ? min(in_common(a, x.starts, x.shared, g), ri_page::rows_of(a, b)) : 0;
}

int64_t scratch_bytes(const ri_paged& p);
// Launches the attention of all requests over what they have in common; `parts` says where its results will be, in d_scratch.
int launch(const char* what, const ri_paged* p, const void* d_q, int64_t q_stride, const int32_t* d_group_start, int32_t groups,
           const int32_t* d_shared, float scale, void* d_scratch, Parts* parts, cudaStream_t s);

}  // namespace ri_shared
