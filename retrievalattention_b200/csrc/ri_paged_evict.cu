// Eviction from a paged cache by accumulated attention weight, in place.
//   Of the slots of a request and KV head, `keep` stay: those of the first n_sink and the last n_recent tokens, then the ones of
//   largest weight, the lower slot first where weights are equal (a NaN is less than any weight).  Slots in front of `keep` that
//   go are filled from behind it, the i-th hole with the i-th slot that stays: keys, values, weights and token numbers.
// Attention does not depend on the order of the slots (rotary positions are in the keys), so nothing else has to move: of n
// slots about keep (n - keep) / n where weights are in no order, and no more than n - keep where a few generated tokens are
// trimmed; sources lie behind `keep` and destinations in front, so no row is read after it was written.
//
// Two kernels.  Selection: a cluster of CTAs per group (request, KV head) maps weights to order-preserving 32-bit keys in shared
// memory (slots beyond that are mapped again when they are needed), finds the keep-th largest by a radix select of four
// 8-bit levels whose histograms the CTAs add up through distributed shared memory, and writes the lists of holes and of the
// slots that fill them, both ascending.  Every thread takes a run of consecutive slots, of odd length against bank conflicts.
// Moves: a half-warp per row, four rows in flight.  Bound by the moved rows, read once and written once.
#include <cooperative_groups.h>

#include "ri_paged.cuh"

namespace {

using namespace ri_page;
namespace cg = cooperative_groups;

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kCachedKeys = 40 * 1024;               // keys of a CTA's slice that shared memory holds
constexpr int kSelMaxCluster = 8;
constexpr int kMoveThreads = 256;
constexpr int kMovesAtOnce = 4;                      // per half-warp
constexpr int kMovesPerBlock = kMoveThreads / 16 * kMovesAtOnce;
constexpr uint32_t kProtected = 0xffffffffu;         // above +infinity

struct EvictArgs {
  Pages pages;
  const int32_t* seen;       // [batch] tokens so far
  uint4* keys;
  uint4* values;
  int32_t* counts;           // [groups]
  int2* moves;               // [groups][most]: (hole, slot that fills it)
  int keep, sink, recent, most;
};

__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);         // -0 becomes +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Exclusive scan over the block, and its total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();                                     // warp_sums may still be read by the scan before
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    const int s = warp_sums[w];
    if (w < warp) before += s;
    total += s;
  }
  return before + incl - v;
}

struct SelShared {
  int hist[4][256];            // per level: this CTA's slots by digit
  int totals[2];               // holes and fillers of this CTA
  int warp_sums[kSelWarps];
  int bin, before;             // the cut's digit, and slots of larger digits
};

__global__ void __launch_bounds__(kSelThreads, 1) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ uint32_t s_keys[];
  __shared__ SelShared sh;
  ri_pdl_enter();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int tid = threadIdx.x, g = blockIdx.x / ctas;
  const Pages& p = a.pages;
  const int b = g / p.hk, h = g - b * p.hk, n = rows_of(p, b);
  if (n <= a.keep) {                                   // the whole cluster leaves
    if (rank == 0 && tid == 0) a.counts[g] = 0;
    return;
  }
  const int slice = (n + ctas - 1) / ctas, lo = min(n, rank * slice), hi = min(n, lo + slice), mine = hi - lo;
  const int newest = a.seen[b] - a.recent;
  auto make_key = [&](int j) {
    const int id = page_of(p, b, j >> p.shift);
    const int64_t at = record_at(p, id, h, j & ((1 << p.shift) - 1));
    const int t = p.token[at];
    return (t < a.sink || t >= newest) ? kProtected : order_key(p.weight[at]);
  };
  for (int i = tid; i < 4 * 256; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
  for (int j = tid; j < min(mine, kCachedKeys); j += kSelThreads) s_keys[j] = make_key(lo + j);
  __syncthreads();
  auto key_of = [&](int j) { return j < kCachedKeys ? s_keys[j] : make_key(lo + j); };

  // the keep-th largest key: digit by digit, `need` slots still to be found among those that agree so far
  uint32_t prefix = 0;
  int need = a.keep;
#pragma unroll 1
  for (int level = 0; level < 4; ++level) {
    const int shift = 24 - 8 * level;
    for (int j = tid; j < mine; j += kSelThreads) {
      const uint32_t k = key_of(j);
      if (level == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sh.hist[level][(k >> shift) & 255u], 1);
    }
    cluster.sync();
    int sum = 0;
    if (tid < 256) {                                   // thread 0 takes the largest digit
      const int digit = 255 - tid;
      for (int c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(&sh.hist[level][0], c)[digit];
    }
    int total;
    const int before = block_scan(sum, sh.warp_sums, total);
    if (tid < 256 && before < need && before + sum >= need) {
      sh.bin = 255 - tid;
      sh.before = before;
    }
    __syncthreads();
    prefix |= (uint32_t)sh.bin << shift;
    need -= sh.before;
    __syncthreads();
  }
  // slots with the cut's key: the first `need` of the group stay
  int equal_before = 0;
  for (int c = 0; c < rank; ++c) equal_before += cluster.map_shared_rank(&sh.hist[3][0], c)[prefix & 255u];

  const int run = ((mine + kSelThreads - 1) / kSelThreads) | 1, first = min(mine, tid * run), last = min(mine, first + run);
  int equal = 0;
  for (int j = first; j < last; ++j) equal += key_of(j) == prefix;
  int total, holes = 0, fillers = 0;
  equal_before += block_scan(equal, sh.warp_sums, total);
  int rank_eq = equal_before;
  for (int j = first; j < last; ++j) {
    const uint32_t k = key_of(j);
    const bool stays = k > prefix || (k == prefix && rank_eq++ < need), front = lo + j < a.keep;
    holes += front && !stays;
    fillers += !front && stays;
  }
  int hole_at = block_scan(holes, sh.warp_sums, total);
  if (tid == 0) sh.totals[0] = total;
  int filler_at = block_scan(fillers, sh.warp_sums, total);
  if (tid == 0) sh.totals[1] = total;
  cluster.sync();
  int all = 0;
  for (int c = 0; c < ctas; ++c) {
    const int* t = cluster.map_shared_rank(sh.totals, c);
    if (c < rank) {
      hole_at += t[0];
      filler_at += t[1];
    }
    all += t[0];
  }
  int2* moves = a.moves + (int64_t)g * a.most;
  rank_eq = equal_before;
  for (int j = first; j < last; ++j) {
    const uint32_t k = key_of(j);
    const bool stays = k > prefix || (k == prefix && rank_eq++ < need), front = lo + j < a.keep;
    if (front && !stays) moves[hole_at++].x = lo + j;
    if (!front && stays) moves[filler_at++].y = lo + j;
  }
  if (rank == 0 && tid == 0) a.counts[g] = all;
  cluster.sync();                                      // nobody's shared memory goes while others may read it
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  ri_pdl_enter();
  const Pages& p = a.pages;
  const int g = blockIdx.y, b = g / p.hk, h = g - b * p.hk, n = a.counts[g];
  const int c = threadIdx.x & 15, half = threadIdx.x >> 4;
  const int2* moves = a.moves + (int64_t)g * a.most;
  for (int i0 = blockIdx.x * kMovesPerBlock + half * kMovesAtOnce; i0 < n; i0 += gridDim.x * kMovesPerBlock) {
    int64_t to_k[kMovesAtOnce], to_v[kMovesAtOnce];    // negative: nothing to move
    uint4 k[kMovesAtOnce], v[kMovesAtOnce];
#pragma unroll
    for (int u = 0; u < kMovesAtOnce; ++u) {
      to_k[u] = -1;
      if (i0 + u >= n) continue;
      const int2 m = moves[i0 + u];
      const int id_to = page_to_write(p, b, m.x >> p.shift), id_of = page_to_write(p, b, m.y >> p.shift), mask = (1 << p.shift) - 1;
      if ((id_to | id_of) < 0) continue;
      const int64_t in_to = ((int64_t)(h << p.shift) + (m.x & mask)) * 16 + c, in_of = ((int64_t)(h << p.shift) + (m.y & mask)) * 16 + c;
      to_k[u] = id_to * (p.key_stride / 8) + in_to;
      to_v[u] = id_to * (p.value_stride / 8) + in_to;
      k[u] = a.keys[id_of * (p.key_stride / 8) + in_of];
      v[u] = a.values[id_of * (p.value_stride / 8) + in_of];
      if (c == 0) {
        const int64_t to = record_at(p, id_to, h, m.x & mask), of = record_at(p, id_of, h, m.y & mask);
        p.weight[to] = p.weight[of];
        p.token[to] = p.token[of];
      }
    }
#pragma unroll
    for (int u = 0; u < kMovesAtOnce; ++u) {
      if (to_k[u] < 0) continue;
      a.keys[to_k[u]] = k[u];
      a.values[to_v[u]] = v[u];
    }
  }
}

int64_t most_moves(const ri_paged& p, int64_t keep) {
  const int64_t room = (int64_t)p.table_stride * p.page_size;
  return keep >= room ? 0 : (keep < room - keep ? keep : room - keep);
}

}  // namespace

extern "C" int64_t ri_paged_evict_scratch_bytes(const ri_paged* p, int32_t keep) {
  const int rc = check(p, "ri_paged_evict");
  if (rc != RI_OK) return rc;
  if (keep < 1) return ri_fail(RI_ERR_INVALID, "ri_paged_evict: keep=%d unsupported", keep);
  const int64_t groups = (int64_t)p->batch * p->kv_heads;
  return ri_align_up(groups * 4, 16) + groups * most_moves(*p, keep) * 8 + 16;
}

extern "C" int ri_paged_evict(const ri_paged* p, const int32_t* d_seen, int32_t keep, int32_t n_sink, int32_t n_recent,
                              void* d_scratch, void* stream) {
  int rc;
  if ((rc = check(p, "ri_paged_evict")) != RI_OK) return rc;
  RI_REQUIRE(p->d_values && p->d_weight && p->d_token && d_seen && d_scratch, "ri_paged_evict: null pointer");
  RI_REQUIRE(keep >= 1 && n_sink >= 0 && n_recent >= 0 && (int64_t)n_sink + n_recent <= keep,
             "ri_paged_evict: keep=%d slots for %d first and %d last tokens", keep, n_sink, n_recent);
  RI_REQUIRE((uintptr_t)d_scratch % 16 == 0, "ri_paged_evict: the scratch must be 16-byte aligned");
  const int64_t groups = (int64_t)p->batch * p->kv_heads, room = (int64_t)p->table_stride * p->page_size;
  if (room <= keep) return RI_OK;                      // no request can hold more
  EvictArgs a = {};
  a.pages = view(*p);
  a.seen = d_seen;
  a.keys = static_cast<uint4*>(const_cast<void*>(p->d_keys));
  a.values = static_cast<uint4*>(const_cast<void*>(p->d_values));
  a.counts = static_cast<int32_t*>(d_scratch);
  a.moves = reinterpret_cast<int2*>(static_cast<uint8_t*>(d_scratch) + ri_align_up(groups * 4, 16));
  a.keep = keep; a.sink = n_sink; a.recent = n_recent;
  a.most = (int)most_moves(*p, keep);
  int sms = 0;
  if ((rc = ri_sm_count(&sms)) != RI_OK) return rc;
  if ((rc = ri_allow_smem<evict_select_kernel>(kCachedKeys * 4)) != RI_OK) return rc;
  int ctas = 1;                                        // as many CTAs to a group as fit the chip at once
  while (ctas < kSelMaxCluster && groups * ctas * 2 <= sms) ctas *= 2;
  const int64_t slice = (room + ctas - 1) / ctas;
  const size_t smem = (size_t)(slice < kCachedKeys ? slice : kCachedKeys) * 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RI_CUDA_OK(ri_launch_pdl_cluster(11, ctas, evict_select_kernel, dim3((unsigned)(groups * ctas)), dim3(kSelThreads), smem, s, a));
  const int64_t blocks = ((int64_t)a.most + kMovesPerBlock - 1) / kMovesPerBlock, wanted = (int64_t)sms * 16 / groups + 1;
  RI_CUDA_OK(ri_launch_pdl_id(11, evict_move_kernel, dim3((unsigned)(blocks < wanted ? blocks : wanted), (unsigned)groups),
                              dim3(kMoveThreads), 0, s, a));
  return RI_OK;
}
