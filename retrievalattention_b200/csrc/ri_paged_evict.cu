// Eviction from a paged cache by accumulated attention weight, in place.
//   Of the slots of a request and KV head, `keep` stay: those of the first n_sink and the last n_recent tokens, then the ones of
//   largest weight, the lower slot first where weights are equal (a NaN is less than any weight).  Slots in front of `keep` that
//   go are filled from behind it, the i-th hole with the i-th slot that stays: keys, values, weights and token numbers.
// Attention does not depend on the order of the slots (rotary positions are in the keys), so nothing else has to move: of n
// slots about keep (n - keep) / n where weights are in no order, and no more than n - keep where a few generated tokens are
// trimmed; sources lie behind `keep` and destinations in front, so no row is read after it was written.
//
// Selection: a cluster of CTAs per group (request, KV head) maps weights to order-preserving 32-bit keys in shared memory (slots
// beyond that are mapped again when they are needed), finds the keep-th largest by a radix select of three levels whose
// histograms the CTAs add up through distributed shared memory, and writes the lists of holes and of the slots that fill them,
// both ascending.  Every thread takes a run of consecutive slots, of odd length against bank conflicts.
// Moves: a half-warp per row, two rows in flight; where there are few, by the same clusters, else by a second kernel over the
// whole chip.  Bound by the moved rows, read once and written once, or by the selection's chain of dependent steps.
// B200, fp16, 4 requests x 8 heads, 20K to 32K -> 8K slots: 60 us, 20 of them the selection; the moves run at 5.3 TB/s, what
// gathers of 256-byte rows reach (four rows in flight of fewer warps: 4.6).  16 x 8, 4160 -> 4096: 13 us, a chain of 30 steps.
#include <cooperative_groups.h>

#include "ri_paged.cuh"

namespace {

using namespace ri_page;
namespace cg = cooperative_groups;

constexpr int kFewThreads = 256, kManyThreads = 512;  // of a CTA of the selection
constexpr int kFewPerSm = 3;                         // CTAs of few threads on an SM
constexpr int kCachedKeys = 40 * 1024;               // keys of a CTA's slice that shared memory holds
constexpr int kSelMaxCluster = 8;
// Slots of a group that are worth another CTA (8 groups, a call; 512 against 2048): 600 slots 14.7 and 16.0 us, 1001 16.6 and 16.0,
// 2000 18.7 and 16.1, 4160 20.7 and 17.1.
constexpr int kSlotsWorthACta = 512;
constexpr int kMoveThreads = 256;
constexpr int kMovesAtOnce = 2;                      // per half-warp
constexpr int kMovesPerBlock = kMoveThreads / 16 * kMovesAtOnce;
// Moves per CTA up to which the selection's clusters do them: with 128 groups of 4096 slots and a few, 256 take 21.7 us inside and 23.4
// by a kernel of their own, 512 33.0 and 30.9.
constexpr int kMovesInside = 256;
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
template <int WARPS, typename T>
__device__ __forceinline__ T block_scan(T v, T* warp_sums, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();                                     // warp_sums may still be read by the scan before
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const T s = warp_sums[w];
    if (w < warp) before += s;
    total += s;
  }
  return before + incl - v;
}

// The moves of group (b, h): half-warp `half` of `halves` takes kMovesAtOnce neighbours at a time, whose rows often lie together.
__device__ __forceinline__ void move_rows(const EvictArgs& a, const int2* moves, int b, int h, int half, int halves, int n) {
  const Pages& p = a.pages;
  const int c = threadIdx.x & 15, mask = (1 << p.shift) - 1;
  for (int i0 = half * kMovesAtOnce; i0 < n; i0 += halves * kMovesAtOnce) {
    int64_t to_k[kMovesAtOnce], to_v[kMovesAtOnce];    // negative: nothing to move
    uint4 k[kMovesAtOnce], v[kMovesAtOnce];
#pragma unroll
    for (int u = 0; u < kMovesAtOnce; ++u) {
      to_k[u] = -1;
      if (i0 + u >= n) continue;
      const int2 m = moves[i0 + u];
      const int id_to = page_to_write(p, b, m.x >> p.shift), id_of = page_to_write(p, b, m.y >> p.shift);
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

constexpr int kLevels = 3, kDigits = 2048;             // 11, 11 and 10 bits of the key
struct SelShared {
  int hist[kLevels][kDigits];  // per level: this CTA's slots by digit
  unsigned long long totals;   // holes and fillers of this CTA, 32 bits each
  unsigned long long warp_sums[kManyThreads / 32];
  int warp_counts[kManyThreads / 32];
  int digit, before;           // the cut's digit, and slots of larger digits
};

// MOVES: the cluster moves the rows itself.  CTAs of few threads are clusters by themselves.
template <int THREADS, bool MOVES>
__global__ void __launch_bounds__(THREADS, THREADS == kFewThreads ? kFewPerSm : 1) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ __align__(16) SelShared sh;
  ri_pdl_enter();
  constexpr int kMaxCtas = THREADS == kFewThreads ? 1 : kSelMaxCluster;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = kMaxCtas > 1 ? (int)cluster.block_rank() : 0, ctas = kMaxCtas > 1 ? (int)cluster.num_blocks() : 1;
  const int tid = threadIdx.x, g = blockIdx.x / ctas;
  const Pages& p = a.pages;
  const int b = g / p.hk, h = g - b * p.hk, n = rows_of(p, b);
  if (n <= a.keep) {                                   // the whole cluster leaves
    if (rank == 0 && tid == 0) a.counts[g] = 0;
    return;
  }
  const int slice = ((n + ctas - 1) / ctas + 3) & ~3, lo = min(n, rank * slice), hi = min(n, lo + slice), mine = hi - lo;
  const int newest = a.seen[b] - a.recent;
  auto meet = [&] {                                    // of the cluster
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  };
  auto record_of = [&](int j) { return record_at(p, page_of(p, b, j >> p.shift), h, j & ((1 << p.shift) - 1)); };
  auto key_from = [&](float w, int t) { return (t < a.sink || t >= newest) ? kProtected : order_key(w); };
  for (int i = tid; i < kLevels * kDigits / 4; i += THREADS) reinterpret_cast<int4*>(&sh.hist[0][0])[i] = make_int4(0, 0, 0, 0);
  // four slots of a page at a time, and four such pieces of a thread on their way together; the slice begins where a piece does
  const int cached = min(mine, kCachedKeys);
  for (int j0 = 4 * tid; j0 < cached; j0 += 16 * THREADS) {
    int64_t at[4];
    float4 w[4];
    int4 t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u] = j0 + 4 * u * THREADS < cached ? record_of(lo + j0 + 4 * u * THREADS) : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at[u] >= 0) {
        w[u] = *reinterpret_cast<const float4*>(p.weight + at[u]);
        t[u] = *reinterpret_cast<const int4*>(p.token + at[u]);
      }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (at[u] >= 0)                                  // up to three slots behind the last one: there is room, and nobody reads them
        *reinterpret_cast<uint4*>(s_keys + j0 + 4 * u * THREADS) =
            make_uint4(key_from(w[u].x, t[u].x), key_from(w[u].y, t[u].y), key_from(w[u].z, t[u].z), key_from(w[u].w, t[u].w));
  }
  __syncthreads();
  auto key_of = [&](int j) {
    if (j < kCachedKeys) return s_keys[j];
    const int64_t at = record_of(lo + j);
    return key_from(p.weight[at], p.token[at]);
  };

  // the keep-th largest key: digit by digit, `need` slots still to be found among those that agree so far
  uint32_t prefix = 0;
  int need = a.keep, ties = 0;                         // ties: slots of the group with the cut's digit
#pragma unroll
  for (int level = 0; level < kLevels; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    const uint32_t mask = level == 2 ? 1023u : 2047u;
    for (int j = tid; j < mine; j += THREADS) {
      const uint32_t k = key_of(j);
      if (level == 0 || (k >> (level == 1 ? 21 : 10)) == (prefix >> (level == 1 ? 21 : 10))) atomicAdd(&sh.hist[level][(k >> shift) & mask], 1);
    }
    meet();
    // each thread adds up kEach neighbouring digits over the cluster, the largest ones at thread 0
    constexpr int kEach = kDigits / THREADS;
    const int digit = kDigits - kEach - kEach * tid;
    int each[kEach], mine_all = 0;
#pragma unroll
    for (int q = 0; q < kEach; q += 4) {
      int4 of[kMaxCtas], sum = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c)
        of[c] = c < ctas ? *reinterpret_cast<const int4*>(cluster.map_shared_rank(&sh.hist[level][0], c) + digit + q) : make_int4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c) { sum.x += of[c].x; sum.y += of[c].y; sum.z += of[c].z; sum.w += of[c].w; }
      each[q] = sum.x; each[q + 1] = sum.y; each[q + 2] = sum.z; each[q + 3] = sum.w;
      mine_all += sum.x + sum.y + sum.z + sum.w;
    }
    int total;
    int before = block_scan<THREADS / 32>(mine_all, sh.warp_counts, total);
    if (before < need && before + mine_all >= need) {
      int d = kEach - 1;
#pragma unroll
      for (int i = kEach - 1; i > 0; --i)
        if (d == i && before + each[i] < need) {
          before += each[i];
          --d;
        }
      sh.digit = digit + d;
      sh.before = before;
    }
    __syncthreads();
    prefix |= (uint32_t)sh.digit << shift;
    need -= sh.before;
  }
  for (int c = 0; c < ctas; ++c) ties += cluster.map_shared_rank(&sh.hist[kLevels - 1][0], c)[prefix & 1023u];
  // the first `need` slots of the group with the cut's key stay; mostly that is all of them
  const int run = ((mine + THREADS - 1) / THREADS) | 1, first = min(mine, tid * run), last = min(mine, first + run);
  int rank_eq = 0;
  if (ties > need) {
    int equal = 0, total;
    for (int c = 0; c < rank; ++c) rank_eq += cluster.map_shared_rank(&sh.hist[kLevels - 1][0], c)[prefix & 1023u];
    for (int j = first; j < last; ++j) equal += key_of(j) == prefix;
    rank_eq += block_scan<THREADS / 32>(equal, sh.warp_counts, total);
  } else {
    need = ties;
  }
  int eq = rank_eq;
  unsigned holes = 0, fillers = 0;
  for (int j = first; j < last; ++j) {
    const uint32_t k = key_of(j);
    const bool stays = k > prefix || (k == prefix && eq++ < need), front = lo + j < a.keep;
    holes += front && !stays;
    fillers += !front && stays;
  }
  unsigned long long total, at = block_scan<THREADS / 32>((unsigned long long)fillers << 32 | holes, sh.warp_sums, total);
  if (tid == 0) sh.totals = total;
  meet();
  unsigned long long all = 0;
  for (int c = 0; c < ctas; ++c) {
    const unsigned long long x = *cluster.map_shared_rank(&sh.totals, c);
    if (c < rank) at += x;
    all += x;
  }
  int hole_at = (int)(unsigned)at, filler_at = (int)(at >> 32);
  int2* moves = a.moves + (int64_t)g * a.most;
  eq = rank_eq;
  if (holes + fillers > 0)
    for (int j = first; j < last; ++j) {
      const uint32_t k = key_of(j);
      const bool stays = k > prefix || (k == prefix && eq++ < need), front = lo + j < a.keep;
      if (front && !stays) moves[hole_at++].x = lo + j;
      if (!front && stays) moves[filler_at++].y = lo + j;
    }
  if (rank == 0 && tid == 0) a.counts[g] = (int)(unsigned)all;
  meet();                                      // the list is there; nobody's shared memory goes while others may read it
  if (MOVES) move_rows(a, moves, b, h, rank * (THREADS / 16) + (tid >> 4), ctas * (THREADS / 16), (int)(unsigned)all);
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs a) {
  ri_pdl_enter();
  const int g = blockIdx.y, b = g / a.pages.hk, half = threadIdx.x >> 4;
  move_rows(a, a.moves + (int64_t)g * a.most, b, g - b * a.pages.hk, blockIdx.x * (kMoveThreads / 16) + half,
            gridDim.x * (kMoveThreads / 16), a.counts[g]);
}

int64_t most_moves(const ri_paged& p, int64_t keep) {
  const int64_t room = slots_of(p);
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
  RI_REQUIRE(((uintptr_t)d_scratch | (uintptr_t)p->d_weight | (uintptr_t)p->d_token) % 16 == 0,
             "ri_paged_evict: weights, token numbers and the scratch must be 16-byte aligned");
  const int64_t groups = (int64_t)p->batch * p->kv_heads, room = slots_of(*p);
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t key_bytes = ri_align_up(room, 4) * 4;
  bool moves;
  if (groups > sms && (key_bytes + (int64_t)sizeof(SelShared) + 1024) * kFewPerSm <= 227 * 1024) {
    // more groups than SMs, each small: three CTAs an SM take them side by side (304 groups, 969 -> 590
    // slots: 46 us with one, 33 with three; 160 groups, 6000 -> 5900: 35 and 27)
    moves = a.most <= kMovesInside;
    const int most = 227 * 1024 / kFewPerSm - 1024 - (int)sizeof(SelShared);
    auto kernel = moves ? evict_select_kernel<kFewThreads, true> : evict_select_kernel<kFewThreads, false>;
    if ((rc = moves ? ri_allow_smem<evict_select_kernel<kFewThreads, true>>(most) : ri_allow_smem<evict_select_kernel<kFewThreads, false>>(most)) != RI_OK)
      return rc;
    RI_CUDA_OK(ri_launch_pdl_id(11, kernel, dim3((unsigned)groups), dim3(kFewThreads), (size_t)key_bytes, s, a));
  } else {
    int ctas = 1;                                      // as many CTAs to a group as fit the chip at once and have enough to do
    while (ctas < kSelMaxCluster && groups * ctas * 2 <= sms && room > (int64_t)ctas * kSlotsWorthACta) ctas *= 2;
    const int64_t slice = ri_align_up((room + ctas - 1) / ctas, 4);
    const size_t smem = (size_t)(slice < kCachedKeys ? slice : kCachedKeys) * 4;
    moves = a.most <= (int64_t)ctas * kMovesInside;
    auto kernel = moves ? evict_select_kernel<kManyThreads, true> : evict_select_kernel<kManyThreads, false>;
    if ((rc = moves ? ri_allow_smem<evict_select_kernel<kManyThreads, true>>(kCachedKeys * 4)
                    : ri_allow_smem<evict_select_kernel<kManyThreads, false>>(kCachedKeys * 4)) != RI_OK)
      return rc;
    RI_CUDA_OK(ri_launch_pdl_cluster(11, ctas, kernel, dim3((unsigned)(groups * ctas)), dim3(kManyThreads), smem, s, a));
  }
  if (moves) return RI_OK;
  const int64_t blocks = ((int64_t)a.most + kMovesPerBlock - 1) / kMovesPerBlock, wanted = (int64_t)sms * 16 / groups + 1;
  RI_CUDA_OK(ri_launch_pdl_id(11, evict_move_kernel, dim3((unsigned)(blocks < wanted ? blocks : wanted), (unsigned)groups),
                              dim3(kMoveThreads), 0, s, a));
  return RI_OK;
}
