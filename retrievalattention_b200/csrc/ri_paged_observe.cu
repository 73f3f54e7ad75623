// The attention weight that the last `window` queries of every request give to the slots of a paged cache.
//   weight_j += sum over query rows r (window query w, query head h of the KV head):  e^{s_rj - lse_r},
//   s_rj = scale q_r.k_j,  lse_r = log sum_j e^{s_rj},  both over the slots that query w sees: j <= length - window + w.
// Rows that see no slot (prompts shorter than the window), or only slots of score -infinity, give nothing.
//
// Two passes over K, both on the tensor cores, with the query rows of a KV head (window x group, 256 at a time) in shared memory:
//   pass 1  S = Q.K^T, M 128 query rows x N 128 keys: a thread holds a query row and keeps its running maximum and sum;
//   pass 2  S^T = K.Q^T, M 128 keys x N query rows: a thread holds a key and adds the probabilities of the rows.
// Either way the reduction stays inside a thread; the operands lie in shared memory the same way for both (rows of 128 channels in
// two 128-byte-swizzled halves), only their roles change.  A slot's weight has one thread, so there are no atomics.
// The split is that of the decode kernels: tiles of 128 slots of all groups behind one another, an equal contiguous range per SM.
// Pass 1 leaves a (maximum, sum) per row and range; pass 2 merges its group's, or where they are many a kernel between the passes.
// Four warps bring in tiles, issue the products and idle, sixteen work on scores: two sides of eight, one per tile of query
// rows in pass 1 (or every second tile of keys, where there is only one), every second tile of keys in pass 2; of a side's
// scores four warps take the first half of the columns and four the second.
// TMEM: 256 columns of scores for each side.  Every wait is bounded; one that runs out is recorded in the
// status word.
// Bound by the exponentials, two for each slot and query row.  B200, 4 requests of 20K to 32K slots, 8 heads, 256 query rows: 165 to 170 us
// by the GPU in a repeated run, 2.5 of the 4.2 exponentials a picosecond that the SMs have at 16 a clock and 1.76 GHz; pass 1 takes 71 us
// from rest (exponentials busy 79 % of the active cycles, tensor pipe 39 %), pass 2 82 (68 %: it also reads each row's lse).  With
// eight score warps 188 us: two warps of a scheduler do not cover each other's loads and barriers.  Some of the exponentials as
// polynomials on the FMA pipe gained nothing with either.
#include <cuda.h>

#include "ri_paged.cuh"
#include "ri_step_sequence.cuh"
#include "ri_tc.cuh"

namespace {

using namespace ri_tc;
using namespace ri_page;
using ri_seq::Place;

constexpr int kTile = 128;                       // slots of a tile
constexpr int kRows = 256;                       // query rows that are worked on together
constexpr int kKeyHalf = kTile * 128, kKeyTile = 2 * kKeyHalf;
constexpr int kRowHalf = kRows * 128, kRowTile = 2 * kRowHalf;
constexpr int kRing = 4;                         // K tiles in shared memory
constexpr int kScoreWarps = 16, kScoreThreads = kScoreWarps * 32;
constexpr int kObsThreads = 128 + kScoreThreads;
constexpr int kPartials = 2 * kRows;             // a (maximum, sum) for each row and half of the columns
constexpr uint32_t kTmemCols = 512;
constexpr int kObsSmem = 1024 + kRowTile + kRing * kKeyTile;
constexpr int kObsMaxCtas = 160;
constexpr int kMergedInside = 16;                // CTAs of a group, see ri_paged_observe

struct ObsArgs : Pages {
  static constexpr int kStep = kTile;
  const uint4* q;                                // [batch][window][hk * gs][16 pieces]
  float2* part;                                  // [slots][half][kRows]: (maximum in the log2 domain, sum)
  float* lse2;                                   // [groups][kRows], +infinity: the row gives nothing; null: pass 2 merges `part`
  int window, gs, first_row, rows;               // rows first_row .. first_row + rows - 1 of window * gs
  int max_ctas;
  float scale2;
  uint32_t idesc;
  int mixed_halves;                              // pages of eight slots: the halves of eight keys lie behind one another
};

// 2^x to within 2^-22 of itself, as exp2f; results below 2^-126 become 0 (they are added to sums of 1 and more, or are weights that
// no eviction tells from 0).  The weights come out within 1.5e-7 of 64 bits where 32-bit torch operations are within 1.0e-7.
__device__ __forceinline__ float ex2(float x) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
constexpr float kFarAbove = 1.2676506e30f;            // 2^100

__device__ __forceinline__ void load_scores(uint32_t taddr, uint32_t (&r)[32]) {
  tc_ld32(taddr, r);
  tc_wait_ld();
  tc_ld_landed(r);
}
// Sum of 2^(s * scale + shift) over 32 scores, added to `sum`; `shift` holds one value a pair of scores.
template <class Shift>
__device__ __forceinline__ void add_exps(const uint32_t (&sr)[32], uint64_t scale, Shift shift, uint64_t (&sum)[2]) {
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const uint64_t e = fma_f2(pack_f2(__uint_as_float(sr[2 * x]), __uint_as_float(sr[2 * x + 1])), scale, shift(x));
    float e0, e1;
    unpack_f2(e, e0, e1);
    sum[x & 1] = add_f2(sum[x & 1], pack_f2(ex2(e0), ex2(e1)));
  }
}
__device__ __forceinline__ float total_of(const uint64_t (&sum)[2]) {
  float a, b;
  unpack_f2(add_f2(sum[0], sum[1]), a, b);
  return a + b;
}
// Pass 1: over 64 scores of a row, one shift for all.
__device__ __forceinline__ float row_sum(uint32_t taddr, float scale, float shift) {
  const uint64_t scale_2 = pack_f2(scale, scale), shift_2 = pack_f2(shift, shift);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t sr[32];
    load_scores(taddr + k * 32, sr);
    add_exps(sr, scale_2, [&](int) { return shift_2; }, sum);
  }
  return total_of(sum);
}
// Pass 2: over a slot's scores with `chunks` * 32 query rows, a shift for each.
__device__ __forceinline__ float column_sum(uint32_t taddr, int chunks, float scale, const float* shift) {
  const uint64_t scale_2 = pack_f2(scale, scale);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll 1
  for (int k = 0; k < chunks; ++k) {
    uint32_t sr[32];
    load_scores(taddr + k * 32, sr);
    const ulonglong2* at = reinterpret_cast<const ulonglong2*>(shift + k * 32);
    add_exps(sr, scale_2, [&](int x) { const ulonglong2 two = at[x >> 1]; return (x & 1) ? two.y : two.x; }, sum);
  }
  return total_of(sum);
}
// The last slot that query row `row` sees in a request of n slots (negative: none).
__device__ __forceinline__ int last_seen(const ObsArgs& a, int n, int row) { return n - a.window + row / a.gs; }

// Where all scores so far are -infinity (or NaN), a reference that leaves them what they are.
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }
struct Sum {                                         // of 2^(x - m)
  float m = -INFINITY, l = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float2 (&x)[N]) {
    float m_new = m, each = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) m_new = fmaxf(m_new, x[i].x);
    const float ref = reference(m_new);
#pragma unroll
    for (int i = 0; i < N; ++i) each += x[i].y * ex2(x[i].x - ref);
    l = l * ex2(m - ref) + each;
    m = m_new;
  }
  __device__ __forceinline__ float lse2() const { return l > 0.f || l != l ? m + log2f(l) : INFINITY; }      // no slot: gives nothing
};
// The CTA that pass 1 gave tile t to.
__device__ __forceinline__ int cta_of(int t, int total, int n_ctas) {
  int c = (int)((int64_t)t * n_ctas / total);
  while (c > 0 && ri_seq::cta_start(c, total, n_ctas) > t) --c;
  while (ri_seq::cta_start(c + 1, total, n_ctas) <= t) ++c;
  return c;
}
// Adds row `row`'s partial results of CTAs c0, c0 + step, ... below c1.
__device__ __forceinline__ void add_partials(const ObsArgs& a, Sum& sum, int g, int row, int c0, int c1, int step) {
  const int each = a.rows <= kTile ? 4 : 2;          // partial results of a CTA: two halves of the columns, and of one or both sides
  for (int c = c0; c < c1; c += 4 * step) {          // four CTAs' on their way together
    float2 x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int u = c + (i >> 2) * step, k = i & 3;
      x[i] = u < c1 && k < each ? a.part[(int64_t)(u + g) * kPartials + (k & 1) * kRows + (k >> 1) * kTile + row] : make_float2(-INFINITY, 0.f);
    }
    sum.add(x);
  }
}

// STATS: pass 1.
template <int DT, bool STATS>
__global__ void __launch_bounds__(kObsThreads, 1) observe_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ ObsArgs a) {
  constexpr int kBuffers = STATS ? 2 : 1;        // of scores, for each side of the score warps: 128 columns each, or 256
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* q_rows = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sQ = base, sK = base + kRowTile;
  __shared__ __align__(8) uint64_t s_bars[1 + 2 * kRing + 8];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  __shared__ __align__(16) float s_neg_lse[kRows];
  __shared__ __align__(16) int s_last[kRows];
  __shared__ float s_sum[2][2][kTile];             // pass 2: what the second half of the query rows gives
  __shared__ int s_nan;                            // some row's lse is no number
  const uint32_t bars = smem_u32(s_bars);
  const uint32_t bar_q = bars;                                              // the group's query rows are there
  auto bar_full = [&](int s) { return bars + 8u * (1 + s); };               // a K tile is there, is free
  auto bar_empty = [&](int s) { return bars + 8u * (1 + kRing + s); };
  auto bar_s_full = [&](int g, int i) { return bars + 8u * (1 + 2 * kRing + 2 * g + i); };      // scores are there, are read
  auto bar_s_empty = [&](int g, int i) { return bars + 8u * (5 + 2 * kRing + 2 * g + i); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(bar_q, kScoreWarps);
    for (int s = 0; s < kRing; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
    for (int g = 0; g < 2; ++g)
      for (int i = 0; i < 2; ++i) { mbar_init(bar_s_full(g, i), 1); mbar_init(bar_s_empty(g, i), kScoreWarps / 2); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  volatile int* abort_flag = &s_abort;
  // Pass 1 lets the next kernel start when the kernel in front of it has ended, not before.  So pass 2, which starts behind
  // pass 1 or beside the merge, finds queries, keys and lengths as they are, and waits only where it reads what those wrote.
  if (STATS) ri_pdl_wait();
  ri_pdl_trigger();

  // this CTA's tiles [lo, hi) of the sequence, segment by segment (the part of a group that falls to it)
  const int total = ri_seq::count_steps(a), n_ctas = min(a.max_ctas, total), c = (int)blockIdx.x;
  const int lo = c < n_ctas ? ri_seq::cta_start(c, total, n_ctas) : 0, hi = c < n_ctas ? ri_seq::cta_start(c + 1, total, n_ctas) : 0;
  // Pass 2 walks its range backwards: what pass 1 read last is still in L2.
  auto tile_at = [&](int i) { return STATS ? lo + i : hi - 1 - i; };
  auto walk_to = [&](Place& at, int t) {
    if (STATS) {
      while (t >= at.first + ri_seq::steps_of<kTile>(at.rows)) ri_seq::next_place(a, at);
    } else {
      while (t < at.first) ri_seq::previous_place(a, at);
    }
  };
  // both sides of the score warps work on the same keys where there are query rows for both, on every second tile otherwise
  const bool both = STATS && a.rows > kTile;

  if (lo < hi) {
    if (warp == 0) {
      // ---------------- K tiles, a box of at most a page per lane ----------------
      Place at = ri_seq::find_place(a, tile_at(0));
      const int box = min(1 << a.shift, kTile), mask = (1 << a.shift) - 1;
      bool ok = true;
      int issued = 0;
      // a tile's boxes, and the page of this lane's; the next tile's page numbers are on their way while a tile's copies are issued
      struct Tile {
        int boxes, id, y;
      };
      auto plan = [&](int i) {
        const int t = tile_at(i);
        walk_to(at, t);
        const int b = at.g / a.hk, h = at.g - b * a.hk, slot0 = (t - at.first) * kTile;
        Tile tile = {(min(kTile, at.rows - slot0) + box - 1) / box, 0, (h << a.shift) + ((slot0 + lane * box) & mask)};
        if (lane < tile.boxes) tile.id = a.table[(int64_t)b * a.table_stride + ((slot0 + lane * box) >> a.shift)];
        return tile;
      };
      Tile next = plan(0);
      for (; issued < hi - lo; ++issued) {
        const Tile tile = next;
        if (issued + 1 < hi - lo) next = plan(issued + 1);
        const int s = issued % kRing;
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty(s), ((issued / kRing) & 1) ^ 1, abort_flag, 81));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(bar_full(s), tile.boxes * box * 256);
        __syncwarp();
        if (lane < tile.boxes) {
          const int id = page_or_first(a, tile.id);
          const uint32_t dst = sK + s * kKeyTile + lane * box * (a.mixed_halves ? 256 : 128);
          tma_load_4d(dst, &map_k, bar_full(s), 0, tile.y, 0, id);
          if (!a.mixed_halves) tma_load_4d(dst + kKeyHalf, &map_k, bar_full(s), 0, tile.y, 1, id);
        }
      }
      if (*abort_flag)         // give the copies still in flight a bounded chance to land before the CTA exits
        for (int t = max(0, issued - kRing); t < issued; ++t) mbar_wait(bar_full(t % kRing), (t / kRing) & 1, abort_flag, 82);
    } else if (warp == 1) {
      // ---------------- products ----------------
      Place at = ri_seq::find_place(a, tile_at(0));
      const uint32_t key_half = a.mixed_halves ? 1024 : kKeyHalf, key_eight = a.mixed_halves ? 2048 : 1024;
      if (lane == 0) {
        bool ok = true;
        int used = 0, groups = 0, made[2] = {0, 0};
        for (; ok && used < hi - lo; ++used) {
          const int g_before = at.g;
          walk_to(at, tile_at(used));
          if (used == 0 || at.g != g_before) ok = mbar_wait(bar_q, groups++ & 1, abort_flag, 83);
          const int s = used % kRing;
          ok = ok && mbar_wait(bar_full(s), (used / kRing) & 1, abort_flag, 84);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (!both && g != (used & 1)) continue;
            const int i = made[g] % kBuffers;
            ok = ok && mbar_wait(bar_s_empty(g, i), ((made[g] / kBuffers) & 1) ^ 1, abort_flag, 85);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = STATS ? tmem + (2 * g + i) * 128 : tmem + g * 256;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              const uint64_t dk = umma_desc_sw128(sK + s * kKeyTile + kb * key_half, key_eight);
              const uint64_t dq = umma_desc_sw128(sQ + kb * kRowHalf + (both && g ? kTile * 128 : 0));
#pragma unroll
              for (int k = 0; k < 4; ++k) tc_mma_f16(d, (STATS ? dq : dk) + 2 * k, (STATS ? dk : dq) + 2 * k, a.idesc, (kb | k) != 0);
            }
            tc_commit(bar_s_full(g, i));
            ++made[g];
          }
          if (ok) tc_commit(bar_empty(s));
        }
      }
    } else if (warp >= 4) {
      // ---------------- scores ----------------
      const int side = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane;
      const int tid = threadIdx.x - 128, g = side;
      const uint32_t t_lane = (uint32_t)(quarter * 32) << 16;
      Place at = ri_seq::find_place(a, tile_at(0));
      bool ok = true;
      int done = 0, used = 0;                          // tiles of this side, of the CTA
      while (used < hi - lo) {
        walk_to(at, tile_at(used));
        const int g_first = at.first, g_end = at.first + ri_seq::steps_of<kTile>(at.rows), n = at.rows;
        // of the group's tiles, those in this CTA's range: up to place `end` of its walk
        const int end = STATS ? min(hi, g_end) - lo : hi - max(lo, g_first);
        const int b = at.g / a.hk, h = at.g - b * a.hk;
        // the group's query rows, their pieces swizzled as TMA would; every product over the rows before has completed, since
        // its scores have been read
        asm volatile("bar.sync 1, %0;" ::"n"(kScoreThreads) : "memory");
        {
          // a half-warp per row, eight rows of a thread on their way together
          const int piece = tid & 15;
          uint4 x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int i = u * 32 + (tid >> 4), r = a.first_row + i, w = r / a.gs;
            x[u] = i < a.rows ? ri_ldg16(a.q + (((int64_t)b * a.window + w) * a.hk * a.gs + h * a.gs + r - w * a.gs) * 16 + piece)
                              : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int i = u * 32 + (tid >> 4);
            *reinterpret_cast<uint4*>(q_rows + (piece >> 3) * kRowHalf + i * 128 + (((piece & 7) ^ (i & 7)) << 4)) = x[u];
          }
          if (!STATS) {
            if (tid == 0) s_nan = 0;
            ri_pdl_wait();
            asm volatile("bar.sync 1, %0;" ::"n"(kScoreThreads) : "memory");
            if (tid < kRows) {
              float lse2;
              if (a.lse2 != nullptr) {
                lse2 = a.lse2[(int64_t)at.g * kRows + tid];
              } else {
                Sum sum;
                const int last_tile = at.first + ri_seq::steps_of<kTile>(n) - 1;
                if (tid < a.rows)
                  add_partials(a, sum, at.g, tid, cta_of(at.first, total, n_ctas), cta_of(last_tile, total, n_ctas) + 1, 1);
                lse2 = sum.lse2();
              }
              s_neg_lse[tid] = -lse2;
              if (lse2 != lse2) s_nan = 1;
              s_last[tid] = tid < a.rows ? last_seen(a, n, a.first_row + tid) : -1;
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync 1, %0;" ::"n"(kScoreThreads) : "memory");
        if (lane == 0) mbar_arrive(bar_q);
        if (STATS) {
          const int r = both ? g * kTile + row : row;
          const int last = r < a.rows ? last_seen(a, n, a.first_row + r) : n - 1;      // rows that fill up a tile hold nobody up
          float m = -INFINITY, l = 0.f;
          for (; used < end; ++used) {
            const int t = tile_at(used);
            if (!both && g != (used & 1)) continue;
            const int i = done % kBuffers;
            ok = ok && __all_sync(0xffffffffu, mbar_wait(bar_s_full(g, i), (done / kBuffers) & 1, abort_flag, 86));
            if (!ok) continue;
            tc_fence_after();
            const uint32_t scores = tmem + (2 * g + i) * 128 + half * 64 + t_lane;
            const int slot0 = (t - at.first) * kTile + half * 64;
            const bool edge = slot0 + 63 > last;      // some scores are masked for this row
            float sum = 0.f;
            // The exponentials need no maximum, just a reference near it: the largest of the first 32 scores, for all tiles.  A
            // tile where the sum grows out of hand against it, or where scores are masked, is done from its own maximum.
            bool again = edge;
            if (!__any_sync(0xffffffffu, edge)) {
              if (__any_sync(0xffffffffu, m == -INFINITY)) {
                uint32_t sr[32];
                load_scores(scores, sr);
                float mx = __uint_as_float(sr[0]);
#pragma unroll
                for (int x = 1; x < 31; x += 2) mx = max3(mx, __uint_as_float(sr[x]), __uint_as_float(sr[x + 1]));
                if (m == -INFINITY) m = fmaxf(mx, __uint_as_float(sr[31])) * a.scale2;
              }
              sum = row_sum(scores, a.scale2, -m);
              again = !(sum < kFarAbove);
            }
            if (__any_sync(0xffffffffu, again)) {
              float mx = -INFINITY;
#pragma unroll 1
              for (int k = 0; k < 2; ++k) {
                uint32_t sr[32];
                load_scores(scores + k * 32, sr);
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (slot0 + k * 32 + x <= last) mx = fmaxf(mx, __uint_as_float(sr[x]));
              }
              const float m_new = fmaxf(m, mx * a.scale2), ref = reference(m_new);
              l *= ex2(m - ref);
              m = m_new;
              sum = 0.f;
#pragma unroll 1
              for (int k = 0; k < 2; ++k) {
                uint32_t sr[32];
                load_scores(scores + k * 32, sr);
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (slot0 + k * 32 + x <= last) sum += ex2(__uint_as_float(sr[x]) * a.scale2 - ref);
              }
            }
            l += sum;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_s_empty(g, i));
            ++done;
          }
          a.part[(int64_t)(c + at.g) * kPartials + half * kRows + side * kTile + row] = make_float2(m, l);
        } else {
          // this thread's slot in the tile at place i of the walk, and the number of its page as the table has it
          auto slot_at = [&](int i) { return (tile_at(i) - at.first) * kTile + row; };
          auto page_at = [&](int i) {
            return i < end && !half && slot_at(i) < n ? a.table[(int64_t)b * a.table_stride + (slot_at(i) >> a.shift)] : 0;
          };
          if (g != (used & 1)) ++used;
          int next_page = page_at(used);
          for (; used < end; used += 2) {
            const int slot = slot_at(used), slot0 = slot - row;
            float* weight = nullptr;
            float old = 0.f;
            const int id = !half && slot < n ? page_or_none(a, next_page) : -1;
            next_page = page_at(used + 2);
            if (id >= 0) {
              weight = a.weight + record_at(a, id, h, slot & ((1 << a.shift) - 1));
              old = *weight;
            }
            ok = ok && __all_sync(0xffffffffu, mbar_wait(bar_s_full(g, 0), done & 1, abort_flag, 87));
            tc_fence_after();
            // some query rows do not see some of the tile's slots
            const bool edge = slot0 + kTile - 1 > n - a.window || s_nan;
            const int chunks = (a.rows + 31) / 32, chunk0 = half ? (chunks + 1) / 2 : 0, my_chunks = half ? chunks / 2 : (chunks + 1) / 2;
            const uint32_t scores = tmem + g * 256 + chunk0 * 32 + t_lane;
            float sum = 0.f;
            // Where every row sees every slot, rows that fill up the last 32 give nothing by their shift of -infinity.  They are zeros,
            // though, and make NaN of an infinite key: a sum that is NaN is done again without them.
            bool masked = edge;
            if (ok && !edge) {
              sum = column_sum(scores, my_chunks, a.scale2, s_neg_lse + chunk0 * 32);
              masked = __any_sync(0xffffffffu, sum != sum);
            }
            if (ok && masked) {        // without `ok` there are no scores to read, but the warp that shares the slots is still met below
              sum = 0.f;
#pragma unroll 1
              for (int k = 0; k < my_chunks; ++k) {
                uint32_t sr[32];
                load_scores(scores + k * 32, sr);
                const int r0 = (chunk0 + k) * 32;
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (slot <= s_last[r0 + x]) sum += ex2(__uint_as_float(sr[x]) * a.scale2 + s_neg_lse[r0 + x]);
              }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_s_empty(g, 0));
            ++done;
            // the two warps that share a slot's query rows meet; the sums of two tiles lie in turn in two places, so that one
            // is read before the meeting after which it is written again
            const int place = done & 1, meeting = 2 + side * 4 + quarter;
            if (half) s_sum[side][place][row] = sum;
            asm volatile("bar.sync %0, 64;" ::"r"(meeting) : "memory");
            if (!half && weight != nullptr) *weight = old + (sum + s_sum[side][place][row]);
          }
          used = end;
        }
      }
    }
  }
  ri_pdl_wait();                                   // CTAs without tiles too: the kernel behind waits for this one alone
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && s_abort) *a.status = s_abort;
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// lse of 32 query rows of one group: the partial results of the CTAs that worked on it, every eighth one by one warp.
__global__ void __launch_bounds__(256) observe_merge_kernel(const __grid_constant__ ObsArgs a) {
  ri_pdl_enter();
  __shared__ float2 s_part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.y, b = g / a.hk;
  const int row = blockIdx.x * 32 + lane, tiles = ri_seq::steps_of<kTile>(rows_of(a, b));
  Sum sum;
  int before = 0, total = 0;
  for (int i = lane; i < a.batch; i += 32) {
    const int t = ri_seq::steps_of<kTile>(rows_of(a, i));
    total += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  total *= a.hk;
  if (tiles > 0 && row < a.rows) {
    const int lo = before * a.hk + (g - b * a.hk) * tiles, n_ctas = min(a.max_ctas, total);
    add_partials(a, sum, g, row, cta_of(lo, total, n_ctas) + warp, cta_of(lo + tiles - 1, total, n_ctas) + 1, 8);
  }
  s_part[warp][lane] = make_float2(sum.m, sum.l);
  __syncthreads();
  if (warp == 0) {
    float2 x[8];
#pragma unroll
    for (int w = 0; w < 8; ++w) x[w] = s_part[w][lane];
    sum = Sum();
    sum.add(x);
    a.lse2[(int64_t)g * kRows + row] = sum.lse2();
  }
}

// Keys as (channel of a half, row of the page's heads, half, page); a box is one half of the channels of at most a page.  Pages of
// eight slots would take 32 boxes of 1 KB a tile, which cost more than their bytes: a box holds both halves there, one behind the
// other (2 requests of 26508 slots, 4 heads, 70 query rows: 48.7 -> 39.1 us).  Boxes of more rows with both halves would leave the
// operand's groups of eight rows at unequal distances, and there are few enough of them: 40 us at 16 slots a page, 37 at 128.
int make_key_map(CUtensorMap* map, const ri_paged& p, bool mixed_halves) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != RI_OK) return rc;
  const cuuint64_t dims[4] = {RI_HEAD_DIM / 2, (cuuint64_t)p.kv_heads * p.page_size, 2, (cuuint64_t)p.n_pages};
  const cuuint64_t strides[3] = {256, 128, (cuuint64_t)p.key_page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)(p.page_size < kTile ? p.page_size : kTile), mixed_halves ? 2u : 1u, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, p.dtype == RI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(p.d_keys), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RI_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return RI_OK;
}

template <int DT>
int launch_observe(ObsArgs a, const CUtensorMap& map_k, cudaStream_t s) {
  int rc;
  if ((rc = ri_allow_smem<observe_kernel<DT, true>>(kObsSmem)) != RI_OK) return rc;
  if ((rc = ri_allow_smem<observe_kernel<DT, false>>(kObsSmem)) != RI_OK) return rc;
  const int rows = a.window * a.gs;
  for (a.first_row = 0; a.first_row < rows; a.first_row += kRows) {
    a.rows = rows - a.first_row < kRows ? rows - a.first_row : kRows;
    a.idesc = idesc_f16(DT, 128, 128);
    RI_CUDA_OK(ri_launch_pdl_id(11, observe_kernel<DT, true>, dim3(a.max_ctas), dim3(kObsThreads), (size_t)kObsSmem, s, map_k, a));
    if (a.lse2 != nullptr) RI_CUDA_OK(ri_launch_pdl_id(11, observe_merge_kernel, dim3(kRows / 32, a.batch * a.hk), dim3(256), 0, s, a));
    a.idesc = idesc_f16(DT, 128, (a.rows + 31) / 32 * 32);      // the scores are read 32 columns at a time
    RI_CUDA_OK(ri_launch_pdl_id(11, observe_kernel<DT, false>, dim3(a.max_ctas), dim3(kObsThreads), (size_t)kObsSmem, s, map_k, a));
  }
  return RI_OK;
}

int64_t obs_slots(const ri_paged& p) { return kObsMaxCtas + (int64_t)p.batch * p.kv_heads; }

}  // namespace

extern "C" int64_t ri_paged_observe_scratch_bytes(const ri_paged* p) {
  const int rc = check(p, "ri_paged_observe");
  if (rc != RI_OK) return rc;
  return obs_slots(*p) * kPartials * 8 + (int64_t)p->batch * p->kv_heads * kRows * 4;
}

extern "C" int ri_paged_observe(const ri_paged* p, const void* d_q, int32_t window, float scale, void* d_scratch, void* stream) {
  int rc;
  if ((rc = check(p, "ri_paged_observe")) != RI_OK) return rc;
  RI_REQUIRE(p->d_weight && d_q && d_scratch, "ri_paged_observe: null pointer");
  RI_REQUIRE(window >= 1 && p->group_size >= 1 && (int64_t)window * p->group_size < (1 << 20),
             "ri_paged_observe: window=%d group_size=%d unsupported", window, p->group_size);
  RI_REQUIRE(((uintptr_t)d_q | (uintptr_t)d_scratch) % 16 == 0, "q and the scratch must be 16-byte aligned");
  RI_REQUIRE(scale > 0.f && scale < 1e30f, "ri_paged_observe: scale must be positive and finite");
  ObsArgs a = {};
  static_cast<Pages&>(a) = view(*p);
  a.q = static_cast<const uint4*>(d_q);
  a.part = static_cast<float2*>(d_scratch);
  // A group that few CTAs share: pass 2 merges its partial results by itself; else a kernel between the passes does, once for all.
  // 1001 slots, 8 heads, 8 CTAs a group: 11.5 us merged inside, 13.2 by a kernel; 4000 slots of one head, 32 CTAs: 17.1 and 16.2.
  const int64_t groups = (int64_t)p->batch * p->kv_heads, tiles = (slots_of(*p) + kTile - 1) / kTile;
  const int64_t most = kObsMaxCtas / groups + 2;
  if ((most < tiles ? most : tiles) > kMergedInside) a.lse2 = reinterpret_cast<float*>(a.part + obs_slots(*p) * kPartials);
  a.window = window;
  a.gs = p->group_size;
  a.scale2 = RI_LOG2E * scale;
  a.mixed_halves = p->page_size == 8;
  int sms = 0;
  if ((rc = ri_sm_count(&sms)) != RI_OK) return rc;
  a.max_ctas = sms < kObsMaxCtas ? sms : kObsMaxCtas;
  CUtensorMap map_k;
  if ((rc = make_key_map(&map_k, *p, a.mixed_halves)) != RI_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p->dtype == RI_BF16 ? launch_observe<RI_BF16>(a, map_k, s) : launch_observe<RI_F16>(a, map_k, s);
}
