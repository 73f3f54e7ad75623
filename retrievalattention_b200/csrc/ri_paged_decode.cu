// Attention of one new token over a paged cache, and the weight that it gives to every slot.
//   out_h = sum_j p_hj v_j,  p_hj = e^{s_hj - lse_h},  s_hj = scale q_h.k_j,  lse_h = log sum_j e^{s_hj}
//   weight_j += sum_h p_hj over the query heads of a KV head (what ri_paged_evict goes by), where asked for
// A request without slots has out 0 and lse -infinity, and so has a head all of whose scores are -infinity.  A score that is NaN or
// +infinity makes its head's out and lse and the group's weights NaN, as the formulas do.
//
// Bound by the rows of K and V, read once: with at most eight query heads to a KV head there are 16 operations for each byte
// read, a sixteenth of what the tensor cores need to be the limit, so m16n8k16 with the heads in M is enough.
// The split is that of the dense cache (ri_step_sequence.cuh): 16-row steps of all groups behind one another, an equal
// contiguous range per SM and again per warp, whatever the requests' lengths; a warp streams its steps through its own ring,
// filled by TMA, a box of 16 rows (8 where a page has no more) of both halves of the channels; the number of the next
// step's page is fetched a step ahead.  Layout in shared memory and the order of the keys in a step: as in ri_dense_decode.cu.
// The probabilities enter the second product as two 16-bit parts: 16 bits of them with bf16, 22 with fp16, whose short exponent a
// moving reference makes up for (see m_run).  Either is a hundredth of the output's own rounding: 0.3 % of bf16 outputs are not the
// ones that 32-bit probabilities give, but their neighbours.  A third part: 0.07 %, and 318 -> 330 us at 4 x 131072 slots.
// A second kernel merges a group's partial results by log-sum-exp in a fixed order.  For the weights the first kernel
// leaves the scores behind (4 bytes a slot and query head, against 512 a slot for K and V), and the second turns them into
// probabilities; every slot has one thread, so the sums have one order and no atomics.
// Short requests that leave the chip room give every group a cluster of CTAs, which does all of this in one kernel.
// With a window the steps between the first slots and the window are left out: they take no part in the split, and nothing of
// them, their page numbers among it, is read.  32 requests, window 8192, 8 heads of 4: 170 to 190 us, 5.7 to 6.3 TB/s.
// Requests that begin alike: this kernel has each one's own slots, beside the one of ri_paged_attend.cu over what they have in common.
// B200, bf16, 8 heads of 4: 4 x 131072 slots 318 to 345 us by the GPU, 6.2 to 6.8 TB/s (a copy: 6.6); 4 requests of 20K to 32K with
// weights 91 us, 4.8 TB/s: the SMs are done after 64 to 78 us, half of them by 68 (some two dozen SMs are the last in every case,
// whatever the page size, the lengths or the groups of a CTA; without the scores all are done 5 us earlier), and the second kernel
// has 10.  CTAs that take work from ones not launched yet ended together, but the units that this takes have few steps a warp and
// many partial results: 340 -> 362 and 98 -> 108 us.
#include <cooperative_groups.h>

#include <type_traits>

#include "ri_paged_shared.cuh"
#include "ri_step_sequence.cuh"
#include "ri_tc.cuh"
#include "ri_wave_attend.cuh"

namespace ri_wave {
namespace {

using namespace ri_tc;
using ri_page::Pages;
using ri_page::page_of;
using ri_page::page_to_write;
using ri_page::record_at;
using ri_seq::Place;
using ri_seq::count_steps;
using ri_seq::cta_start;
using ri_seq::find_place;
using ri_seq::next_place;
__device__ __forceinline__ int steps_of(int rows) { return ri_seq::steps_of<16>(rows); }

constexpr int kPagedWarps = 8;
constexpr int kPagedThreads = kPagedWarps * 32;
constexpr int kPagedMaxCtas = 160;                    // the grid is one CTA per SM, at most this many
constexpr int kPagedRing = kPagedWarps * kStages * kStageBytes;   // 192 KB, on a 1024-byte boundary
constexpr int kPagedSmem = 1024 + kPagedRing;
constexpr int kFinishThreads = 256;
constexpr int kMaxCluster = 8;
constexpr int kApart = 8;                             // steps whose products the tensor cores add up among themselves
// More steps than that to a warp, if every request were as long as its table has room for: sums in two levels.  32 steps that are
// cut off lose 64 * 2^-25 at most, 2e-6; the second level costs 0.4 us (8 heads: 8000 slots 14.0 and 14.4 us).
constexpr int kLongSteps = 32;

struct PagedArgs : Pages {
  static constexpr int kStep = 16;
  const uint4* q;
  float* part_o;             // [slots][gs][128]
  float2* part_ml;           // [slots][gs]: (maximum in the log2 domain, sum)
  float* scores;             // [step][gs][16] in the log2 domain, or null; inside a step the order of the lanes that made them
  float* lse;                // [groups][gs] or null
  uint16_t* out;
  int64_t q_stride;          // 16-byte pieces from request to request
  int gs, max_ctas;
  float scale2;
};
__device__ __forceinline__ int used_ctas(int total, int max_ctas) { return ri_seq::used_ctas<kPagedWarps>(total, max_ctas); }

// Where a request's rows lie among its slots.
struct AllSlots {
  __device__ __forceinline__ int slot(int row) const { return row; }
  __device__ __forceinline__ bool sees(int row, int rows) const { return row < rows; }
  __device__ __forceinline__ bool sees_step(int row, int rows) const { return row + 16 <= rows; }      // all of it
};
__device__ __forceinline__ AllSlots span_of(const PagedArgs&, int) { return {}; }

// A window: only the last `window` slots and the first `sink` are seen.  Between the two whole steps are left out, so that rows
// count on behind the first slots' last step where the window's first one begins; the slots of those two that are not seen are masked.
struct WindowArgs : PagedArgs {
  int window, sink;
};
struct WindowSpan {
  int front, skip, low, sink;            // rows in front of the gap, slots left out, the window's first slot
  __device__ __forceinline__ int slot(int row) const { return row < front ? row : row + skip; }
  __device__ __forceinline__ bool sees(int row, int rows) const { return row < rows && (slot(row) >= low || slot(row) < sink); }
  __device__ __forceinline__ bool sees_step(int row, int rows) const {
    return row + 16 <= rows && max(slot(row), sink) >= min(slot(row) + 16, low);
  }
};
__device__ __forceinline__ WindowSpan span_of(const WindowArgs& a, int b) {
  const int n = ri_page::rows_of(static_cast<const Pages&>(a), b), low = max(0, n - a.window), front = (min(a.sink, low) + 15) & ~15;
  return {front, max(0, (low & ~15) - front), low, a.sink};
}
__device__ __forceinline__ int rows_of(const WindowArgs& a, int b) {
  return ri_page::rows_of(static_cast<const Pages&>(a), b) - span_of(a, b).skip;
}

// The slots of its own that a request has behind those it has in common with others, whose partial results are there already.
struct SharedArgs : PagedArgs {
  ri_shared::Parts common;
};
__device__ __forceinline__ WindowSpan span_of(const SharedArgs& a, int b) {
  const int low = ri_shared::common_of(a, a.common, b);
  return {0, low & ~15, low, 0};
}
__device__ __forceinline__ int rows_of(const SharedArgs& a, int b) {
  const int n = ri_page::rows_of(static_cast<const Pages&>(a), b), low = ri_shared::common_of(a, a.common, b);
  return n > low ? n - (low & ~15) : 0;
}

// The scores of a step lie in the order of the lanes that made them: place i holds key (i / 2 % 2) * 8 + i / 4 + (i % 2) * 4.
__device__ __forceinline__ int slot_in_step(int place) { return (place & ~15) + ((place >> 1) & 1) * 8 + ((place >> 2) & 3) + (place & 1) * 4; }

// Two probabilities as two 16-bit parts each.  One that fp16 has no value for takes the smallest and what is too much of it, so
// that it gives finite values nothing and an infinite one its infinity.
template <int DT>
__device__ __forceinline__ uint2 two_parts(float p0, float p1) {
  if (DT != RI_F16) return split2<DT>(p0, p1);
  constexpr float kSmallest = 5.9604645e-8f;           // 2^-24
  const uint32_t hi = Elem<DT>::pack2(p0 > 0.f ? fmaxf(p0, kSmallest) : p0, p1 > 0.f ? fmaxf(p1, kSmallest) : p1);
  return make_uint2(hi, Elem<DT>::pack2(p0 - Elem<DT>::from_bits((uint16_t)(hi & 0xffffu)), p1 - Elem<DT>::from_bits((uint16_t)(hi >> 16))));
}

// BOX: rows of a TMA box.  CLUSTER: a group per cluster, which shares out the group's steps, joins the partial results through
// distributed shared memory and adds the weights: no second kernel.  LONG: see kLongSteps.  Args: PagedArgs or WindowArgs.
template <int DT, int BOX, bool WEIGHTS, bool CLUSTER, bool LONG, class Args>
__global__ void __launch_bounds__(kPagedThreads, 1) paged_decode_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v,
                                                                     const __grid_constant__ Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ __align__(8) uint64_t s_full[kPagedWarps][kStages];
  __shared__ int s_abort;
  __shared__ float sm_m[kPagedWarps][kMaxHeads], sm_l[kPagedWarps][kMaxHeads];
  __shared__ float2 s_ml[kMaxHeads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, t = lane & 3, gs = a.gs;
  const int sr = ((r & 1) << 2) | (r >> 1);              // the lane's row and pieces, see ri_dense_decode.cu
  if (tid == 0) s_abort = 0;
  if (lane == 0) {                                       // a warp's barriers are set up and fed by the same lane
    for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&s_full[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  volatile int* abort_flag = &s_abort;
  // The next kernel may start when the kernel in front of this one has ended, not before: it finds lengths and page tables as
  // they are without waiting for this one.
  // SharedArgs: the kernel in front is the one over what requests have in common, which has waited for those before it, and nothing
  // of its results is read here: this one streams rows on the SMs that the other is done with, and waits at its end.
  constexpr bool kBeside = std::is_same_v<Args, SharedArgs>;
  if (!kBeside) ri_pdl_wait();
  ri_pdl_trigger();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = CLUSTER ? (int)cluster.num_blocks() : 1, rank = CLUSTER ? (int)cluster.block_rank() : 0;
  const int c = (int)blockIdx.x;
  int c_lo, c_hi;                                        // this CTA's steps: of the whole sequence, or of its group
  Place c_first;
  int64_t score_step = 0;                                // where the group's scores begin, if steps are counted by group
  if (CLUSTER) {
    const int g = c / ctas, b = g / a.hk, rows = rows_of(a, b), n = steps_of(rows);
    if (n == 0) {                                        // the whole cluster leaves
      for (int i = tid + rank * kPagedThreads; i < gs * RI_HEAD_DIM; i += ctas * kPagedThreads) a.out[(int64_t)g * gs * RI_HEAD_DIM + i] = 0;
      if (rank == 0 && tid < gs && a.lse != nullptr) a.lse[g * gs + tid] = -INFINITY;
      ri_pdl_wait();
      return;
    }
    c_first = {g, 0, rows};
    c_lo = (int)((int64_t)n * rank / ctas);
    c_hi = (int)((int64_t)n * (rank + 1) / ctas);
    score_step = (int64_t)g * steps_of(a.width << a.shift);
  } else {
    const int total = count_steps(a), n_ctas = used_ctas(total, a.max_ctas);
    if (c >= n_ctas || total == 0) {
      ri_pdl_wait();
      return;
    }
    c_lo = cta_start(c, total, n_ctas);
    c_hi = cta_start(c + 1, total, n_ctas);
    c_first = find_place(a, c_lo);
  }
  const int c_n = c_hi - c_lo, lo = c_lo + c_n * warp / kPagedWarps, hi = c_lo + c_n * (warp + 1) / kPagedWarps;
  const bool merged = CLUSTER || c_hi <= c_first.first + steps_of(c_first.rows);      // the CTA's range lies inside one group

  // a stage: K, then V; of each the boxes one behind the other, a box as two halves of 64 channels
  constexpr int kTensor = kStageBytes / 2, kBox = BOX * 256, kHalf = BOX * 128, kStageStride = kPagedWarps * kStageBytes;
  uint8_t* my_ring = ring + warp * kStageBytes;
  const uint32_t my_ring_u32 = smem_u32(my_ring), my_full = smem_u32(&s_full[warp][0]);
  auto row_at = [&](int row) { return BOX == 16 ? row * 128 : (row >> 3) * kBox + (row & 7) * 128; };

  // Head r: a reference near the largest score so far, and the sum of the probabilities against it (this lane's share, reduced over
  // the quad at the end).  The reference is a whole number, so that it seldom moves and a power of two does the rescaling.
  // bf16 holds probabilities of any size.  fp16 ends at 2^-24: there the reference lies kAbove below the largest score, so that
  // probabilities go up to 2^15, and follows steps down whose largest is kSmallSteps smaller, to kDeepest below the largest
  // of all (`peak`; sums stay below 2^105).  What a probability may lose is 2^-25 against the 2^6 and more of its step's largest.
  constexpr float kAbove = DT == RI_F16 ? 15.f : 0.f, kSmallSteps = 8.f, kDeepest = 60.f;
  float m_run = -INFINITY, l_run = 0.f, peak = -INFINITY;
  // Tensor cores cut a sum off where an addition rounds to nearest, always towards zero, and over hundreds of steps that adds up
  // (400 steps: 5 % of fp16 outputs rounded to the wrong side).  So where there may be many (LONG) the products of up to kApart steps
  // are summed by themselves, in `last`, and `acc` holds those before them against the reference that they had, `m_acc`.
  float acc[8][4], last[8][4], m_acc = -INFINITY;
  int apart = 0;                           // steps in `last`
  auto heads_2t = [&](float f, float& f0, float& f1) {      // what belongs to heads 2t and 2t + 1, of which this lane has the sums
    f0 = __shfl_sync(0xffffffffu, f, (2 * t) * 4);
    f1 = __shfl_sync(0xffffffffu, f, (2 * t + 1) * 4);
  };
  auto add_up = [&](float (&sum)[8][4]) {      // sum = acc + last
    float f0, f1;
    heads_2t(exp2f(m_acc - (m_run == -INFINITY ? 0.f : m_run)), f0, f1);
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[x][i] = fmaf(acc[x][i], i & 1 ? f1 : f0, last[x][i]);
  };
  auto clear = [&] {
    m_run = m_acc = peak = -INFINITY;
    l_run = 0.f;
    apart = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[x][i] = last[x][i] = 0.f;
  };
  auto reduce_sum = [&] {
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  };
  // sums to rows of 128 floats, one per head (heads 2t and 2t+1 are this lane's)
  auto put = [&](float* o) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int ch = (x < 4) ? 8 * sr + 2 * x : 64 + 8 * sr + 2 * (x - 4);
      if (2 * t < gs) *reinterpret_cast<float2*>(o + (2 * t) * RI_HEAD_DIM + ch) = make_float2(last[x][0], last[x][2]);
      if (2 * t + 1 < gs) *reinterpret_cast<float2*>(o + (2 * t + 1) * RI_HEAD_DIM + ch) = make_float2(last[x][1], last[x][3]);
    }
  };
  // Slots: along the sequence (warp, group) goes up by one of the two at a time, so their sum names a partial result.
  auto store_partial = [&](int g) {
    const int64_t slot = (int64_t)(c * kPagedWarps + warp) + g;
    reduce_sum();
    if (LONG) add_up(last);
    put(a.part_o + slot * gs * RI_HEAD_DIM);
    if (t == 0 && r < gs) a.part_ml[slot * gs + r] = make_float2(m_run, l_run);
  };

  clear();
  if (lo < hi) {
    Place at_issue = CLUSTER ? c_first : find_place(a, lo), at = at_issue;
    // pages of the next step to issue; the second one only where a page is half a step
    int id0 = 0, id1 = 0;
    auto span_issue = span_of(a, at_issue.g / a.hk), span = span_issue;
    auto fetch_ids = [&](int s) {
      if (s >= at_issue.first + steps_of(at_issue.rows)) {
        do next_place(a, at_issue);
        while (s >= at_issue.first + steps_of(at_issue.rows));
        span_issue = span_of(a, at_issue.g / a.hk);
      }
      const int b = at_issue.g / a.hk, row = (s - at_issue.first) * 16, slot = span_issue.slot(row);
      id0 = page_of(a, b, slot >> a.shift);
      if (BOX == 8 && row + 8 < at_issue.rows) id1 = page_of(a, b, (slot + 8) >> a.shift);
    };
    auto issue = [&](int s, int stage) {
      if (lane == 0) {
        const uint32_t dst = my_ring_u32 + stage * kStageStride, bar = my_full + 8 * stage;
        const int row = (s - at_issue.first) * 16, slot = span_issue.slot(row);
        const int in_page = ((at_issue.g % a.hk) << a.shift) + (slot & ((1 << a.shift) - 1));
        const bool second = BOX == 8 && row + 8 < at_issue.rows;
        mbar_arrive_expect_tx(bar, (BOX == 16 || second) ? kStageBytes : kStageBytes / 2);
        tma_load_4d(dst, &map_k, bar, 0, in_page, 0, id0);
        tma_load_4d(dst + kTensor, &map_v, bar, 0, in_page, 0, id0);
        if (second) {
          const int in_next = ((at_issue.g % a.hk) << a.shift) + ((slot + 8) & ((1 << a.shift) - 1));
          tma_load_4d(dst + kBox, &map_k, bar, 0, in_next, 0, id1);
          tma_load_4d(dst + kTensor + kBox, &map_v, bar, 0, in_next, 0, id1);
        }
      }
    };
    int s_issue = lo;
#pragma unroll
    for (int st = 0; st < kStages; ++st)
      if (s_issue < hi) {
        fetch_ids(s_issue);
        issue(s_issue++, st);
      }
    if (s_issue < hi) fetch_ids(s_issue);
    uint4 qa[4];
    auto load_q = [&] {
      const int b = at.g / a.hk, h = at.g - b * a.hk;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        qa[kk] = r < gs ? ri_ldg16(a.q + b * a.q_stride + (h * gs + r) * 16 + t + kk * 4) : make_uint4(0, 0, 0, 0);
    };
    load_q();
    int stage = 0, phase = 0;
    bool ok = true;
#pragma unroll 1
    for (int s = lo; s < hi; ++s) {
      if (s >= at.first + steps_of(at.rows)) {
        store_partial(at.g);
        clear();
        do next_place(a, at);
        while (s >= at.first + steps_of(at.rows));
        span = span_of(a, at.g / a.hk);
        load_q();
      }
      const int base = (s - at.first) * 16;
      ok = __all_sync(0xffffffffu, mbar_wait(my_full + 8 * stage, phase, abort_flag, 71));
      if (!ok) break;
      const uint8_t* src = my_ring + stage * kStageStride;
      float s2[2][2];
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        float c1[4] = {0.f, 0.f, 0.f, 0.f}, c2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint4 kb = *reinterpret_cast<const uint4*>(src + (kk >> 1) * kHalf + row_at(8 * jj + sr) +
                                                           (((t ^ sr) << 4) ^ ((kk & 1) << 6)));
          Elem<DT>::mma16816(c1, qa[kk].x, 0u, qa[kk].y, 0u, kb.x, kb.y);
          Elem<DT>::mma16816(c2, qa[kk].z, 0u, qa[kk].w, 0u, kb.z, kb.w);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          s2[jj][e] = span.sees(base + jj * 8 + t + 4 * e, at.rows) ? (c1[e] + c2[e]) * a.scale2 : -INFINITY;
      }
      if (WEIGHTS && r < gs)
        reinterpret_cast<float4*>(a.scores)[((score_step + s) * gs + r) * 4 + t] = make_float4(s2[0][0], s2[0][1], s2[1][0], s2[1][1]);
      // softmax for head r against a running reference
      float mx = fmaxf(fmaxf(s2[0][0], s2[0][1]), fmaxf(s2[1][0], s2[1][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float here = ceilf(mx) - kAbove;               // NaN where all scores are: that moves nothing
      float m_new = fmaxf(m_run, here);
      if (DT == RI_F16) {
        peak = fmaxf(peak, here);
        if (here < m_run - kSmallSteps) m_new = fmaxf(here, peak - kDeepest);
      }
      const float m_safe = m_new == -INFINITY ? 0.f : m_new;
      if (LONG && apart == kApart) {
        add_up(acc);
        m_acc = m_run;
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) last[x][i] = 0.f;
        apart = 0;
      }
      ++apart;
      const float alpha = exp2f(m_run - m_safe);
      float p[2][2], psum = 0.f;
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[jj][e] = exp2f(s2[jj][e] - m_safe);
          psum += p[jj][e];
        }
      l_run = l_run * alpha + psum;
      m_run = m_new;
      float f0, f1;
      heads_2t(alpha, f0, f1);
#pragma unroll
      for (int x = 0; x < 8; ++x) { last[x][0] *= f0; last[x][1] *= f1; last[x][2] *= f0; last[x][3] *= f1; }
      uint4 v[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* at_v = src + kTensor + row_at(t + 4 * i) + (((sr ^ t) << 4) ^ ((i & 1) << 6));
        v[i][0] = *reinterpret_cast<const uint4*>(at_v);
        v[i][1] = *reinterpret_cast<const uint4*>(at_v + kHalf);
      }
      __syncwarp();
      if (s_issue < hi) {                             // the stage is in registers: refill it before the products
        issue(s_issue++, stage);
        if (s_issue < hi) fetch_ids(s_issue);
      }
      // what lies behind a group's rows, or in front of its window, may be anything
      if (!span.sees_step(base, at.rows)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!span.sees(base + t + 4 * i, at.rows)) v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
      }
      const uint2 b0 = two_parts<DT>(p[0][0], p[0][1]), b1 = two_parts<DT>(p[1][0], p[1][1]);
      pv_step<DT, true>(last, v, b0.x, b1.x, b0.y, b1.y);
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
    if (!ok) {               // leave a bounded chance to the copies in flight before their memory goes
      if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_wait(my_full + 8 * ((stage + i) % kStages), phase ^ (stage + i >= kStages), abort_flag, 72);
        *a.status = s_abort;
      }
      __syncwarp();
    } else if (!merged) {
      store_partial(at.g);
    }
  }
  ri_pdl_wait();
  if (!merged) return;

  reduce_sum();
  if (LONG) add_up(last);
  if (t == 0) { sm_m[warp][r] = m_run; sm_l[warp][r] = l_run; }
  auto warp_o = [&](int w) { return reinterpret_cast<float*>(ring + w * kStageBytes); };
  float* cta_o = reinterpret_cast<float*>(ring + kPagedWarps * kStageBytes);      // CLUSTER: this CTA's partial result
  put(warp_o(warp));
  __syncthreads();
  const int64_t slot = (int64_t)c * kPagedWarps + c_first.g;
  for (int idx = tid; idx < gs * RI_HEAD_DIM; idx += kPagedThreads) {
    const int h = idx >> 7;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) M = fmaxf(M, sm_m[w][h]);
    const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      const float f = exp2f(sm_m[w][h] - Ms);
      L += sm_l[w][h] * f;
      O += warp_o(w)[idx] * f;
    }
    if (CLUSTER) {
      cta_o[idx] = O;
      if ((idx & 127) == 0) s_ml[h] = make_float2(M, L);
    } else {
      a.part_o[slot * gs * RI_HEAD_DIM + idx] = O;
      if ((idx & 127) == 0) a.part_ml[slot * gs + h] = make_float2(M, L);
    }
  }
  if (!CLUSTER) return;

  cluster.sync();
  // reference and sum of head h over the cluster
  auto joined = [&](int h, float2 (&ml)[kMaxCluster]) {
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxCluster; ++i) {
      ml[i] = i < ctas ? *cluster.map_shared_rank(&s_ml[h], i) : make_float2(-INFINITY, 0.f);
      M = fmaxf(M, ml[i].x);
    }
    M = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < kMaxCluster; ++i) L += ml[i].y * exp2f(ml[i].x - M);
    return make_float2(M, L);
  };
  for (int idx = tid + rank * kPagedThreads; idx < gs * RI_HEAD_DIM; idx += ctas * kPagedThreads) {
    float2 ml[kMaxCluster];
    float o[kMaxCluster], O = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxCluster; ++i) o[i] = i < ctas ? cluster.map_shared_rank(cta_o, i)[idx] : 0.f;
    const float2 all = joined(idx >> 7, ml);
#pragma unroll
    for (int i = 0; i < kMaxCluster; ++i) O += o[i] * exp2f(ml[i].x - all.x);
    a.out[(int64_t)c_first.g * gs * RI_HEAD_DIM + idx] = Elem<DT>::bits(all.y == 0.f ? 0.f : O / all.y);
    if ((idx & 127) == 0 && a.lse != nullptr) a.lse[c_first.g * gs + (idx >> 7)] = all.y == 0.f ? -INFINITY : (all.x + log2f(all.y)) * 0.69314718055994531f;
  }
  if (WEIGHTS) {
    if (tid < gs) {
      float2 ml[kMaxCluster];
      const float2 all = joined(tid, ml);
      sm_l[0][tid] = all.y == 0.f ? INFINITY : all.x + log2f(all.y);      // nothing to give: 0
    }
    __syncthreads();
    const int b = c_first.g / a.hk, h_kv = c_first.g - b * a.hk;
    for (int place = c_lo * 16 + tid; place < c_hi * 16; place += kPagedThreads) {      // this CTA's own scores
      const int i = place & 15, at = slot_in_step(place);
      const int id = at < c_first.rows ? page_to_write(a, b, at >> a.shift) : -1;
      if (id < 0) continue;
      const float* of = a.scores + ((score_step + (place >> 4)) * gs) * 16 + i;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < kMaxHeads; ++h)
        if (h < gs) sum += exp2f(of[h * 16] - sm_l[0][h]);
      a.weight[record_at(a, id, h_kv, at & ((1 << a.shift) - 1))] += sum;
    }
  }
  cluster.sync();                                        // nobody's shared memory goes while others may read it
}

// A group's rows, the first of its steps in the sequence, and (warp 0) how many partial results it has, which `slots` takes.
struct Own {
  int rows, lo, count;
};
template <class Args>
__device__ __forceinline__ Own list_own(const Args& a, int b, int h_kv, int g, int* slots) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0, all = 0, rows = 0;                     // steps in front of the request (of one KV head), of all; its rows
  for (int i = lane; i < a.batch; i += 32) {
    const int r = rows_of(a, i), steps = steps_of(r);
    all += steps;
    if (i < b) before += steps;
    if (i == b) rows = r;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
    rows += __shfl_xor_sync(0xffffffffu, rows, o);
  }
  all *= a.hk;
  const int n = steps_of(rows), lo = before * a.hk + h_kv * n, hi = lo + n;
  int count = 0;
  if (warp == 0 && n > 0) {
    const int n_ctas = used_ctas(all, a.max_ctas);
    int c0 = (int)((int64_t)lo * n_ctas / all);          // the CTA that holds step lo
    while (c0 > 0 && cta_start(c0, all, n_ctas) > lo) --c0;
    while (cta_start(c0 + 1, all, n_ctas) <= lo) ++c0;
    for (int c_base = c0; c_base < n_ctas && cta_start(c_base, all, n_ctas) < hi; c_base += 4) {      // 4 CTAs a warp step
      const int c = c_base + (lane >> 3), w = lane & 7;
      bool mine = false;
      if (c < n_ctas) {
        const int c_lo = cta_start(c, all, n_ctas), c_n = cta_start(c + 1, all, n_ctas) - c_lo;
        if (c_lo >= lo && c_lo + c_n <= hi) {            // merged by the CTA
          mine = w == 0;
        } else {
          const int w_lo = c_lo + c_n * w / kPagedWarps, w_hi = c_lo + c_n * (w + 1) / kPagedWarps;
          mine = max(w_lo, lo) < min(w_hi, hi);
        }
      }
      const unsigned votes = __ballot_sync(0xffffffffu, mine);
      if (mine) slots[count + __popc(votes & ((1u << lane) - 1))] = c * kPagedWarps + w + g;
      count += __popc(votes);
    }
  }
  return {rows, lo, count};
}

// What is left once every partial result is there, a group per blockIdx.y: its blocks join the partial results, a query head at
// a time, and with weights turn the group's scores into probabilities, kFoldSlots slots at a time, a thread per slot.  Every
// block works out lse of all heads (warp h of head h), so none waits for another.  Which partial results the group has
// follows from the lengths, so a warp lists them, in the order of the sequence, before the wait for the kernel that makes them.
constexpr int kFoldEach = 2, kFoldSlots = kFoldEach * kFinishThreads;
constexpr int kFinishBlocks = 4;                         // of an SM
constexpr int kTogether = 4;                             // partial results of a warp on their way
template <int DT, class Args>
__global__ void __launch_bounds__(kFinishThreads, kFinishBlocks) paged_finish_kernel(const __grid_constant__ Args a) {
  extern __shared__ int s_slot[];                        // [most partial results of a group]
  __shared__ float s_m[kMaxHeads], s_l[kMaxHeads], s_o[kFinishThreads / 32][RI_HEAD_DIM];
  __shared__ int s_n;
  ri_pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.y, gs = a.gs, b = g / a.hk, h_kv = g - b * a.hk;
  const Own own = list_own(a, b, h_kv, g, s_slot);
  const int rows = own.rows, n = steps_of(rows), lo = own.lo;
  int count = own.count;
  // a tile of slots: pages (their tables do not change either), then scores and weights
  int id[kFoldEach] = {};
  float sc[kFoldEach][kMaxHeads], old[kFoldEach];
  auto slot_of = [&](int tile, int e) { return slot_in_step(tile * kFoldSlots + e * kFinishThreads + tid); };
  auto weight_at = [&](int tile, int e) { return a.weight + record_at(a, id[e], h_kv, slot_of(tile, e) & ((1 << a.shift) - 1)); };
  auto find_pages = [&](int tile) {
#pragma unroll
    for (int e = 0; e < kFoldEach; ++e) {
      const int slot = slot_of(tile, e);
      id[e] = slot < rows ? page_to_write(a, b, slot >> a.shift) : -1;
    }
  };
  auto fetch = [&](int tile) {
#pragma unroll
    for (int e = 0; e < kFoldEach; ++e) {
      const int place = tile * kFoldSlots + e * kFinishThreads + tid;
      const float* of = a.scores + ((int64_t)(lo + (place >> 4)) * gs) * 16 + (place & 15);
#pragma unroll
      for (int h = 0; h < kMaxHeads; ++h)
        if (h < gs && id[e] >= 0) sc[e][h] = of[h * 16];
      if (id[e] >= 0) old[e] = *weight_at(tile, e);
    }
  };
  const bool folds = a.weight != nullptr && (int)blockIdx.x * kFoldSlots < rows;
  if (folds) find_pages(blockIdx.x);
  if (tid == 0) s_n = count;
  ri_pdl_wait();
  if (n == 0) {
    for (int h = blockIdx.x; h < gs; h += gridDim.x) {
      if (tid < RI_HEAD_DIM) a.out[((int64_t)g * gs + h) * RI_HEAD_DIM + tid] = 0;
      if (tid == 0 && a.lse != nullptr) a.lse[g * gs + h] = -INFINITY;
    }
    return;
  }
  if (folds) fetch(blockIdx.x);
  __syncthreads();
  count = s_n;
  if (warp < gs) {
    float M = -INFINITY, L = 0.f;
    for (int i0 = 0; i0 < count; i0 += 32 * kTogether) {
      float2 ml[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int i = i0 + u * 32 + lane;
        ml[u] = i < count ? a.part_ml[(int64_t)s_slot[i] * gs + warp] : make_float2(-INFINITY, 0.f);
      }
      float most = M;
#pragma unroll
      for (int u = 0; u < kTogether; ++u) most = fmaxf(most, ml[u].x);
      const float ref = most == -INFINITY ? 0.f : most;
      L *= exp2f(M - ref);
#pragma unroll
      for (int u = 0; u < kTogether; ++u) L += ml[u].y * exp2f(ml[u].x - ref);
      M = most;
    }
    const float own = M;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float Ms = M == -INFINITY ? 0.f : M;
    L *= exp2f(own - Ms);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) {
      s_m[warp] = Ms;
      s_l[warp] = L;
      if (blockIdx.x == 0 && a.lse != nullptr) a.lse[g * gs + warp] = (M + log2f(L)) * 0.69314718055994531f;
    }
  }
  for (int head = blockIdx.x; head < gs; head += gridDim.x) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);          // a warp per partial result, four channels a lane
    float M = -INFINITY;                                 // this warp's reference; it need not wait for the head's
    for (int i0 = warp; i0 < count; i0 += kTogether * (kFinishThreads / 32)) {
      float4 x[kTogether];
      float m[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        const int i = i0 + u * (kFinishThreads / 32);
        m[u] = -INFINITY;
        if (i < count) {
          const int64_t at = (int64_t)s_slot[i] * gs + head;
          m[u] = a.part_ml[at].x;
          x[u] = reinterpret_cast<const float4*>(a.part_o + at * RI_HEAD_DIM)[lane];
        }
      }
      float most = M;
#pragma unroll
      for (int u = 0; u < kTogether; ++u) most = fmaxf(most, m[u]);
      if (most == -INFINITY) continue;
      const float f0 = exp2f(M - most);
      o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
      for (int u = 0; u < kTogether; ++u)
        if (i0 + u * (kFinishThreads / 32) < count) {
          const float f = exp2f(m[u] - most);
          o.x += x[u].x * f; o.y += x[u].y * f; o.z += x[u].z * f; o.w += x[u].w * f;
        }
      M = most;
    }
    __syncthreads();                                     // the head's maximum and sum are there, the last head's rows are read
    const float f = exp2f(M - s_m[head]);
    reinterpret_cast<float4*>(s_o[warp])[lane] = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    __syncthreads();
    if (tid < RI_HEAD_DIM) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kFinishThreads / 32; ++w) sum += s_o[w][tid];
      a.out[((int64_t)g * gs + head) * RI_HEAD_DIM + tid] = Elem<DT>::bits(s_l[head] == 0.f ? 0.f : sum / s_l[head]);
    }
  }
  if (!folds) return;
  __syncthreads();
  float lse2[kMaxHeads];
#pragma unroll
  for (int h = 0; h < kMaxHeads; ++h) lse2[h] = h < gs && s_l[h] != 0.f ? s_m[h] + log2f(s_l[h]) : INFINITY;      // nothing to give: 0
  for (int tile = blockIdx.x; tile * kFoldSlots < rows; tile += gridDim.x) {
    if (tile != (int)blockIdx.x) {
      find_pages(tile);
      fetch(tile);
    }
#pragma unroll
    for (int e = 0; e < kFoldEach; ++e) {
      if (id[e] < 0) continue;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < kMaxHeads; ++h)
        if (h < gs) sum += exp2f(sc[e][h] - lse2[h]);
      *weight_at(tile, e) = old[e] + sum;
    }
  }
}

// The same where requests have slots in common: a block per group joins the partial results over those and over the request's own, a
// thread for each query head and four channels, several of them with every n-th part each.  (As a part of the kernel above, a block for
// each query head: 64 requests of 8 heads of 4, 14 us.)  What it goes by are the call's inputs, so that it is looked up before the wait.
constexpr int kSharedThreads = 512;
template <int DT>
__global__ void __launch_bounds__(kSharedThreads, 2) shared_finish_kernel(const __grid_constant__ SharedArgs a) {
  extern __shared__ int s_slot[];
  __shared__ int s_n;
  __shared__ float4 s_o[kSharedThreads];
  __shared__ float2 s_ml[kSharedThreads];
  ri_pdl_trigger();
  const int gs = a.gs, g = blockIdx.x, b = g / a.hk, h_kv = g - b * a.hk;
  const int each = gs * (RI_HEAD_DIM / 4), teams = kSharedThreads / each, team = threadIdx.x / each, t = threadIdx.x - team * each;
  const int quad = t / gs, r = t - quad * gs;
  const ri_shared::Parts& x = a.common;
  int item = -1, item_rows = 0, item_row = 0;              // the group's item, if there is one
  if (ri_shared::common_of(a, x, b) > 0) {
    const int of = ri_shared::group_of(x.starts, x.groups, b);
    const int b0 = ri_shared::clamped(x.starts[of], a.batch), b1 = ri_shared::clamped(x.starts[of + 1], a.batch);
    const int first = b0 + (b - b0) / x.pair * x.pair;
    item = h_kv * a.batch + first;
    item_rows = min(x.pair, b1 - first) * gs;
    item_row = (b - first) * gs + r;
  }
  const Own own = list_own(a, b, h_kv, g, s_slot);
  if (threadIdx.x == 0) s_n = own.count;
  ri_pdl_wait();
  int extra = 0;
  int64_t part = 0;
  if (item >= 0) {
    const int c0 = ri_shared::clamped(x.ctas[2 * item], x.max_ctas - 1);
    extra = max(0, ri_shared::clamped(x.ctas[2 * item + 1], x.max_ctas - 1) - c0 + 1);
    part = (int64_t)c0 * x.part_rows + (int64_t)item * gs;
  }
  __syncthreads();
  const int count = extra + s_n;
  auto ml_of = [&](int i) {
    return i < extra ? x.ml[part + (int64_t)i * x.part_rows + item_row] : a.part_ml[(int64_t)s_slot[i - extra] * gs + r];
  };
  auto four_of = [&](int i) {
    return i < extra ? reinterpret_cast<const float4*>(x.o + (part + (int64_t)i * x.part_rows) * RI_HEAD_DIM)[((quad >> 1) * item_rows + item_row) * 2 + (quad & 1)]
                     : reinterpret_cast<const float4*>(a.part_o + ((int64_t)s_slot[i - extra] * gs + r) * RI_HEAD_DIM)[quad];
  };
  constexpr int kWide = 4;                                 // partial results on their way
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  // adds parts against the largest reference so far; one far below it, or what was there, still counts enough to hand on an infinite value
  auto factor = [](float m, float ref) { return m == -INFINITY ? 0.f : fmaxf(exp2f(m - ref), 1.17549435e-38f); };
  auto add = [&](const float2* ml, const float4* v, int n) {
    float most = M;
    for (int u = 0; u < n; ++u) most = fmaxf(most, ml[u].x);
    const float ref = most == -INFINITY ? 0.f : most, old = factor(M, ref);
    L *= old;
    o.x *= old; o.y *= old; o.z *= old; o.w *= old;
    for (int u = 0; u < n; ++u) {
      const float f = factor(ml[u].x, ref);
      L += ml[u].y * f;
      o.x += v[u].x * f; o.y += v[u].y * f; o.z += v[u].z * f; o.w += v[u].w * f;
    }
    M = most;
  };
  if (team < teams)
    for (int i0 = team; i0 < count; i0 += kWide * teams) {
      float2 ml[kWide];
      float4 v[kWide];
#pragma unroll
      for (int u = 0; u < kWide; ++u) {
        const int i = i0 + u * teams;
        ml[u] = make_float2(-INFINITY, 0.f);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < count) {
          ml[u] = ml_of(i);
          v[u] = four_of(i);
        }
      }
      add(ml, v, kWide);
    }
  s_ml[threadIdx.x] = make_float2(M, L);
  s_o[threadIdx.x] = o;
  __syncthreads();
  if (team > 0) return;
  for (int u = 1; u < teams; ++u) add(&s_ml[u * each + t], &s_o[u * each + t], 1);
  const float f = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2*>(a.out + ((int64_t)g * gs + r) * RI_HEAD_DIM + quad * 4) =
      make_uint2(Elem<DT>::pack2(o.x * f, o.y * f), Elem<DT>::pack2(o.z * f, o.w * f));
  if (quad == 0 && a.lse != nullptr) a.lse[g * gs + r] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

int64_t paged_slots(const ri_paged& p) { return (int64_t)kPagedMaxCtas * kPagedWarps + (int64_t)p.batch * p.kv_heads; }
int64_t paged_most_steps(const ri_paged& p) {
  return (int64_t)p.batch * p.kv_heads * ((ri_page::slots_of(p) + 15) / 16);
}

// Pages as (64 channels, row of the page's heads, half, page).
int make_page_map(CUtensorMap* map, const void* base, const ri_paged& p, int64_t page_stride, int box) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != RI_OK) return rc;
  const cuuint64_t dims[4] = {64, (cuuint64_t)p.kv_heads * p.page_size, 2, (cuuint64_t)p.n_pages};
  const cuuint64_t strides[3] = {256, 128, (cuuint64_t)page_stride * 2};
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 2, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, p.dtype == RI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RI_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return RI_OK;
}

// How many clusters of `ctas` CTAs the device holds at once: they lie inside one GPC, so that is not SMs / ctas.
int clusters_at_once(int ctas, int* out) {
  static std::atomic<int> known[64][kMaxCluster + 1];
  int dev = 0, rc;
  RI_CUDA_OK(cudaGetDevice(&dev));
  const bool track = dev >= 0 && dev < 64;
  if (track && (*out = known[dev][ctas].load(std::memory_order_relaxed)) > 0) return RI_OK;
  auto* kernel = paged_decode_kernel<RI_BF16, 16, true, true, false, PagedArgs>;      // all of them have the same shared memory and threads
  if ((rc = ri_allow_smem<paged_decode_kernel<RI_BF16, 16, true, true, false, PagedArgs>>(kPagedSmem)) != RI_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPagedThreads);
  cfg.dynamicSmemBytes = kPagedSmem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  RI_CUDA_OK(cudaOccupancyMaxActiveClusters(out, kernel, &cfg));
  if (track) known[dev][ctas].store(*out, std::memory_order_relaxed);
  return RI_OK;
}
// CTAs of a cluster where every group can have a cluster at once and the longest request that fits the tables is short; 0: no
// clusters.  A second kernel costs 2 us of host and device time; an even split over all SMs gains more than that from five steps a
// warp on (8 heads of 4, a call: 777 slots 11.3 us with two kernels, 9.6 with clusters; 4000 slots, four steps a warp, 11.6 and
// 9.7; 8000 slots 13.9 and 14.9).
constexpr int kClusterSteps = 4;                       // of a warp, at most
int cluster_size(const PagedArgs& a, int64_t most, int* ctas) {
  const int64_t groups = (int64_t)a.batch * a.hk, steps = (most + 15) / 16;
  *ctas = 0;
  if (groups > a.max_ctas || steps > kMaxCluster * kPagedWarps * kClusterSteps) return RI_OK;
  for (int n = 1; n <= kMaxCluster; n *= 2) {
    int fit = 0;
    const int rc = clusters_at_once(n, &fit);
    if (rc != RI_OK) return rc;
    if (groups <= fit && (*ctas == 0 || steps > (int64_t)*ctas * kPagedWarps)) *ctas = n;
  }
  if (steps > (int64_t)*ctas * kPagedWarps * kClusterSteps) *ctas = 0;
  return RI_OK;
}
// The most rows that a request may have.
int64_t most_rows(const PagedArgs& a) { return (int64_t)a.width << a.shift; }
int64_t most_rows(const WindowArgs& a) {
  const int64_t all = most_rows(static_cast<const PagedArgs&>(a)), seen = (int64_t)a.window + a.sink + 30;      // two steps begun
  return seen < all ? seen : all;
}
template <int DT, int BOX, bool WEIGHTS, bool LONG, class Args>
int launch_split(const Args& a, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t s) {
  const int rc = ri_allow_smem<paged_decode_kernel<DT, BOX, WEIGHTS, false, LONG, Args>>(kPagedSmem);
  if (rc != RI_OK) return rc;
  RI_CUDA_OK(ri_launch_pdl_id(11, paged_decode_kernel<DT, BOX, WEIGHTS, false, LONG, Args>, dim3(a.max_ctas), dim3(kPagedThreads), (size_t)kPagedSmem,
                              s, map_k, map_v, a));
  return RI_OK;
}
template <int DT, int BOX, bool WEIGHTS, class Args>
int launch_steps(const Args& a, const CUtensorMap& map_k, const CUtensorMap& map_v, int ctas, cudaStream_t s) {
  int rc;
  if constexpr (!std::is_same_v<Args, SharedArgs>) if (ctas > 0) {
    if ((rc = ri_allow_smem<paged_decode_kernel<DT, BOX, WEIGHTS, true, false, Args>>(kPagedSmem)) != RI_OK) return rc;
    RI_CUDA_OK(ri_launch_pdl_cluster(11, ctas, paged_decode_kernel<DT, BOX, WEIGHTS, true, false, Args>, dim3(a.batch * a.hk * ctas), dim3(kPagedThreads),
                                     (size_t)kPagedSmem, s, map_k, map_v, a));
    return RI_OK;
  }
  const int64_t steps = (int64_t)a.batch * a.hk * ((most_rows(a) + 15) / 16);
  return steps > (int64_t)a.max_ctas * kPagedWarps * kLongSteps ? launch_split<DT, BOX, WEIGHTS, true>(a, map_k, map_v, s)
                                                                : launch_split<DT, BOX, WEIGHTS, false>(a, map_k, map_v, s);
}
template <int DT, int BOX>
int launch_steps(const PagedArgs& a, const CUtensorMap& map_k, const CUtensorMap& map_v, int ctas, cudaStream_t s) {
  return a.weight ? launch_steps<DT, BOX, true, PagedArgs>(a, map_k, map_v, ctas, s) : launch_steps<DT, BOX, false, PagedArgs>(a, map_k, map_v, ctas, s);
}
template <int DT, int BOX>
int launch_steps(const SharedArgs& a, const CUtensorMap& map_k, const CUtensorMap& map_v, int ctas, cudaStream_t s) {
  return launch_steps<DT, BOX, false, SharedArgs>(a, map_k, map_v, 0, s);
}
template <int DT, int BOX>
int launch_steps(const WindowArgs& a, const CUtensorMap& map_k, const CUtensorMap& map_v, int ctas, cudaStream_t s) {
  return launch_steps<DT, BOX, false, WindowArgs>(a, map_k, map_v, ctas, s);
}
template <int DT, class Args>
int launch_paged(const Args& a, const CUtensorMap& map_k, const CUtensorMap& map_v, int box, cudaStream_t s) {
  const int64_t most = most_rows(a);
  int ctas = 0, rc;
  if (!std::is_same_v<Args, SharedArgs> && (rc = cluster_size(a, most, &ctas)) != RI_OK) return rc;
  rc = box == 8 ? launch_steps<DT, 8>(a, map_k, map_v, ctas, s) : launch_steps<DT, 16>(a, map_k, map_v, ctas, s);
  if (rc != RI_OK || ctas > 0) return rc;
  // partial results of a group: its steps, or all that there are and one more
  const int64_t groups = (int64_t)a.batch * a.hk, steps = (most + 15) / 16, parts = (int64_t)a.max_ctas * kPagedWarps;
  const size_t smem = (size_t)(steps < parts ? steps : parts) * 4 + 4;
  if constexpr (std::is_same_v<Args, SharedArgs>) {
    RI_CUDA_OK(ri_launch_pdl_id(11, shared_finish_kernel<DT>, dim3((unsigned)groups), dim3(kSharedThreads), smem, s, a));
  } else {
    // blocks of a group: for its heads, or with weights its tiles of slots, as many as the chip holds at once
    const int64_t tiles = a.weight ? (most + kFoldSlots - 1) / kFoldSlots : 0, room = kFinishBlocks * (int64_t)a.max_ctas / groups;
    int64_t blocks = tiles > a.gs ? tiles : a.gs;
    if (blocks > room) blocks = room > 1 ? room : 1;
    RI_CUDA_OK(ri_launch_pdl_id(11, paged_finish_kernel<DT, Args>, dim3((unsigned)blocks, (unsigned)groups), dim3(kFinishThreads), smem, s, a));
  }
  return RI_OK;
}

}  // namespace
}  // namespace ri_wave

extern "C" int64_t ri_paged_decode_scratch_bytes(const ri_paged* p) {
  const int rc = ri_page::check(p, "ri_paged_decode");
  if (rc != RI_OK) return rc;
  if (p->group_size < 1 || p->group_size > ri_wave::kMaxHeads) return ri_fail(RI_ERR_INVALID, "ri_paged_decode: group_size=%d unsupported", p->group_size);
  int64_t floats = ri_wave::paged_slots(*p) * p->group_size * (RI_HEAD_DIM + 2);
  if (p->d_weight) floats += 4 + ri_wave::paged_most_steps(*p) * p->group_size * 16;
  return floats * 4;
}

namespace ri_wave {
namespace {

// Checks of a call, and what all of its kernels go by.
int prepare(const char* what, const ri_paged* p, const void* d_q, int64_t q_stride, void* d_out, float* d_lse, float scale, void* d_scratch,
            PagedArgs& a) {
  int rc;
  if ((rc = ri_page::check(p, what)) != RI_OK) return rc;
  RI_REQUIRE(p->d_values && d_q && d_out && d_scratch, "%s: null pointer", what);
  RI_REQUIRE(p->group_size >= 1 && p->group_size <= kMaxHeads, "%s: group_size=%d unsupported (1 to %d)", what, p->group_size, kMaxHeads);
  RI_REQUIRE(q_stride >= (int64_t)p->kv_heads * p->group_size * RI_HEAD_DIM && q_stride % 8 == 0, "%s: queries overlap or lie at odd places", what);
  RI_REQUIRE(((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_scratch) % 16 == 0, "q, out and the scratch must be 16-byte aligned");
  RI_REQUIRE(scale > 0.f && scale < 1e30f, "%s: scale must be positive and finite", what);
  static_cast<ri_page::Pages&>(a) = ri_page::view(*p);
  a.q = static_cast<const uint4*>(d_q);
  a.q_stride = q_stride / 8;
  a.gs = p->group_size;
  a.part_o = static_cast<float*>(d_scratch);
  float* next = a.part_o + paged_slots(*p) * a.gs * RI_HEAD_DIM;
  a.part_ml = reinterpret_cast<float2*>(next);
  next += paged_slots(*p) * a.gs * 2;
  if (p->d_weight) a.scores = reinterpret_cast<float*>(ri_align16((size_t)next));
  a.lse = d_lse;
  a.out = static_cast<uint16_t*>(d_out);
  a.scale2 = RI_LOG2E * scale;
  int sms = 0;
  if ((rc = ri_sm_count(&sms)) != RI_OK) return rc;
  a.max_ctas = sms < kPagedMaxCtas ? sms : kPagedMaxCtas;
  return RI_OK;
}
template <class Args>
int launch(const ri_paged& p, const Args& a, void* stream) {
  int rc;
  const int box = p.page_size < 16 ? 8 : 16;
  CUtensorMap map_k, map_v;
  if ((rc = make_page_map(&map_k, p.d_keys, p, p.key_page_stride, box)) != RI_OK) return rc;
  if ((rc = make_page_map(&map_v, p.d_values, p, p.value_page_stride, box)) != RI_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p.dtype == RI_BF16 ? launch_paged<RI_BF16>(a, map_k, map_v, box, s) : launch_paged<RI_F16>(a, map_k, map_v, box, s);
}

// Requests that begin alike are attended together where all slots there may be are more than this many bytes of K and V.  It takes a
// kernel more, and requests that are attended one by one find much of what others have read in L2: 8 heads of 4, L2 flushed, 8 requests of
// 4096 slots in common and 500 of their own (151 MB) 42 us together and 34 one by one, 16 requests (302 MB) 48 and 52, 8 requests over
// 16384 slots (554 MB) 60 and 85; 64 over 32768 (9.1 GB), not flushed, 138 and 1140.
constexpr int64_t kAlikeBytes = 160 << 20;
bool apart(const ri_paged& p) { return (int64_t)p.batch * p.kv_heads * ri_page::slots_of(p) * 4 * RI_HEAD_DIM <= kAlikeBytes; }
int64_t own_bytes(const ri_paged& p) { return ri_align_up(paged_slots(p) * p.group_size * (RI_HEAD_DIM + 2) * 4, 16); }

}  // namespace
}  // namespace ri_wave

extern "C" int ri_paged_decode(const ri_paged* p, const void* d_q, int64_t q_stride, void* d_out, float* d_lse, float scale,
                               void* d_scratch, void* stream) {
  ri_wave::PagedArgs a = {};
  const int rc = ri_wave::prepare("ri_paged_decode", p, d_q, q_stride, d_out, d_lse, scale, d_scratch, a);
  return rc != RI_OK ? rc : ri_wave::launch(*p, a, stream);
}

extern "C" int ri_paged_decode_window(const ri_paged* p, const void* d_q, int64_t q_stride, int32_t window, int32_t sink, void* d_out,
                                      float* d_lse, float scale, void* d_scratch, void* stream) {
  RI_REQUIRE(window >= 1 && sink >= 0, "ri_paged_decode_window: window=%d sink=%d unsupported", window, sink);
  RI_REQUIRE(p == nullptr || p->d_weight == nullptr, "ri_paged_decode_window: weights are added up over all slots, not over a window");
  ri_wave::WindowArgs a = {};
  const int rc = ri_wave::prepare("ri_paged_decode_window", p, d_q, q_stride, d_out, d_lse, scale, d_scratch, a);
  a.window = window;
  a.sink = sink;
  return rc != RI_OK ? rc : ri_wave::launch(*p, a, stream);
}

extern "C" int64_t ri_paged_shared_decode_scratch_bytes(const ri_paged* p, int32_t groups) {
  const int rc = ri_page::check(p, "ri_paged_shared_decode");
  if (rc != RI_OK) return rc;
  if (p->group_size < 1 || p->group_size > ri_wave::kMaxHeads)
    return ri_fail(RI_ERR_INVALID, "ri_paged_shared_decode: group_size=%d unsupported", p->group_size);
  if (groups < 1 || groups > p->batch) return ri_fail(RI_ERR_INVALID, "ri_paged_shared_decode: groups=%d unsupported", groups);
  return ri_wave::own_bytes(*p) + (ri_wave::apart(*p) ? 0 : ri_shared::scratch_bytes(*p));
}

extern "C" int ri_paged_shared_decode(const ri_paged* p, const void* d_q, int64_t q_stride, const int32_t* d_group_start, int32_t groups,
                                      const int32_t* d_shared, void* d_out, float* d_lse, float scale, void* d_scratch, void* stream) {
  const int64_t bytes = ri_paged_shared_decode_scratch_bytes(p, groups);
  if (bytes < 0) return (int)bytes;
  RI_REQUIRE(d_shared && d_group_start, "ri_paged_shared_decode: null pointer");
  RI_REQUIRE(p->d_weight == nullptr, "ri_paged_shared_decode: weights are not added up where slots are in common");
  ri_wave::SharedArgs a = {};
  int rc = ri_wave::prepare("ri_paged_shared_decode", p, d_q, q_stride, d_out, d_lse, scale, d_scratch, a);
  if (rc != RI_OK) return rc;
  if (ri_wave::apart(*p)) return ri_wave::launch(*p, static_cast<const ri_wave::PagedArgs&>(a), stream);
  rc = ri_shared::launch("ri_paged_shared_decode", p, d_q, q_stride, d_group_start, groups, d_shared, scale,
                         static_cast<char*>(d_scratch) + ri_wave::own_bytes(*p), &a.common, static_cast<cudaStream_t>(stream));
  return rc != RI_OK ? rc : ri_wave::launch(*p, a, stream);
}
