// Attention of many query rows over a paged cache, on the tensor cores.
//   out_r = sum_j p_rj v_j,  p_rj = e^{s_rj - lse_r},  s_rj = scale q_r.k_j,  lse_r = log sum_j e^{s_rj},  over the slots j that row r sees:
// ri_paged_prompt         several new tokens of every request: the token at slot s sees j <= s with j > s - window or j < sink;
// ri_paged_shared_decode  one new token of every request, where groups of requests have their first slots in common: a group's rows over
//                         those slots are worked on together here; each request's own slots and the join are ri_paged_decode.cu's.
// A row that sees nothing, or only scores of -infinity, has out 0 and lse -infinity; a NaN or +infinity among its scores makes both NaN.
//
// The rows of a tile of 128 are tokens (or requests) times the query heads of one KV head, so K and V serve a whole group of heads and a
// tile spans few tokens: with four heads 32, which is what keeps the masked part of a window small.  An item is up to two neighbouring
// tiles and a KV head; it walks the boxes (of a page, at most 128 slots) that its rows may see, its first slots' and then its window's,
// 128 slots a step.  Boxes that no row sees are not read but filled with zeros.
//   S_g = Q_g.K^T     M 128 x N 128 x K 128, both operands by TMA with the 128-byte swizzle, pages through the page table;
//   softmax           a thread per query row (= TMEM lane), online, against a lazy reference maximum; P goes back over S as 16-bit pairs.
//                     Prompts: one part, rounded (8 bits of bf16, 11 of fp16), as in ri_prefill_attn.cu: a second one makes half of a step's
//                     products twice as many.  Against 64 bits the outputs are 2.2e-3 off where the rounding of the result alone gives 1.65e-3
//                     (fp16 2.6e-4 and 2.0e-4).  What requests have in common: two parts, as ri_paged_decode.cu has for requests that are
//                     attended one by one, so that what a request gets does not hang on which of the two the call takes (64 requests over
//                     32768 slots, the call: 124 us with one part, 138 with two);
//   O_g += P_g.V      A from TMEM, B the V tile as it lies (MN-major), the accumulator in TMEM for the whole walk.
// Items of two tiles: a group of four softmax warps for each, which share every tile of K and V.  Items of one tile: the groups take
// its even and its odd steps, and join what they have at the end.
// Work: the steps of all items, head by head, are cut into one contiguous range per CTA, of equal length; every CTA works out where its own
// begins.  An item that falls to several CTAs leaves partial results behind, which a second kernel joins in the order of the sequence.
// TMEM: S_0 | S_1 | O_0 | O_1.  Warps: TMA producer, MMA issuer, the one that hands out segments (the part of an item that falls to the
// CTA), one that clears what lies behind a request's last slot, eight softmax warps.  Every wait is bounded; one that runs out is recorded in the status word.
// A tile's slots that a row does not see have a probability of 0, and what they hold is finite where it was written as such; where it
// was not, 0 * infinity leaves a NaN, and the segment is done once more (kAgain).  Slots behind a request's last one may
// hold anything: they are zeros in shared memory before the product.
// B200, bf16, 8 heads of 4, one prompt, a call among others: 8192 tokens 512 to 532 us over all slots (the dense prompt kernel: 464), 297 to
// 305 over a window of 2048, 70 over one of 128; 32768 tokens over 2048 1.20 ms, 1.43 under the power cap (2.1 PFLOP over what is seen,
// 650 us at the cuBLAS rate).  What bounds it: a
// step of two tiles keeps the tensor pipe's queue full for 3200 clocks (16 products of M 128 N 128 K 16 a tile, at 100 clocks each where
// shared memory's bandwidth would allow 64; the pipe counts as active for half of them); an item costs 7000 more, for the first scores, the
// outputs and masked columns; a launch 12 us until its first probabilities, most of it code that runs for the first time.  Measured and
// not kept: four tiles of K and V in the ring instead of five (no difference), outputs through shared memory in whole lines (61 -> 75 us
// at window 128), leaving out exponentials of columns that no row of a warp sees (505 -> 525, by its code), scores read twice, 32 columns
// at a time, for a quarter of the code (505 -> 533), descriptions of the copies fetched ahead (31.5 -> 32.3 for four short pieces).
#include <cuda.h>

#include <type_traits>

#include "ri_paged_shared.cuh"
#include "ri_tc.cuh"

namespace {

using namespace ri_tc;
using namespace ri_page;
using ri_shared::clamped;

constexpr int kTile = 128;                 // query rows of a tile, slots of a step
constexpr int kHalf = kTile * 128;         // bytes of a 128-row x 64-channel half-tile
constexpr int kRing = 5;                   // tiles of K and V in shared memory: K0, V0, K1, V1, ...
constexpr int kThreads = 384;
constexpr int kSegments = 4;               // segments on their way from the warp that hands them out
constexpr int kTails = 4;                 // V tiles in the ring that a request's slots end in: it holds three V tiles
constexpr uint32_t kTmemCols = 512;
constexpr int kLowPart = kTile / 2;        // SHARED: columns of S_g that the probabilities' second parts begin at
constexpr int kMaxCtas = 160;
constexpr int kMaxRequests = 16384;        // of a call, or groups
constexpr int kMaxEntries = 8192;          // of the table of steps
// An item's end this many steps from the end of a CTA's range becomes the end of the range: a part of an item costs as much again
// for its partial result and the second kernel.  Items of at most twice as many are never cut.  With 2, 4 and 6: four pieces of prompts
// behind 6000 slots 38, 32 and 30 us, a prompt of 2048 tokens over all slots 62, 65 and 71.
constexpr int kSnap = 4;
// What an item costs beside its steps (7000 clocks; a step 3400).  8192 tokens over all slots, whose items have 1 to 64 steps: 541 us shared
// out by steps, 505 by cost.
constexpr int kItemCost = 2;
// Of a CTA, over what groups have in common: more parts of an item than that are slower to join than they are to make (one KV head of 8,
// 32768 slots: 148 parts 52 us, 65 parts 35; 2 x 6016 slots of 4 heads 51 and 48).
constexpr int kLeastCost = 4;
// Where a row's outputs come out NaN while its sum is a number, a slot that it does not see, or gives a probability that vanishes, holds a
// NaN or an infinity.  The segments that this happened to are done once more, behind the CTA's last one, over tiles of V in which all that
// is not finite has been made 0; the softmax warps look up what it was, where a row's score says that the slot counts.  So what lies in
// the cache makes no call more than some ten times as long, and no wait of the pipeline long.  8192 tokens of 8 heads of 4 over all slots:
// 0.54 ms; with a NaN in the value of slot 4000 1.6, of slot 8100 1.1, in all values 1.8, an infinity in one channel of every slot 5.6.
// Window 1024 with four first slots, infinities behind those in their page: 0.19 and 0.50.
constexpr int kAgain = 1024;               // bits; segment i has the i-th modulo that: a second time is right for any
constexpr int kHeadsMost = 8;              // query heads of a KV head
constexpr int kMeta = 8;                   // ints that a CTA leaves for the kernel that joins

// An item's steps go over places: the boxes that hold its first slots, then those from its window's first one on.
__device__ __forceinline__ int slot_of(int place, int front, int skip) { return place < front ? place : place + skip; }
struct Segment {
  int step, n;                             // the first of the item's steps here, and how many; 0: no more segments
  int two;                                 // two tiles of rows
  int front, skip;                         // places in front of the gap; slots left out
  int table_row, head;
  int q_row, n_tok;                        // the item's first token (or request), and how many
  int low, high, sink;                     // slots that some row of the item sees: [low, high) and [0, sink)
  int end;                                 // the place behind the request's last slot
  int slot0;                               // ri_paged_prompt: the first token's slot
  int part;                                // rows of partial results in front of this segment's, -1: the item is whole
  int clean;                               // 0, or 1 + what of K and V was loaded before, in tiles modulo 2 kRing: see kAgain
  __device__ __forceinline__ int steps(int g) const { return two ? n : (n + 1 - g) >> 1; }      // of group g, and its j-th one
  __device__ __forceinline__ int nth(int g, int j) const { return step + (two ? j : 2 * j + g); }
};

// Shared memory.  It has no room to spare, so the barriers and the rest stand behind the ring, in what 227 KB leave.
struct Control {
  uint64_t bars[14 + kTails + 2 * kRing + 2 * kSegments];
  Segment segments[kSegments];
  float2 stat[2][kTile];                   // items of one tile: a row's (maximum, sum) in either group
  int scan[kThreads / 32 + 1];
  int begin[4], end[4];                    // where the CTA's range begins and ends: head, sequence, pair of tiles, step
  int first;                               // the first sequence with rows
  int descends;                            // some sequence's rows begin in front of those of the one before it
  uint32_t again[kAgain / 32];             // segments that are done once more
  int any_again;
  uint32_t odd[kRing][kTile / 32];         // done once more: rows of the tile of V that held something else than numbers
  uint32_t tmem;
  int abort;
};
constexpr int kTiles = (4 + 2 * kRing) * kHalf;
constexpr int kSmem = kTiles + (int)ri_align16(sizeof(Control));
static_assert(kSmem <= 227 * 1024, "shared memory");
static_assert((kMaxRequests + 1 + kMaxEntries + 1) * 4 <= 2 * kRing * kHalf, "the tables of the plan lie in the ring");

struct Args : Pages {
  const int32_t* starts;     // rows of the requests [batch + 1]; SHARED: requests of the groups [groups + 1]
  const int32_t* shared;     // SHARED: [groups] slots in common
  const uint16_t* q;
  const void* keys;
  const void* values;
  int64_t q_stride;          // elements
  uint16_t* out;
  float* lse;                // or null
  float* part_o;             // rows of 128, a segment's in the order [channels / 8][rows][8]
  float2* part_ml;           // (reference in the log2 domain, sum)
  int* meta;                 // prompt: [CTAs][kMeta]; SHARED: CTAs (first, last) of the items
  int n_seq, n_rows;         // sequences: requests, or groups; rows of q
  int gs, tile_tokens, max_ctas, part_rows;      // tokens of a tile; rows of a CTA's part of the partial results
  int window, sink;          // window 0: none
  float scale2;
  uint32_t idesc_qk, idesc_pv;
};

// ---- what there is to do: sequences of rows over a request's slots, cut into pairs of tiles ----------------------------
struct Seq {
  int n, q_row, table_row;               // tokens (or requests), the first one's row of q, whose page table
  int rows;                              // slots that count
};
struct Item {
  int n_tok, front, skip, low, high, sink, steps;
  __device__ __forceinline__ int cost() const { return steps + kItemCost; }
};
template <bool SHARED>
__device__ __forceinline__ Seq seq_of(const Args& a, int v) {
  Seq s = {0, 0, v, 0};
  if (!SHARED) {
    s.q_row = clamped(a.starts[v], a.n_rows);
    s.n = max(0, clamped(a.starts[v + 1], a.n_rows) - s.q_row);
    s.rows = rows_of(a, v);
  } else {
    s.q_row = clamped(a.starts[v], a.batch);
    s.table_row = min(s.q_row, a.batch - 1);
    s.rows = ri_shared::in_common(a, a.starts, a.shared, v);
    s.n = s.rows > 0 ? max(0, clamped(a.starts[v + 1], a.batch) - s.q_row) : 0;
  }
  return s;
}
__device__ __forceinline__ int pairs_of(const Args& a, const Seq& s) { return (s.n + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens); }
template <bool SHARED>
__device__ __forceinline__ Item item_of(const Args& a, const Seq& s, int p) {
  Item it;
  const int first = p * 2 * a.tile_tokens;
  it.n_tok = min(s.n - first, 2 * a.tile_tokens);
  it.low = 0;
  it.high = s.rows;
  it.sink = 0;
  if (!SHARED) {
    const int slot = s.rows - s.n + first;                // of the first token
    it.high = clamped(slot + it.n_tok, s.rows);
    if (a.window > 0) it.low = clamped(slot - a.window + 1, it.high);
    it.sink = min(a.sink, it.low);
  }
  const int box = min(1 << a.shift, kTile);
  it.front = (it.sink + box - 1) & -box;
  it.skip = max(0, (it.low & -box) - it.front);
  it.steps = max(1, (it.high - it.skip + kTile - 1) / kTile);      // rows that see nothing still have outputs
  return it;
}

// ---- the CTA's range ----------------------------------------------------------------------------------------------------
// Exclusive sum of x over the CTA's threads; `total` becomes the sum of all.
__device__ __forceinline__ int block_scan(int x, int* tmp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) tmp[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += tmp[w];
    total += tmp[w];
  }
  __syncthreads();
  return before + incl - x;
}
// The last i < n with table[i] <= x (table[0] <= x).
__device__ __forceinline__ int last_at_most(const int* table, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (table[mid] <= x ? lo : hi) = mid;
  }
  return lo;
}
// Tables of the pairs in front of every sequence and of the steps in front of every 2^k pairs (of one KV head) are made by all
// threads together; then one looks up where the CTA's range begins, another where it ends.
__device__ __forceinline__ void plan(const Args& a, int* table, Control& s) {
  const int tid = threadIdx.x;
  int* pairs = table;
  int* steps = table + a.n_seq + 1;
  int total = 0;
  {
    const int each = (a.n_seq + kThreads - 1) / kThreads, v0 = min(tid * each, a.n_seq), v1 = min(v0 + each, a.n_seq);
    int sum = 0, first = a.n_seq;
    for (int v = v0; v < v1; ++v) {
      if (a.starts[v + 1] < a.starts[v]) s.descends = 1;
      const int n = pairs_of(a, seq_of<false>(a, v));
      pairs[v] = sum;
      if (n > 0) first = min(first, v);
      sum += n;
    }
    if (first < a.n_seq) atomicMin(&s.first, first);
    const int before = block_scan(sum, s.scan, total);
    for (int v = v0; v < v1; ++v) pairs[v] += before;
    if (tid == 0) pairs[a.n_seq] = total;
  }
  __syncthreads();
  // Rows that several requests claim could be more than there are, and more than what is counted here has bits for: nothing is done.
  if (s.descends != 0 && tid == 0) *a.status = RI_STATUS_ROW_START;
  const int n_pairs = s.descends != 0 ? 0 : total;
  int k = 0;
  while ((n_pairs - 1) >> k >= kMaxEntries) ++k;
  const int entries = n_pairs > 0 ? ((n_pairs - 1) >> k) + 1 : 0;
  {
    const int each = (entries + kThreads - 1) / kThreads, e0 = min(tid * each, entries), e1 = min(e0 + each, entries);
    int sum = 0;
    if (e0 < e1) {
      int at = e0 << k, v = last_at_most(pairs, a.n_seq, at);
      Seq seq = seq_of<false>(a, v);
      for (int e = e0; e < e1; ++e) {
        steps[e] = sum;
        for (const int end = min((e + 1) << k, n_pairs); at < end; ++at) {
          if (at >= pairs[v + 1]) {
            do ++v;
            while (at >= pairs[v + 1]);
            seq = seq_of<false>(a, v);
          }
          sum += item_of<false>(a, seq, at - pairs[v]).cost();
        }
      }
    }
    const int before = block_scan(sum, s.scan, total);
    for (int e = e0; e < e1; ++e) steps[e] += before;
  }
  __syncthreads();
  if (tid < 2) {
    const int64_t all = (int64_t)total * a.hk;
    const int n_ctas = (int)min((int64_t)a.max_ctas, all), c = (int)blockIdx.x + tid;
    int* place = tid == 0 ? s.begin : s.end;
    const int64_t x = c < n_ctas ? all * c / n_ctas : all;
    int head = a.hk, v = 0, p = 0, step = 0;
    if (x < all) {
      head = (int)(x / total);
      const int y = (int)(x - (int64_t)head * total), e = last_at_most(steps, entries, y);
      int at = e << k, before = steps[e];
      v = last_at_most(pairs, a.n_seq, at);
      Seq seq = seq_of<false>(a, v);
      for (;;) {
        p = at - pairs[v];
        const Item it = item_of<false>(a, seq, p);
        const int n = it.steps;
        if (y - before < it.cost()) {
          step = max(0, y - before - kItemCost);
          if (step > 0) {
            if (step <= kSnap || a.meta == nullptr) {      // no room for partial results: no item is long enough to be cut
              step = 0;
              break;
            }
            if (n - step > kSnap) break;
            step = 0;                      // the next item, which may be the next head's first
            if (++at == n_pairs) {
              ++head;
              v = p = 0;
              if (head < a.hk) v = last_at_most(pairs, a.n_seq, 0);
              break;
            }
            while (at >= pairs[v + 1]) ++v;
            p = at - pairs[v];
          }
          break;
        }
        before += it.cost();
        ++at;
        if (at >= pairs[v + 1]) {
          do ++v;
          while (at >= pairs[v + 1]);
          seq = seq_of<false>(a, v);
        }
      }
    }
    place[0] = head;
    place[1] = head < a.hk ? v : 0;
    place[2] = head < a.hk ? p : 0;
    place[3] = head < a.hk ? step : 0;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // TMA writes over the tables
  __syncthreads();
}

// 32 bytes, a whole sector of L2, in one instruction where the tensor lies so that it can be.
__device__ __forceinline__ void store32(void* p, const uint32_t (&u)[8], bool wide) {
  if (!wide) {
    static_cast<uint4*>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
    static_cast<uint4*>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
    return;
  }
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]),
               "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
// Products and their completion by the one lane for which `one` is set, for whole warps.
__device__ __forceinline__ void mma_by(uint32_t one, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts_by(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t one, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one)
      : "memory");
}
// Whether a request's slots end inside a box of this tile: what the box brings in behind them may be anything.
__device__ __forceinline__ bool ends_in_box(int end, int tile, int shift) {
  const int r = end - tile * kTile;
  return r > 0 && r < kTile && (r & (min(1 << shift, kTile) - 1)) != 0;
}

__device__ __forceinline__ float ex2(float x) {       // 2^x; results below 2^-126 become 0
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
// A tile is read four times over: 32 columns a mask, bit i of which says whether column i is seen.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

// What a thread's row sees: places [low, high) and [0, sink).
struct Sight {
  int low, high, sink;
  __device__ __forceinline__ bool all_of(int place) const { return place >= low && place + kTile <= high; }
  __device__ __forceinline__ uint32_t mask(int place) const {      // of 32 places
    return bits_below(high - place) & (~bits_below(low - place) | bits_below(sink - place));
  }
};

// ---- segments that are done once more ------------------------------------------------------------------------------------
template <int DT>
struct Exponent {
  static constexpr uint32_t kAll = DT == RI_BF16 ? 0x7f80u : 0x7c00u;      // of a NaN or an infinity
};
// Eight values; what is not finite becomes 0.  Whether there was any.
template <int DT>
__device__ __forceinline__ bool make_finite(uint4& x) {
  constexpr uint32_t kBoth = Exponent<DT>::kAll * 0x10001u;
  auto odd = [](uint32_t& u) {
    const uint32_t m = __vcmpeq2(u & kBoth, kBoth);
    u &= ~m;
    return m;
  };
  return (odd(x.x) | odd(x.y) | odd(x.z) | odd(x.w)) != 0;
}
// Which channels a row gets +infinity (words 0 to 3), -infinity (4 to 7) or, with both, NaN from; channel 4 i + e is bit i of word e.
// Of the step's slots `odd` (a bit for each of 128), those whose score is more than -infinity count, however little; eight of them at a
// time, for their values' way here.  A row all of whose channels are NaN learns nothing more.
template <int DT>
__device__ __noinline__ void note_odd(const Args& a, const Segment& sg, const uint32_t* odd, uint32_t tmem_s, int place, uint32_t* got) {
  constexpr int kTogether = 8;
  const int lane = threadIdx.x & 31;
  const uint16_t* head = static_cast<const uint16_t*>(a.values) + ((int64_t)sg.head << a.shift) * RI_HEAD_DIM + 4 * lane;
  uint32_t sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = got[i];
#pragma unroll 1
  for (int x = 0; x < kTile / 32; ++x) {
    const uint32_t here = odd[x];
    if (!__any_sync(0xffffffffu, here != 0)) continue;
    uint32_t part[32], counts = 0;
    tc_ld32(tmem_s + x * 32, part);
    tc_wait_ld();
    tc_ld_landed(part);
#pragma unroll
    for (int y = 0; y < 32; ++y)
      if (__uint_as_float(part[y]) * a.scale2 != -INFINITY) counts |= 1u << y;
    const uint32_t all = sum[0] & sum[1] & sum[2] & sum[3] & sum[4] & sum[5] & sum[6] & sum[7];
    counts = all == 0xffffffffu ? 0u : counts & here;
    uint32_t left = __reduce_or_sync(0xffffffffu, counts);
    const int slot = slot_of(place + x * 32 + lane, sg.front, sg.skip), row = slot & ((1 << a.shift) - 1);      // of this lane's place
    const int id = left & (1u << lane) ? page_of(a, sg.table_row, slot >> a.shift) : 0;
    while (left != 0) {
      uint32_t bit[kTogether];
      uint2 u[kTogether];
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        bit[k] = left & (0u - left);
        left ^= bit[k];
        const int of = __ffs(bit[k] != 0 ? bit[k] : bit[0]) - 1;
        u[k] = *reinterpret_cast<const uint2*>(head + __shfl_sync(0xffffffffu, id, of) * a.value_stride + __shfl_sync(0xffffffffu, row, of) * RI_HEAD_DIM);
      }
#pragma unroll
      for (int k = 0; k < kTogether; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t v = ((e < 2 ? u[k].x : u[k].y) >> (16 * (e & 1))) & 0xffffu, size = v & 0x7fffu;
          const bool nan = size > Exponent<DT>::kAll, inf = size == Exponent<DT>::kAll;
          const uint32_t plus = __ballot_sync(0xffffffffu, nan || (inf && v == size)), minus = __ballot_sync(0xffffffffu, nan || (inf && v != size));
          if (counts & bit[k]) {
            sum[e] |= plus;
            sum[4 + e] |= minus;
          }
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) got[i] = sum[i];
}
// Puts them into the row's accumulator, whose products are done.
__device__ __noinline__ void put_odd(uint32_t tmem_o, const uint32_t* got) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) any |= got[i];
  if (!__any_sync(0xffffffffu, any != 0)) return;
#pragma unroll 1
  for (int x = 0; x < 4; ++x) {
    uint32_t o[32];
    tc_ld32(tmem_o + x * 32, o);
    tc_wait_ld();
    tc_ld_landed(o);
#pragma unroll
    for (int y = 0; y < 32; ++y) {
      const uint32_t bit = 1u << (8 * x + y / 4);
      const bool plus = got[y & 3] & bit, minus = got[4 + (y & 3)] & bit;
      if (plus || minus) o[y] = plus && minus ? 0x7fffffffu : (plus ? 0x7f800000u : 0xff800000u);
    }
    tc_st32(tmem_o + x * 32, o);
  }
  tc_wait_st();
}

// ---- softmax of a segment's steps, by the warp that has the rows ---------------------------------------------------------
// l_run and m_ref become a row's sum and the reference that it and the outputs go by; `phase`: of the scores' barrier.  False: it gave up.
// The reference follows the running maximum in steps of more than 2^kLazy, kAbove below it: fp16's short exponent then holds
// probabilities down to 2^-(24 + kAbove) of the largest, which are at most 2^(kAbove + kLazy).
template <int DT, bool SHARED, bool CLEAN>
__device__ __forceinline__ bool softmax_steps(const Args& a, Control& s, const Segment& sg, const Sight& sight, uint32_t tmem_s, uint32_t tmem_o,
                                              int grp, uint32_t phase, float& m_ref, float& l_run, uint32_t* got) {
  constexpr float kLazy = 4.f, kAbove = DT == RI_F16 ? 10.f : 0.f;
  const int lane = threadIdx.x & 31;
  const uint32_t bars = smem_u32(s.bars);
  volatile int* abort_flag = &s.abort;
  const uint64_t scale_2 = pack_f2(a.scale2, a.scale2);
  for (int j = 0; j < sg.steps(grp); ++j) {
    const int place = sg.nth(grp, j) * kTile;
    if (!__all_sync(0xffffffffu, mbar_wait(bars + 8u * (4 + grp), (phase ^ j) & 1, abort_flag, 11))) return false;
    tc_fence_after();
    // Columns that are not seen become -infinity where they lie, 32 at a time: a tile's few tokens begin and end seeing close together,
    // so most of four times 32 columns are seen by all rows of a warp, and a loop is a quarter of the instructions.
    if (__any_sync(0xffffffffu, !sight.all_of(place))) {
#pragma unroll 1
      for (int x = 0; x < 4; ++x) {
        const uint32_t seen = sight.mask(place + x * 32);
        if (!__any_sync(0xffffffffu, seen != 0xffffffffu)) continue;
        uint32_t part[32];
        tc_ld32(tmem_s + x * 32, part);
        tc_wait_ld();
        tc_ld_landed(part);
#pragma unroll
        for (int y = 0; y < 32; ++y)
          if (!(seen & (1u << y))) part[y] = 0xff800000u;      // -inf
        tc_st32(tmem_s + x * 32, part);
      }
      tc_wait_st();
    }
    if constexpr (CLEAN) {                               // what the step's tile of V held is known once it is clean
      const int tile = sg.clean + 2 * (sg.nth(grp, j) - sg.step), at = tile % kRing;
      if (!__all_sync(0xffffffffu, mbar_wait(bars + 8u * (14 + kTails + at), (tile / kRing) & 1, abort_flag, 11))) return false;
      note_odd<DT>(a, sg, s.odd[at], tmem_s, place, got);
    }
    uint32_t sr[4][32];
#pragma unroll
    for (int x = 0; x < 4; ++x) tc_ld32(tmem_s + x * 32, sr[x]);
    tc_wait_ld();
#pragma unroll
    for (int x = 0; x < 4; ++x) tc_ld_landed(sr[x]);

    float mx[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      mx[x] = fmaxf(__uint_as_float(sr[x][0]), __uint_as_float(sr[x][1]));
#pragma unroll
      for (int y = 2; y < 32; y += 2) mx[x] = max3(mx[x], __uint_as_float(sr[x][y]), __uint_as_float(sr[x][y + 1]));
    }
    const float m_tile = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * a.scale2 - kAbove;
    const bool move = m_tile > m_ref + kLazy;              // also true for the first finite tile (m_ref = -inf)
    if (__any_sync(0xffffffffu, move)) {
      // the warp's accumulator rows are multiplied anyway, so every row of it catches up with its maximum
      const float m_new = fmaxf(m_ref, m_tile);
      const float factor = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m_new);      // 1 when the maximum stays
      l_run *= factor;
      m_ref = m_new;
      if (j > 0) {                                         // rare: bring this warp's rows of O to the new reference
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          uint32_t orow[32];
          tc_ld32(tmem_o + x * 32, orow);
          tc_wait_ld();
          tc_ld_landed(orow);
#pragma unroll
          for (int y = 0; y < 32; ++y) orow[y] = __float_as_uint(__uint_as_float(orow[y]) * factor);
          tc_st32(tmem_o + x * 32, orow);
        }
      }
    }
    // probabilities p = 2^(s * scale - m), packed as the 16-bit operand of the second product: word y of the row = slots 2y, 2y+1
    const float ref = m_ref == -INFINITY ? 0.f : m_ref;
    const uint64_t neg_m = pack_f2(-ref, -ref);
    uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t pw[16], low[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const uint64_t e = fma_f2(pack_f2(__uint_as_float(sr[x][2 * y]), __uint_as_float(sr[x][2 * y + 1])), scale_2, neg_m);
        float e0, e1;
        unpack_f2(e, e0, e1);
        const float p0 = ex2(e0), p1 = ex2(e1);
        sum2[y & 1] = add_f2(sum2[y & 1], pack_f2(p0, p1));
        pw[y] = Elem<DT>::pack2(p0, p1);
        if (SHARED) low[y] = Elem<DT>::pack2(p0 - Elem<DT>::from_bits((uint16_t)(pw[y] & 0xffffu)), p1 - Elem<DT>::from_bits((uint16_t)(pw[y] >> 16)));
      }
      tc_st16(tmem_s + x * 16, pw);
      if (SHARED) tc_st16(tmem_s + kLowPart + x * 16, low);
      if (x == 1) {          // the product over the first 64 slots may start
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + 8u * (6 + grp));
      }
    }
    float s0, s1;
    unpack_f2(add_f2(sum2[0], sum2[1]), s0, s1);
    l_run += s0 + s1;
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + 8u * (8 + grp));
  }
  return true;
}
// The same over clean tiles, and what those held goes into the accumulators.  Called where nothing of the ordinary steps is in registers.
struct Sums {
  float m, l;
  bool ok;
};
template <int DT, bool SHARED>
__device__ __noinline__ Sums clean_steps(const Args& a, Control& s, const Segment& sg, Sight sight, uint32_t tmem_s, uint32_t tmem_o, int grp,
                                         uint32_t phases, float m_ref) {
  Sums sums = {m_ref, 0.f, true};
  uint32_t got[8] = {};
  sums.ok = softmax_steps<DT, SHARED, true>(a, s, sg, sight, tmem_s, tmem_o, grp, phases & 1, sums.m, sums.l, got);
  if (sums.ok && sg.steps(grp) > 0) {
    sums.ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(s.bars) + 8u * (10 + grp), (phases >> (1 + grp)) & 1, &s.abort, 11));
    tc_fence_after();
    if (sums.ok) put_odd(tmem_o, got);
    tc_fence_before();
  }
  return sums;
}

template <int DT, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
paged_attend_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Control& s = *reinterpret_cast<Control*>(smem + kTiles);
  const uint32_t sQ = smem_u32(smem), sKV = sQ + 4 * kHalf, bars = smem_u32(s.bars);
  auto bar_q = [&](int g) { return bars + 8u * g; };
  auto bar_q_empty = [&](int g) { return bars + 8u * (2 + g); };
  auto bar_s_full = [&](int g) { return bars + 8u * (4 + g); };
  auto bar_p_part = [&](int g) { return bars + 8u * (6 + g); };
  auto bar_p_full = [&](int g) { return bars + 8u * (8 + g); };
  auto bar_o_full = [&](int g) { return bars + 8u * (10 + g); };
  auto bar_join = [&](int i) { return bars + 8u * (12 + i); };
  auto bar_tail = [&](int i) { return bars + 8u * (14 + i % kTails); };
  auto bar_full = [&](int i) { return bars + 8u * (14 + kTails + i); };
  auto bar_empty = [&](int i) { return bars + 8u * (14 + kTails + kRing + i); };
  auto bar_seg = [&](int i) { return bars + 8u * (14 + kTails + 2 * kRing + i); };
  auto bar_seg_empty = [&](int i) { return bars + 8u * (14 + kTails + 2 * kRing + kSegments + i); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = (int)blockIdx.x;

  if (threadIdx.x == 0) {
    // the swizzle of the tiles goes by addresses: shared memory that does not begin on a boundary of 1 KB gives up at once
    s.abort = (sQ & 1023u) ? 10 : 0;
    s.first = 0x7fffffff;
    s.descends = 0;
    s.any_again = 0;
    for (int g = 0; g < 2; ++g) {
      mbar_init(bar_q(g), 1); mbar_init(bar_q_empty(g), 1); mbar_init(bar_s_full(g), 1);
      mbar_init(bar_p_part(g), 4); mbar_init(bar_p_full(g), 4); mbar_init(bar_o_full(g), 1); mbar_init(bar_join(g), 8);
    }
    for (int i = 0; i < kRing; ++i) { mbar_init(bar_full(i), 1); mbar_init(bar_empty(i), 1); }
    for (int i = 0; i < kSegments; ++i) { mbar_init(bar_seg(i), 1); mbar_init(bar_seg_empty(i), 11); }
    for (int i = 0; i < kTails; ++i) mbar_init(bar_tail(i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < kAgain / 32) s.again[threadIdx.x] = 0;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  volatile int* abort_flag = &s.abort;
  ri_pdl_wait();
  ri_pdl_trigger();                        // the kernels behind wait for the end of this one where they read what it writes
  const bool aligned = s.abort == 0;       // of the whole CTA
  if (!SHARED && aligned) plan(a, reinterpret_cast<int*>(smem + 4 * kHalf), s);

  // every role goes through the segments one by one, whole warps
  auto take = [&](int i) {
    return __all_sync(0xffffffffu, mbar_wait(bar_seg(i % kSegments), (i / kSegments) & 1, abort_flag, 10)) && s.segments[i % kSegments].n > 0;
  };
  auto release = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_seg_empty(i % kSegments));
  };

  // Behind the last segment, once, all of them: whether there are some to be done once more.  They follow as the first ones did.
  auto all_done = [&](int i) {
    release(i);
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    return __any_sync(0xffffffffu, *static_cast<volatile int*>(&s.any_again) != 0 && *abort_flag == 0);
  };

  if (aligned) {
  int pass = 0;
  // registers at launch: 384 x 168; after the split 128 x 96 + 256 x 200, which is less
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 0) {
      // ---------------- TMA producer: Q_0, K0, Q_1, V0, K1, V1, ... of one segment after the other; a box per lane ----------------
      const int box = min(1 << a.shift, kTile), mask = (1 << a.shift) - 1, place_of_lane = lane * box;
      const uint32_t q_bytes = (uint32_t)(a.tile_tokens * a.gs) * 256;
      int issued = 0, q_issued[2] = {0, 0}, tails = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (!take(i)) {
          if (pass++ == 1 || !all_done(i)) break;
          continue;
        }
        const Segment& sg = s.segments[i % kSegments];
        const int first = sg.step, n = sg.n, two = sg.two, front = sg.front, skip = sg.skip, clean = sg.clean;
        const int head = sg.head, low = sg.low, high = sg.high, sink = sg.sink, end = sg.end;
        const int32_t* table = a.table + (int64_t)sg.table_row * a.table_stride;
        auto load_q = [&](int g) {
          if (!__all_sync(0xffffffffu, mbar_wait(bar_q_empty(g), (q_issued[g] & 1) ^ 1, abort_flag, 12))) return false;
          if (lane == 0) {
            mbar_arrive_expect_tx(bar_q(g), q_bytes);
            for (int kb = 0; kb < 2; ++kb)
              tma_load_4d(sQ + (g * 2 + kb) * kHalf, &map_q, bar_q(g), 0, head * a.gs, kb, sg.q_row + g * a.tile_tokens);
          }
          __syncwarp();
          ++q_issued[g];
          return true;
        };
        // this lane's box of the j-th step; one that no row sees is looked up nowhere, and comes from behind the pool, as zeros
        auto slot_at = [&](int j) { return slot_of((first + j) * kTile + place_of_lane, front, skip); };
        auto seen = [&](int slot) { return place_of_lane < kTile && slot < high && (slot + box > low || slot < sink); };
        auto page_at = [&](int j) { return seen(slot_at(j)) ? table[slot_at(j) >> a.shift] : -1; };
        int next = page_at(0);
        ok = load_q(0);
        for (int j = 0; ok && j < n; ++j) {
          const int id = seen(slot_at(j)) ? page_or_first(a, next) : a.n_pages;
          const int y = (head << a.shift) + (slot_at(j) & mask);
          if (j + 1 < n) next = page_at(j + 1);
          for (int t = 0; ok && t < 2; ++t) {
            const int at = issued % kRing;
            ok = __all_sync(0xffffffffu, mbar_wait(bar_empty(at), ((issued / kRing) & 1) ^ 1, abort_flag, 13));
            if (!ok) break;
            // a V tile that the request's slots end in is full when what lies behind them has been cleared; a clean one like it
            const uint32_t bar = t == 1 && (clean != 0 || ends_in_box(end, first + j, a.shift)) ? bar_tail(tails++) : bar_full(at);
            if (lane == 0) mbar_arrive_expect_tx(bar, 2 * kHalf);
            __syncwarp();
            if (place_of_lane < kTile)
              for (int kb = 0; kb < 2; ++kb)
                tma_load_4d(sKV + (at * 2 + kb) * kHalf + place_of_lane * 128, t ? &map_v : &map_k, bar, 0, y, kb, id);
            ++issued;
            if (j == 0 && t == 0 && two) ok = load_q(1);
          }
        }
        release(i);
      }
      if (pass == 0) all_done(0);
      if (*abort_flag) {     // give the copies still in flight a bounded chance to land before the CTA exits
        for (int g = 0; g < 2; ++g)
          if (q_issued[g] > 0) mbar_wait(bar_q(g), (q_issued[g] - 1) & 1, abort_flag, 14);
        for (int t = max(0, tails - kTails); t < tails; ++t) mbar_wait(bar_tail(t), (t / kTails) & 1, abort_flag, 14);
        for (int t = max(0, issued - kRing); t < issued; ++t) mbar_wait(bar_full(t % kRing), (t / kRing) & 1, abort_flag, 14);
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      // Per step: P_0.V, then S_0 of the group's next tile, then the same for group 1; behind the last step of a segment come the
      // first scores of the next one.  S_g of the next tile overwrites the columns P_g was read from: both are products of this
      // thread, which the tensor pipe takes in order.
      // The whole warp goes along without a branch that its lanes could take differently, and one lane's predicate stands before each
      // product: their operands' places are then in uniform registers, where the instruction takes them from.  The groups are loops,
      // not copies of the code: all roles together have to fit the instruction cache (8192 tokens, window 128: 67 -> 63 us).
      const uint32_t one = lane == 0;
      const uint32_t tmem_u = __reduce_max_sync(0xffffffffu, tmem);
      auto wait = [&](uint32_t bar, uint32_t parity, int where) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        const unsigned long long t0 = global_ns();
        for (uint32_t spin = 0;; ++spin) {
          if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
          if ((spin & 255u) == 255u) {
            if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
            if (__any_sync(0xffffffffu, global_ns() - t0 > kWaitLimitNs)) { *abort_flag = where; return false; }
          }
          if (spin > (1u << 28)) { *abort_flag = where + 100; return false; }      // second bound, independent of the timer
        }
      };
      int at = 0, phase = 0;               // the segment's next tile in the ring; the ring's turn
      uint32_t q_used = 0, p_used = 0;     // parities, a bit for each group
      // place and parity of the tile that lies `ahead` of the next one
      auto slot = [&](int ahead) { const int x = at + ahead; return x >= kRing ? x - kRing : x; };
      auto turn = [&](int ahead) { return (uint32_t)(at + ahead >= kRing ? phase ^ 1 : phase); };
      auto wait_tile = [&](int ahead) { return wait(bar_full(slot(ahead)), turn(ahead), 15); };
      auto issue_pv = [&](int g, int tile, int k0, bool first) {
        const uint64_t db = umma_desc_mn_sw128(sKV + tile * 2 * kHalf, kHalf);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mma_ts_by(one, tmem_u + (2 + g) * kTile, tmem_u + g * kTile + 8 * (k0 + k), db + 128 * (k0 + k), a.idesc_pv, !first || (k0 + k) != 0);
          if (SHARED)
            mma_ts_by(one, tmem_u + (2 + g) * kTile, tmem_u + g * kTile + kLowPart + 8 * (k0 + k), db + 128 * (k0 + k), a.idesc_pv, 1u);
        }
      };
      auto issue_qk = [&](int g, int q, int tile) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint64_t da = umma_desc_sw128(sQ + (q * 2 + kb) * kHalf), db = umma_desc_sw128(sKV + (tile * 2 + kb) * kHalf);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_by(one, tmem_u + g * kTile, da + 2 * k, db + 2 * k, a.idesc_qk, (kb | k) != 0);
        }
        commit_by(one, bar_s_full(g));       // also says that P_g.V of the tile before has completed
      };
      auto advance = [&] {                   // by a step: K and V
        at += 2;
        if (at >= kRing) { at -= kRing; phase ^= 1; }
      };
      // P_g.V of a step whose V tile is there: its first half as soon as there are probabilities for it
      auto product = [&](int g, int tile, bool first) {
        if (!wait(bar_p_part(g), (p_used >> g) & 1, 17)) return false;
        tc_fence_after();
        issue_pv(g, tile, 0, first);
        if (!wait(bar_p_full(g), (p_used >> g) & 1, 18)) return false;
        tc_fence_after();
        issue_pv(g, tile, 4, false);
        p_used ^= 1u << g;
        return true;
      };
      auto query = [&](int g) {
        const bool there = wait(bar_q(g), (q_used >> g) & 1, 16);
        q_used ^= 1u << g;
        return there;
      };
      // two tiles: both groups use every tile of K and V
      auto two_tiles = [&](int n) {
        if (!wait_tile(0)) return false;
#pragma unroll 1
        for (int g = 0; g < 2; ++g) {
          if (!query(g)) return false;
          tc_fence_after();
          issue_qk(g, g, slot(0));
          if (n == 1) commit_by(one, bar_q_empty(g));
        }
        commit_by(one, bar_empty(slot(0)));
        for (int j = 0; j < n; ++j) {
#pragma unroll 1
          for (int g = 0; g < 2; ++g) {
            if ((g == 0 && !wait_tile(1)) || !product(g, slot(1), j == 0)) return false;
            if (j + 1 < n) {
              if (g == 0 && !wait_tile(2)) return false;
              tc_fence_after();
              issue_qk(g, g, slot(2));
              if (j + 2 == n) commit_by(one, bar_q_empty(g));
            } else {
              commit_by(one, bar_o_full(g));
            }
          }
          commit_by(one, bar_empty(slot(1)));
          if (j + 1 < n) commit_by(one, bar_empty(slot(2)));
          advance();
        }
        return true;
      };
      // one tile: group 0 takes the even steps and group 1 the odd ones, so that step i is computed behind the scores of step i + 1
      auto one_tile = [&](int n) {
        if (!wait_tile(0) || !query(0)) return false;
        tc_fence_after();
        issue_qk(0, 0, slot(0));
        if (n == 1) commit_by(one, bar_q_empty(0));
        commit_by(one, bar_empty(slot(0)));
        if (n > 1) {
          if (!wait_tile(2)) return false;
          tc_fence_after();
          issue_qk(1, 0, slot(2));
          if (n == 2) commit_by(one, bar_q_empty(0));
          commit_by(one, bar_empty(slot(2)));
        }
        for (int i = 0; i < n; i += 2) {
#pragma unroll 1
          for (int g = 0; g < 2; ++g) {
            if (i + g >= n) continue;
            if (!wait_tile(1) || !product(g, slot(1), i == 0)) return false;
            commit_by(one, bar_empty(slot(1)));
            advance();
            if (i + g + 2 < n) {             // the group's next step, one behind the other group's
              if (!wait_tile(2)) return false;
              tc_fence_after();
              issue_qk(g, 0, slot(2));
              if (i + g + 3 == n) commit_by(one, bar_q_empty(0));
              commit_by(one, bar_empty(slot(2)));
            } else {
              commit_by(one, bar_o_full(g));
            }
          }
        }
        return true;
      };
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (!wait(bar_seg(i % kSegments), (i / kSegments) & 1, 10)) break;
        const int n = (int)__reduce_max_sync(0xffffffffu, (unsigned)s.segments[i % kSegments].n);
        const bool two = __any_sync(0xffffffffu, s.segments[i % kSegments].two);
        if (n == 0) {
          if (pass++ == 1 || !all_done(i)) break;
          continue;
        }
        release(i);
        ok = two ? two_tiles(n) : one_tile(n);
      }
      if (pass == 0) all_done(0);
    } else if (warp == 3) {
      // ---------------- V tiles that a request's slots end in: zeros behind them, up to the end of their box; clean tiles ----------------
      int tile0 = 0, tails = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (!take(i)) {
          if (pass++ == 1 || !all_done(i)) break;
          continue;
        }
        const int first = s.segments[i % kSegments].step, n = s.segments[i % kSegments].n, end = s.segments[i % kSegments].end;
        const bool clean = s.segments[i % kSegments].clean != 0;
        release(i);
        for (int j = 0; j < n; ++j) {
          if (!clean && !ends_in_box(end, first + j, a.shift)) continue;
          const int at = (tile0 + 2 * j + 1) % kRing, box = min(1 << a.shift, kTile), r0 = end - (first + j) * kTile, r1 = (r0 + box - 1) & -box;
          ok = __all_sync(0xffffffffu, mbar_wait(bar_tail(tails), (tails / kTails) & 1, abort_flag, 15));
          if (!ok) break;
          uint8_t* v = smem + 4 * kHalf + at * 2 * kHalf;
          if (clean) {                       // what lies behind the last slot may stay where it is finite: probabilities of 0
#pragma unroll 1
            for (int w = 0; w < kTile / 32; ++w) {
              uint32_t rows = 0;
#pragma unroll 1
              for (int kb = 0; kb < 2; ++kb) {
                uint4* piece = reinterpret_cast<uint4*>(v + kb * kHalf + w * 32 * 128) + lane;      // eight lanes a row
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                  uint4 x = piece[32 * y];
                  const bool odd = make_finite<DT>(x);
                  if (odd) piece[32 * y] = x;
                  const uint32_t votes = __ballot_sync(0xffffffffu, odd);
#pragma unroll
                  for (int r = 0; r < 4; ++r)
                    if ((votes >> (8 * r)) & 0xffu) rows |= 1u << (4 * y + r);
                }
              }
              if (lane == 0) s.odd[at][w] = rows;
            }
          } else {
            for (int x = r0 * 8 + lane; x < r1 * 8; x += 32)
              for (int kb = 0; kb < 2; ++kb) *reinterpret_cast<uint4*>(v + kb * kHalf + x * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_full(at));
          ++tails;
        }
        tile0 += 2 * n;
      }
      if (pass == 0) all_done(0);
    } else if (warp == 2) {
      // ---------------- segments ----------------
      int given = 0, index = 0, tiles = 0;   // the segment's number; tiles of K and V in front of it, modulo 2 kRing
      Segment sg = {};
      auto give = [&] {                      // by one lane
        if (pass == 1 && sg.n > 0) {
          const int k = index++ % kAgain;
          if (!((s.again[k / 32] >> (k % 32)) & 1u)) return true;
        }
        sg.clean = pass == 0 ? 0 : 1 + tiles;
        tiles = (tiles + 2 * sg.n) % (2 * kRing);
        const int at = given % kSegments;
        if (!mbar_wait(bar_seg_empty(at), ((given / kSegments) & 1) ^ 1, abort_flag, 19)) return false;
        s.segments[at] = sg;
        mbar_arrive(bar_seg(at));
        ++given;
        return true;
      };
      auto again = [&] {                     // as all_done, but this warp has nothing to release
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
        return __any_sync(0xffffffffu, *static_cast<volatile int*>(&s.any_again) != 0 && *abort_flag == 0);
      };
      // steps `step` to `end` - 1 of an item
      auto describe = [&](const Seq& seq, const Item& it, int h, int p, int step, int end) {
        sg.table_row = seq.table_row;
        sg.head = h;
        sg.q_row = seq.q_row + p * 2 * a.tile_tokens;
        sg.n_tok = it.n_tok;
        sg.step = step;
        sg.n = end - step;
        sg.front = it.front;
        sg.skip = it.skip;
        sg.low = it.low;
        sg.high = it.high;
        sg.sink = it.sink;
        sg.end = seq.rows - it.skip;
        sg.slot0 = seq.rows - seq.n + p * 2 * a.tile_tokens;
        sg.two = it.n_tok > a.tile_tokens;
      };
#pragma unroll 1
      do {
        if (SHARED) {
          // All items of a group have the same steps, so the range is found without tables, by the warp: what code runs once costs by
          // the instruction (6016 slots, 24 requests: the kernel 21 us with tables).
          auto cost_of = [&](int g) {
            if (g >= a.n_seq) return 0;
            const Seq seq = seq_of<true>(a, g);
            return pairs_of(a, seq) * ((seq.rows + kTile - 1) / kTile + kItemCost);
          };
          int total = 0;
          for (int g = lane; g < a.n_seq; g += 32) total += cost_of(g);
          total = __reduce_add_sync(0xffffffffu, total);
          const int64_t all = (int64_t)total * a.hk;
          const int n_ctas = (int)min((int64_t)a.max_ctas, (all + kLeastCost - 1) / kLeastCost);
          const int64_t lo = c < n_ctas ? all * c / n_ctas : all, hi = c < n_ctas ? all * (c + 1) / n_ctas : all;
          if (lo < hi && lane == 0) {
            int h = (int)(lo / total), g = 0;
            int64_t at = (int64_t)h * total;   // the item's place in the sequence
            bool ok = true;
            while (ok && at < hi) {
              const Seq seq = seq_of<true>(a, g);
              const int pairs = pairs_of(a, seq), steps = (seq.rows + kTile - 1) / kTile, cost = steps + kItemCost;
              int p = at < lo ? (int)min((int64_t)pairs, (lo - at) / cost) : 0;
              at += (int64_t)p * cost;
              for (; ok && p < pairs && at < hi; ++p, at += cost) {
                const int step = (int)max((int64_t)0, lo - at - kItemCost), end = (int)min((int64_t)steps, max((int64_t)0, hi - at - kItemCost));
                if (step >= end) continue;
                describe(seq, item_of<true>(a, seq, p), h, p, step, end);
                const int item = h * a.batch + sg.q_row;
                sg.part = c * a.part_rows + item * a.gs;
                if (step == 0) a.meta[2 * item] = c;
                if (end == steps) a.meta[2 * item + 1] = c;
                ok = give();
              }
              if (++g == a.n_seq) {
                g = 0;
                ++h;
              }
            }
            sg.n = 0;
            if (ok) give();
          } else if (lane == 0) {
            give();
          }
        } else if (lane == 0) {
          int h = s.begin[0], v = s.begin[1], p = s.begin[2], step = s.begin[3];
          const int h1 = s.end[0], v1 = s.end[1], p1 = s.end[2], step1 = s.end[3], first = s.first;
          int tail = 0, head = 0;              // rows of a segment that others go on with; whether the first one is another CTA's item
          Seq seq = {};
          int pairs = 0, of = -1;
          bool ok = true;
          while (ok && h < a.hk) {
            const bool last = h == h1 && v == v1 && p == p1;
            if (last && step == step1) break;
            if (of != v) {
              seq = seq_of<false>(a, v);
              pairs = pairs_of(a, seq);
              of = v;
            }
            const Item it = item_of<false>(a, seq, p);
            const int end = last ? step1 : it.steps;
            const bool begins = step == 0, ends = end == it.steps;
            describe(seq, it, h, p, step, end);
            sg.part = begins && ends ? -1 : (2 * c + begins) * a.part_rows;
            if (!begins) head = ends ? 1 : 2;  // it ends here, or goes on behind
            if (begins && !ends) {
              tail = sg.n_tok;
              a.meta[c * kMeta + 2] = h;
              a.meta[c * kMeta + 3] = sg.q_row;
            }
            ok = give();
            step = 0;
            if (last) break;
            if (++p == pairs) {
              p = 0;
              do ++v;
              while (v < a.n_seq && !(v == v1 && h == h1) && pairs_of(a, seq_of<false>(a, v)) == 0);
              if (v == a.n_seq) {
                v = first;
                ++h;
              }
            }
          }
          if (a.meta != nullptr) {
            a.meta[c * kMeta] = tail;
            a.meta[c * kMeta + 1] = head;
          }
          sg.n = 0;
          if (ok) give();
        }
        __syncwarp();
      } while (pass++ == 0 && again());
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- softmax and epilogue: thread = query row = TMEM lane; group g owns S_g and O_g ----------------
    const int grp = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;      // a warp may touch only its quarter of the lanes
    const uint32_t t_lane = (uint32_t)(quarter * 32) << 16;
    const uint32_t tmem_s = tmem + grp * kTile + t_lane, tmem_o = tmem + (2 + grp) * kTile + t_lane;
    bool ok = true;
    // parities of what is waited for next: bit 0 scores, 1 and 2 outputs of the two groups, 3 joins.  A row of scores takes 128
    // registers, so little else is kept over the steps: what the segment says is read from shared memory where it is needed.
    uint32_t phases = 0;
    auto meet = [&](int i) {                               // of all eight warps
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_join(i));
      return (bool)__all_sync(0xffffffffu, mbar_wait(bar_join(i), (phases >> 3) & 1, abort_flag, 10));
    };
    for (int i = 0; ok; ++i) {
      if (!take(i)) {
        if (pass++ == 1 || !all_done(i)) break;
        continue;
      }
      const Segment& sg = s.segments[i % kSegments];         // stays until the end of the segment
      // the row in its item, its token; rows that fill up a tile are like the last one, so that they hold nobody up
      auto row_in_item = [&] { return (sg.two ? grp * a.tile_tokens * a.gs : 0) + row; };
      auto token = [&] { return sg.q_row + min(row_in_item(), sg.n_tok * a.gs - 1) / a.gs; };
      auto sight_of_row = [&] {
        const int q_row = token();
        Sight x = {sg.low - sg.skip, 0, 0};
        if (!SHARED) {
          const int slot = sg.slot0 + q_row - sg.q_row;
          x.high = min(max(slot + 1, 0), sg.end + sg.skip) - sg.skip;
          x.low = a.window > 0 ? max(0, slot - a.window + 1) - sg.skip : 0;
          x.sink = a.sink;
        } else {
          x.high = min(sg.high, rows_of(a, q_row)) - sg.skip;
        }
        return x;
      };
      const Sight sight = sight_of_row();
      // Rows that fill up a tile hold what was there before, or are another request's: they take no part in what a warp decides together,
      // so that results repeat to the bit.  No score is above their reference.
      auto is_row = [&] { return row < a.tile_tokens * a.gs && row_in_item() < sg.n_tok * a.gs; };
      float m_ref = is_row() ? -INFINITY : INFINITY, l_run = 0.f;
      if (sg.clean == 0) {
        ok = softmax_steps<DT, SHARED, false>(a, s, sg, sight, tmem_s, tmem_o, grp, phases & 1, m_ref, l_run, nullptr);
      } else {
        const Sums sums = clean_steps<DT, SHARED>(a, s, sg, sight, tmem_s, tmem_o, grp, phases, m_ref);
        m_ref = sums.m;
        l_run = sums.l;
        ok = sums.ok;
      }
      phases ^= sg.steps(grp) & 1;
      // ---- epilogue, one row per thread.  Two tiles: each group its own.  One: the groups exchange (maximum, sum) through shared
      //      memory, then each joins half of the channels of both accumulators; the second barrier keeps an accumulator until the
      //      other group has read it ----
      float m = m_ref, l = l_run, w0 = 1.f, w1 = 0.f;        // of the row; weights of the accumulators read below
      const bool two = sg.two;
      if (!two) {
        s.stat[grp][row] = make_float2(m_ref, l_run);
        ok = ok && meet(0);
        const float2 other = s.stat[grp ^ 1][row];
        m = fmaxf(m_ref, other.x);
        const float f_own = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m), f_other = other.x == -INFINITY ? 0.f : exp2f(other.x - m);
        l = l_run * f_own + other.y * f_other;
        w0 = grp ? f_other : f_own;
        w1 = grp ? f_own : f_other;
      }
      const float f = sg.part < 0 ? (l == 0.f ? 0.f : 1.f / l) : 1.f;      // NaN stays one
      w0 *= f;
      w1 *= f;
      if (sg.clean != 0) {                                   // an infinite value is one however little its group counts
        constexpr float kLeast = 1.17549435e-38f;
        w0 = w0 < kLeast && l != 0.f ? kLeast : w0;
        w1 = w1 < kLeast && l != 0.f ? kLeast : w1;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
        if (sg.steps(g) > 0) {             // the other group's outputs count even where nobody here waits for them
          if (!two || g == grp) ok = ok && __all_sync(0xffffffffu, mbar_wait(bar_o_full(g), (phases >> (1 + g)) & 1, abort_flag, 11));
          phases ^= 2u << g;
        }
      if (ok) {
        tc_fence_after();
        const bool both = !two && sg.steps(1) > 0;
        const int n_rows = sg.n_tok * a.gs, item_row = row_in_item(), q_row = token();
        const bool valid = is_row();
        const int x0 = two ? 0 : grp * 2, x1 = two ? 4 : x0 + 2;
        const int h = sg.head * a.gs + item_row % a.gs;
        const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
        bool bad = false;
#pragma unroll 1
        for (int x = x0; x < x1; ++x) {                        // 32 channels at a time: it runs once an item, so its code is kept short
          uint32_t part[32];
          float o[32];
          tc_ld32(tmem + (2 + (two ? grp : 0)) * kTile + t_lane + x * 32, part);
          tc_wait_ld();
          tc_ld_landed(part);
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __uint_as_float(part[y]) * w0;
          if (both) {
            tc_ld32(tmem + 3 * kTile + t_lane + x * 32, part);
            tc_wait_ld();
            tc_ld_landed(part);
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] += __uint_as_float(part[y]) * w1;
          }
          if (valid) {
#pragma unroll
            for (int y = 0; y < 32; ++y) bad |= o[y] != o[y];
            if (sg.part < 0) {
              uint16_t* dst = a.out + ((int64_t)q_row * a.hk * a.gs + h) * RI_HEAD_DIM + x * 32;
#pragma unroll
              for (int y = 0; y < 32; y += 16) {
                uint32_t u[8];
#pragma unroll
                for (int v = 0; v < 8; ++v) u[v] = Elem<DT>::pack2(o[y + 2 * v], o[y + 2 * v + 1]);
                store32(dst + y, u, wide);
              }
            } else {
              float4* dst = reinterpret_cast<float4*>(a.part_o + (int64_t)sg.part * RI_HEAD_DIM) + (x * 4 * n_rows + item_row) * 2;
#pragma unroll
              for (int y = 0; y < 32; y += 4) dst[y / 8 * 2 * n_rows + (y / 4 & 1)] = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            }
          }
        }
        if (valid && (two || grp == 0)) {
          if (sg.part >= 0) a.part_ml[sg.part + item_row] = make_float2(m, l);
          else if (a.lse != nullptr) a.lse[(int64_t)q_row * a.hk * a.gs + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
        }
        if (__any_sync(0xffffffffu, valid && bad && l == l) && pass == 0 && lane == 0) {
          atomicOr(&s.again[i % kAgain / 32], 1u << (i % 32));
          s.any_again = 1;
        }
      }
      if (!two) {
        ok = ok && meet(1);
        phases ^= 8;
      }
      release(i);
    }
    if (pass == 0) all_done(0);
  }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && s.abort) *a.status = s.abort;
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// ---- the parts of an item that fell to several CTAs, joined in their order ---------------------------------------------------
// Factor of a part against the largest reference; one that is far below it still counts enough to hand on an infinite value.
__device__ __forceinline__ float part_factor(float m, float most) {
  return m == -INFINITY ? 0.f : fmaxf(exp2f(m - most), 1.17549435e-38f);
}
struct Joined {
  float m = -INFINITY, l = 0.f;
  __device__ __forceinline__ void add(float2 ml) {
    const float most = fmaxf(m, ml.x), ref = most == -INFINITY ? 0.f : most;
    l = l * exp2f(m - ref) + ml.y * exp2f(ml.x - ref);
    m = most;
  }
  __device__ __forceinline__ float lse() const { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f; }
  __device__ __forceinline__ float scale() const { return l == 0.f ? 0.f : 1.f / l; }
};

// ri_paged_prompt: a block per CTA whose range ends inside an item that begins in it, and 32 rows of that item; a lane per row, four
// times four channels a warp.
constexpr int kJoinRows = 32, kJoinThreads = 256;
template <int DT>
__global__ void __launch_bounds__(kJoinThreads) prompt_join_kernel(const __grid_constant__ Args a) {
  ri_pdl_enter();
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y * kJoinRows + lane;
  const int* meta = a.meta + c * kMeta;
  const int h = clamped(meta[2], a.hk - 1), q_row = clamped(meta[3], a.n_rows - 1), n_tok = min(meta[0], min(2 * a.tile_tokens, a.n_rows - q_row));
  const int n_rows = n_tok * a.gs;
  if (n_tok <= 0 || row >= n_rows) return;
  int last = c;                                            // the CTA that has the item's end
  while (last + 1 < a.max_ctas && meta[(last + 1 - c) * kMeta + 1] == 2) ++last;
  if (last + 1 < a.max_ctas && meta[(last + 1 - c) * kMeta + 1] == 1) ++last;
  auto part_at = [&](int i) { return (int64_t)(2 * i + (i == c)) * a.part_rows; };
  Joined all;
  for (int i = c; i <= last; ++i) all.add(a.part_ml[part_at(i) + row]);
  float4 o[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = c; i <= last; ++i) {
    const float f = part_factor(a.part_ml[part_at(i) + row].x, all.m);
    const float4* src = reinterpret_cast<const float4*>(a.part_o + part_at(i) * RI_HEAD_DIM) + (warp * 2 * n_rows + row) * 2;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float4 y = src[(x >> 1) * 2 * n_rows + (x & 1)];
      o[x].x += f * y.x; o[x].y += f * y.y; o[x].z += f * y.z; o[x].w += f * y.w;
    }
  }
  const float f = all.scale();
  const int64_t at = ((int64_t)q_row + row / a.gs) * a.hk * a.gs + h * a.gs + row % a.gs;
  uint4* dst = reinterpret_cast<uint4*>(a.out + at * RI_HEAD_DIM) + warp * 2;
#pragma unroll
  for (int x = 0; x < 2; ++x)
    dst[x] = make_uint4(Elem<DT>::pack2(o[2 * x].x * f, o[2 * x].y * f), Elem<DT>::pack2(o[2 * x].z * f, o[2 * x].w * f),
                        Elem<DT>::pack2(o[2 * x + 1].x * f, o[2 * x + 1].y * f), Elem<DT>::pack2(o[2 * x + 1].z * f, o[2 * x + 1].w * f));
  if (warp == 0 && a.lse != nullptr) a.lse[at] = all.lse();
}

// ---- host ----------------------------------------------------------------------------------------------------------------
// Queries as (channel of a half, head, half, row): a box is one half of the query heads of a KV head, of a tile's tokens.
int make_query_map(CUtensorMap* map, const void* q, int64_t q_stride, int q_heads, int rows, int gs, int tokens, int dtype) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != RI_OK) return rc;
  const cuuint64_t dims[4] = {RI_HEAD_DIM / 2, (cuuint64_t)q_heads, 2, (cuuint64_t)rows};
  const cuuint64_t strides[3] = {256, 128, (cuuint64_t)q_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)gs, 1, (cuuint32_t)tokens}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, dtype == RI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(q),
                         dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RI_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return RI_OK;
}
// Keys or values as (channel of a half, row of the page's heads, half, page): a box is one half of the channels of at most a page.
int make_pool_map(CUtensorMap* map, const void* base, const ri_paged& p, int64_t page_stride) {
  EncodeTiledFn enc;
  const int rc = get_encode_fn(&enc);
  if (rc != RI_OK) return rc;
  const cuuint64_t dims[4] = {RI_HEAD_DIM / 2, (cuuint64_t)p.kv_heads * p.page_size, 2, (cuuint64_t)p.n_pages};
  const cuuint64_t strides[3] = {256, 128, (cuuint64_t)page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)(p.page_size < kTile ? p.page_size : kTile), 1, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, p.dtype == RI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RI_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return RI_OK;
}

int64_t most_items_rows(const ri_paged& p, int rows) {      // rows of an item, at most
  const int pair = 2 * (kTile / p.group_size);
  return (int64_t)(rows < pair ? rows : pair) * p.group_size;
}
// Steps of an item, at most.
int64_t most_steps(const ri_paged& p, int rows, int window, int sink) {
  const int64_t all = (slots_of(p) + kTile - 1) / kTile;
  if (window == 0) return all;
  const int64_t pair = 2 * (kTile / p.group_size), box = p.page_size < kTile ? p.page_size : kTile;
  const int64_t seen = ((int64_t)window + sink + (rows < pair ? rows : pair) + 2 * box + kTile - 1) / kTile;      // first slots and window in boxes begun
  return seen < all ? seen : all;
}
// Whether an item may be cut.
bool may_cut(const ri_paged& p, int rows, int window, int sink) { return most_steps(p, rows, window, sink) > 2 * kSnap; }

int check_call(const char* what, const ri_paged* p, int64_t sequences) {
  const int rc = check(p, what);
  if (rc != RI_OK) return rc;
  RI_REQUIRE(p->group_size >= 1 && p->group_size <= kHeadsMost, "%s: group_size=%d unsupported (1 to %d)", what, p->group_size, kHeadsMost);
  RI_REQUIRE(sequences >= 1 && sequences <= kMaxRequests, "%s: %lld requests or groups unsupported (%d at most)", what, (long long)sequences,
             kMaxRequests);
  return RI_OK;
}

template <int DT, bool SHARED>
int launch(const Args& a, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, bool join, cudaStream_t s) {
  const int rc = ri_allow_smem<paged_attend_kernel<DT, SHARED>>(kSmem);
  if (rc != RI_OK) return rc;
  RI_CUDA_OK(ri_launch_pdl_id(11, paged_attend_kernel<DT, SHARED>, dim3(a.max_ctas), dim3(kThreads), (size_t)kSmem, s, map_q, map_k, map_v, a));
  if (join) {
    RI_CUDA_OK(ri_launch_pdl_id(11, prompt_join_kernel<DT>, dim3(a.max_ctas, (a.part_rows + kJoinRows - 1) / kJoinRows), dim3(kJoinThreads), 0, s, a));
  }
  return RI_OK;
}

template <bool SHARED>
int attend(const char* what, const ri_paged* p, const void* d_q, int64_t q_stride, int rows, Args a, void* d_out, float* d_lse, float scale,
           bool join, cudaStream_t s) {
  int rc;
  RI_REQUIRE(p->d_values && d_q && (SHARED || d_out) && a.starts, "%s: null pointer", what);
  const int64_t pairs = (int64_t)rows / (2 * (kTile / p->group_size)) + a.n_seq;
  RI_REQUIRE(pairs * (most_steps(*p, rows, a.window, a.sink) + kItemCost) < (1ll << 31), "%s: too large", what);      // they are counted in 32 bits
  RI_REQUIRE(q_stride >= (int64_t)p->kv_heads * p->group_size * RI_HEAD_DIM && q_stride % 8 == 0, "%s: queries overlap or lie at odd places", what);
  RI_REQUIRE(((uintptr_t)d_q | (uintptr_t)d_out) % 16 == 0, "%s: tensors must be 16-byte aligned", what);
  RI_REQUIRE(scale > 0.f && scale < 1e30f, "%s: scale must be positive and finite", what);
  static_cast<Pages&>(a) = view(*p);
  a.q = static_cast<const uint16_t*>(d_q);
  a.q_stride = q_stride;
  a.out = static_cast<uint16_t*>(d_out);
  a.lse = d_lse;
  a.n_rows = rows;
  a.gs = p->group_size;
  a.tile_tokens = kTile / a.gs;
  a.part_rows = (int)most_items_rows(*p, rows);
  a.scale2 = RI_LOG2E * scale;
  a.keys = p->d_keys;
  a.values = p->d_values;
  a.idesc_qk = idesc_f16(p->dtype, kTile, kTile);
  a.idesc_pv = a.idesc_qk | (1u << 16);      // B = V is MN-major (channels contiguous)
  int sms = 0;
  if ((rc = ri_sm_count(&sms)) != RI_OK) return rc;
  a.max_ctas = sms < kMaxCtas ? sms : kMaxCtas;
  CUtensorMap map_q, map_k, map_v;
  if ((rc = make_query_map(&map_q, d_q, q_stride, p->kv_heads * a.gs, rows, a.gs, a.tile_tokens, p->dtype)) != RI_OK) return rc;
  if ((rc = make_pool_map(&map_k, p->d_keys, *p, p->key_page_stride)) != RI_OK) return rc;
  if ((rc = make_pool_map(&map_v, p->d_values, *p, p->value_page_stride)) != RI_OK) return rc;
  return p->dtype == RI_BF16 ? launch<RI_BF16, SHARED>(a, map_q, map_k, map_v, join, s) : launch<RI_F16, SHARED>(a, map_q, map_k, map_v, join, s);
}

// Workspaces: meta, sums, outputs of the parts.
int64_t prompt_part_rows(const ri_paged& p, int rows) { return 2 * kMaxCtas * most_items_rows(p, rows); }
constexpr int64_t kPromptMeta = (int64_t)kMaxCtas * kMeta * 4;
int64_t shared_meta(const ri_paged& p) { return ri_align_up(8 * (int64_t)p.batch * p.kv_heads, 16); }
int64_t shared_rows(const ri_paged& p) { return (int64_t)kMaxCtas * most_items_rows(p, p.batch) + (int64_t)p.batch * p.kv_heads * p.group_size; }
void place(Args& a, void* d_scratch, int64_t meta, int64_t rows) {
  a.meta = static_cast<int*>(d_scratch);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(d_scratch) + meta);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * RI_HEAD_DIM);
}

}  // namespace

extern "C" int64_t ri_paged_prompt_scratch_bytes(const ri_paged* p, int32_t rows, int32_t window, int32_t sink) {
  const int rc = check_call("ri_paged_prompt", p, p ? p->batch : 1);
  if (rc != RI_OK) return rc;
  if (rows < 1 || window < 0 || sink < 0) return ri_fail(RI_ERR_INVALID, "ri_paged_prompt: rows=%d window=%d sink=%d unsupported", rows, window, sink);
  return may_cut(*p, rows, window, sink) ? kPromptMeta + prompt_part_rows(*p, rows) * (RI_HEAD_DIM + 2) * 4 : 0;
}

extern "C" int ri_paged_prompt(const ri_paged* p, const void* d_q, int64_t q_stride, int32_t rows, const int32_t* d_row_start, int32_t window,
                               int32_t sink, void* d_out, float* d_lse, float scale, void* d_scratch, void* stream) {
  const int64_t bytes = ri_paged_prompt_scratch_bytes(p, rows, window, sink);
  if (bytes < 0) return (int)bytes;
  RI_REQUIRE((bytes == 0 || d_scratch) && (uintptr_t)d_scratch % 16 == 0, "ri_paged_prompt: the scratch must be there and 16-byte aligned");
  Args a = {};
  a.starts = d_row_start;
  a.n_seq = p->batch;
  a.window = window;
  a.sink = sink;
  if (bytes > 0) place(a, d_scratch, kPromptMeta, prompt_part_rows(*p, rows));
  return attend<false>("ri_paged_prompt", p, d_q, q_stride, rows, a, d_out, d_lse, scale, bytes > 0, static_cast<cudaStream_t>(stream));
}

int64_t ri_shared::scratch_bytes(const ri_paged& p) { return shared_meta(p) + shared_rows(p) * (RI_HEAD_DIM + 2) * 4; }

int ri_shared::launch(const char* what, const ri_paged* p, const void* d_q, int64_t q_stride, const int32_t* d_group_start, int32_t groups,
                      const int32_t* d_shared, float scale, void* d_scratch, Parts* parts, cudaStream_t s) {
  const int rc = check_call(what, p, groups);
  if (rc != RI_OK) return rc;
  Args a = {};
  a.starts = d_group_start;
  a.shared = d_shared;
  a.n_seq = groups;
  place(a, d_scratch, shared_meta(*p), shared_rows(*p));
  int sms = 0;
  const int rc2 = ri_sm_count(&sms);
  if (rc2 != RI_OK) return rc2;
  *parts = {d_group_start, d_shared, a.meta, a.part_o, a.part_ml, groups, 2 * (kTile / p->group_size), (int)most_items_rows(*p, p->batch),
            sms < kMaxCtas ? sms : kMaxCtas};
  return attend<true>(what, p, d_q, q_stride, p->batch, a, nullptr, nullptr, scale, false, s);
}
