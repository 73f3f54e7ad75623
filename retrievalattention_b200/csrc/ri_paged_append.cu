// Rotary positions with several axes on a fused QKV projection, queries out, keys and values into a paged cache.
//   for i < 64, (c, s) the table's row at the row's position on axis axis_of[i], columns i and 64 + i:
//     x'_i = x_i c - x_{i+64} s,    x'_{i+64} = x_{i+64} c + x_i s          (query and key heads; values as they are)
// One axis is the ordinary rotary embedding; text, images and video take (time, height, width).
// (reference: model_hub/llama.py:232-235 the split, :312-320 the rotation; cache_hub/flash_attn_cache.py:133-151 the append)
//
// Bound by the projection, read once and written once.  A row of it lies in one piece and comes in by one bulk copy, three rows
// on their way to each of three CTAs of an SM, which take neighbouring rows.  Two warps issue the copies and fetch what the rows
// need beside them: 128 cosines and sines, each by its own axis, which serve all heads from shared memory, and the row's place
// in the cache (request, slot, page: three loads that depend on one another).  Eight warps rotate, a half-warp per head and 16
// bytes per lane.
// Every wait is bounded; one that runs out is recorded in the status word.
// 32768 rows of 32 + 8 heads, bf16: 149 us, 5.5 TB/s (a copy: 6.6).  A CTA per row, plain loads: 200; the next row's loads in
// registers: 170; bulk copies, four CTAs of four rows each with the CTAs' rows interleaved: 157, with neighbouring rows 154;
// three of three 149, three of six 185, two of eight 161: more rows in flight than the memory needs spread its accesses.
// Short rows (half of kUnitHeads or less) go up to four together, or the latency of a row's place and angles is what counts: 30000
// rows of 8 + 1 heads 77 -> 52 us, 15000 of 4 + 4 39 -> 31.  Longer rows have a kernel of their own without the bookkeeping, which
// costs them more than it gives (32768 rows of 32 + 8 heads: 163 us with it).
#include "ri_paged.cuh"
#include "ri_tc.cuh"

namespace {

using namespace ri_page;
using namespace ri_tc;

constexpr int kWorkWarps = 8, kServiceWarps = 2;
constexpr int kWorkThreads = kWorkWarps * 32;
constexpr int kAppendThreads = kWorkThreads + kServiceWarps * 32;
constexpr int kAppendCtas = 3;                         // of an SM
constexpr int kStages = 3;                             // units on their way to a CTA
constexpr int kUnitHeads = 48;                         // 12 KB: a row, a part of one, or a few short ones
constexpr int kUnitRows = 4;                           // at most

struct AxisOf {
  uint8_t of[64];
};
struct AppendArgs {
  Pages pages;
  const uint4* qkv;
  const float* cos_sin;
  const int64_t* positions;     // [axes][rows]
  const int32_t* row_start;     // [batch + 1] or null: row b is request b's
  const int32_t* seen;          // [batch]; with token numbers only
  uint4* q;
  uint4* k;                     // [rows][hk] or null
  uint4* v;
  uint4* keys;
  uint4* values;
  int64_t qkv_stride;           // 16-byte pieces
  int64_t max_positions;
  int rows, hq;
  int unit_rows, unit_heads, units_per_row;      // a unit: that many rows, of each that many heads
  AxisOf axis;
};

template <int DT>
__device__ __forceinline__ uint4 rotate(const uint4& mine, const uint4& other, const float* cs, float sign) {
  const uint32_t a[4] = {mine.x, mine.y, mine.z, mine.w}, b[4] = {other.x, other.y, other.z, other.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float r[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = Elem<DT>::from_bits((uint16_t)(a[i] >> (16 * e))), y = Elem<DT>::from_bits((uint16_t)(b[i] >> (16 * e)));
      r[e] = x * cs[2 * i + e] + sign * y * cs[8 + 2 * i + e];
    }
    o[i] = Elem<DT>::pack2(r[0], r[1]);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// What a row needs beside its pieces, fetched by a service warp.
struct alignas(16) RowPlan {
  float cs[128];             // cosines, sines; read 16 bytes at a time
  int id, row, token;        // page (-1: none), row in it, token number
};

// The plans of rows row0 .. row0 + n - 1 (n <= ROWS), whose loads are on their way together: lane r looks for row r's place.
template <int ROWS>
__device__ __forceinline__ void plan_rows(const AppendArgs& a, int row0, int n, int lane, RowPlan* plans) {
  const Pages& p = a.pages;
  int64_t pos[ROWS][2];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (r < n) pos[r][i] = a.positions[(int64_t)a.axis.of[lane + 32 * i] * a.rows + row0 + r];
  int b = row0 + lane;
  if (a.row_start != nullptr) {
    b = 0;
    for (int b0 = 0;; b0 += 32) {                      // requests that end at or before the first row
      const bool passed = b0 + lane < p.batch && a.row_start[b0 + lane + 1] <= row0;
      const unsigned votes = __ballot_sync(0xffffffffu, passed);
      b += __popc(votes);
      if (votes != 0xffffffffu) break;
    }
    if (ROWS > 1 && lane < n)
      while (b < p.batch && a.row_start[b + 1] <= row0 + lane) ++b;
  }
  // rows that belong to no request (i < 0) are rotated, no more
  int i_row = -1, length = 0, token = 0;
  if (lane < n && b < p.batch) {
    i_row = row0 + lane - (a.row_start != nullptr ? a.row_start[b] : b);
    length = p.lengths[b];
    token = a.seen != nullptr ? a.seen[b] : length;
  }
  float cs[ROWS][4];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (r < n) {
        const int64_t at = (pos[r][i] < 0 ? 0 : (pos[r][i] >= a.max_positions ? a.max_positions - 1 : pos[r][i])) * 128 + lane + 32 * i;
        cs[r][i] = a.cos_sin[at];
        cs[r][2 + i] = a.cos_sin[at + 64];
      }
  if (lane < n) {
    const int64_t slot = (int64_t)max(length, 0) + i_row;
    int id = -1;
    if (i_row >= 0) {
      if (slot < ((int64_t)p.width << p.shift)) id = page_to_write(p, b, (int)(slot >> p.shift));
      else *p.status = RI_STATUS_PAGES_FULL;
    }
    plans[lane].id = id;
    plans[lane].row = (int)slot & ((1 << p.shift) - 1);
    plans[lane].token = token + i_row;
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r < n) plans[r].cs[lane + 32 * i] = cs[r][i];
}

// Work goes by units: an equal part of a row's heads where there are more than kUnitHeads, else a row or a few.
// ROWS: rows of a unit, at most.
template <int DT, int ROWS>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) rope_append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ __align__(128) uint8_t s_rows[];       // [kStages][unit_heads * 256]
  __shared__ RowPlan s_plan[kStages][ROWS];
  __shared__ __align__(8) uint64_t s_full[kStages], s_empty[kStages];
  __shared__ int s_abort;
  const Pages& p = a.pages;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = a.hq + 2 * p.hk, unit_rows = ROWS == 1 ? 1 : a.unit_rows, unit_bytes = unit_rows * a.unit_heads * 256;
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&s_full[s]), 2);                  // the copy, the plan
      mbar_init(smem_u32(&s_empty[s]), kWorkWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  volatile int* abort_flag = &s_abort;
  ri_pdl_enter();
  // a contiguous range per CTA: neighbouring rows lie in one page
  const int units = ROWS == 1 ? a.rows * a.units_per_row : (a.rows + unit_rows - 1) / unit_rows;
  const int u_lo = (int)((int64_t)blockIdx.x * units / gridDim.x), mine = (int)((int64_t)(blockIdx.x + 1) * units / gridDim.x) - u_lo;
  bool ok = true;
  if (warp >= kWorkWarps) {
    // ---------------- service warps: every second unit each ----------------
    int i = warp - kWorkWarps;
    for (; ok && i < mine; i += kServiceWarps) {
      const int s = i % kStages, u = u_lo + i, row = ROWS == 1 ? u / a.units_per_row : u * unit_rows;
      const int head0 = ROWS == 1 ? (u - row * a.units_per_row) * a.unit_heads : 0, n_rows = ROWS == 1 ? 1 : min(unit_rows, a.rows - row);
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_empty[s]), ((i / kStages) & 1) ^ 1, abort_flag, 91));
      if (!ok) break;
      const uint32_t full = smem_u32(&s_full[s]), bytes = (uint32_t)min(a.unit_heads, heads - head0) * 256;
      if (lane == 0) mbar_arrive_expect_tx(full, n_rows * bytes);
      __syncwarp();
      if (lane < n_rows)
        bulk_load(smem_u32(s_rows) + s * unit_bytes + lane * bytes, a.qkv + (row + lane) * a.qkv_stride + head0 * 16, bytes, full);
      plan_rows<ROWS>(a, row, n_rows, lane, s_plan[s]);
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    }
    if (!ok && lane == 0)      // give this warp's copies in flight a bounded chance to land before the CTA exits
      for (int j = i - kServiceWarps; j >= 0 && j >= i - kStages; j -= kServiceWarps)
        mbar_wait(smem_u32(&s_full[j % kStages]), (j / kStages) & 1, abort_flag, 92);
  } else {
    const int c = tid & 15, half = tid >> 4;
    const float sign = c < 8 ? -1.f : 1.f;
    for (int i = 0; ok && i < mine; ++i) {
      const int s = i % kStages, u = u_lo + i, row0 = ROWS == 1 ? u / a.units_per_row : u * unit_rows;
      const int head0 = ROWS == 1 ? (u - row0 * a.units_per_row) * a.unit_heads : 0, n_rows = ROWS == 1 ? 1 : min(unit_rows, a.rows - row0);
      const int n = min(a.unit_heads, heads - head0);      // heads of each row
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[s]), (i / kStages) & 1, abort_flag, 93));
      if (!ok) break;
      const uint4* src = reinterpret_cast<const uint4*>(s_rows + s * unit_bytes);
      if (head0 == 0) {
        for (int k = tid; k < n_rows * p.hk; k += kWorkThreads) {
          const RowPlan& plan = s_plan[s][ROWS == 1 ? 0 : k / p.hk];
          if (plan.id < 0) continue;
          const int64_t at = record_at(p, plan.id, ROWS == 1 ? k : k % p.hk, plan.row);
          if (p.weight != nullptr) p.weight[at] = 0.f;
          if (p.token != nullptr) p.token[at] = plan.token;
        }
      }
      float cs[16];                                    // this piece's eight cosines, then its eight sines
      int r = -1, id = -1, at = 0;                     // of row r of the unit
      for (int j = half; j < n_rows * n; j += kWorkThreads / 16) {
        if (r < 0 || (ROWS > 1 && j >= (r + 1) * n)) {
          r = ROWS == 1 ? 0 : j / n;
          const RowPlan& plan = s_plan[s][r];
          id = plan.id;
          at = plan.row;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 f = reinterpret_cast<const float4*>(plan.cs)[(k >> 1) * 16 + (c & 7) * 2 + (k & 1)];
            cs[4 * k] = f.x; cs[4 * k + 1] = f.y; cs[4 * k + 2] = f.z; cs[4 * k + 3] = f.w;
          }
        }
        const int row = row0 + r, head = head0 + j - r * n, h = head - a.hq, hv = h - p.hk;
        const uint4 x = src[j * 16 + c];
        const uint4 res = hv >= 0 ? x : rotate<DT>(x, src[j * 16 + (c ^ 8)], cs, sign);
        if (h < 0) {
          a.q[((int64_t)row * a.hq + head) * 16 + c] = res;
        } else {
          uint4* dense = hv >= 0 ? a.v : a.k;
          if (dense != nullptr) dense[((int64_t)row * p.hk + (hv >= 0 ? hv : h)) * 16 + c] = res;
          if (id >= 0) {
            const int64_t in_page = ((int64_t)((hv >= 0 ? hv : h) << p.shift) + at) * 16 + c;
            if (hv >= 0) a.values[id * (p.value_stride / 8) + in_page] = res;
            else a.keys[id * (p.key_stride / 8) + in_page] = res;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_empty[s]));
    }
  }
  if (!ok && lane == 0) *p.status = s_abort;
}

}  // namespace

extern "C" int ri_rope_paged_append(const ri_paged* p, const void* d_qkv, int64_t qkv_stride, const float* d_cos_sin,
                                    int64_t max_positions, const int64_t* d_positions, const uint8_t* h_axis_of, int32_t axes,
                                    int32_t rows, const int32_t* d_row_start, const int32_t* d_seen, void* d_q, void* d_k, void* d_v,
                                    void* stream) {
  int rc;
  if ((rc = check(p, "ri_rope_paged_append")) != RI_OK) return rc;
  RI_REQUIRE(p->d_values && d_qkv && d_cos_sin && d_positions && h_axis_of && d_q, "ri_rope_paged_append: null pointer");
  RI_REQUIRE(!p->d_token || d_seen, "ri_rope_paged_append: token numbers need the count of tokens seen");
  RI_REQUIRE(rows >= 1 && max_positions >= 1 && axes >= 1 && axes <= 64 && p->group_size >= 1 && p->group_size <= 65535,
             "ri_rope_paged_append: rows=%d axes=%d group_size=%d unsupported", rows, axes, p->group_size);
  RI_REQUIRE(d_row_start || rows == p->batch, "ri_rope_paged_append: %d rows for %d requests need row_start", rows, p->batch);
  const int64_t hq = (int64_t)p->group_size * p->kv_heads;
  RI_REQUIRE(hq + 2 * p->kv_heads < (1 << 24) && qkv_stride >= (hq + 2 * p->kv_heads) * RI_HEAD_DIM && qkv_stride % 8 == 0,
             "ri_rope_paged_append: rows of the projection overlap or lie at odd places");
  RI_REQUIRE(((uintptr_t)d_qkv | (uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v) % 16 == 0,
             "ri_rope_paged_append: tensors must be 16-byte aligned");
  AppendArgs a = {};
  for (int i = 0; i < 64; ++i) {
    RI_REQUIRE(h_axis_of[i] < axes, "ri_rope_paged_append: frequency %d follows axis %d of %d", i, h_axis_of[i], axes);
    a.axis.of[i] = h_axis_of[i];
  }
  a.pages = view(*p);
  a.qkv = static_cast<const uint4*>(d_qkv);
  a.qkv_stride = qkv_stride / 8;
  a.cos_sin = d_cos_sin;
  a.max_positions = max_positions;
  a.positions = d_positions;
  a.row_start = d_row_start;
  a.seen = d_seen;
  a.q = static_cast<uint4*>(d_q);
  a.k = static_cast<uint4*>(d_k);
  a.v = static_cast<uint4*>(d_v);
  a.keys = static_cast<uint4*>(const_cast<void*>(p->d_keys));
  a.values = static_cast<uint4*>(const_cast<void*>(p->d_values));
  a.rows = rows;
  a.hq = (int)hq;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int sms = 0;
  if ((rc = ri_sm_count(&sms)) != RI_OK) return rc;
  const int heads = (int)hq + 2 * p->kv_heads;
  a.units_per_row = (heads + kUnitHeads - 1) / kUnitHeads;
  a.unit_heads = (heads + a.units_per_row - 1) / a.units_per_row;
  // short rows go a few together, where there is more than a unit for every CTA: with fewer they would leave CTAs idle
  a.unit_rows = 1;
  const int64_t most = (int64_t)sms * kAppendCtas;
  while (a.unit_rows < kUnitRows && (a.unit_rows + 1) * heads <= kUnitHeads && rows > most * a.unit_rows) ++a.unit_rows;
  const int64_t units = a.units_per_row > 1 ? (int64_t)rows * a.units_per_row : ((int64_t)rows + a.unit_rows - 1) / a.unit_rows;
  RI_REQUIRE(units < (1ll << 30), "ri_rope_paged_append: too large");
  const dim3 grid((unsigned)(units < most ? units : most));
  const size_t smem = (size_t)kStages * a.unit_rows * a.unit_heads * 256;
  auto go = [&](auto kernel) { return ri_launch_pdl_id(8, kernel, grid, dim3(kAppendThreads), smem, s, a); };
  constexpr int kMost = kStages * kUnitHeads * 256;
  if (a.unit_rows > 1) {
    if ((rc = ri_allow_smem<rope_append_kernel<RI_BF16, kUnitRows>>(kMost)) != RI_OK ||
        (rc = ri_allow_smem<rope_append_kernel<RI_F16, kUnitRows>>(kMost)) != RI_OK)
      return rc;
    RI_CUDA_OK(p->dtype == RI_BF16 ? go(rope_append_kernel<RI_BF16, kUnitRows>) : go(rope_append_kernel<RI_F16, kUnitRows>));
  } else {
    if ((rc = ri_allow_smem<rope_append_kernel<RI_BF16, 1>>(kMost)) != RI_OK ||
        (rc = ri_allow_smem<rope_append_kernel<RI_F16, 1>>(kMost)) != RI_OK)
      return rc;
    RI_CUDA_OK(p->dtype == RI_BF16 ? go(rope_append_kernel<RI_BF16, 1>) : go(rope_append_kernel<RI_F16, 1>));
  }
  return RI_OK;
}
