// Rotary positions with several axes on a fused QKV projection, queries out, keys and values into a paged cache.
//   for i < 64, (c, s) the table's row at the row's position on axis axis_of[i], columns i and 64 + i:
//     x'_i = x_i c - x_{i+64} s,    x'_{i+64} = x_{i+64} c + x_i s          (query and key heads; values as they are)
// One axis is the ordinary rotary embedding; text, images and video take (time, height, width).
// With norms a query or key head is first  x_i <- x_i w_i / sqrt(mean x^2 + eps),  in 32 bits up to the one rounding behind the rotation;
// the half-warp that has a head has its sum of squares in four shuffles.  The root is taken behind the rotation, and weights that are
// the same for all heads go into the row's cosines and sines, which a service warp multiplies: the rotation is what it was, and the
// rotating warps, which would be what counts otherwise, have a third more to do, not twice as much.  32768 rows of 32 + 8 heads: 155 to 167 us
// (146 to 149 without norms; with the weights loaded and multiplied head by head 210).  Weights for each head are multiplied by the lane that has
// the piece, and the piece that it is rotated with comes from the lane beside it: 176 to 180 us (198 with both pieces weighted by both lanes).
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
  const uint4* q_norm;          // [16 pieces] or [heads][16]: the strides say which
  const uint4* k_norm;
  int q_norm_stride, k_norm_stride;              // pieces from head to head: 0 or 16
  float eps;
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

// Eight channels as pairs in 32 bits.
template <int DT>
__device__ __forceinline__ void unpack_pairs(const uint4& x, uint64_t (&p)[4]) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = pack_f2(Elem<DT>::from_bits((uint16_t)(u[i] & 0xffffu)), Elem<DT>::from_bits((uint16_t)(u[i] >> 16)));
}
// The rotation behind an RMS norm: (x A + y B) / rms, pairs at a time.  Sixteen lanes, those of `half_warp`, have a head's pieces.
template <int DT>
__device__ __forceinline__ uint4 rotate_normed(const uint64_t (&x)[4], const uint64_t (&y)[4], const uint64_t (&a)[4], const uint64_t (&b)[4],
                                               float inv) {
  const uint64_t by = pack_f2(inv, inv);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpack_f2(mul_f2(fma_f2(x[i], a[i], mul_f2(y[i], b[i])), by), lo, hi);
    o[i] = Elem<DT>::pack2(lo, hi);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ float head_squares(const uint64_t (&x)[4], unsigned half_warp) {
  uint64_t two = mul_f2(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) two = fma_f2(x[i], x[i], two);
  float sum, odd;
  unpack_f2(two, sum, odd);
  sum += odd;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(half_warp, sum, o);
  return sum;
}

// What a row needs beside its pieces, fetched by a service warp.
enum Norm { kNone, kOneWeight, kHeadWeights };      // norms: none, with a weight for all heads, with one for each
template <int NORM>
struct alignas(16) RowPlan {
  // cosines, sines; kOneWeight: for query and key heads what every channel is multiplied by, and the one it is rotated with, weights
  // included.  Read 16 bytes at a time
  float cs[NORM == kOneWeight ? 512 : 128];
  int id, row, token;        // page (-1: none), row in it, token number
};

// The plans of rows row0 .. row0 + n - 1 (n <= ROWS), whose loads are on their way together: lane r looks for row r's place.
// w: kOneWeight, the weights of query and key heads for channels lane + 32 i and, behind them, 64 on.
template <int ROWS, int NORM>
__device__ __forceinline__ void plan_rows(const AppendArgs& a, int row0, int n, int lane, const float (&w)[2][4], RowPlan<NORM>* plans) {
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
      if (r < n) {
        if (NORM != kOneWeight) {
          plans[r].cs[lane + 32 * i] = cs[r][i];
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {                  // channel lane + 32 i; it is rotated with the one 64 from it
            plans[r].cs[256 * k + lane + 32 * i] = w[k][i] * cs[r][i & 1];
            plans[r].cs[256 * k + 128 + lane + 32 * i] = (i < 2 ? -1.f : 1.f) * w[k][i ^ 2] * cs[r][2 + (i & 1)];
          }
        }
      }
}

// Work goes by units: an equal part of a row's heads where there are more than kUnitHeads, else a row or a few.
// ROWS: rows of a unit, at most.  NORM: whether and with what weights query and key heads are normalised before they are rotated.
template <int DT, int ROWS, int NORM>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) rope_append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ __align__(128) uint8_t s_rows[];       // [kStages][unit_heads * 256]
  __shared__ RowPlan<NORM> s_plan[kStages][ROWS];
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
    float w[2][4] = {};
    if (NORM == kOneWeight) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        w[0][x] = Elem<DT>::from_bits(reinterpret_cast<const uint16_t*>(a.q_norm)[lane + 32 * x]);
        w[1][x] = Elem<DT>::from_bits(reinterpret_cast<const uint16_t*>(a.k_norm)[lane + 32 * x]);
      }
    }
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
      plan_rows<ROWS, NORM>(a, row, n_rows, lane, w, s_plan[s]);
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    }
    if (!ok && lane == 0)      // give this warp's copies in flight a bounded chance to land before the CTA exits
      for (int j = i - kServiceWarps; j >= 0 && j >= i - kStages; j -= kServiceWarps)
        mbar_wait(smem_u32(&s_full[j % kStages]), (j / kStages) & 1, abort_flag, 92);
  } else {
    const int c = tid & 15, half = tid >> 4;
    const unsigned half_warp = 0xffffu << (lane & 16);
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
          const RowPlan<NORM>& plan = s_plan[s][ROWS == 1 ? 0 : k / p.hk];
          if (plan.id < 0) continue;
          const int64_t at = record_at(p, plan.id, ROWS == 1 ? k : k % p.hk, plan.row);
          if (p.weight != nullptr) p.weight[at] = 0.f;
          if (p.token != nullptr) p.token[at] = plan.token;
        }
      }
      int r = -1, id = -1, at = 0;                     // of row r of the unit
      // where head `head` of that row goes
      auto put = [&](int row, int head, const uint4& res) {
        const int h = head - a.hq, hv = h - p.hk;
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
      };
      if constexpr (NORM == kNone) {
        float cs[16];                                  // this piece's eight cosines, then its eight sines
        for (int j = half; j < n_rows * n; j += kWorkThreads / 16) {
          if (r < 0 || (ROWS > 1 && j >= (r + 1) * n)) {
            r = ROWS == 1 ? 0 : j / n;
            const RowPlan<NORM>& plan = s_plan[s][r];
            id = plan.id;
            at = plan.row;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float4 f = reinterpret_cast<const float4*>(plan.cs)[(k >> 1) * 16 + (c & 7) * 2 + (k & 1)];
              cs[4 * k] = f.x; cs[4 * k + 1] = f.y; cs[4 * k + 2] = f.z; cs[4 * k + 3] = f.w;
            }
          }
          const int head = head0 + j - r * n;
          const uint4 x = src[j * 16 + c];
          put(row0 + r, head, head >= a.hq + p.hk ? x : rotate<DT>(x, src[j * 16 + (c ^ 8)], cs, sign));
        }
      } else {
        uint64_t fa[4], fb[4];                         // factors of this piece's channels, and of those it is rotated with
        bool of_keys = false;                          // kOneWeight: whose they are
        for (int j = half; j < n_rows * n; j += kWorkThreads / 16) {
          const bool next = r < 0 || (ROWS > 1 && j >= (r + 1) * n);
          if (next) {
            r = ROWS == 1 ? 0 : j / n;
            id = s_plan[s][r].id;
            at = s_plan[s][r].row;
          }
          const int head = head0 + j - r * n;
          const bool key = head >= a.hq;
          const uint4 mine16 = src[j * 16 + c];
          if (head >= a.hq + p.hk) {
            put(row0 + r, head, mine16);
            continue;
          }
          if (next || (NORM == kOneWeight && key != of_keys)) {
            of_keys = key;
            const float* from = s_plan[s][r].cs + (NORM == kOneWeight ? (key ? 256 : 0) + 8 * c : 8 * (c & 7));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float4 f = reinterpret_cast<const float4*>(from)[k], g = reinterpret_cast<const float4*>(from + (NORM == kOneWeight ? 128 : 64))[k];
              const float turn = NORM == kOneWeight ? 1.f : sign;
              fa[2 * k] = pack_f2(f.x, f.y);
              fa[2 * k + 1] = pack_f2(f.z, f.w);
              fb[2 * k] = pack_f2(turn * g.x, turn * g.y);
              fb[2 * k + 1] = pack_f2(turn * g.z, turn * g.w);
            }
          }
          uint64_t x[4], y[4];
          unpack_pairs<DT>(mine16, x);
          const float inv = rsqrtf(head_squares(x, half_warp) * (1.f / RI_HEAD_DIM) + a.eps);
          if (NORM == kHeadWeights) {                  // the piece it is rotated with comes, weighted, from the lane that has it
            const uint4* w = key ? a.k_norm + (head - a.hq) * a.k_norm_stride : a.q_norm + head * a.q_norm_stride;
            uint64_t wx[4];
            unpack_pairs<DT>(ri_ldg16(w + c), wx);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              x[k] = mul_f2(x[k], wx[k]);
              y[k] = __shfl_xor_sync(half_warp, (unsigned long long)x[k], 8);
            }
          } else {
            unpack_pairs<DT>(src[j * 16 + (c ^ 8)], y);
          }
          put(row0 + r, head, rotate_normed<DT>(x, y, fa, fb, inv));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_empty[s]));
    }
  }
  if (!ok && lane == 0) *p.status = s_abort;
}

template <int DT, int ROWS, int NORM>
int launch_kernel(const AppendArgs& a, dim3 grid, size_t smem, cudaStream_t s) {
  const int rc = ri_allow_smem<rope_append_kernel<DT, ROWS, NORM>>(kStages * kUnitHeads * 256);
  if (rc != RI_OK) return rc;
  RI_CUDA_OK(ri_launch_pdl_id(8, rope_append_kernel<DT, ROWS, NORM>, grid, dim3(kAppendThreads), smem, s, a));
  return RI_OK;
}
template <int DT, int ROWS>
int launch(const AppendArgs& a, dim3 grid, size_t smem, cudaStream_t s) {
  if (a.q_norm == nullptr) return launch_kernel<DT, ROWS, kNone>(a, grid, smem, s);
  return a.q_norm_stride == 0 && a.k_norm_stride == 0 ? launch_kernel<DT, ROWS, kOneWeight>(a, grid, smem, s)
                                                      : launch_kernel<DT, ROWS, kHeadWeights>(a, grid, smem, s);
}

struct Norms {
  const void* q;
  const void* k;
  int32_t q_heads, k_heads;     // that have a weight of their own: 1 or all
  float eps;
};

int append(const char* what, const ri_paged* p, const void* d_qkv, int64_t qkv_stride, const float* d_cos_sin, int64_t max_positions,
           const int64_t* d_positions, const uint8_t* h_axis_of, int32_t axes, int32_t rows, const int32_t* d_row_start,
           const int32_t* d_seen, const Norms* norms, void* d_q, void* d_k, void* d_v, void* stream) {
  int rc;
  if ((rc = check(p, what)) != RI_OK) return rc;
  RI_REQUIRE(p->d_values && d_qkv && d_cos_sin && d_positions && h_axis_of && d_q, "%s: null pointer", what);
  RI_REQUIRE(!p->d_token || d_seen, "%s: token numbers need the count of tokens seen", what);
  RI_REQUIRE(rows >= 1 && max_positions >= 1 && axes >= 1 && axes <= 64 && p->group_size >= 1 && p->group_size <= 65535,
             "%s: rows=%d axes=%d group_size=%d unsupported", what, rows, axes, p->group_size);
  RI_REQUIRE(d_row_start || rows == p->batch, "%s: %d rows for %d requests need row_start", what, rows, p->batch);
  const int64_t hq = (int64_t)p->group_size * p->kv_heads;
  RI_REQUIRE(hq + 2 * p->kv_heads < (1 << 24) && qkv_stride >= (hq + 2 * p->kv_heads) * RI_HEAD_DIM && qkv_stride % 8 == 0,
             "%s: rows of the projection overlap or lie at odd places", what);
  RI_REQUIRE(((uintptr_t)d_qkv | (uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v) % 16 == 0,
             "%s: tensors must be 16-byte aligned", what);
  AppendArgs a = {};
  for (int i = 0; i < 64; ++i) {
    RI_REQUIRE(h_axis_of[i] < axes, "%s: frequency %d follows axis %d of %d", what, i, h_axis_of[i], axes);
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
  if (norms != nullptr) {
    RI_REQUIRE(norms->q && norms->k, "%s: null pointer", what);
    RI_REQUIRE(((uintptr_t)norms->q | (uintptr_t)norms->k) % 16 == 0, "%s: tensors must be 16-byte aligned", what);
    RI_REQUIRE((norms->q_heads == 1 || norms->q_heads == hq) && (norms->k_heads == 1 || norms->k_heads == p->kv_heads),
               "%s: weights of %d and %d heads for %d and %d", what, norms->q_heads, norms->k_heads, (int)hq, p->kv_heads);
    RI_REQUIRE(norms->eps >= 0.f && norms->eps < 1e30f, "%s: eps must be finite and not negative", what);
    a.q_norm = static_cast<const uint4*>(norms->q);
    a.k_norm = static_cast<const uint4*>(norms->k);
    a.q_norm_stride = norms->q_heads > 1 ? 16 : 0;
    a.k_norm_stride = norms->k_heads > 1 ? 16 : 0;
    a.eps = norms->eps;
  }
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
  RI_REQUIRE(units < (1ll << 30), "%s: too large", what);
  const dim3 grid((unsigned)(units < most ? units : most));
  const size_t smem = (size_t)kStages * a.unit_rows * a.unit_heads * 256;
  if (a.unit_rows > 1) return p->dtype == RI_BF16 ? launch<RI_BF16, kUnitRows>(a, grid, smem, s) : launch<RI_F16, kUnitRows>(a, grid, smem, s);
  return p->dtype == RI_BF16 ? launch<RI_BF16, 1>(a, grid, smem, s) : launch<RI_F16, 1>(a, grid, smem, s);
}

}  // namespace

extern "C" int ri_rope_paged_append(const ri_paged* p, const void* d_qkv, int64_t qkv_stride, const float* d_cos_sin,
                                    int64_t max_positions, const int64_t* d_positions, const uint8_t* h_axis_of, int32_t axes,
                                    int32_t rows, const int32_t* d_row_start, const int32_t* d_seen, void* d_q, void* d_k, void* d_v,
                                    void* stream) {
  return append("ri_rope_paged_append", p, d_qkv, qkv_stride, d_cos_sin, max_positions, d_positions, h_axis_of, axes, rows, d_row_start,
                d_seen, nullptr, d_q, d_k, d_v, stream);
}

extern "C" int ri_rope_paged_append_norm(const ri_paged* p, const void* d_qkv, int64_t qkv_stride, const float* d_cos_sin,
                                         int64_t max_positions, const int64_t* d_positions, const uint8_t* h_axis_of, int32_t axes,
                                         int32_t rows, const int32_t* d_row_start, const int32_t* d_seen, const void* d_q_norm,
                                         const void* d_k_norm, int32_t q_norm_heads, int32_t k_norm_heads, float eps, void* d_q,
                                         void* d_k, void* d_v, void* stream) {
  const Norms norms = {d_q_norm, d_k_norm, q_norm_heads, k_norm_heads, eps};
  return append("ri_rope_paged_append_norm", p, d_qkv, qkv_stride, d_cos_sin, max_positions, d_positions, h_axis_of, axes, rows,
                d_row_start, d_seen, &norms, d_q, d_k, d_v, stream);
}
