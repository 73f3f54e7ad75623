// Rotary positions with several axes on a fused QKV projection, queries out, keys and values into a paged cache.
//   for i < 64, (c, s) the table's row at the row's position on axis axis_of[i], columns i and 64 + i:
//     x'_i = x_i c - x_{i+64} s,    x'_{i+64} = x_{i+64} c + x_i s          (query and key heads; values as they are)
// One axis is the ordinary rotary embedding; text, images and video take (time, height, width).
// (reference: model_hub/llama.py:232-235 the split, :312-320 the rotation; cache_hub/flash_attn_cache.py:133-151 the append)
//
// Bound by the projection, read once and written once.  One CTA per row: a head is sixteen 16-byte pieces, a half-warp per
// head, and a piece's partner (the channels 64 away) comes by shuffle.  The row's 128 cosines and sines are fetched once, each
// by its own axis, and serve all heads from shared memory; they and the row's place in the cache (request, slot, page: three
// dependent loads) come in while the row's pieces do.
#include "ri_paged.cuh"

namespace {

using namespace ri_page;

constexpr int kAppendThreads = 256;
constexpr int kHeadsAtOnce = kAppendThreads / 16;      // one round of the CTA
constexpr int kRounds = 4;                             // rounds whose loads are in flight together

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

template <int DT>
__global__ void __launch_bounds__(kAppendThreads) rope_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ float s_cs[128];
  __shared__ int s_id, s_row, s_token;
  ri_pdl_enter();
  const Pages& p = a.pages;
  const int row = blockIdx.x, tid = threadIdx.x, c = tid & 15, first = tid >> 4;
  const int heads = a.hq + 2 * p.hk;
  const uint4* src = a.qkv + row * a.qkv_stride;
  uint4 x[kRounds];
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const int head = first + u * kHeadsAtOnce;
    x[u] = head < heads ? ri_ldg16(src + head * 16 + c) : make_uint4(0, 0, 0, 0);
  }
  if (tid < 128) {
    int64_t pos = a.positions[(int64_t)a.axis.of[tid & 63] * a.rows + row];
    pos = pos < 0 ? 0 : (pos >= a.max_positions ? a.max_positions - 1 : pos);
    s_cs[tid] = a.cos_sin[pos * 128 + tid];
  } else if (tid >= kAppendThreads - 32) {             // the last warp: which request, slot and page
    const int lane = tid & 31;
    int b = row;
    if (a.row_start != nullptr) {
      b = 0;
      for (int b0 = 0;; b0 += 32) {                    // requests that end at or before this row
        const bool passed = b0 + lane < p.batch && a.row_start[b0 + lane + 1] <= row;
        const unsigned votes = __ballot_sync(0xffffffffu, passed);
        b += __popc(votes);
        if (votes != 0xffffffffu) break;
      }
    }
    if (lane == 0) {
      s_id = -1;
      s_row = s_token = 0;
      const int i = b < p.batch ? row - (a.row_start != nullptr ? a.row_start[b] : b) : -1;
      if (i >= 0) {                                    // rows that belong to no request are rotated, no more
        const int64_t slot = (int64_t)max(p.lengths[b], 0) + i;
        if (slot < ((int64_t)p.table_stride << p.shift)) {
          s_id = page_to_write(p, b, (int)(slot >> p.shift));
          s_row = (int)slot & ((1 << p.shift) - 1);
          s_token = (a.seen != nullptr ? a.seen[b] : (int)slot - i) + i;
        } else {
          *p.status = RI_STATUS_PAGES_FULL;
        }
      }
    }
  }
  __syncthreads();
  const int id = s_id, at = s_row;
  float cs[16];                                        // this piece's eight cosines, then its eight sines
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = s_cs[(c & 7) * 8 + i];
    cs[8 + i] = s_cs[64 + (c & 7) * 8 + i];
  }
  const float sign = c < 8 ? -1.f : 1.f;
  if (id >= 0) {
    for (int h = tid; h < p.hk; h += kAppendThreads) {
      if (p.weight != nullptr) p.weight[record_at(p, id, h, at)] = 0.f;
      if (p.token != nullptr) p.token[record_at(p, id, h, at)] = s_token;
    }
  }
  for (int base = 0; base < heads; base += kRounds * kHeadsAtOnce) {
#pragma unroll
    for (int u = 0; u < kRounds; ++u) {
      const int head = base + first + u * kHeadsAtOnce;
      uint4 other;
      other.x = __shfl_xor_sync(0xffffffffu, x[u].x, 8);
      other.y = __shfl_xor_sync(0xffffffffu, x[u].y, 8);
      other.z = __shfl_xor_sync(0xffffffffu, x[u].z, 8);
      other.w = __shfl_xor_sync(0xffffffffu, x[u].w, 8);
      if (head >= heads) continue;
      const int h = head - a.hq, hv = h - p.hk;
      const uint4 res = hv >= 0 ? x[u] : rotate<DT>(x[u], other, cs, sign);
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
    const int next = base + kRounds * kHeadsAtOnce;
    if (next < heads) {
#pragma unroll
      for (int u = 0; u < kRounds; ++u) {
        const int head = next + first + u * kHeadsAtOnce;
        x[u] = head < heads ? ri_ldg16(src + head * 16 + c) : make_uint4(0, 0, 0, 0);
      }
    }
  }
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
  auto go = [&](auto kernel) { return ri_launch_pdl_id(8, kernel, dim3(rows), dim3(kAppendThreads), 0, s, a); };
  RI_CUDA_OK(p->dtype == RI_BF16 ? go(rope_append_kernel<RI_BF16>) : go(rope_append_kernel<RI_F16>));
  return RI_OK;
}
