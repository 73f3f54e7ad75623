// What the kernels over a paged cache share: its addressing, and the checks of the struct that describes it.
//
// A pool holds pages [n_pages][kv_heads][page_size] of rows of 128 channels, keys and values in two tensors whose pages may
// lie further apart than they are large; weight and token number of every slot lie dense beside them.  Slot j of request b
// is row j % page_size of page table[b][j / page_size], for every KV head.  Page sizes are powers of two of 8 and more, so
// that a box of 8 rows never leaves a page.
#pragma once

#include "ri_common.cuh"

namespace ri_page {

struct Pages {
  const int32_t* table;      // [batch][table_stride]
  const int32_t* lengths;    // [batch]
  float* weight;             // [n_pages][hk][page_size] or null
  int32_t* token;            // the same, or null
  int* status;               // 0, or what went wrong
  int64_t key_stride, value_stride;   // elements from page to page
  int batch, hk, n_pages, table_stride, width, shift;   // width: table entries that count; page_size = 1 << shift
};

// Slots of request b that are in use: its length as far as its page table counts.
__device__ __forceinline__ int rows_of(const Pages& p, int b) {
  return (int)min((int64_t)max(p.lengths[b], 0), (int64_t)p.width << p.shift);
}
// A page number out of a table, for readers.  One that names no page is reported, and page 0 stands in for it: nothing outside
// the pool is touched, and the call's results for that request mean nothing.
__device__ __forceinline__ int page_or_first(const Pages& p, int id) {
  if ((unsigned)id < (unsigned)p.n_pages) return id;
  *p.status = RI_STATUS_PAGE_ID;
  return 0;
}
// The same for writers: -1 where there is no such page, and nothing is written.
__device__ __forceinline__ int page_or_none(const Pages& p, int id) {
  if ((unsigned)id < (unsigned)p.n_pages) return id;
  *p.status = RI_STATUS_PAGE_ID;
  return -1;
}
// Page i of request b.
__device__ __forceinline__ int page_of(const Pages& p, int b, int i) { return page_or_first(p, p.table[(int64_t)b * p.table_stride + i]); }
__device__ __forceinline__ int page_to_write(const Pages& p, int b, int i) {
  return page_or_none(p, p.table[(int64_t)b * p.table_stride + i]);
}
// Row `row` of head h in page `id`: its place in the tensors of weights and token numbers.
__device__ __forceinline__ int64_t record_at(const Pages& p, int id, int h, int row) {
  return (((int64_t)id * p.hk + h) << p.shift) + row;
}

inline int width_of(const ri_paged& p) { return p.table_width > 0 ? p.table_width : p.table_stride; }
inline int64_t slots_of(const ri_paged& p) { return (int64_t)width_of(p) * p.page_size; }      // of the longest request there may be

inline Pages view(const ri_paged& p) {
  Pages v = {};
  v.table = p.d_table;
  v.lengths = p.d_lengths;
  v.weight = p.d_weight;
  v.token = p.d_token;
  v.status = p.d_status;
  v.key_stride = p.key_page_stride;
  v.value_stride = p.value_page_stride;
  v.batch = p.batch; v.hk = p.kv_heads; v.n_pages = p.n_pages; v.table_stride = p.table_stride;
  v.width = width_of(p);
  while ((1 << v.shift) < p.page_size) ++v.shift;
  return v;
}

inline int check(const ri_paged* p, const char* what) {
  RI_REQUIRE(p && p->d_keys && p->d_table && p->d_lengths && p->d_status, "%s: null pointer", what);
  RI_REQUIRE(p->batch >= 1 && p->kv_heads >= 1 && (int64_t)p->batch * p->kv_heads <= 65535, "%s: batch=%d kv_heads=%d unsupported",
             what, p->batch, p->kv_heads);
  RI_REQUIRE(p->page_size >= 8 && p->page_size <= 1024 && (p->page_size & (p->page_size - 1)) == 0,
             "%s: page_size=%d unsupported (a power of two from 8 to 1024)", what, p->page_size);
  RI_REQUIRE(p->n_pages >= 1 && p->table_stride >= 1, "%s: n_pages=%d table_stride=%d unsupported", what, p->n_pages, p->table_stride);
  RI_REQUIRE(p->table_width >= 0 && p->table_width <= p->table_stride, "%s: table_width=%d of table_stride=%d unsupported", what,
             p->table_width, p->table_stride);
  RI_REQUIRE(slots_of(*p) < (1ll << 31) - 1024 && (int64_t)p->batch * p->kv_heads * (slots_of(*p) / 8 + 1) < (1ll << 31) - 1024,
             "%s: the page table reaches too far", what);
  RI_REQUIRE(p->dtype == RI_BF16 || p->dtype == RI_F16, "dtype=%d unsupported", p->dtype);
  const int64_t page = (int64_t)p->kv_heads * p->page_size * RI_HEAD_DIM;
  RI_REQUIRE(p->key_page_stride >= page && p->key_page_stride % 8 == 0 && (!p->d_values || (p->value_page_stride >= page && p->value_page_stride % 8 == 0)),
             "%s: pages overlap or lie at odd places", what);
  RI_REQUIRE(((uintptr_t)p->d_keys | (uintptr_t)p->d_values) % 16 == 0, "%s: the pools must be 16-byte aligned", what);
  RI_REQUIRE(((uintptr_t)p->d_weight | (uintptr_t)p->d_token | (uintptr_t)p->d_table | (uintptr_t)p->d_lengths) % 4 == 0,
             "%s: misaligned pointer", what);
  return RI_OK;
}

}  // namespace ri_page
