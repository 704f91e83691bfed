// The paged int8 key/value cache as the kernels see it, and the way from a row of a call to its
// place in the pool.
#pragma once
#include "quant_common.cuh"
#include "sdq_internal.h"

namespace sdq {

__host__ __device__ __forceinline__ int32_t table_at(const int32_t* p, int64_t i) {
#ifdef __CUDA_ARCH__
  return __ldg(p + i);
#else
  return p[i];
#endif
}

// Division of a position by the page size: floor(p / d) = (p * m) >> 32 with m = ceil(2^32 / d) is
// exact while p * (m * d - 2^32) < 2^32, and m * d - 2^32 < d, so for p * d < 2^32; beyond that the
// hardware's own division is used.
struct PageDiv {
  uint32_t size, magic, most;  // most: largest position the multiplication serves
  __host__ explicit PageDiv(uint32_t d)
      : size(d), magic(d > 1 ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u),
        most(d > 1 ? (uint32_t)(((1ull << 32) - 1) / d) : 0u) {}
  __host__ __device__ __forceinline__ uint32_t page(uint32_t p) const {
    return size > 1 && p <= most ? (uint32_t)(((uint64_t)p * magic) >> 32) : p / size;
  }
};

struct KvArgs {
  int8_t* k;            // [pages, heads, page_size, D]
  int8_t* v;
  float* k_scale;       // [pages, heads, page_size]
  float* v_scale;
  const int32_t* row_start;   // [batch + 1]
  const int32_t* kv_len;      // [batch]
  const int32_t* page_table;  // [batch, max_pages]
  PageDiv page;
  int32_t pages, heads, page_size, D, batch, max_pages;
  int32_t rows;
};

struct AttendArgs {
  const void* q;    // [rows, heads, D], ldq elements from row to row
  void* out;        // the same shape and type, ldo elements from row to row
  int64_t ldq, ldo;
  int32_t heads;    // query heads, a multiple of the cache's
  int32_t causal;
  float scale;
};

// Row range of sequence b, whatever the table holds: [first, last) inside [0, rows].
__host__ __device__ __forceinline__ void seq_rows(const KvArgs& a, int b, int& first, int& last) {
  const int32_t f = table_at(a.row_start, b), l = table_at(a.row_start, b + 1);
  first = f < 0 ? 0 : f > a.rows ? a.rows : f;
  last = l < first ? first : l > a.rows ? a.rows : l;
}

// The sequence that owns a row: the last b with row_start[b] <= row; -1 in front of the first one
// and behind the last.
__host__ __device__ __forceinline__ int seq_of_row(const KvArgs& a, int row) {
  int lo = 0, hi = a.batch;   // row_start[lo - 1] <= row < row_start[hi]
  if (row >= table_at(a.row_start, a.batch)) return -1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (table_at(a.row_start, mid) <= row) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

// Pool row of position p of sequence b for cache head 0 (head h lies h * page_size further), or -1
// where the table has no such page.
__host__ __device__ __forceinline__ int pool_row(const KvArgs& a, int b, int p) {
  if (p < 0) return -1;
  const uint32_t i = a.page.page((uint32_t)p);
  if (i >= (uint32_t)a.max_pages) return -1;
  const int page = table_at(a.page_table, (int64_t)b * a.max_pages + i);
  if ((uint32_t)page >= (uint32_t)a.pages) return -1;
  return page * a.heads * a.page_size + (p - (int)i * a.page_size);
}

// Pool row (head 0) that row `row` of a call stands for: the rows of a sequence are its last ones.
__host__ __device__ __forceinline__ int pool_row_of(const KvArgs& a, int row) {
  const int b = seq_of_row(a, row);
  if (b < 0) return -1;
  const int last = table_at(a.row_start, b + 1);
  const int64_t p = (int64_t)table_at(a.kv_len, b) - last + row;
  return p > INT32_MAX ? -1 : p < 0 ? -1 : pool_row(a, b, (int)p);
}

cudaError_t launch_kv_io(const KvArgs& a, void* k, void* v, int dtype, int64_t ld, bool append, cudaStream_t s);
cudaError_t launch_kv_attention(const KvArgs& a, const AttendArgs& t, int dtype, cudaStream_t s);

}  // namespace sdq
