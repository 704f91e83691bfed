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
  int* status;      // device word for a wait that gave up
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

// Row tiles.  The rows of a sequence and one cache head are its new tokens times the `group` query heads
// that share the head, row = token * group + head; a tile takes T of them.  Tiles are numbered from the
// longest sequence down, and inside one from its last rows (which see the most keys) back: blocks run in
// about that order, so the GPU ends on short pieces.  That takes comparing all sequences with all, which
// pays up to 64 of them; beyond, sequence b's numbers begin at row_start[b] * group / T + b, which leaves
// room for a ragged last tile (ceil(n / T) <= floor((s + n) / T) - floor(s / T) + 1), and a number that is no
// tile ends at once.  Called by whole warps.
struct Tile {
  int b, first_row, rows;   // sequence; first (token, head) row; how many
  int first, n, len;        // first row of the call, new tokens, keys of the sequence
};
__device__ __forceinline__ bool find_tile(const KvArgs& a, int group, int T, int id, Tile* t) {
  const int lane = threadIdx.x & 31;
  int in_seq;   // number inside the sequence
  if (a.batch <= 64) {
    int len[2], tiles[2], before[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int b = lane + 32 * i;
      len[i] = -1;
      tiles[i] = 0;
      if (b < a.batch) {
        int f, l;
        seq_rows(a, b, f, l);
        len[i] = max(0, table_at(a.kv_len, b));
        tiles[i] = ((l - f) * group + T - 1) / T;
      }
    }
    for (int j = 0; j < a.batch; j++) {
      const int lj = __shfl_sync(0xffffffffu, j < 32 ? len[0] : len[1], j & 31), tj = __shfl_sync(0xffffffffu, j < 32 ? tiles[0] : tiles[1], j & 31);
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (lj > len[i] || (lj == len[i] && j < lane + 32 * i)) before[i] += tj;
    }
    int b = -1, at = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t it = __ballot_sync(0xffffffffu, id >= before[i] && id < before[i] + tiles[i]);
      if (it) {
        const int src = __ffs(it) - 1;
        b = src + 32 * i;
        at = __shfl_sync(0xffffffffu, before[i] + tiles[i] - 1, src);
      }
    }
    if (b < 0) return false;
    t->b = b;
    in_seq = at - id;
  } else {
    // the last b whose tiles begin at or before id: their first numbers do not decrease, 32 at a time
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      bool at_or_before = false;
      if (b0 + lane < a.batch) {
        int f, l;
        seq_rows(a, b0 + lane, f, l);
        at_or_before = (int64_t)f * group / T + b0 + lane <= id;
      }
      const uint32_t all = __ballot_sync(0xffffffffu, at_or_before);
      before += __popc(all);
      if (all != 0xffffffffu) break;
    }
    if (before == 0) return false;
    t->b = before - 1;
    int f, l;
    seq_rows(a, t->b, f, l);
    in_seq = id - (int)((int64_t)f * group / T + t->b);
  }
  int last;
  seq_rows(a, t->b, t->first, last);
  t->n = last - t->first;
  t->first_row = in_seq * T;
  t->rows = min(T, t->n * group - t->first_row);
  if (t->rows <= 0 || in_seq < 0) return false;   // (below zero only where row_start decreases)
  const int64_t most = (int64_t)a.max_pages * a.page_size;
  t->len = (int)max((int64_t)0, min((int64_t)table_at(a.kv_len, t->b), most));
  return true;
}

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) {   // 2 ulp; 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Bytes `sel` of w (each xored with 0x80 beforehand: v + 128) as two fp16 numbers: 0x6400 is 1024 with a
// last place of 1, so 1024 + 128 + v is exact and so is its difference from 1152.
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t w, uint32_t sel) {
  const uint32_t t = __byte_perm(w, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&t), __floats2half2_rn(1152.0f, 1152.0f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // 2^e, e in -126..127

cudaError_t launch_kv_io(const KvArgs& a, void* k, void* v, int dtype, int64_t ld, bool append, cudaStream_t s);
cudaError_t launch_kv_attention(const KvArgs& a, const AttendArgs& t, int dtype, cudaStream_t s);
// the many-row kernel on tcgen05: kv_attention_tcgen05.cu
cudaError_t launch_kv_attend_many(const KvArgs& a, const AttendArgs& t, int dtype, cudaStream_t s);
// at sdq_init, for its device: the kernels' shared memory and cluster sizes
int kv_attend_few_setup(std::string* why);
int kv_attend_many_setup(std::string* why);

}  // namespace sdq
