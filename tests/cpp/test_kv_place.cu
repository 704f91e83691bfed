// Host run of the cache's index arithmetic (the functions the kernels use): page division, the
// sequence that owns a row, and the pool row of a position -- good tables and bad ones.  No GPU.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv_common.cuh"

using namespace sdq;

static int failures = 0;
#define CHECK(c)                                               \
  do {                                                         \
    if (!(c)) { failures++; std::printf("FAIL line %d: %s\n", __LINE__, #c); } \
  } while (0)

static KvArgs make(const std::vector<int32_t>& start, const std::vector<int32_t>& len, const std::vector<int32_t>& table,
                   int max_pages, int pages, int heads, int page_size, int rows) {
  return KvArgs{nullptr, nullptr, nullptr, nullptr, start.data(), len.data(), table.data(), PageDiv((uint32_t)page_size),
                pages, heads, page_size, 64, (int32_t)len.size(), max_pages, rows};
}

int main() {
  for (uint32_t d : {1u, 2u, 3u, 7u, 16u, 48u, 64u, 100u, 128u, 1000u, 65537u, 1u << 24}) {
    PageDiv div(d);
    for (uint64_t p = 0; p < 4 * (uint64_t)d && p < 100000; p++) CHECK(div.page((uint32_t)p) == (uint32_t)p / d);
    for (uint32_t p : {0x7fffffffu, 0x7ffffffeu, 0x40000000u, 0xffffffffu / d, 0xffffffffu / d - 1, 0xffffffffu / d + 1})
      CHECK(div.page(p) == p / d);
    std::mt19937 rng(d);
    for (int i = 0; i < 20000; i++) { const uint32_t p = rng() & 0x7fffffffu; CHECK(div.page(p) == p / d); }
  }
  {  // rows of sequences, an empty one among them; rows in front and behind belong to nobody
    const std::vector<int32_t> start = {2, 5, 5, 9}, len = {10, 4, 6}, table = {3, 1, 0, 2, 5, 4};
    const KvArgs a = make(start, len, table, 2, 6, 3, 5, 12);
    const int want[12] = {-1, -1, 0, 0, 0, 2, 2, 2, 2, -1, -1, -1};
    for (int r = 0; r < 12; r++) CHECK(seq_of_row(a, r) == want[r]);
    CHECK(pool_row_of(a, 2) == 1 * 15 + 2);    // position 7 of sequence 0: its second page, offset 2
    CHECK(pool_row_of(a, 4) == 1 * 15 + 4);
    CHECK(pool_row_of(a, 5) == 5 * 15 + 2);    // position 2 of sequence 2
    CHECK(pool_row_of(a, 8) == 4 * 15 + 0);
    CHECK(pool_row_of(a, 0) == -1 && pool_row_of(a, 9) == -1);
    CHECK(pool_row(a, 0, 10) == -1 && pool_row(a, 0, -1) == -1 && pool_row(a, 0, INT32_MAX) == -1);
  }
  {  // more rows than positions, page numbers outside the pool, lengths that are no lengths
    const std::vector<int32_t> start = {0, 4, 8, 12}, len = {2, INT32_MAX, INT32_MIN}, table = {-1, 7, 6, INT32_MIN, 0, 1};
    const KvArgs a = make(start, len, table, 2, 6, 1, 4, 12);
    for (int r = 0; r < 12; r++) CHECK(pool_row_of(a, r) == -1);
    CHECK(pool_row(a, 2, 3) == 3 && pool_row(a, 2, 4) == 4 && pool_row(a, 2, 8) == -1);
    CHECK(pool_row(a, 0, 0) == -1 && pool_row(a, 0, 4) == -1 && pool_row(a, 1, 0) == -1);
  }
  {  // tables that decrease or leave [0, rows]: any answer lies inside
    std::mt19937 rng(5);
    for (int trial = 0; trial < 2000; trial++) {
      const int B = 1 + rng() % 6, rows = 1 + rng() % 30, pages = 1 + rng() % 8, heads = 1 + rng() % 3, ps = 1 + rng() % 9;
      std::vector<int32_t> start(B + 1), len(B), table(B * 3);
      for (auto& x : start) x = (int32_t)(rng() % 60) - 20;
      for (auto& x : len) x = (int32_t)(rng() % 80) - 20;
      for (auto& x : table) x = (int32_t)(rng() % 12) - 2;
      const KvArgs a = make(start, len, table, 3, pages, heads, ps, rows);
      for (int r = 0; r < rows; r++) {
        const int b = seq_of_row(a, r), s = pool_row_of(a, r);
        CHECK(b >= -1 && b < B);
        CHECK(s >= -1 && s < pages * heads * ps - (heads - 1) * ps);
      }
      for (int b = 0; b < B; b++) {
        int f, l;
        seq_rows(a, b, f, l);
        CHECK(0 <= f && f <= l && l <= rows);
      }
    }
  }
  std::printf(failures ? "%d failures\n" : "ok\n", failures);
  return failures ? 1 : 0;
}
