// Attention of many new rows over the paged int8 cache, on tcgen05.
//
// One CTA per (128 rows, cache head); a row is a (token, query head) pair, so the heads that share a
// cache head fill one tile together.  20 warps, in warpgroups of their own register counts:
//   warps 0..7   : softmax, one thread per row and half of a block's 128 keys (two threads share a row)
//   warps 8..11  : converters of keys: the cache's int8 pages -> fp16 operand tiles in shared memory
//   warps 12..15 : converters of values, transposed on the way
//   warp 16      : MMA issuer of the scores, S = Q K^T
//   warp 17      : MMA issuer of O += P V, P in tensor memory (written in place over S)
// S is double-buffered in tensor memory, so the softmax of a block overlaps the products of its neighbours.
//
// bf16 and fp16 queries: the two halves of a block's keys are two independent attentions, each with running
// offsets, sums and an O of its own (tensor memory: O 0..127 and 128..255, S / P 256..383 and 384..511; Q in
// shared memory), which meet at the end; the two groups of softmax warps never wait for each other, and one's
// exponentials run beside the other's maxima.  fp32 queries have two fp16 numbers per element of Q and of
// the weights and need shared memory to add O up in (see below): Q lies in tensor memory (hi 0..63, lo
// 64..127), there is one O (128..255), and the two threads of a row agree on every block's maximum.
//
// The cached integers are exact in fp16, so a product takes one MMA for each fp16 number that the other
// factor is made of: one for bf16 and fp16 queries, two (hi + lo, 22 bits) for fp32 ones.  The keys' scales
// enter with the scores and the values' with the weights, w = p * v_scale / 2^ev, where 2^ev bounds the
// sequence's v scales (found in a pass over them: 4 of the 2 (D + 4) bytes of a key).
//
// Softmax in one sweep with a running offset m of each row: p = 2^6 2^(s - m); the offset moves, and O and
// the row's sum are scaled down, only when a block's maximum exceeds it by more than 9 log2 units, so a
// weight stays below 2^15 and inside fp16, whose grid ends at 2^-30 of the weight at the offset and of the
// largest v scale: each key's share is off by 2^-23 of that scale at most, however small its own is.  A larger
// power than 2^6 would move that down and the offset more often, which scales O and costs as much as a
// block's exponentials: fp32, 2 x 1000 rows, 8000 keys, 24 heads: 361 us, 11 % more with 2^8, 29 % with 2^10.  With fp32 queries O is taken out of tensor memory every kDrain blocks and added up in
// shared memory in fp32: the tensor core's accumulator truncates, and over thousands of keys that would be
// the largest error there is (1e-5 of the result at 4k keys).
//
// Bound by: the softmax (a block's 128 x 128 weights take 1024 cycles of the exponential unit and ~1200 of
// issue) with the conversion beside it (~450); the MMAs need 512..1024 per product.  bf16, 3 sequences, 1537
// rows, 16k keys, 32 query heads on 8: 574 us, 174 at the tensor cores' rate; 496 with the conversion left out.
//
// Every mbarrier wait is bounded like the GEMM kernels'.
#include <cooperative_groups.h>

#include "kv_common.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace sdq {
namespace {
using namespace tc;

constexpr int kRowsT = 128;        // rows of a tile
constexpr int kKeys = 128;         // keys of a block
constexpr int kPlane = kKeys * 128 * 2;        // 32 KiB: a block's keys or values in fp16
constexpr int kThreadsT = 640;
// registers of a thread: 640 threads are launched with 96 each; 256 * 136 + 256 * 80 + 128 * 40 = 60416 of 61440
constexpr int kRegsSoftmax = 136, kRegsConvert = 80, kRegsIssue = 40;
constexpr int kDrain = 4;          // blocks between two drains of O (fp32 queries)
constexpr uint32_t kColQhi = 0, kColQlo = 64, kColS = 256;
__host__ __device__ constexpr uint32_t kColO(int planes, int grp) { return planes == 2 ? 128u : 128u * grp; }
constexpr float kShift = 6.0f;     // weights are 2^6 times p
constexpr float kStepUp = 9.0f;    // log2 units by which a block's maximum may exceed the running offset

// Shared memory behind the operand tiles.
struct Book {
  float ks[4][kKeys], vs[4][kKeys];   // scales of the blocks under way
  uint32_t there[4][4];               // which of their keys exist
  uint32_t odd[4][4];                 // which of the v scales are not finite
  int rows[2][4][kKeys];              // pool rows, as the converters of keys and of values looked them up
  float meet[2][2][kRowsT];           // what the two threads of a row tell each other
  float sum[2][kRowsT], off[2][kRowsT];   // sums and offsets of the two halves
  float all_sum[kRowsT], all_off[kRowsT], factor[kRowsT];   // of this block's share of the keys, for the cluster
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pready[2][2], pvdone[2][2], scales[4], qready, lready, ofull, pair[4];
  uint32_t v_top;
  uint32_t tmem;
  int abort;
};
constexpr int kJoinRow = 132;      // floats from row to row of a block's results: 8 rows side by side fill the banks once
static_assert(kRowsT * kJoinRow * 4 <= 4 * kPlane, "the results lie over the operand tiles");
constexpr int kSlack = 1024;       // to bring the dynamic base to a 1024-byte boundary
template <int P>
constexpr int kSmemMany = 4 * kPlane + (P == 2 ? 128 * kRowsT * 4 : kPlane) + (int)sizeof(Book) + kSlack;

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t rest_bits(uint32_t hi, float x, float y) {   // fp16 of what `hi` leaves of x and y
  const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return half2_bits(x - back.x, y - back.y);
}

// Two fp32 numbers to an instruction.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 floats_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// SPLIT: clusters of `blocks` CTAs share a tile's keys; without, `blocks` is 1 and known to the compiler
// (which otherwise spills: 3 to 6 % of the time).
template <int DT, bool SPLIT>
__global__ void __launch_bounds__(kThreadsT, 1) kv_attend_many(const KvArgs a, const AttendArgs t, const int blocks, const int vec_q, const int vec_out) {
  const int ck = SPLIT ? blocks : 1;
  constexpr int P = DT == SDQ_F32 ? 2 : 1;
  constexpr int EPV = Vec<DT>::EPV;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t smem_v = base + 2 * kPlane;
  const uint32_t smem_q = base + 4 * kPlane;                      // 16-bit queries: q as operand tile
  float* drained = reinterpret_cast<float*>(smem + 4 * kPlane);   // fp32 queries: [d][row], O so far
  float* joined = reinterpret_cast<float*>(smem);                 // [row][d], this block's result for its cluster
  Book& bk = *reinterpret_cast<Book*>(smem + 4 * kPlane + (P == 2 ? 128 * kRowsT * 4 : kPlane));
  volatile int* abort_flag = &bk.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLIT ? blockIdx.x % ck : 0, kh = blockIdx.x / ck % a.heads, group = t.heads / a.heads;

  wait_prior_grids();
  Tile tile;
  if (!find_tile(a, group, kRowsT, blockIdx.x / ck / a.heads, &tile)) return;
  const int last_token = (tile.first_row + tile.rows - 1) / group;
  const int last_pos = t.causal ? (int)max((int64_t)-1, (int64_t)table_at(a.kv_len, tile.b) - tile.n + last_token) : INT_MAX;
  const int all_keys = max(0, t.causal ? (last_pos < tile.len ? last_pos + 1 : tile.len) : tile.len);
  // the blocks of a cluster take runs of whole key blocks; below, keys count from this block's first one
  const int per = (int)((((uint32_t)all_keys + kKeys - 1) / kKeys + ck - 1) / ck);
  const int key0 = !SPLIT ? 0 : (int)min((int64_t)all_keys, (int64_t)rank * per * kKeys);
  const int keys = SPLIT ? (int)min((int64_t)(all_keys - key0), (int64_t)per * kKeys) : all_keys;
  const int nblk = (int)(((uint32_t)keys + kKeys - 1) / kKeys);
  auto place = [&](int p) {   // pool row of key p for this cache head, -1: absent
    const int r = p < keys ? pool_row(a, tile.b, key0 + p) : -1;
    return r < 0 ? -1 : r + kh * a.page_size;
  };
  auto bar = [&](const uint64_t& b) { return smem_u32(&b); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(bar(bk.kfull[i]), 4);
      mbar_init(bar(bk.kempty[i]), 1);
      mbar_init(bar(bk.vfull[i]), 4);
      mbar_init(bar(bk.vempty[i]), 1);
      mbar_init(bar(bk.sfull[i]), 1);
      for (int h = 0; h < 2; h++) {
        mbar_init(bar(bk.pready[i][h]), P == 2 ? 8 : 4);
        mbar_init(bar(bk.pvdone[i][h]), 1);
      }
    }
    for (int i = 0; i < 4; i++) {
      mbar_init(bar(bk.scales[i]), 4);
      mbar_init(bar(bk.pair[i]), 2);
    }
    mbar_init(bar(bk.qready), 8);
    mbar_init(bar(bk.lready), 8);
    mbar_init(bar(bk.ofull), 1);
    bk.abort = 0;
    bk.v_top = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(&bk.tmem), 512);
    tmem_relinquish();
  }
  // the largest v scale of the keys
  {
    float top = 0.0f;
    for (int p0 = threadIdx.x; p0 < keys; p0 += 8 * kThreadsT) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int r = place(p0 + i * kThreadsT);
        x[i] = r >= 0 ? fabsf(__ldg(a.v_scale + r)) : 0.0f;
        x[i] = x[i] <= 3.402823466e38f ? x[i] : 0.0f;   // an infinity or NaN says nothing of the others
      }
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, x[i]);
    }
    top = warp_max(top);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (lane == 0) atomicMax(&bk.v_top, __float_as_uint(top));   // positive floats order as integers
    __syncthreads();
  }
  const uint32_t tmem_base = bk.tmem;
  const int ev = min(max((int)(bk.v_top >> 23) - 126, -126), 126);   // v_scale < 2^ev (where it is finite)

  auto key_of = [&](int j) { return j < nblk ? place(j * kKeys + (int)(threadIdx.x & 127)) : -1; };
  if (warp >= 8 && warp < 12) {
    // ---------------------------------------------------------------- converters of keys
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    const int tt = threadIdx.x & 127;
    const int piece = tt & 7, krow = tt >> 3;             // 16 bytes of d, key krow + 16 i
    const bool has_k = piece * 16 < a.D;
    const float unit = pow2f(-ev);
    uint4 kr[8];
    auto load_k = [&](int j) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int row = bk.rows[0][j & 3][krow + 16 * i];
        kr[i] = make_uint4(0, 0, 0, 0);
        if (row >= 0 && has_k) kr[i] = __ldg(reinterpret_cast<const uint4*>(a.k + (int64_t)row * a.D + piece * 16));
      }
    };
    int row_now = key_of(0), row_next = key_of(1);
    bk.rows[0][0][tt] = row_now;
    bk.rows[0][1][tt] = row_next;
    float ks = row_now >= 0 ? __ldg(a.k_scale + row_now) : 0.0f, vs = row_now >= 0 ? __ldg(a.v_scale + row_now) : 0.0f;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (nblk > 0) load_k(0);
    bool ok = true;   // after a wait that gave up the loop only keeps the warps' meetings
    for (int j = 0; j < nblk; j++) {
      const int row_2 = key_of(j + 2);
      const uint32_t slot = j & 1, ph = (j >> 1) & 1;
      ok = ok && mbar_wait_warp(bar(bk.kempty[slot]), ph ^ 1u, abort_flag, t.status, 0xc00 | 1);
      if (ok) {
        const uint32_t st = base + slot * kPlane + (piece >> 2) * 16384;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint32_t x[4] = {kr[i].x ^ 0x80808080u, kr[i].y ^ 0x80808080u, kr[i].z ^ 0x80808080u, kr[i].w ^ 0x80808080u};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            h[2 * e] = bytes_to_half2(x[e], 0x4140);
            h[2 * e + 1] = bytes_to_half2(x[e], 0x4342);
          }
          const int key = krow + 16 * i, c0 = 2 * (piece & 3);
          const uint32_t row = st + key * 128;
          // the second 64 values of d store their odd chunk first: the two halves use other banks
          if (piece < 4) {
            st_shared_v4_b32(row + ((c0 ^ (key & 7)) << 4), h[0], h[1], h[2], h[3]);
            st_shared_v4_b32(row + (((c0 + 1) ^ (key & 7)) << 4), h[4], h[5], h[6], h[7]);
          } else {
            st_shared_v4_b32(row + (((c0 + 1) ^ (key & 7)) << 4), h[4], h[5], h[6], h[7]);
            st_shared_v4_b32(row + ((c0 ^ (key & 7)) << 4), h[0], h[1], h[2], h[3]);
          }
        }
        bk.ks[j & 3][tt] = ks;
        bk.vs[j & 3][tt] = vs * unit;
        const uint32_t there = __ballot_sync(0xffffffffu, row_now >= 0);
        const uint32_t odd = __ballot_sync(0xffffffffu, !(fabsf(vs) <= 3.402823466e38f));
        if (lane == 0) {
          bk.there[j & 3][warp - 8] = there;
          bk.odd[j & 3][warp - 8] = odd;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(bk.kfull[slot]));
          mbar_arrive(bar(bk.scales[j & 3]));
        }
        if (j + 1 < nblk) load_k(j + 1);   // behind the fence, which would wait for it
      }
      row_now = row_next;
      row_next = row_2;
      bk.rows[0][(j + 2) & 3][tt] = row_2;
      ks = row_now >= 0 ? __ldg(a.k_scale + row_now) : 0.0f;
      vs = row_now >= 0 ? __ldg(a.v_scale + row_now) : 0.0f;
      asm volatile("bar.sync 1, 128;" ::: "memory");   // the next rows are there
    }
  } else if (warp >= 12 && warp < 16) {
    // ---------------------------------------------------------------- converters of values
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    const int w = warp - 12, tt = threadIdx.x & 127;
    // 16 values of d of 8 of this warp's 32 keys.  Neighbouring lanes differ in the keys, and those of odd
    // pieces store their words in pairs swapped, so that 8 lanes write to 8 different groups of banks (lanes
    // that differed in d alone would all write to one: 8 times as long, 200 of 880 us).
    const int piece = lane >> 2, kg = lane & 3, odd = piece & 1;
    const bool has_v = piece * 16 < a.D;
    uint4 vr[8];
    auto load_v = [&](int j) {
      const int4* rp = reinterpret_cast<const int4*>(&bk.rows[1][j & 3][w * 32 + kg * 8]);
      const int4 r0 = rp[0], r1 = rp[1];
      const int rows[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        vr[e] = make_uint4(0, 0, 0, 0);
        if (rows[e] >= 0 && has_v) vr[e] = __ldg(reinterpret_cast<const uint4*>(a.v + (int64_t)rows[e] * a.D + piece * 16));
      }
    };
    bk.rows[1][0][tt] = key_of(0);
    bk.rows[1][1][tt] = key_of(1);
    asm volatile("bar.sync 2, 128;" ::: "memory");
    if (nblk > 0) load_v(0);
    bool ok = true;
    for (int j = 0; j < nblk; j++) {
      const int row_2 = key_of(j + 2);
      const uint32_t slot = j & 1, ph = (j >> 1) & 1;
      ok = ok && mbar_wait_warp(bar(bk.vempty[slot]), ph ^ 1u, abort_flag, t.status, 0xc00 | 2);
      if (ok) {
        if (has_v) {
          const uint32_t st = smem_v + slot * kPlane + (w >> 1) * 16384;
          const int chunk = (w & 1) * 4 + kg;
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint32_t h[4][4];   // [value of d][pair of keys]
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              auto word = [&](const uint4& x) {   // q ^ odd of x
                return q < 2 ? ((q ^ odd) ? x.y : x.x) : ((q ^ odd) == 3 ? x.w : x.z);
              };
              const uint32_t u = word(vr[e]), v = word(vr[e + 1]);
              const uint32_t x = __byte_perm(u, v, 0x5140) ^ 0x80808080u, y = __byte_perm(u, v, 0x7362) ^ 0x80808080u;
              h[0][e / 2] = bytes_to_half2(x, 0x4140);
              h[1][e / 2] = bytes_to_half2(x, 0x4342);
              h[2][e / 2] = bytes_to_half2(y, 0x4140);
              h[3][e / 2] = bytes_to_half2(y, 0x4342);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int d = 16 * piece + 4 * (q ^ odd) + i;
              st_shared_v4_b32(st + d * 128 + ((chunk ^ (d & 7)) << 4), h[i][0], h[i][1], h[i][2], h[i][3]);
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(bk.vfull[slot]));
        if (j + 1 < nblk) load_v(j + 1);
      }
      bk.rows[1][(j + 2) & 3][tt] = row_2;
      asm volatile("bar.sync 2, 128;" ::: "memory");
    }
  } else if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == 16 && lane == 0 && nblk > 0) {
      // -------------------------------------------------------------- scores
      constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRowsT >> 4) << 24);
      bool ok = mbar_wait_spin(bar(bk.qready), 0, abort_flag, t.status, 0xc00 | 3);
      for (int j = 0; ok && j < nblk; j++) {
        const uint32_t slot = j & 1, ph = (j >> 1) & 1;
        ok = mbar_wait_spin(bar(bk.kfull[slot]), ph, abort_flag, t.status, 0xc00 | 4);
        if (ok && j >= 2) ok = mbar_wait_spin(bar(bk.pvdone[slot][0]), ph ^ 1u, abort_flag, t.status, 0xc00 | 5);
        if (P == 1 && ok && j >= 2) ok = mbar_wait_spin(bar(bk.pvdone[slot][1]), ph ^ 1u, abort_flag, t.status, 0xc00 | 5);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + kColS + slot * kKeys, st = base + slot * kPlane;
        for (int ks = 0; ks < a.D / 16; ks++) {
          const uint64_t k = make_smem_desc(st + (ks >> 2) * 16384) + (uint64_t)((ks & 3) * 2);
          if constexpr (P == 2) {
            umma_f16_ts(d, tmem_base + kColQlo + ks * 8, k, kIdesc, ks != 0);
            umma_f16_ts(d, tmem_base + kColQhi + ks * 8, k, kIdesc, 1u);
          } else {
            umma_f16_ss(d, make_smem_desc(smem_q + (ks >> 2) * 16384) + (uint64_t)((ks & 3) * 2), k, kIdesc, ks != 0);
          }
        }
        umma_commit(bar(bk.kempty[slot]));
        umma_commit(bar(bk.sfull[slot]));
      }
    }
    if (warp == 17 && lane == 0 && nblk > 0) {
      // -------------------------------------------------------------- P V
      const uint32_t idesc = (1u << 4) | ((uint32_t)(a.D >> 3) << 17) | ((uint32_t)(kRowsT >> 4) << 24);
      bool ok = true;
      for (int j = 0; ok && j < nblk; j++) {
        const uint32_t slot = j & 1, ph = (j >> 1) & 1;
        ok = mbar_wait_spin(bar(bk.vfull[slot]), ph, abort_flag, t.status, 0xc00 | 7);
        const bool fresh = P == 2 ? j % kDrain == 0 : j == 0;   // O was taken out (or is new)
        const uint32_t p0 = tmem_base + kColS + slot * kKeys;
        for (int h = 0; ok && h < (P == 2 ? 1 : 2); h++) {
          ok = mbar_wait_spin(bar(bk.pready[slot][h]), ph, abort_flag, t.status, 0xc00 | 6);
          if (!ok) break;
          tc_fence_after();
          const uint32_t o = tmem_base + kColO(P, h);
          constexpr int kSteps = P == 2 ? kKeys / 16 : kKeys / 32;
#pragma unroll
          for (int i = 0; i < kSteps; i++) {
            const int ks = h * kSteps + i;
            const uint64_t v = make_smem_desc(smem_v + slot * kPlane + (ks >> 2) * 16384) + (uint64_t)((ks & 3) * 2);
            // the weights of keys 32 c + 16 i .. lie in 8 columns: hi at 32 c + 8 i, lo 16 further
            const uint32_t p = p0 + (ks >> 1) * 32 + (ks & 1) * 8;
            if constexpr (P == 2) umma_f16_ts(o, p + 16, v, idesc, !(fresh && i == 0));
            umma_f16_ts(o, p, v, idesc, P == 2 || !(fresh && i == 0));
          }
          umma_commit(bar(bk.pvdone[slot][h]));
        }
        if (!ok) break;
        umma_commit(bar(bk.vempty[slot]));
      }
      if (ok) umma_commit(bar(bk.ofull));
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------------------------------------------------------- softmax
    const int quarter = warp & 3, grp = warp >> 2, r = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int rr = tile.first_row + r, token = rr / group, head = kh * group + (rr - token * group);
    const bool live = r < tile.rows;
    const int seen = !live ? 0 : t.causal ? max(0, last_pos - last_token + token + 1 - key0) : INT_MAX;   // keys in front of the row's end
    uint32_t pair_ph = 0;
    bool ok = true;
    auto pair_sync = [&]() {   // this warp and the one with the other half of the same rows
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bk.pair[quarter]));
      const bool done = mbar_wait_warp(bar(bk.pair[quarter]), pair_ph, abort_flag, t.status, 0xc00 | 8);
      pair_ph ^= 1u;
      return done;
    };
    // ---- q: this thread's half of the row, 64 values of d ----
    float factor;
    {
      float q[64];
      float mx = 0.0f;
      const int64_t at = (int64_t)(tile.first + token) * t.ldq + (int64_t)head * a.D + grp * 64;
#pragma unroll
      for (int i = 0; i < 64; i += 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) q[i + e] = 0.0f;
        if (live && grp * 64 + i < a.D) {
          if (vec_q) {
#pragma unroll
            for (int e = 0; e < 8; e += EPV) {
              float y[EPV];
              Vec<DT>::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(t.q) + (at + i + e) * (16 / EPV))), y);
#pragma unroll
              for (int f = 0; f < EPV; f++) q[i + e + f] = y[f];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) q[i + e] = load_src<DT>(t.q, at + i + e);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fold_abs(mx, q[i + e]);
      }
      bk.meet[0][grp][r] = mx;
      ok = pair_sync();
      mx = fmaxf(mx, bk.meet[0][grp ^ 1][r]);
      // largest |q| of the row into [2^14, 2^15); a row with an infinity has no softmax: all NaN
      const bool finite = mx <= 3.402823466e38f;
      const int e = mx > 0.0f && finite ? max(ilogbf(mx) - 14, -126) : 0;
      const float inv = finite ? pow2f(-e) : __uint_as_float(0x7fc00000u);
      factor = fmaxf(pow2f(e) * t.scale * kLog2e, 1.17549435e-38f);   // not zero: -inf times it has to stay -inf
      uint32_t hi[32];
#pragma unroll
      for (int i = 0; i < 32; i++) hi[i] = half2_bits(q[2 * i] * inv, q[2 * i + 1] * inv);
      if constexpr (P == 2) {
        tmem_st_32x32(tmem_base + kColQhi + grp * 32 + lane_base, hi);
        uint32_t lo[32];
#pragma unroll
        for (int i = 0; i < 32; i++) lo[i] = rest_bits(hi[i], q[2 * i] * inv, q[2 * i + 1] * inv);
        tmem_st_32x32(tmem_base + kColQlo + grp * 32 + lane_base, lo);
        tmem_st_wait();
        tc_fence_before();
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
          st_shared_v4_b32(smem_q + grp * 16384 + r * 128 + ((i ^ (r & 7)) << 4), hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
        fence_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bk.qready));
    }
    float m = -INFINITY, e_off = 0.0f, l = 0.0f;
    for (int j = 0; ok && j < nblk; j++) {
      const uint32_t slot = j & 1, ph = (j >> 1) & 1;
      ok = mbar_wait_warp(bar(bk.scales[j & 3]), (j >> 2) & 1, abort_flag, t.status, 0xc00 | 9);
      if (ok) ok = mbar_wait_warp(bar(bk.sfull[slot]), ph, abort_flag, t.status, 0xc00 | 10);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_col = tmem_base + kColS + slot * kKeys + grp * 64 + lane_base;
      uint32_t s[2][32];
      tmem_ld_32x32(s_col, s[0]);
      tmem_ld_32x32(s_col + 32, s[1]);
      tmem_ld_wait();
      const float4* ks = reinterpret_cast<const float4*>(&bk.ks[j & 3][grp * 64]);
      const float4* vs = reinterpret_cast<const float4*>(&bk.vs[j & 3][grp * 64]);
      const int left = seen - (j * kKeys + grp * 64);   // keys of this half that the row sees
      uint32_t sees[2];
#pragma unroll
      for (int h = 0; h < 2; h++)
        sees[h] = bk.there[j & 3][grp * 2 + h] & (left >= 32 * h + 32 ? 0xffffffffu : left <= 32 * h ? 0u : (1u << (left - 32 * h)) - 1);
      const bool all = __all_sync(0xffffffffu, (sees[0] & sees[1]) == 0xffffffffu);
      // One pass with the offset as it stands, while every key is seen and no maximum runs away from it:
      // the maximum is found beside the weights instead of in front of them.
      if constexpr (P == 1) {
        if (all && __all_sync(0xffffffffu, m > -INFINITY)) {
          const uint64_t f2 = pair_of(factor, factor), e2 = pair_of(e_off, e_off);
          const ulonglong2* k2 = reinterpret_cast<const ulonglong2*>(ks);
          const ulonglong2* v2 = reinterpret_cast<const ulonglong2*>(vs);
          float top[4] = {m, m, m, m};
          uint64_t sum[4] = {};
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint64_t x[4], k[4], v[4];
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const ulonglong2 kk = k2[h * 8 + i / 4 + e], vv = v2[h * 8 + i / 4 + e];
                k[2 * e] = kk.x; k[2 * e + 1] = kk.y;
                v[2 * e] = vv.x; v[2 * e + 1] = vv.y;
              }
#pragma unroll
              for (int e = 0; e < 4; e++) {
                x[e] = mul2(pair_of(__uint_as_float(s[h][i + 2 * e]), __uint_as_float(s[h][i + 2 * e + 1])), k[e]);
                const float2 y = floats_of(x[e]);
                top[e] = fmaxf(top[e], fmaxf(y.x, y.y));
              }
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float2 y = floats_of(fma2(x[e], f2, e2));
                x[e] = pair_of(exp2_fast(y.x), exp2_fast(y.y));
              }
#pragma unroll
              for (int e = 0; e < 4; e++) {
                sum[e] = add2(sum[e], x[e]);
                const float2 y = floats_of(mul2(x[e], v[e]));
                w[i / 2 + e] = half2_bits(y.x, y.y);
              }
            }
            tmem_st_32x16(s_col + 32 * h, w);   // over scores that the registers still hold
          }
          const float bm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          if (!__any_sync(0xffffffffu, (bm - m) * factor > kStepUp)) {
            const float2 y = floats_of(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
            l += y.x + y.y;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(bk.pready[slot][grp]));
            continue;
          }
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // independent chains
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 k4 = ks[h * 8 + i / 4];
          const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
          for (int e = 0; e < 4; e++) s[h][i + e] = __float_as_uint(__uint_as_float(s[h][i + e]) * kk[e]);
        }
        if (!all) {
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (!((sees[h] >> i) & 1)) s[h][i] = 0xff800000u;   // -inf
        }
#pragma unroll
        for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(s[h][i]));
      }
      float bm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if constexpr (P == 2) {
        bk.meet[j & 1][grp][r] = bm;    // alternating, so that one meeting a block is enough
        ok = pair_sync();
        if (!ok) break;
        bm = fmaxf(bm, bk.meet[j & 1][grp ^ 1][r]);
      }
      const bool grow = (bm - m) * factor > kStepUp;   // true in the row's first block with a key
      const bool drain = P == 2 && j > 0 && j % kDrain == 0;
      const bool any = __any_sync(0xffffffffu, grow);
      if (any || drain) {
        float f = 1.0f;
        if (grow) {
          f = exp2_fast((m - bm) * factor);
          m = bm;
          e_off = kShift - m * factor;
          l *= f;
        }
        if (j > 0) {
          // O holds the blocks so far: the last P V must be done before O is scaled or taken out (the
          // next one waits for this block's weights)
          ok = mbar_wait_warp(bar(bk.pvdone[(j - 1) & 1][P == 2 ? 0 : grp]), ((j - 1) >> 1) & 1, abort_flag, t.status, 0xc00 | 11);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = P == 2 ? 2 * grp : 0; c < (P == 2 ? 2 * grp + 2 : 4); c++) {
            if (c * 32 >= a.D) break;
            uint32_t o[32];
            tmem_ld_32x32(tmem_base + kColO(P, grp) + c * 32 + lane_base, o);
            tmem_ld_wait();
            if constexpr (P == 2) {
              float* d = drained + c * 32 * kRowsT + r;
              if (drain) {
#pragma unroll
                for (int i = 0; i < 32; i++) d[i * kRowsT] = j == kDrain ? __uint_as_float(o[i]) * f : (d[i * kRowsT] + __uint_as_float(o[i])) * f;
                continue;
              }
              if (j >= kDrain) {
#pragma unroll
                for (int i = 0; i < 32; i++) d[i * kRowsT] *= f;
              }
            }
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_32x32(tmem_base + kColO(P, grp) + c * 32 + lane_base, o);
          }
        }
      }
      float lb[4] = {};   // the block's sum by itself: fewer roundings than one long chain
      // each 32 columns of scores become 16 of fp16 pairs of weights (hi), then 16 of what is left (lo)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t hi[32];
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          const float4 va = vs[h * 8 + i / 4], vb = vs[h * 8 + i / 4 + 1];
          const float vv[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; e++) p[e] = exp2_fast(fmaf(__uint_as_float(s[h][i + e]), factor, e_off));
#pragma unroll
          for (int e = 0; e < 8; e++) {
            lb[e & 3] += p[e];
            p[e] *= vv[e];
          }
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const uint32_t x = half2_bits(p[e], p[e + 1]);
            hi[(i + e) / 2] = x;
            if constexpr (P == 2) hi[16 + (i + e) / 2] = rest_bits(x, p[e], p[e + 1]);
          }
        }
        if constexpr (P == 2) {
          tmem_st_32x32(s_col + 32 * h, hi);
        } else {
          uint32_t h16[16];
#pragma unroll
          for (int i = 0; i < 16; i++) h16[i] = hi[i];
          tmem_st_32x16(s_col + 32 * h, h16);
        }
      }
      l += (lb[0] + lb[1]) + (lb[2] + lb[3]);
      if (!all && (bk.odd[j & 3][grp * 2] | bk.odd[j & 3][grp * 2 + 1]) != 0) {
        // 0 * infinity, which only rows that see the key may have.  Rare, so the weights are taken back for it:
        // a choice at each of them above took 3 to 7 % of all calls.
        tmem_st_wait();
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
          const int left_h = seen - (j * kKeys + grp * 64) - 32 * h;
          const uint32_t sees_h = bk.there[j & 3][grp * 2 + h] & (left_h >= 32 ? 0xffffffffu : left_h <= 0 ? 0u : (1u << left_h) - 1);
          uint32_t w[32];
          tmem_ld_32x32(s_col + 32 * h, w);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const uint32_t keep = ((sees_h >> (2 * i)) & 1 ? 0xffffu : 0u) | ((sees_h >> (2 * i + 1)) & 1 ? 0xffff0000u : 0u);
            w[i] &= keep;
            if constexpr (P == 2) w[16 + i] &= keep;
          }
          tmem_st_32x32(s_col + 32 * h, w);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bk.pready[slot][P == 2 ? 0 : grp]));
    }
    // ---- both halves' sums, then O / l ----
    if (ok) {
      bk.sum[grp][r] = l;
      bk.off[grp][r] = m;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bk.lready));
      ok = mbar_wait_warp(bar(bk.lready), 0, abort_flag, t.status, 0xc00 | 12);
    }
    if (ok && nblk > 0) ok = mbar_wait_warp(bar(bk.ofull), 0, abort_flag, t.status, 0xc00 | 13);
    if (ok) {
      tc_fence_after();
      float f[2] = {1.0f, 1.0f};   // brings the halves to one offset
      const float top = fmaxf(bk.off[0][r], bk.off[1][r]);
      if constexpr (P == 1) {
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (top != -INFINITY) f[h] = exp2_fast((bk.off[h][r] - top) * factor);
      }
      l = bk.sum[0][r] * f[0] + bk.sum[1][r] * f[1];
      const float inv = l != 0.0f ? (1.0f / l) * pow2f(ev) : 0.0f;   // a row that sees no key is zero
      const int64_t at = (int64_t)(tile.first + token) * t.ldo + (int64_t)head * a.D;
      if (SPLIT && grp == 0) {
        bk.all_sum[r] = l;
        bk.all_off[r] = top;
        bk.factor[r] = factor;
      }
#pragma unroll 1
      for (int c = 2 * grp; c < 2 * grp + 2; c++) {
        if (c * 32 >= a.D) break;
        float o[32];
        if (nblk > 0) {
          uint32_t x[32];
          tmem_ld_32x32(tmem_base + kColO(P, 0) + c * 32 + lane_base, x);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i++) o[i] = __uint_as_float(x[i]) * f[0];
          if constexpr (P == 1) {
            tmem_ld_32x32(tmem_base + kColO(P, 1) + c * 32 + lane_base, x);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] += __uint_as_float(x[i]) * f[1];
          }
#pragma unroll
          for (int i = 0; i < 32; i++) {
            if constexpr (P == 2) {
              if (nblk > kDrain) o[i] += drained[(c * 32 + i) * kRowsT + r];
            }
            o[i] = l != 0.0f ? o[i] * inv : 0.0f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++) o[i] = 0.0f;
        }
        if constexpr (SPLIT) {   // over the operand tiles, whose products are done
          float4* dst = reinterpret_cast<float4*>(joined + r * kJoinRow + c * 32);
#pragma unroll
          for (int i = 0; i < 32; i += 4) dst[i / 4] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += EPV) {
            if (c * 32 + i >= a.D) break;
            float y[EPV];
#pragma unroll
            for (int e = 0; e < EPV; e++) y[e] = o[i + e];
            if (vec_out) {
              *reinterpret_cast<uint4*>(static_cast<char*>(t.out) + (at + c * 32 + i) * (16 / EPV)) = Vec<DT>::pack(y);
            } else {
#pragma unroll
              for (int e = 0; e < EPV; e++) store_dst<DT>(t.out, at + c * 32 + i + e, y[e]);
            }
          }
        }
      }
      tc_fence_before();
    }
  }

  // ---- the blocks of a cluster: each has softmax(its keys) V and the sum and offset behind it ----
  if constexpr (SPLIT) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (warp < 8 && !*abort_flag) {
      const int share = kRowsT / ck;   // rows that this block finishes, 16 threads to a row, 8 values of d to a thread
      for (int it = threadIdx.x; it < share * 16; it += 256) {
        const int r = rank * share + (it >> 4), d0 = (it & 15) * 8;
        if (r >= tile.rows || d0 >= a.D) continue;
        const float factor = bk.factor[r];
        float top = -INFINITY, l = 0.0f, o[8] = {};
        for (int k = 0; k < ck; k++) top = fmaxf(top, cluster.map_shared_rank(&bk.all_off[r], k)[0]);
        for (int k = 0; k < ck; k++) {
          const float off = cluster.map_shared_rank(&bk.all_off[r], k)[0];
          const float w = cluster.map_shared_rank(&bk.all_sum[r], k)[0] * (top != -INFINITY ? exp2_fast((off - top) * factor) : 1.0f);
          const float4* src = reinterpret_cast<const float4*>(cluster.map_shared_rank(joined, k) + r * kJoinRow + d0);
          const float4 x = src[0], y = src[1];
          const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          l += w;
#pragma unroll
          for (int e = 0; e < 8; e++) o[e] = fmaf(w, v[e], o[e]);
        }
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;   // a row that sees no key is zero
        const int rr = tile.first_row + r, token = rr / group;
        const int64_t at = (int64_t)(tile.first + token) * t.ldo + (int64_t)(kh * group + (rr - token * group)) * a.D + d0;
#pragma unroll
        for (int i = 0; i < 8; i += EPV) {
          float y[EPV];
#pragma unroll
          for (int e = 0; e < EPV; e++) y[e] = o[i + e] * inv;
          if (vec_out) {
            *reinterpret_cast<uint4*>(static_cast<char*>(t.out) + (at + i) * (16 / EPV)) = Vec<DT>::pack(y);
          } else {
#pragma unroll
            for (int e = 0; e < EPV; e++) store_dst<DT>(t.out, at + i + e, y[e]);
          }
        }
      }
    }
    cluster.sync();   // nobody leaves while its results may be read
  }

  // -------------------------------------------------------------------- common exit
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (*abort_flag) {
    for (int i = 0; i < 1000; i++) __nanosleep(1000);   // let MMAs in flight end (~1 ms)
    __syncthreads();
  }
  if (warp == 16) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int DT>
cudaError_t launch_typed(const KvArgs& a, const AttendArgs& t, cudaStream_t s) {
  constexpr int P = DT == SDQ_F32 ? 2 : 1, size = DT == SDQ_F32 ? 4 : 2;
  const int group = t.heads / a.heads;
  const int64_t tiles = (int64_t)a.rows * group / kRowsT + a.batch;
  const int vec_q = (reinterpret_cast<uintptr_t>(t.q) & 15) == 0 && t.ldq * size % 16 == 0;
  const int vec_out = (reinterpret_cast<uintptr_t>(t.out) & 15) == 0 && t.ldo * size % 16 == 0;
  int ck = 1;
  const int64_t mean = ((int64_t)a.rows * group + a.batch - 1) / a.batch, work = (mean + kRowsT - 1) / kRowsT * a.batch * a.heads;
  const int64_t most = (int64_t)a.max_pages * a.page_size;
  // Clusters share a tile's keys while all of them run at a time (one CTA to an SM), and a CTA has two blocks
  // of keys.  One sequence of 32k keys, 8 heads, 64 rows: 528 us without, 152 with 4, 90 with 8; 256 rows, 16
  // clusters of 8, which do not fit: 160, 140 with 4.
  static const int kFit[3] = {74, 34, 14};
  for (int i = 0; i < 3 && work <= kFit[i] && most >= (int64_t)ck * 2 * 2 * kKeys; i++) ck *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.heads * ck));
  cfg.blockDim = dim3(kThreadsT);
  cfg.dynamicSmemBytes = kSmemMany<P>;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)ck, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = ck > 1 ? 2 : 1;
  return ck > 1 ? cudaLaunchKernelEx(&cfg, kv_attend_many<DT, true>, a, t, ck, vec_q, vec_out)
                : cudaLaunchKernelEx(&cfg, kv_attend_many<DT, false>, a, t, ck, vec_q, vec_out);
}

template <int DT>
cudaError_t allow_smem() {
  constexpr int kSmem = kSmemMany<DT == SDQ_F32 ? 2 : 1>;
  const cudaError_t e = cudaFuncSetAttribute(kv_attend_many<DT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kv_attend_many<DT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
}

}  // namespace

int kv_attend_many_setup(std::string* why) {
  cudaError_t e = allow_smem<SDQ_F32>();
  if (e == cudaSuccess) e = allow_smem<SDQ_BF16>();
  if (e == cudaSuccess) e = allow_smem<SDQ_F16>();
  if (e != cudaSuccess) {
    if (why) *why = std::string("cache attention set-up: ") + cudaGetErrorString(e);
    return SDQ_ERR_CUDA;
  }
  return SDQ_OK;
}

cudaError_t launch_kv_attend_many(const KvArgs& a, const AttendArgs& t, int dtype, cudaStream_t s) {
  if (dtype == SDQ_F32) return launch_typed<SDQ_F32>(a, t, s);
  if (dtype == SDQ_BF16) return launch_typed<SDQ_BF16>(a, t, s);
  return launch_typed<SDQ_F16>(a, t, s);
}

}  // namespace sdq
