// Products of few rows with 4-bit weights and group scales.
//
//   w[n,k] = sc[n, k/g] * q[n,k],  q in [-8, 7]
//   y[m,n] = sum_G sc[n,G] * sum_{k in G} a[m,k] q[n,k]   (* a_scale[m] for int8 rows, + bias, GELU)
//
// Layout of an uploaded weight: tiles of 16 rows x 128 columns, 1 KB and their scales, the tiles of 16 rows one
// after the other along k.  Lane 4 g + c of a warp owns two pieces of 16 bytes, 512 apart, for 64
// columns each: words 2 i and 2 i + 1 of a piece hold its share of columns 32 i .. 32 i + 31, which is
// columns 8c .. 8c + 7 of rows g and g + 8.  Nibbles (0,4) are row g, columns 8c + 4h, + 1 of word
// 2 i + h; (1,5) row g + 8, the same columns; (2,6) row g, columns 8c + 4h + 2, + 3; (3,7) row g + 8 of
// those.  A nibble is q + 8; rows and columns beyond the matrix hold 8 (zero).  The scales of a tile
// follow its weights, [group][row % 8][row / 8]: a tile is one run of memory.
#include <cooperative_groups.h>

#include <algorithm>

#include "epilogue.cuh"
#include "quant_common.cuh"
#include "sdq_internal.h"

namespace cg = cooperative_groups;

namespace sdq {
namespace {

constexpr int kBlock = 256;

// ---- quantizer: a warp per (row, group) ----
template <int DT, int ST>
__global__ void __launch_bounds__(kBlock) w4_quantize_kernel(const void* __restrict__ src, int64_t N, int64_t K,
                                                             int group, uint8_t* __restrict__ q, void* __restrict__ scale) {
  wait_prior_grids();
  const int lane = threadIdx.x & 31;
  const int64_t groups = (K + group - 1) / group, row_bytes = (K + 1) / 2;
  const int64_t warps = (int64_t)gridDim.x * (kBlock / 32);
  for (int64_t w = (int64_t)blockIdx.x * (kBlock / 32) + (threadIdx.x >> 5); w < N * groups; w += warps) {
    const int64_t n = w / groups, g = w - n * groups;
    const int64_t k0 = g * group;
    const int cols = (int)min((int64_t)group, K - k0);
    float x[4], mx = 0.0f;   // pairs of columns: 2 * lane, 2 * lane + 1, and 64 further
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int c = 64 * (i >> 1) + 2 * lane + (i & 1);
      x[i] = c < cols ? load_src<DT>(src, n * K + k0 + c) : 0.0f;
      mx = fold_abs(mx, x[i]);
    }
    mx = warp_max(mx);
    const float most = ST == SDQ_F16 ? 65504.0f : ST == SDQ_BF16 ? 3.3895313892515355e38f : 3.4028234663852886e38f;
    const float sc = round_to<ST>(fminf(__fdiv_rn(mx, 7.0f), most));
    if (lane == 0) store_dst<ST>(scale, w, sc);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const int c = 32 * i + 2 * lane;
      if (c >= cols) continue;
      int v[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float r = sc > 0.0f ? rintf(__fdiv_rn(x[i + j], sc)) : 0.0f;
        v[j] = (int)fminf(fmaxf(r, -7.0f), 7.0f) + 8;
      }
      q[n * row_bytes + (k0 + c) / 2] = (uint8_t)(v[0] | (v[1] << 4));
    }
  }
}

// Bytes of a tile.
__host__ __device__ constexpr int kTileBytes(int ss, int group) { return 1024 + 128 / group * 16 * ss; }

// ---- upload: [N, ceil(K/2)] bytes, low nibble first, and [N, groups] scales into the tiles ----
// `tile_words` 32-bit words a tile; SIZE bytes a scale.
template <int SIZE>
__global__ void __launch_bounds__(kBlock) w4_layout_kernel(const uint8_t* __restrict__ q, const void* __restrict__ scale, int64_t N,
                                                           int64_t K, int group, int tile_words, int64_t words,
                                                           uint32_t* __restrict__ out) {
  const int64_t row_bytes = (K + 1) / 2, k_tiles = (K + 127) / 128, groups = (K + group - 1) / group;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < words; i += (int64_t)gridDim.x * kBlock) {
    const int64_t tile = i / tile_words, nt = tile / k_tiles, kt = tile - nt * k_tiles;
    const int at = (int)(i - tile * tile_words);
    uint32_t w = 0;
    if (at < 256) {
      const int j = at & 3, lane = (at >> 2) & 31, piece = at >> 7;
#pragma unroll
      for (int p = 0; p < 8; p++) {
        const int64_t n = nt * 16 + (lane >> 2) + 8 * (p & 1);
        const int64_t k = kt * 128 + piece * 64 + (j >> 1) * 32 + 8 * (lane & 3) + 4 * (j & 1) + 2 * ((p >> 1) & 1) + (p >> 2);
        uint32_t v = 8;
        if (n < N && k < K) v = (q[n * row_bytes + (k >> 1)] >> (4 * (k & 1))) & 15u;
        w |= v << (4 * p);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 4 / SIZE; h++) {
        const int e = (at - 256) * (4 / SIZE) + h;   // scale of the tile: [group][row % 8][row / 8]
        const int64_t n = nt * 16 + ((e & 15) >> 1) + 8 * (e & 1), g = kt * (128 / group) + (e >> 4);
        if (n < N && g < groups) {
          if constexpr (SIZE == 4) w = static_cast<const uint32_t*>(scale)[n * groups + g];
          else w |= (uint32_t) static_cast<const uint16_t*>(scale)[n * groups + g] << (16 * h);
        }
      }
    }
    out[i] = w;
  }
}

// ---- products ----
// A warp owns 16 weight rows and streams their tiles; a tile is one 16-byte load of each lane.  The
// nibbles become fp16 (or bf16) integers in registers, which are the A operand of m16n8k16 tensor
// instructions; the activations, 8 rows of x to an instruction, are the B operand.  Sums of 64 columns
// (32 with groups of 32) stay in the accumulators and leave them by one fused multiply-add with the
// group's scale.
//
// Exactness: q is an integer of 4 bits, exact in either 16-bit type.  fp16 and int8 rows enter as fp16
// and bf16 rows as bf16, as they are; fp32 rows as two fp16 numbers (hi + lo, 22 bits) times a power of
// two for each row and tile.  int8 sums are whole numbers below 2^24 and exact.
__device__ __forceinline__ uint32_t lop3_and_or(uint32_t a, uint32_t mask, uint32_t or_) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(or_));   // (a & mask) | or_
  return r;
}
template <bool BF>
__device__ __forceinline__ void nibbles_to_16(uint32_t w, uint32_t (&a)[4]) {
  if constexpr (BF) {
    // 0x4300 is 128 with a last place of 1: 128 + v is exact, and so is the difference from 136
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.0f, 136.0f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t t = lop3_and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t), off);
      a[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  } else {
    // 0x6400 is 1024 with a last place of 1: 1024 + v or 1024 + 16 v, then v - 8 by one exact operation
    const __half2 off = __floats2half2_rn(1032.0f, 1032.0f), sixteenth = __floats2half2_rn(0.0625f, 0.0625f),
                  off16 = __floats2half2_rn(-72.0f, -72.0f);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t t = lop3_and_or(w >> (8 * i), 0x000f000fu, 0x64006400u);
      const uint32_t u = lop3_and_or(w >> (8 * i), 0x00f000f0u, 0x64006400u);
      const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&t), off);
      const __half2 s = __hfma2(*reinterpret_cast<const __half2*>(&u), sixteenth, off16);
      a[2 * i] = *reinterpret_cast<const uint32_t*>(&r);
      a[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&s);
    }
  }
}
template <bool BF, bool FIRST>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
#define SDQ_MMA(TYPE, C0, C1, C2, C3)                                                                              \
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " \
               "{%10,%11,%12,%13};"                                                                                \
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                    \
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(C0), "f"(C1), "f"(C2), "f"(C3))
  if constexpr (BF && FIRST) SDQ_MMA("bf16", 0.0f, 0.0f, 0.0f, 0.0f);
  else if constexpr (BF) SDQ_MMA("bf16", c[0], c[1], c[2], c[3]);
  else if constexpr (FIRST) SDQ_MMA("f16", 0.0f, 0.0f, 0.0f, 0.0f);
  else SDQ_MMA("f16", c[0], c[1], c[2], c[3]);
#undef SDQ_MMA
}
// Asynchronous 16-byte copies into shared memory.
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Scales of rows g and g + 8, stored side by side.
template <int ST>
__device__ __forceinline__ float2 scale_pair(const uint8_t* p) {
  if constexpr (ST == SDQ_F32) {
    return *reinterpret_cast<const float2*>(p);
  } else if constexpr (ST == SDQ_BF16) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(p));
  }
}

// How a launch is cut.  A cluster of `ck` blocks owns `strip` (or one less) 16-row tiles of the weight;
// its blocks split k, `slice` tiles of 128 columns each.  A block keeps its slice of x in shared memory,
// in stages of `stage` tiles where it does not fit, and deals the (row tile, k tile) pairs of a stage out
// to its warps in contiguous runs: every warp streams the same number of weight bytes, without a pause at
// the end of a row tile, and a row tile that crosses warps is summed afterwards.
struct W4Plan {
  int ck, strips_long, strip, slice, stage, slots;
  int x, exp, red, part;   // offsets in shared memory, in bytes
};

constexpr int kWarps = kBlock / 32;
constexpr int kRows = 8;    // rows of x to a block
// Weight tiles that a warp has under way.  Loads into registers do not get that far: the hardware
// counts them in six classes, so a wait for an old one is a wait for younger ones too.
constexpr int kAhead = 4;
constexpr int kBlocksPerSm = 2;
// n values of x from column k on; zeros behind the end of the row.
template <int XT>
__device__ __forceinline__ void x_scalars(const W4Args& a, int64_t row, int k, int n, float* v) {
  for (int j = 0; j < n; j++) {
    float f = 0.0f;
    if (k + j < a.K) {
      if constexpr (XT == SDQ_I8) f = (float)static_cast<const int8_t*>(a.x)[row * a.ldx + k + j];
      else f = load_src<XT>(a.x, row * a.ldx + k + j);
    }
    v[j] = f;
  }
}
__device__ __forceinline__ uint32_t half2_bits(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// x of columns [k0, k0 + 128 tiles) into shared memory as [k32][plane][row][32], 16-bit elements.
template <int XT>
__device__ __forceinline__ void fill_x(const W4Args& a, int m0, int rows, int k0, int tiles, int vec, uint8_t* smem,
                                       float* row_exp) {
  auto floats4 = [&](int r, int k, float (&f)[4]) {
    if (vec) {
      const float4 q = k < a.K ? __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.x) + (m0 + r) * a.ldx + k))
                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      f[0] = q.x; f[1] = q.y; f[2] = q.z; f[3] = q.w;
    } else {
      x_scalars<XT>(a, m0 + r, k, 4, f);
    }
  };
  if constexpr (XT == SDQ_F32) {
    // A warp takes one row of one tile, 4 columns to a lane: its largest finite |x| into [2^14, 2^15), where
    // fp16 holds it, and lo's last place lies 2^-39 below it.
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pairs = rows * tiles;
    const uint32_t by_rows = (65536u + rows - 1) / rows;   // p / rows by a product: right while p * (rows - 1) < 2^16,
                                                           // and no stage has 2^13 pairs (shared memory holds 512 B of each)
    constexpr int U = 7;
    for (int p0 = warp; p0 < pairs; p0 += kWarps * U) {
      float f[U][4];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int p = p0 + u * kWarps, tile = (int)((uint32_t)p * by_rows >> 16);
#pragma unroll
        for (int e = 0; e < 4; e++) f[u][e] = 0.0f;
        if (p < pairs) floats4(p - tile * rows, k0 + tile * 128 + lane * 4, f[u]);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int p = p0 + u * kWarps, tile = (int)((uint32_t)p * by_rows >> 16), r = p - tile * rows;
        if (p >= pairs) break;
        uint32_t mag[4], mx;   // |x| as bits, which order like the numbers; infinities and NaN come last
#pragma unroll
        for (int e = 0; e < 4; e++) mag[e] = __float_as_uint(f[u][e]) & 0x7fffffffu;
        mx = __reduce_max_sync(0xffffffffu, max(max(mag[0], mag[1]), max(mag[2], mag[3])));
        const bool finite = mx < 0x7f800000u;
        if (!finite) {
#pragma unroll
          for (int e = 0; e < 4; e++) mag[e] = mag[e] < 0x7f800000u ? mag[e] : 0u;
          mx = __reduce_max_sync(0xffffffffu, max(max(mag[0], mag[1]), max(mag[2], mag[3])));
        }
        const int e2 = max((int)(mx >> 23) - 127 - 14, -126);   // -126..113
        const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
        if (lane == 0) row_exp[tile * kRows + r] = __uint_as_float((uint32_t)(e2 + 127) << 23);
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float x = f[u][2 * e] * inv, y = f[u][2 * e + 1] * inv;
          hi[e] = half2_bits(x, y);
          float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
          float rx = x - back.x, ry = y - back.y;
          if (!finite) {   // an infinity has no rest
            rx = isinf(back.x) ? 0.0f : rx;
            ry = isinf(back.y) ? 0.0f : ry;
          }
          lo[e] = half2_bits(rx, ry);
        }
        uint2* dst = reinterpret_cast<uint2*>(smem) + ((tile * 4 + (lane >> 3)) * 2 * rows + r) * 8 + (lane & 7);
        dst[0] = make_uint2(hi[0], hi[1]);
        dst[rows * 8] = make_uint2(lo[0], lo[1]);
      }
    }
  } else if constexpr (XT == SDQ_I8) {
    const int nv = tiles * 8;
    uint4* dst = reinterpret_cast<uint4*>(smem);
#pragma unroll 2
    for (int i = threadIdx.x; i < nv * rows; i += kBlock) {
      const int r = i / nv, v = i - r * nv, k = k0 + v * 16;
      float f[16];
      if (vec) {
        const uint4 q = k < a.K ? __ldg(reinterpret_cast<const uint4*>(static_cast<const int8_t*>(a.x) + (m0 + r) * a.ldx + k))
                                : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 16; e++) f[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3)));
      } else {
        x_scalars<XT>(a, m0 + r, k, 16, f);
      }
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = half2_bits(f[2 * e], f[2 * e + 1]);
      const int at = ((v >> 1) * rows + r) * 4 + (v & 1) * 2;
      dst[at] = make_uint4(h[0], h[1], h[2], h[3]);
      dst[at + 1] = make_uint4(h[4], h[5], h[6], h[7]);
    }
  } else {
    const int nv = tiles * 16;
    uint4* dst = reinterpret_cast<uint4*>(smem);
#pragma unroll 4
    for (int i = threadIdx.x; i < nv * rows; i += kBlock) {
      const int r = i / nv, v = i - r * nv, k = k0 + v * 8;
      uint4 q = make_uint4(0, 0, 0, 0);
      const uint16_t* src = static_cast<const uint16_t*>(a.x) + (m0 + r) * a.ldx + k;
      if (vec) {
        if (k < a.K) q = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
        uint32_t w[4] = {};
        for (int e = 0; e < 8; e++)
          if (k + e < a.K) w[e >> 1] |= (uint32_t)src[e] << (16 * (e & 1));
        q = make_uint4(w[0], w[1], w[2], w[3]);
      }
      dst[((v >> 2) * rows + r) * 4 + (v & 3)] = q;
    }
  }
}

// XT, ST: types of the activations and of the scales.
template <int XT, int ST, int GROUP>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm) w4_rows_kernel(const W4Args a, const W4Plan p, const int vec) {
  constexpr bool BF = XT == SDQ_BF16;
  constexpr int P = XT == SDQ_F32 ? 2 : 1;
  constexpr int SS = ST == SDQ_F32 ? 4 : 2, kTile = kTileBytes(SS, GROUP), kScalePieces = (kTile - 1024) / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  float* row_exp = reinterpret_cast<float*>(smem + p.exp);   // fp32 rows: 2^e of every tile and row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % p.ck, strip = blockIdx.x / p.ck;
  // the first strips_long strips have p.strip row tiles, the others one less
  const int strip_rows = strip < p.strips_long ? p.strip : p.strip - 1;
  const int row0 = strip * p.strip - max(0, strip - p.strips_long);
  const int m0 = blockIdx.y * kRows;
  const int rows = (int)min((int64_t)kRows, a.M - m0);
  const int k_tiles = (int)((a.K + 127) / 128);
  const int slice0 = min(k_tiles, rank * p.slice), slice1 = min(k_tiles, slice0 + p.slice);
  float* red = reinterpret_cast<float*>(smem + p.red);     // [warp][slot][row of x][16]
  float* part = reinterpret_cast<float*>(smem + p.part);   // [row tile][row of x][16]
  const int box = rows * 16;
  const uint8_t* ring = smem + warp * (kAhead * kTile);
  const uint32_t to_ring = (uint32_t)__cvta_generic_to_shared(ring);

  allow_dependent_launch();
  bool first = true;
  __shared__ int first_row[kWarps];   // row tile that each warp's run begins in
  const int share = threadIdx.x / box, within = threadIdx.x - share * box, shares = kBlock / box;   // of the sums below
  for (int s0 = slice0; s0 < slice1 || first; s0 += p.stage) {   // once at least: a block without columns adds zeros
    const int tiles = max(0, min(p.stage, slice1 - s0));
    const int run = (strip_rows * tiles + kWarps - 1) / kWarps;
    const int i0 = min(warp * run, strip_rows * tiles), i1 = min(i0 + run, strip_rows * tiles);
    const int r0 = tiles > 0 ? i0 / tiles : 0, t0 = i0 - r0 * tiles;
    // what the next fetch takes: tiles lie behind one another up to the end of the stage's row tile
    const uint8_t* src = reinterpret_cast<const uint8_t*>(a.q) + ((int64_t)(row0 + r0) * k_tiles + s0 + t0) * kTile + lane * 16;
    const int64_t skip = (int64_t)(k_tiles - tiles) * kTile;
    int to_end = tiles - t0, left = i1 - i0;
    auto fetch = [&](uint32_t slot) {
      if (left > 0) {
        left--;
        const uint32_t dst = to_ring + slot * kTile + lane * 16;
        copy_async(dst, src);
        copy_async(dst + 512, src + 512);
        if (kScalePieces == 32 || lane < kScalePieces) copy_async(dst + 1024, src + 1024);
        src += kTile;
        if (--to_end == 0) {
          src += skip;
          to_end = tiles;
        }
      }
      copies_commit();   // one group a tile, an empty one behind the last, so that their number tells which have landed
    };
#pragma unroll
    for (int i = 0; i < kAhead; i++) fetch(i);
    if (first) wait_prior_grids();   // the weights are there from the upload on; x, bias and out belong to the stream
    fill_x<XT>(a, m0, rows, s0 * 128, tiles, vec, smem + p.x, row_exp);
    __syncthreads();
    float y[4] = {}, acc[4];
    const float2* exb = reinterpret_cast<const float2*>(row_exp) + t0 * (kRows / 2) + c;   // rows 2 c, 2 c + 1
    // lanes of columns that no row of x fills read the last row: what they compute is never stored
    const uint4* x_lane = reinterpret_cast<const uint4*>(smem + p.x) + min(g, rows - 1) * 4 + c;
    const uint4* xb = x_lane + t0 * (4 * P * 4) * rows;
    int to_store = tiles - t0, slot = 0;
    uint32_t at = 0;
    for (int i = i0; i < i1; i++) {
      copies_wait<kAhead - 1>();
      __syncwarp();   // the scales are other lanes' copies
      const uint8_t* piece = ring + at * kTile;
      const uint4 w0 = *reinterpret_cast<const uint4*>(piece + lane * 16), w1 = *reinterpret_cast<const uint4*>(piece + lane * 16 + 512);
      float2 ex = make_float2(1.0f, 1.0f);
      if constexpr (P == 2) {
        ex = *exb;   // of rows that are none: whatever lies there, for sums that are never stored
        exb += kRows / 2;
      }
      const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {      // 32 columns
        uint4 b[P];
#pragma unroll
        for (int pl = 0; pl < P; pl++) b[pl] = xb[(j * P + pl) * 4 * rows];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t af[4];
          nibbles_to_16<BF>(words[2 * j + h], af);
#pragma unroll
          for (int pl = 0; pl < P; pl++) {
            const uint2 bb = h == 0 ? make_uint2(b[pl].x, b[pl].y) : make_uint2(b[pl].z, b[pl].w);
            if (pl == 0 && h == 0 && (32 * j) % GROUP % 64 == 0) mma16816<BF, true>(acc, af, bb);
            else mma16816<BF, false>(acc, af, bb);
          }
        }
        if ((32 * (j + 1)) % GROUP % 64 == 0) {   // at the end of a group, and after 64 columns of a long one
          const float2 f = scale_pair<ST>(piece + 1024 + (32 * j / GROUP) * (16 * SS) + g * (2 * SS));
          if constexpr (P == 2) {
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] *= e & 1 ? ex.y : ex.x;
          }
          y[0] = fmaf(acc[0], f.x, y[0]);
          y[1] = fmaf(acc[1], f.x, y[1]);
          y[2] = fmaf(acc[2], f.y, y[2]);
          y[3] = fmaf(acc[3], f.y, y[3]);
        }
      }
      xb += (4 * P * 4) * rows;
      __syncwarp();
      fetch(at);   // the words of this slot are used up
      at = at + 1 == kAhead ? 0 : at + 1;
      if (--to_store == 0 || i + 1 == i1) {   // the row tile, or this warp's share of it, is done
        float* dst = red + (warp * p.slots + slot) * box + g;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          if (2 * c + j < rows) {
            dst[(2 * c + j) * 16] = y[j];
            dst[(2 * c + j) * 16 + 8] = y[j + 2];
          }
        }
        y[0] = y[1] = y[2] = y[3] = 0.0f;
        to_store = tiles;
        xb = x_lane;
        exb = reinterpret_cast<const float2*>(row_exp) + c;
        slot++;
      }
    }
    copies_wait<0>();
    if (lane == 0) first_row[warp] = r0;
    __syncthreads();
    // ---- the block's sums: row tile r lies in the warps whose runs touch [r, r + 1) * tiles ----
    if (share < shares) {
      for (int r = share; r < strip_rows; r += shares) {
        float s = first ? 0.0f : part[r * box + within];
#pragma unroll
        for (int k = 0; k < kWarps; k++)
          if (k * run < (r + 1) * tiles && (k + 1) * run > r * tiles) s += red[(k * p.slots + r - first_row[k]) * box + within];
        part[r * box + within] = s;
      }
    }
    first = false;
    if (s0 + p.stage < slice1) __syncthreads();   // x and the sums are read before the next stage writes them
  }
  auto finish = [&](int r, float s) {   // element `within` of row tile r
    const int m = within >> 4, i = within;
    const int64_t n = ((int64_t)row0 + r) * 16 + (i & 15);
    if (n >= a.N) return;
    if (XT == SDQ_I8) s *= a.x_scale[m0 + m];
    if (a.bias) s += a.bias[n];
    if (a.gelu) s = gelu_tanh(s);
    const int64_t o = (m0 + m) * a.N + n;
    if (a.out_dtype == SDQ_F32) store_dst<SDQ_F32>(a.out, o, s);
    else if (a.out_dtype == SDQ_BF16) store_dst<SDQ_BF16>(a.out, o, s);
    else store_dst<SDQ_F16>(a.out, o, s);
  };
  if (p.ck == 1) {
    if (share < shares)
      for (int r = share; r < strip_rows; r += shares) finish(r, part[r * box + within]);   // each thread its own sums
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (share < shares) {
      for (int r = rank * shares + share; r < strip_rows; r += shares * p.ck) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = k < p.ck ? cluster.map_shared_rank(part, k)[r * box + within] : 0.0f;
        finish(r, ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
      }
    }
    cluster.sync();   // nobody leaves while its sums may be read
  }
}

constexpr int kSmemMost = 108 * 1024;   // of a block: two of them share an SM

// The cut for clusters of ck blocks in `waves` rounds; false where shared memory does not hold even one
// tile of x beside the rest.
bool w4_cut(int64_t N, int64_t K, int rows, int planes, int ring, int ck, int waves, W4Plan* p, int* smem) {
  const int clusters = ck == 1 ? 296 : ck == 2 ? 148 : ck == 4 ? 71 : 33;   // that run at a time, two blocks to an SM
  const int n_tiles = (int)((N + 15) / 16), k_tiles = (int)((K + 127) / 128);
  const int strips = (int)std::min<int64_t>(n_tiles, (int64_t)clusters * waves);
  p->ck = ck;
  p->strip = (n_tiles + strips - 1) / strips;
  p->strips_long = n_tiles - strips * (p->strip - 1);
  p->slice = (k_tiles + ck - 1) / ck;
  const int tile_bytes = 128 * 2 * planes * rows;
  for (int stages = 1; stages <= p->slice; stages++) {
    p->stage = (p->slice + stages - 1) / stages;
    // a run of ceil(strip * t / warps) pairs, t to a row tile, touches at most (run + t - 2) / t + 1 row
    // tiles, which is no more than strip / warps + 2 for any t
    p->slots = p->strip / kWarps + 2;
    p->x = ring * kWarps;
    p->exp = p->x + p->stage * tile_bytes;
    p->red = p->exp + (planes == 2 ? p->stage * kRows * 4 : 0);
    p->part = p->red + kWarps * p->slots * rows * 64;
    *smem = p->part + p->strip * rows * 64;
    if (*smem <= kSmemMost) return true;
  }
  return false;
}

// The cheapest of the four cluster sizes.  A larger cluster means a shorter slice of x to convert in every
// block and a finer division of the row tiles, and costs a meeting of its blocks.  In clocks, fitted to
// such measurements: 600 for a tile of a warp (1040 with fp32 rows, two products), 10 / 12 / 56 for 256 elements of x (16
// bits / int8 / fp32), 0 / 900 / 1500 / 2000 for the meeting and 8 % for blocks that wait for each other.
// One bf16 row, 4096 x 28672: 16.5 us without clusters, 16.9 / 17.8 / 19.6 with 2 / 4 / 8; 8 fp32 rows,
// 14336 x 5003: 51.9 us without, 33.3 / 24.6 / 22.3 with.
W4Plan w4_plan(const W4Args& a, int rows, int ring, int* smem) {
  const int planes = a.x_dtype == SDQ_F32 ? 2 : 1;
  W4Plan best{};
  double least = 1e300;
  for (int i = 0, ck = 1; i < 4; i++, ck *= 2) {
    W4Plan p;
    int bytes, waves = 1 + (int)(a.N / (16 * 160) * ck / 296);   // no strip of more than 160 tiles fits anyway
    while (!w4_cut(a.N, a.K, rows, planes, ring, ck, waves, &p, &bytes)) waves++;
    static const double kMeet[4] = {0, 900, 1500, 2000};
    const double tiles = (p.strip * p.slice + kWarps - 1) / kWarps * (planes == 2 ? 1040.0 : 600.0);
    const double fill = p.slice * 128.0 * rows / kBlock * (planes == 2 ? 56 : a.x_dtype == SDQ_I8 ? 12 : 10);
    const double cost = waves * ((tiles + fill) * (ck > 1 ? 1.08 : 1.0) + kMeet[i]);
    if (cost < least) { least = cost; best = p; *smem = bytes; }
  }
  return best;
}

template <int XT, int ST, int GROUP>
cudaError_t launch_rows(const W4Args& a, cudaStream_t s) {
  int smem = 0;
  const W4Plan p = w4_plan(a, (int)std::min<int64_t>(a.M, kRows), kAhead * kTileBytes(ST == SDQ_F32 ? 4 : 2, GROUP), &smem);
  const int n_tiles = (int)((a.N + 15) / 16);
  const int strips = p.strips_long + (n_tiles - p.strips_long * p.strip) / std::max(1, p.strip - 1);
  const int size = XT == SDQ_F32 ? 4 : XT == SDQ_I8 ? 1 : 2;
  const int vec = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.ldx * size % 16 == 0 && a.K * size % 16 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(strips * p.ck), (unsigned)((a.M + kRows - 1) / kRows));
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)p.ck, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = p.ck > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, w4_rows_kernel<XT, ST, GROUP>, a, p, vec);
}
template <int XT, int ST, int GROUP>
cudaError_t allow_rows() {
  return cudaFuncSetAttribute(w4_rows_kernel<XT, ST, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
}
template <int XT, int ST>
cudaError_t allow_group() {
  cudaError_t e = allow_rows<XT, ST, 32>();
  if (e == cudaSuccess) e = allow_rows<XT, ST, 64>();
  return e == cudaSuccess ? allow_rows<XT, ST, 128>() : e;
}
template <int XT>
cudaError_t allow_scales() {
  cudaError_t e = allow_group<XT, SDQ_F32>();
  if (e == cudaSuccess) e = allow_group<XT, SDQ_BF16>();
  return e == cudaSuccess ? allow_group<XT, SDQ_F16>() : e;
}
template <int XT, int ST>
cudaError_t launch_group(const W4Args& a, cudaStream_t s) {
  return a.group == 32 ? launch_rows<XT, ST, 32>(a, s) : a.group == 64 ? launch_rows<XT, ST, 64>(a, s) : launch_rows<XT, ST, 128>(a, s);
}
template <int XT>
cudaError_t launch_scales(const W4Args& a, cudaStream_t s) {
  return a.scale_dtype == SDQ_F32    ? launch_group<XT, SDQ_F32>(a, s)
         : a.scale_dtype == SDQ_BF16 ? launch_group<XT, SDQ_BF16>(a, s) : launch_group<XT, SDQ_F16>(a, s);
}

template <int DT>
cudaError_t quantize_typed(const void* src, int64_t N, int64_t K, int group, uint8_t* q, void* scale, int scale_dtype,
                           unsigned grid, cudaStream_t s) {
  if (scale_dtype == SDQ_F32) return launch_overlapped(w4_quantize_kernel<DT, SDQ_F32>, dim3(grid), dim3(kBlock), 0, s, src, N, K, group, q, scale);
  if (scale_dtype == SDQ_BF16) return launch_overlapped(w4_quantize_kernel<DT, SDQ_BF16>, dim3(grid), dim3(kBlock), 0, s, src, N, K, group, q, scale);
  return launch_overlapped(w4_quantize_kernel<DT, SDQ_F16>, dim3(grid), dim3(kBlock), 0, s, src, N, K, group, q, scale);
}

}  // namespace

size_t w4_bytes(int64_t N, int64_t K, int group, int scale_dtype) {
  return (size_t)((N + 15) / 16) * (size_t)((K + 127) / 128) * kTileBytes(scale_dtype == SDQ_F32 ? 4 : 2, group);
}

cudaError_t launch_w4_quantize(const void* src, int src_dtype, int64_t N, int64_t K, int group, uint8_t* q, void* scale,
                               int scale_dtype, cudaStream_t s) {
  const int64_t blocks = (N * ((K + group - 1) / group) + kBlock / 32 - 1) / (kBlock / 32);
  const unsigned grid = (unsigned)(blocks < 148 * 64 ? blocks : 148 * 64);
  count_launch();
  if (src_dtype == SDQ_F32) return quantize_typed<SDQ_F32>(src, N, K, group, q, scale, scale_dtype, grid, s);
  if (src_dtype == SDQ_BF16) return quantize_typed<SDQ_BF16>(src, N, K, group, q, scale, scale_dtype, grid, s);
  return quantize_typed<SDQ_F16>(src, N, K, group, q, scale, scale_dtype, grid, s);
}

cudaError_t launch_w4_layout(const uint8_t* q, const void* scale, int scale_dtype, int64_t N, int64_t K, int group,
                             uint32_t* out, cudaStream_t s) {
  const int64_t words = (int64_t)(w4_bytes(N, K, group, scale_dtype) / 4);
  const int tile_words = kTileBytes(scale_dtype == SDQ_F32 ? 4 : 2, group) / 4;
  const unsigned grid = (unsigned)std::min<int64_t>(148 * 16, (words + kBlock - 1) / kBlock);
  count_launch();
  if (scale_dtype == SDQ_F32) w4_layout_kernel<4><<<grid, kBlock, 0, s>>>(q, scale, N, K, group, tile_words, words, out);
  else w4_layout_kernel<2><<<grid, kBlock, 0, s>>>(q, scale, N, K, group, tile_words, words, out);
  return cudaGetLastError();
}

int w4_setup(std::string* why) {
  cudaError_t e = allow_scales<SDQ_F32>();
  if (e == cudaSuccess) e = allow_scales<SDQ_BF16>();
  if (e == cudaSuccess) e = allow_scales<SDQ_F16>();
  if (e == cudaSuccess) e = allow_scales<SDQ_I8>();
  if (e != cudaSuccess) {
    if (why) *why = std::string("4-bit product set-up: ") + cudaGetErrorString(e);
    return SDQ_ERR_CUDA;
  }
  return SDQ_OK;
}

cudaError_t launch_w4_matmul(const W4Args& a, cudaStream_t s) {
  count_launch();
  switch (a.x_dtype) {
    case SDQ_F32: return launch_scales<SDQ_F32>(a, s);
    case SDQ_BF16: return launch_scales<SDQ_BF16>(a, s);
    case SDQ_F16: return launch_scales<SDQ_F16>(a, s);
    default: return launch_scales<SDQ_I8>(a, s);
  }
}

}  // namespace sdq
