// Attention of new tokens over the paged int8 cache.
//   out = sum_j p_j v_j / sum_j p_j,   p_j = 2^(s_j - m),   s_j = log2(e) * scale * k_scale_j * (q . kq_j)
//   v_j = v_scale_j * vq_j
//
// The cached integers are exact in fp16, so the tensor cores take them as they are and every rounding
// lies on the other factor: a row of q becomes one fp16 number per element times a power of two (exact
// for bf16 and fp16 queries, 11 bits of the row's largest element at least), or two for fp32 queries (22
// bits); so do the weights p_j * v_scale_j.  A power of two near the largest v_scale seen keeps the
// weights inside fp16's range, however far the scales of a cache lie apart.
#include <cooperative_groups.h>

#include "kv_common.cuh"

namespace cg = cooperative_groups;

namespace sdq {
namespace {

constexpr float kLowest = -1e30f;   // below any score; finite, so that a row without a key has no inf - inf

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit elements, two to a lane, transposed within the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// ---- few rows: a warp streams keys, 32 at a time, for 8 or 16 rows ----
// Bound by HBM (2 (D + 4) bytes a key and cache head against 4 D products for a few rows).  A warp keeps
// kDepth steps of keys under way as asynchronous copies.  Keys and values are the A operands of
// m16n8k16 instructions, 16 keys (or 16 values of d) by 16, and the rows, 8 to an instruction, the other:
// S^T = K Q^T and O^T = V^T P^T, so that a single token's rows do not leave half of an instruction empty,
// and the softmax has 16 x 8 scores to do.  The order of d and of the keys inside an instruction is chosen
// so that a lane's 16-byte reads of k and v hold whole operands.  Warps of a block take steps in turn,
// blocks of a cluster take contiguous pieces of the sequence, and their results meet in (distributed)
// shared memory: one launch, no scratch.
constexpr int kWarps = 4;
constexpr int kBlock = kWarps * 32;
constexpr int kDepth = 3;
constexpr int kStep = 32;   // keys of a step: two halves of 16, whose products do not wait for one another

// NJ: 64 values of d at a time, 1 (D <= 64) or 2.
template <int NJ>
struct Stage {
  static constexpr int kRow = 64 * NJ;              // bytes of a key's or value's row
  static constexpr int kV = kStep * kRow;           // offsets: keys, values, scales of both, mask
  static constexpr int kScale = 2 * kStep * kRow;
  static constexpr int kMask = kScale + 2 * kStep * 4;
  static constexpr int kBytes = kMask + 16;
  // where 16-byte chunk `chunk` of key `key` lies in its row: the xors spread the reads over the banks
  __device__ static __forceinline__ int key_chunk(int key, int chunk) { return NJ == 2 ? chunk ^ ((key & 1) << 2) : chunk; }
  __device__ static __forceinline__ int value_chunk(int key, int chunk) {
    return NJ == 2 ? chunk ^ (key & 6) : chunk ^ ((key >> 1) & 3);
  }
};

// NT: rows in units of 8.
template <int DT, int NJ, int NT>
__global__ void __launch_bounds__(kBlock, 2) kv_attend_few(const KvArgs a, const AttendArgs t, const int ck, const int vec) {
  constexpr int P = DT == SDQ_F32 ? 2 : 1;
  constexpr int DP = 64 * NJ;            // D, filled up
  constexpr int R = 8 * NT;
  constexpr bool kKeepQ = P * NT * NJ <= 2;   // q stays in registers (at most 16 of them)
  using St = Stage<NJ>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) uint16_t qs[P][R][DP + 8];   // fp16
  __shared__ int q_exp[R];
  __shared__ float2 ml[kWarps][R];       // running maximum and sum of every warp
  __shared__ float2 block_ml[R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % ck, kh = blockIdx.x / ck % a.heads;
  const int group = t.heads / a.heads;

  allow_dependent_launch();
  wait_prior_grids();
  Tile tile;
  if (!find_tile(a, group, R, blockIdx.x / ck / a.heads, &tile)) return;   // the same in all blocks of a cluster
  // keys that the tile's last token sees
  const int last_token = (tile.first_row + tile.rows - 1) / group;
  const int last_pos = t.causal ? (int)max((int64_t)-1, (int64_t)table_at(a.kv_len, tile.b) - tile.n + last_token) : INT_MAX;
  const int keys = max(0, t.causal ? (last_pos < tile.len ? last_pos + 1 : tile.len) : tile.len);
  const int steps = (keys + kStep - 1) / kStep;   // no sequence has more than 2^30 places
  const int per = (steps + ck - 1) / ck;
  const int s0 = min(steps, rank * per), s1 = min(steps, s0 + per);

  // ---- the warp's stream: steps s0 + warp, + kWarps, ... ----
  uint8_t* ring = smem + warp * (kDepth * St::kBytes);
  const uint32_t to_ring = (uint32_t)__cvta_generic_to_shared(ring);
  const int chunk = lane % (4 * NJ), key_in = lane / (4 * NJ);   // this lane copies chunk `chunk` of keys key_in + 8 / NJ * i
  const bool copies = chunk * 16 < a.D;
  const bool whole = a.page_size % 16 == 0;   // half a step lies inside one page
  const int lane_src = key_in * a.D + chunk * 16, more = 8 / NJ * a.D;
  const uint32_t to_k = key_in * St::kRow + St::key_chunk(key_in, chunk) * 16;
  const uint32_t to_v0 = St::kV + key_in * St::kRow + St::value_chunk(key_in, chunk) * 16;
  const uint32_t to_v1 = St::kV + (key_in + 8 / NJ) * St::kRow + St::value_chunk(key_in + 8 / NJ, chunk) * 16;
  auto place = [&](int p) {   // pool row of key p for this cache head
    const int r = p < keys ? pool_row(a, tile.b, p) : -1;
    return r < 0 ? -1 : r + kh * a.page_size;
  };
  // Where the next steps lie: with whole halves, lanes 2 i and 2 i + 1 look up the i-th of 16 steps at a
  // time; else every lane its key of one step.
  int rows_ahead = -1, looked_up = 16;
  auto fetch = [&](int s, int slot) {
    if (s < s1) {
      const uint32_t dst = to_ring + slot * St::kBytes;
      uint32_t there = 0;
      if (whole) {
        if (looked_up == 16) {
          const int ahead = s + (lane >> 1) * kWarps;
          rows_ahead = ahead < s1 ? place(ahead * kStep + (lane & 1) * 16) : -1;
          looked_up = 0;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int row = __shfl_sync(0xffffffffu, rows_ahead, 2 * looked_up + h);
          if (row >= 0) {
            const int left = keys - s * kStep - 16 * h;
            there |= (left >= 16 ? 0xffffu : (1u << left) - 1) << (16 * h);
            if (copies) {
              const int64_t at = (int64_t)row * a.D + lane_src;
              const int8_t *ksrc = a.k + at, *vsrc = a.v + at;
#pragma unroll
              for (int i = 0; i < 2 * NJ; i++) {
                // key_in + 8 / NJ * i has key_in's last bit, and its other bits repeat with every second i
                copy_async16(dst + to_k + (16 * h + 8 / NJ * i) * St::kRow, ksrc);
                copy_async16(dst + (i & 1 ? to_v1 - 8 / NJ * St::kRow : to_v0) + (16 * h + 8 / NJ * i) * St::kRow, vsrc);
                ksrc += more;
                vsrc += more;
              }
            }
            const int key = lane & 15;
            copy_async4(dst + St::kScale + (lane < 16 ? 0 : kStep * 4) + (16 * h + key) * 4, (lane < 16 ? a.k_scale : a.v_scale) + row + key);
          }
        }
        looked_up++;
      } else {
        const int row = place(s * kStep + lane);
        there = __ballot_sync(0xffffffffu, row >= 0);
#pragma unroll
        for (int i = 0; i < 4 * NJ; i++) {
          const int key = key_in + 8 / NJ * i;
          const int r = __shfl_sync(0xffffffffu, row, key);
          if (r >= 0 && copies) {
            const int64_t at = (int64_t)r * a.D + chunk * 16;
            copy_async16(dst + key * St::kRow + St::key_chunk(key, chunk) * 16, a.k + at);
            copy_async16(dst + St::kV + key * St::kRow + St::value_chunk(key, chunk) * 16, a.v + at);
          }
        }
        if (row >= 0) {
          copy_async4(dst + St::kScale + lane * 4, a.k_scale + row);
          copy_async4(dst + St::kScale + (kStep + lane) * 4, a.v_scale + row);
        }
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(ring + slot * St::kBytes + St::kMask) = there;
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kDepth; i++) fetch(s0 + warp + i * kWarps, i);

  // ---- q: 16 threads to a row ----
  for (int i16 = threadIdx.x; i16 < 16 * R; i16 += kBlock) {
    const int r = i16 >> 4, part = i16 & 15, d0 = part * 8;
    float x[8] = {};
    if (r < tile.rows && d0 < a.D) {
      const int rr = tile.first_row + r, token = rr / group;
      const int64_t at = (int64_t)(tile.first + token) * t.ldq + (int64_t)(kh * group + rr - token * group) * a.D + d0;
      if (vec) {
        constexpr int EPV = Vec<DT>::EPV;
#pragma unroll
        for (int j = 0; j < 8 / EPV; j++) {
          float y[EPV];
          Vec<DT>::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(t.q) + at * (16 / EPV)) + j), y);
#pragma unroll
          for (int e = 0; e < EPV; e++) x[j * EPV + e] = y[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = load_src<DT>(t.q, at + e);
      }
    }
    float mx = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) mx = fold_abs(mx, x[e]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    // largest |q| of the row into [2^14, 2^15); a row with an infinity has no softmax: all NaN
    const bool finite = mx <= 3.402823466e38f;
    const int e = mx > 0.0f && finite ? max(ilogbf(mx) - 14, -126) : 0;
    if (part == 0) q_exp[r] = e;
    const float inv = finite ? pow2f(-e) : __uint_as_float(0x7fc00000u);
    if (d0 < DP) {
      uint32_t hi[4];
#pragma unroll
      for (int i = 0; i < 4; i++) hi[i] = half2_bits(x[2 * i] * inv, x[2 * i + 1] * inv);
      *reinterpret_cast<uint4*>(&qs[0][r][d0]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (P == 2) {
        uint32_t lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
          lo[i] = half2_bits(x[2 * i] * inv - back.x, x[2 * i + 1] * inv - back.y);
        }
        *reinterpret_cast<uint4*>(&qs[P - 1][r][d0]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  }
  __syncthreads();
  // q as B operands: lane (g, c) holds d = 16 (c + 4 j) + 4 i .. + 3 of row 8 n + g for instruction (j, i)
  auto q_pieces = [&](int p, int n, int j, int h) { return *reinterpret_cast<const uint4*>(&qs[p][n * 8 + g][(c + 4 * j) * 16 + 8 * h]); };
  uint4 q_kept[P][NT][NJ][2];
  if constexpr (kKeepQ) {
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
          for (int h = 0; h < 2; h++) q_kept[p][n][j][h] = q_pieces(p, n, j, h);
  }
  // rows 8 n + 2 c, + 1 of the tile: what turns a product into a score, and the last key they see
  float factor[NT][2];
  int pos[NT][2];
#pragma unroll
  for (int n = 0; n < NT; n++) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = n * 8 + 2 * c + e, rr = tile.first_row + min(r, tile.rows - 1);
      factor[n][e] = pow2f(q_exp[r]) * t.scale * kLog2e;
      pos[n][e] = t.causal ? last_pos - (last_token - rr / group) : INT_MAX;
    }
  }
  const int least_pos = t.causal ? last_pos - (last_token - tile.first_row / group) : INT_MAX;

  float o[4 * NJ][NT][4] = {};
  float m[NT][2], l[NT][2] = {};
#pragma unroll
  for (int n = 0; n < NT; n++) m[n][0] = m[n][1] = kLowest;
  uint32_t v_top = 0;          // bits of the largest v_scale so far; the weights are in units of 2^v_exp
  int v_exp = -126;
  float unit = pow2f(126);
  int slot = 0;
  for (int s = s0 + warp; s < s1; s += kWarps) {
    copies_wait<kDepth - 1>();
    __syncwarp();
    const uint8_t* st = ring + slot * St::kBytes;
    // ---- scores: keys 16 u + g and + 8 by rows 2 c, 2 c + 1 ----
    float sc[2][NT][4] = {};
#pragma unroll
    for (int j = 0; j < NJ; j++) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        uint32_t kw[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int key = 16 * u + 8 * h + g;
          const uint4 w = *reinterpret_cast<const uint4*>(st + key * St::kRow + St::key_chunk(key, c + 4 * j) * 16);
          kw[h][0] = w.x ^ 0x80808080u;
          kw[h][1] = w.y ^ 0x80808080u;
          kw[h][2] = w.z ^ 0x80808080u;
          kw[h][3] = w.w ^ 0x80808080u;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t a0 = bytes_to_half2(kw[0][i], 0x4140), a2 = bytes_to_half2(kw[0][i], 0x4342);
          const uint32_t a1 = bytes_to_half2(kw[1][i], 0x4140), a3 = bytes_to_half2(kw[1][i], 0x4342);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int p = 0; p < P; p++) {
              const uint4 q = kKeepQ ? q_kept[p][n][j][i >> 1] : q_pieces(p, n, j, i >> 1);
              mma_f16(sc[u][n], a0, a1, a2, a3, i & 1 ? q.z : q.x, i & 1 ? q.w : q.y);
            }
        }
      }
    }
    // ---- softmax ----
    const uint32_t there = *reinterpret_cast<const uint32_t*>(st + St::kMask);
    float ks[4], vs[4];   // of keys g + 8 i
    bool ok[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      ok[i] = (there >> (g + 8 * i)) & 1;
      ks[i] = *reinterpret_cast<const float*>(st + St::kScale + (g + 8 * i) * 4);
      vs[i] = *reinterpret_cast<const float*>(st + St::kScale + (kStep + g + 8 * i) * 4);
      if (!ok[i]) vs[i] = 0.0f;
    }
    const int key0 = s * kStep + g;
    const bool all = there == 0xffffffffu && s * kStep + kStep - 1 <= least_pos;
    float mn[NT][2];
    bool higher = false;
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float& x = sc[i >> 1][n][2 * (i & 1) + e];
          x = x * factor[n][e] * ks[i];
        }
      }
      if (!all) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (!ok[i] || key0 + 8 * i > pos[n][e]) sc[i >> 1][n][2 * (i & 1) + e] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = fmaxf(fmaxf(sc[0][n][e], sc[0][n][e + 2]), fmaxf(sc[1][n][e], sc[1][n][e + 2]));
        x = fmaxf(x, m[n][e]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        mn[n][e] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        higher |= mn[n][e] > m[n][e];
      }
    }
    auto mag = [&](int i) { return __float_as_uint(vs[i]) & 0x7fffffffu; };   // positive floats order as integers, infinities and NaN last
    const uint32_t top = max(max(mag(0), mag(1)), max(mag(2), mag(3)));
    bool odd = false;   // a v scale of the step is not finite (the largest finite one says nothing of it)
    if (__any_sync(0xffffffffu, higher || top > v_top)) {   // rescale what has been summed
      float by = 1.0f;
      uint32_t all_top = __reduce_max_sync(0xffffffffu, top);
      odd = all_top >= 0x7f800000u;
      if (odd) {
        uint32_t finite = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) finite = max(finite, mag(i) < 0x7f800000u ? mag(i) : 0u);
        all_top = __reduce_max_sync(0xffffffffu, finite);
      }
      if (all_top > v_top) {
        v_top = all_top;
        const int e = max((int)(v_top >> 23) - 127 - 14, -126);   // the largest scale into [2^14, 2^15)
        by = pow2f(max(v_exp - e, -126));
        v_exp = e;
        unit = pow2f(-e);   // e in -126..114
      }
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          f[e] = exp2_fast(m[n][e] - mn[n][e]);
          l[n][e] *= f[e];
          f[e] *= by;
          m[n][e] = mn[n][e];
        }
#pragma unroll
        for (int i = 0; i < 4 * NJ; i++) {
#pragma unroll
          for (int e = 0; e < 4; e++) o[i][n][e] *= f[e & 1];
        }
      }
    }
    uint32_t pb[2][P][NT][2];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float vu = vs[i] * unit;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float wt[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float p = exp2_fast(sc[i >> 1][n][2 * (i & 1) + e] - m[n][e]);
          l[n][e] += p;
          wt[e] = p * vu;
        }
        const uint32_t hi = half2_bits(wt[0], wt[1]);
        pb[i >> 1][0][n][i & 1] = transpose8(hi);
        if constexpr (P == 2) {
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          pb[i >> 1][P - 1][n][i & 1] = transpose8(half2_bits(wt[0] - back.x, wt[1] - back.y));
        }
      }
    }
    if (odd && !all) {   // 0 * infinity, which only rows that see the key may have
#pragma unroll
      for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const bool here = (there >> (g + 8 * i)) & 1;
          const uint32_t keep = transpose8((here && key0 + 8 * i <= pos[n][0] ? 0xffffu : 0u) | (here && key0 + 8 * i <= pos[n][1] ? 0xffff0000u : 0u));
#pragma unroll
          for (int p = 0; p < P; p++) pb[i >> 1][p][n][i & 1] &= keep;
        }
      }
    }
    // ---- values: a lane reads its keys 16 u + 2 c, + 1, + 8, + 9 at d = 16 g .. (8 g .. with NJ = 1) ----
#pragma unroll
    for (int u = 0; u < 2; u++) {
      uint32_t w[4][2 * NJ];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int key = 16 * u + (i >> 1) * 8 + 2 * c + (i & 1);
        const uint8_t* row = st + St::kV + key * St::kRow;
        if constexpr (NJ == 2) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + St::value_chunk(key, g) * 16);
          w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(row + St::value_chunk(key, g >> 1) * 16 + (g & 1) * 8);
          w[i][0] = x.x; w[i][1] = x.y;
        }
      }
#pragma unroll
      for (int j = 0; j < 2 * NJ; j++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {   // two of a word's four columns: rows g and g + 8 of an instruction
          const uint32_t x = __byte_perm(w[0][j], w[1][j], h ? 0x7362 : 0x5140) ^ 0x80808080u;
          const uint32_t y = __byte_perm(w[2][j], w[3][j], h ? 0x7362 : 0x5140) ^ 0x80808080u;
          const uint32_t a0 = bytes_to_half2(x, 0x4140), a1 = bytes_to_half2(x, 0x4342);
          const uint32_t a2 = bytes_to_half2(y, 0x4140), a3 = bytes_to_half2(y, 0x4342);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int p = 0; p < P; p++) mma_f16(o[j * 2 + h][n], a0, a1, a2, a3, pb[u][p][n][0], pb[u][p][n][1]);
        }
      }
    }
    __syncwarp();
    fetch(s + kDepth * kWarps, slot);
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  }
  copies_wait<0>();

  // ---- the warps' results meet: [warp][row][DP] over the ring ----
  __syncthreads();
  float* box = reinterpret_cast<float*>(smem);
  const float back = pow2f(v_exp);
#pragma unroll
  for (int n = 0; n < NT; n++) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
      const int r = n * 8 + 2 * c + e;
      if (g == 0) ml[warp][r] = make_float2(m[n][e], l[n][e]);
      if (r < tile.rows) {
        // instruction i holds d = 8 NJ g + 2 i, + 1
        float* dst = box + (warp * R + r) * DP + g * 8 * NJ;
#pragma unroll
        for (int i = 0; i < 4 * NJ; i += 2)
          *reinterpret_cast<float4*>(dst + 2 * i) =
              make_float4(o[i][n][e] * back, o[i][n][2 + e] * back, o[i + 1][n][e] * back, o[i + 1][n][2 + e] * back);
      }
    }
  }
  __syncthreads();
  // parts with maxima of their own, relative to the largest (a row of NaN scores has none, but a NaN sum)
  auto store = [&](int r, int d, float v) {
    const int rr = tile.first_row + r, token = rr / group;
    store_dst<DT>(t.out, (int64_t)(tile.first + token) * t.ldo + (int64_t)(kh * group + rr - token * group) * a.D + d, v);
  };
  const int count = tile.rows * DP;
  for (int i = threadIdx.x; i < count; i += kBlock) {
    const int r = i / DP, d = i % DP;
    float top = kLowest, sum = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; w++) top = fmaxf(top, ml[w][r].x);
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
      const float2 x = ml[w][r];
      const float f = exp2_fast(x.x - top);
      sum += x.y * f;
      v += box[(w * R + r) * DP + d] * f;
    }
    if (ck == 1) {
      if (d < a.D) store(r, d, sum != 0.0f ? v / sum : 0.0f);
    } else {
      box[r * DP + d] = v;    // of warp 0: this thread alone reads and writes the element
      if (d == 0) block_ml[r] = make_float2(top, sum);
    }
  }
  if (ck == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = rank * kBlock + threadIdx.x; i < count; i += kBlock * ck) {
    const int r = i / DP, d = i % DP;
    float top = kLowest, sum = 0.0f, v = 0.0f;
    for (int k = 0; k < ck; k++) top = fmaxf(top, cluster.map_shared_rank(block_ml, k)[r].x);
    for (int k = 0; k < ck; k++) {
      const float2 x = cluster.map_shared_rank(block_ml, k)[r];
      const float f = exp2_fast(x.x - top);
      sum += x.y * f;
      v += cluster.map_shared_rank(box, k)[i] * f;
    }
    if (d < a.D) store(r, d, sum != 0.0f ? v / sum : 0.0f);
  }
  cluster.sync();   // nobody leaves while its sums may be read
}

// As many blocks to a sequence and cache head as fill the GPU at two to an SM, and leave a warp a step.
// One sequence of 32k keys, 8 heads: 246 us with 1 block, 68 with 4, 38 with 8, 31 with 16; 64 of 4k: 75 with
// 1, 93 with 2, 121 with 4.
int split_few(const KvArgs& a) {
  int ck = 1;
  const int64_t work = (int64_t)a.batch * a.heads, most = (int64_t)a.max_pages * a.page_size;
  while (ck < 16 && work * ck * 2 <= 296 && most >= (int64_t)ck * 2 * kWarps * kStep) ck *= 2;
  return ck;
}

template <int NJ, int NT>
constexpr int kSmemFew = kWarps * kDepth * Stage<NJ>::kBytes > kWarps * 8 * NT * 64 * NJ * 4 ? kWarps * kDepth * Stage<NJ>::kBytes
                                                                                            : kWarps * 8 * NT * 64 * NJ * 4;
template <int DT, int NJ, int NT>
cudaError_t allow_few() {
  const cudaError_t e = cudaFuncSetAttribute(kv_attend_few<DT, NJ, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemFew<NJ, NT>);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kv_attend_few<DT, NJ, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
template <int DT>
cudaError_t allow_typed() {
  cudaError_t e = allow_few<DT, 1, 1>();
  if (e == cudaSuccess) e = allow_few<DT, 1, 2>();
  if (e == cudaSuccess) e = allow_few<DT, 2, 1>();
  return e == cudaSuccess ? allow_few<DT, 2, 2>() : e;
}

template <int DT, int NJ, int NT>
cudaError_t launch_few(const KvArgs& a, const AttendArgs& t, int vec, cudaStream_t s) {
  const int group = t.heads / a.heads;
  const int64_t tiles = (int64_t)a.rows * group / (8 * NT) + a.batch;   // with numbers that are no tile, see Tile
  const int ck = split_few(a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.heads * ck));
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = kSmemFew<NJ, NT>;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)ck, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = ck > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kv_attend_few<DT, NJ, NT>, a, t, ck, vec);
}
template <int DT>
cudaError_t launch_typed(const KvArgs& a, const AttendArgs& t, cudaStream_t s) {
  const int size = DT == SDQ_F32 ? 4 : 2;
  const int vec = (reinterpret_cast<uintptr_t>(t.q) & 15) == 0 && t.ldq * size % 16 == 0;
  // tiles of 8 rows while the average sequence has no more
  const int group = t.heads / a.heads;
  const bool narrow = (int64_t)a.rows * group <= (int64_t)8 * a.batch;
  if (a.D <= 64) return narrow ? launch_few<DT, 1, 1>(a, t, vec, s) : launch_few<DT, 1, 2>(a, t, vec, s);
  return narrow ? launch_few<DT, 2, 1>(a, t, vec, s) : launch_few<DT, 2, 2>(a, t, vec, s);
}

}  // namespace

int kv_attend_few_setup(std::string* why) {
  cudaError_t e = allow_typed<SDQ_F32>();
  if (e == cudaSuccess) e = allow_typed<SDQ_BF16>();
  if (e == cudaSuccess) e = allow_typed<SDQ_F16>();
  if (e != cudaSuccess) {
    if (why) *why = std::string("cache attention set-up: ") + cudaGetErrorString(e);
    return SDQ_ERR_CUDA;
  }
  return SDQ_OK;
}

cudaError_t launch_kv_attention(const KvArgs& a, const AttendArgs& t, int dtype, cudaStream_t s) {
  count_launch();
  // Tiles of 128 rows on tcgen05 from 33 rows to a sequence (a row: a token and a query head) on the average,
  // once the blocks here would go round more than 1.3 times.  bf16, here / there, us: 64 sequences of 2k keys,
  // 8 heads: 32 rows 131 / 157, 48 rows 176 / 169, 128 rows 432 / 230; one of 32k, 8 heads: 48 rows 79 / 92
  // (384 blocks), 64 rows 115 / 91 (512); one of 32k, 1 head: 128 rows 40 / 81, 256 rows 69 / 82 (256 blocks),
  // 512 rows 112 / 83; one of 2k, 4 heads, the rule's worst: 128 rows 37 / 26 (256 blocks).
  const int64_t mean = ((int64_t)a.rows * (t.heads / a.heads) + a.batch - 1) / a.batch;
  if (mean > 32 && (mean + 15) / 16 * a.batch * a.heads * split_few(a) > 384) return launch_kv_attend_many(a, t, dtype, s);
  if (dtype == SDQ_F32) return launch_typed<SDQ_F32>(a, t, s);
  if (dtype == SDQ_BF16) return launch_typed<SDQ_BF16>(a, t, s);
  return launch_typed<SDQ_F16>(a, t, s);
}

}  // namespace sdq
