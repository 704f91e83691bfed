// Products of few rows with 4-bit weights and group scales.
//
//   w[n,k] = sc[n, k/g] * q[n,k],  q in [-8, 7]
//   y[m,n] = sum_G sc[n,G] * sum_{k in G} a[m,k] q[n,k]   (* a_scale[m] for int8 rows, + bias, GELU)
//
// Layout of an uploaded weight: tiles of 16 rows x 64 columns, 512 bytes each, the tiles of 16 rows
// one after the other along k.  Lane 4 g + c of a warp owns 16 bytes of a tile: word j holds its share
// of columns 16 j .. 16 j + 15, nibbles (0,4) row g columns 2c, 2c+1; (1,5) row g + 8, the same
// columns; (2,6) row g, columns 2c + 8, 2c + 9; (3,7) row g + 8 of those.  A nibble is q + 8; rows and
// columns beyond the matrix hold 8 (zero).  Scales lie as [16-row tile][group][16].
#include "epilogue.cuh"
#include "quant_common.cuh"
#include "sdq_internal.h"

namespace sdq {
namespace {

constexpr int kBlock = 256;

template <int DT>
__device__ __forceinline__ float scale_at(const void* p, int64_t i) { return load_src<DT>(p, i); }

// ---- quantizer: one thread per 8 columns... one warp per (row, group) ----
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

// ---- upload: [N, ceil(K/2)] bytes, low nibble first, into the tiles ----
__global__ void __launch_bounds__(kBlock) w4_layout_kernel(const uint8_t* __restrict__ q, int64_t N, int64_t K,
                                                           int64_t words, uint32_t* __restrict__ out) {
  const int64_t row_bytes = (K + 1) / 2, k_tiles = (K + 63) / 64;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < words; i += (int64_t)gridDim.x * kBlock) {
    const int j = (int)(i & 3), lane = (int)(i >> 2) & 31;
    const int64_t tile = i >> 7, nt = tile / k_tiles, kt = tile - nt * k_tiles;
    uint32_t w = 0;
#pragma unroll
    for (int p = 0; p < 8; p++) {
      const int64_t n = nt * 16 + (lane >> 2) + 8 * (p & 1);
      const int64_t k = kt * 64 + j * 16 + 2 * (lane & 3) + 8 * ((p >> 1) & 1) + (p >> 2);
      uint32_t v = 8;
      if (n < N && k < K) v = (q[n * row_bytes + (k >> 1)] >> (4 * (k & 1))) & 15u;
      w |= v << (4 * p);
    }
    out[i] = w;
  }
}
template <int SIZE>
__global__ void __launch_bounds__(kBlock) w4_scale_layout_kernel(const void* __restrict__ src, int64_t N, int64_t groups,
                                                                 int64_t count, void* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < count; i += (int64_t)gridDim.x * kBlock) {
    const int64_t n = (i >> 4) / groups * 16 + (i & 15), g = (i >> 4) % groups;
    if constexpr (SIZE == 4)
      static_cast<uint32_t*>(out)[i] = n < N ? static_cast<const uint32_t*>(src)[n * groups + g] : 0u;
    else
      static_cast<uint16_t*>(out)[i] = n < N ? static_cast<const uint16_t*>(src)[n * groups + g] : (uint16_t)0;
  }
}

__device__ __forceinline__ float any_scale(const void* p, int64_t i, int dt) {
  return dt == SDQ_F32 ? load_src<SDQ_F32>(p, i) : dt == SDQ_BF16 ? load_src<SDQ_BF16>(p, i) : load_src<SDQ_F16>(p, i);
}
__device__ __forceinline__ float any_act(const void* p, int64_t i, int dt) {
  return dt == SDQ_I8 ? (float)static_cast<const int8_t*>(p)[i] : any_scale(p, i, dt);
}

// One warp per output: lanes along k.
__global__ void __launch_bounds__(kBlock) w4_simple_kernel(const W4Args a) {
  wait_prior_grids();
  const int lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * (kBlock / 32) + (threadIdx.x >> 5);
  if (i >= a.M * a.N) return;
  const int64_t m = i / a.N, n = i - m * a.N;
  const int64_t k_tiles = (a.K + 63) / 64, groups = (a.K + a.group - 1) / a.group;
  const int64_t nt = n >> 4;
  const int r = (int)(n & 15);
  float y = 0.0f;
  for (int64_t k = lane; k < a.K; k += 32) {
    const int kk = (int)(k & 15);
    const int64_t word = ((nt * k_tiles + (k >> 6)) * 32 + (r & 7) * 4 + ((kk & 7) >> 1)) * 4 + ((k >> 4) & 3);
    const int p = (r >> 3) + 2 * (kk >> 3) + 4 * (kk & 1);
    const float q = (float)((int)((a.q[word] >> (4 * p)) & 15u) - 8);
    y = fmaf(any_act(a.x, m * a.ldx + k, a.x_dtype) * q, any_scale(a.scale, (nt * groups + k / a.group) * 16 + r, a.scale_dtype), y);
  }
  for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (lane != 0) return;
  if (a.x_scale) y *= a.x_scale[m];
  if (a.bias) y += a.bias[n];
  if (a.gelu) y = gelu_tanh(y);
  if (a.out_dtype == SDQ_F32) store_dst<SDQ_F32>(a.out, i, y);
  else if (a.out_dtype == SDQ_BF16) store_dst<SDQ_BF16>(a.out, i, y);
  else store_dst<SDQ_F16>(a.out, i, y);
}

template <int DT>
cudaError_t quantize_typed(const void* src, int64_t N, int64_t K, int group, uint8_t* q, void* scale, int scale_dtype,
                           unsigned grid, cudaStream_t s) {
  if (scale_dtype == SDQ_F32) return launch_overlapped(w4_quantize_kernel<DT, SDQ_F32>, dim3(grid), dim3(kBlock), 0, s, src, N, K, group, q, scale);
  if (scale_dtype == SDQ_BF16) return launch_overlapped(w4_quantize_kernel<DT, SDQ_BF16>, dim3(grid), dim3(kBlock), 0, s, src, N, K, group, q, scale);
  return launch_overlapped(w4_quantize_kernel<DT, SDQ_F16>, dim3(grid), dim3(kBlock), 0, s, src, N, K, group, q, scale);
}

}  // namespace

size_t w4_bytes(int64_t N, int64_t K) { return (size_t)((N + 15) / 16) * (size_t)((K + 63) / 64) * 512; }
size_t w4_scale_bytes(int64_t N, int64_t K, int group, int scale_dtype) {
  return (size_t)((N + 15) / 16) * 16 * (size_t)((K + group - 1) / group) * (scale_dtype == SDQ_F32 ? 4 : 2);
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
                             uint32_t* q_out, void* scale_out, cudaStream_t s) {
  const int64_t words = (int64_t)(w4_bytes(N, K) / 4), groups = (K + group - 1) / group;
  const int64_t scales = (N + 15) / 16 * 16 * groups;
  count_launch(2);
  w4_layout_kernel<<<148 * 8, kBlock, 0, s>>>(q, N, K, words, q_out);
  if (scale_dtype == SDQ_F32) w4_scale_layout_kernel<4><<<148 * 2, kBlock, 0, s>>>(scale, N, groups, scales, scale_out);
  else w4_scale_layout_kernel<2><<<148 * 2, kBlock, 0, s>>>(scale, N, groups, scales, scale_out);
  return cudaGetLastError();
}

cudaError_t launch_w4_matmul(const W4Args& a, cudaStream_t s) {
  count_launch();
  return launch_overlapped(w4_simple_kernel, dim3((unsigned)((a.M * a.N + kBlock / 32 - 1) / (kBlock / 32))), dim3(kBlock), 0, s, a);
}

}  // namespace sdq
