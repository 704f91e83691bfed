// RMS norm with the residual's addition in front and int8 rows behind it, in one pass.
//
//   s = round_T(x + residual)                       (T: the type of the stream; s = x without a residual)
//   r = fp32(1 / sqrt(sum_k s_k^2 / K + eps))       the sum and the root in 64 bits
//   h = (s * r) * weight                            two fp32 roundings (one without a weight)
//   a_scale = max|h| * (1/127) (1 if that is 0),  aq = clamp(rne(h * (1 / a_scale)), -127, 127)
//
// The last line is the activation quantization of the int8 linears but for the scale's last bit (a
// multiplication where that one divides).  The sum is held in
// 64 bits so that r is the correctly rounded value whatever the order of the additions: two kernels,
// two grids or a CPU restatement all get the same r, hence the same bytes.  (The SM's fp64 pipe adds
// one element per lane every other cycle, several times the rate at which HBM delivers them.)
//
// Bound by HBM: x, residual and s once each, one byte per element for aq.
#include "quant_common.cuh"
#include "sdq_internal.h"

namespace sdq {
namespace {

constexpr int kBlock = 256;

// Sum / maximum over the TPR threads that share a row.  `red`: one slot per warp of the block.
template <int TPR>
__device__ __forceinline__ double row_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < TPR / 32 ? red[((threadIdx.x / TPR) * (TPR / 32)) + lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* red) {
  v = warp_max(v);
  if constexpr (TPR > 32) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_max(lane < TPR / 32 ? red[((threadIdx.x / TPR) * (TPR / 32)) + lane] : 0.0f);
  }
  return v;
}

// fp32(1 / sqrt(sum / K + eps)).  Two Newton steps on the fp32 estimate (2^-22 -> 2^-43 -> 2^-86, held to
// 64 bits' 2^-52) give the root as exactly as a division and a square root do, in a tenth of their time.
__device__ __forceinline__ float inv_rms(double sum, double inv_k, float eps) {
  const double x = fma(sum, inv_k, (double)eps);
  if (!(x > 1e-37 && x < 1e37)) return (float)(1.0 / sqrt(x));   // beyond the estimate's range; 0, inf, NaN
  double y = (double)rsqrtf((float)x);
  y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
  y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
  return (float)y;
}

struct NormArgs {
  const void* x;
  const void* residual;   // null: none
  void* sum;              // null without a residual; may be x or residual itself
  const float* weight;    // null: all ones
  int8_t* aq;             // null: only h is wanted
  float* a_scale;
  void* h;                // null: not wanted
  int64_t M, K, ldx, ldr, lds;
  float eps;
};

// A row in the registers of TPR threads, VPT 16-byte vectors each.  Needs K a multiple of the
// vector, 16-byte aligned rows, K <= TPR * VPT vectors.
template <int DT, int TPR, int VPT>
__global__ void __launch_bounds__(TPR > kBlock ? TPR : kBlock) rmsnorm_regs(const NormArgs a) {
  constexpr int EPV = Vec<DT>::EPV;
  constexpr int kWarps = (TPR > kBlock ? TPR : kBlock) / 32;
  constexpr int kRows = TPR > kBlock ? 1 : kBlock / TPR;   // rows of a block
  __shared__ double red_sum[kWarps];
  __shared__ float red_max[kWarps];
  allow_dependent_launch();
  wait_prior_grids();
  const int t = threadIdx.x % TPR;
  const int nv = (int)(a.K / EPV);
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  const bool live = row < a.M;   // rows of a block share its barriers: an idle one goes along
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const char*>(a.x) + row * a.ldx * (16 / EPV));
  float v[VPT][EPV];
  uint4 raw[VPT], res[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int at = t + i * TPR;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (live && at < nv) raw[i] = __ldcs(x + at);
  }
  if (a.residual) {
    const uint4* r = reinterpret_cast<const uint4*>(static_cast<const char*>(a.residual) + row * a.ldr * (16 / EPV));
    uint4* sum = reinterpret_cast<uint4*>(static_cast<char*>(a.sum) + row * a.lds * (16 / EPV));
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int at = t + i * TPR;
      res[i] = make_uint4(0, 0, 0, 0);
      if (live && at < nv) res[i] = __ldcs(r + at);
    }
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int at = t + i * TPR;
      float b[EPV];
      Vec<DT>::unpack(raw[i], v[i]);
      Vec<DT>::unpack(res[i], b);
#pragma unroll
      for (int e = 0; e < EPV; e++) v[i][e] = __fadd_rn(v[i][e], b[e]);
      raw[i] = Vec<DT>::pack(v[i]);
      if (live && at < nv) sum[at] = raw[i];
      Vec<DT>::unpack(raw[i], v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; i++) Vec<DT>::unpack(raw[i], v[i]);
  }
  // with one vector to a thread (few rows) the weights are on their way while the squares are added up
  auto weight4 = [&](int at, int j) { return __ldg(reinterpret_cast<const float4*>(a.weight) + at * (EPV / 4) + j); };
  float4 wt[EPV / 4];
  if (VPT == 1 && a.weight && t < nv) {
#pragma unroll
    for (int j = 0; j < EPV / 4; j++) wt[j] = weight4(t, j);
  }
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < VPT; i++)
#pragma unroll
    for (int e = 0; e < EPV; e++) ss = fma((double)v[i][e], (double)v[i][e], ss);
  const float r = inv_rms(row_sum<TPR>(ss, red_sum), 1.0 / (double)a.K, a.eps);
  float mx = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int at = t + i * TPR;
    if (live && at < nv) {
#pragma unroll
      for (int e = 0; e < EPV; e++) v[i][e] = __fmul_rn(v[i][e], r);
      if (a.weight) {
#pragma unroll
        for (int j = 0; j < EPV / 4; j++) {
          const float4 wj = VPT == 1 ? wt[j] : weight4(at, j);
          v[i][4 * j] = __fmul_rn(v[i][4 * j], wj.x);
          v[i][4 * j + 1] = __fmul_rn(v[i][4 * j + 1], wj.y);
          v[i][4 * j + 2] = __fmul_rn(v[i][4 * j + 2], wj.z);
          v[i][4 * j + 3] = __fmul_rn(v[i][4 * j + 3], wj.w);
        }
      }
#pragma unroll
      for (int e = 0; e < EPV; e++) mx = fold_abs(mx, v[i][e]);
      if (a.h) reinterpret_cast<uint4*>(a.h)[row * nv + at] = Vec<DT>::pack(v[i]);
    }
  }
  if (!a.aq) return;
  mx = row_max<TPR>(mx, red_max);
  const float sc = int8_row_scale(mx);
  if (!live) return;
  if (t == 0) a.a_scale[row] = sc;
  const float inv = __fdiv_rn(1.0f, sc);
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int at = t + i * TPR;
    if (at < nv) {
      uint32_t w[EPV / 4];
#pragma unroll
      for (int j = 0; j < EPV / 4; j++)
        w[j] = pack4(act_round(__fmul_rn(v[i][4 * j], inv)), act_round(__fmul_rn(v[i][4 * j + 1], inv)),
                     act_round(__fmul_rn(v[i][4 * j + 2], inv)), act_round(__fmul_rn(v[i][4 * j + 3], inv)));
      if constexpr (EPV == 8) reinterpret_cast<uint2*>(a.aq)[row * nv + at] = make_uint2(w[0], w[1]);
      else reinterpret_cast<uint32_t*>(a.aq)[row * nv + at] = w[0];
    }
  }
}

// Any K, stride and alignment: three sweeps over the row, the later ones served by L1 / L2.  A
// thread reads back only elements that it wrote itself, so sum may be x or residual.
template <int DT>
__global__ void __launch_bounds__(kBlock) rmsnorm_any(const NormArgs a) {
  constexpr int64_t kSize = DT == SDQ_F32 ? 4 : 2;
  __shared__ double red_sum[kBlock / 32];
  __shared__ float red_max[kBlock / 32];
  allow_dependent_launch();
  wait_prior_grids();
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const void* s = static_cast<const char*>(a.x) + row * a.ldx * kSize;
    double ss = 0.0;
    if (a.residual) {
      const void* res = static_cast<const char*>(a.residual) + row * a.ldr * kSize;
      void* sum = static_cast<char*>(a.sum) + row * a.lds * kSize;
      for (int64_t k = threadIdx.x; k < a.K; k += kBlock) {
        const float v = round_to<DT>(__fadd_rn(load_src<DT>(s, k), load_src<DT>(res, k)));
        store_dst<DT>(sum, k, v);
        ss = fma((double)v, (double)v, ss);
      }
      s = sum;
    } else {
      for (int64_t k = threadIdx.x; k < a.K; k += kBlock) {
        const float v = load_src<DT>(s, k);
        ss = fma((double)v, (double)v, ss);
      }
    }
    const float r = inv_rms(row_sum<kBlock>(ss, red_sum), 1.0 / (double)a.K, a.eps);
    auto value = [&](int64_t k) {
      const float v = __fmul_rn(load_src<DT>(s, k), r);
      return a.weight ? __fmul_rn(v, a.weight[k]) : v;
    };
    float mx = 0.0f;
    for (int64_t k = threadIdx.x; k < a.K; k += kBlock) {
      const float v = value(k);
      mx = fold_abs(mx, v);
      if (a.h) store_dst<DT>(a.h, row * a.K + k, v);
    }
    mx = row_max<kBlock>(mx, red_max);
    if (a.aq) {
      const float sc = int8_row_scale(mx);
      if (threadIdx.x == 0) a.a_scale[row] = sc;
      const float inv = __fdiv_rn(1.0f, sc);
      for (int64_t k = threadIdx.x; k < a.K; k += kBlock)
        a.aq[row * a.K + k] = (int8_t)act_round(__fmul_rn(value(k), inv));
    }
    __syncthreads();  // the next row reuses red_sum / red_max
  }
}

template <int DT, int TPR, int VPT>
cudaError_t launch_regs(const NormArgs& a, cudaStream_t s) {
  constexpr int kRows = TPR > kBlock ? 1 : kBlock / TPR;
  return launch_overlapped(rmsnorm_regs<DT, TPR, VPT>, dim3((unsigned)((a.M + kRows - 1) / kRows)),
                           dim3(TPR > kBlock ? TPR : kBlock), 0, s, a);
}

template <int DT>
cudaError_t launch_typed(const NormArgs& a, cudaStream_t s) {
  constexpr int EPV = Vec<DT>::EPV;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int64_t nv = a.K / EPV;
  bool vec = a.K % EPV == 0 && aligned(a.x) && a.ldx % EPV == 0 && aligned(a.weight) &&
             (reinterpret_cast<uintptr_t>(a.aq) & 7) == 0 && aligned(a.h) && nv <= 4096 && a.M <= 0x7fffffff;
  if (a.residual) vec = vec && aligned(a.residual) && aligned(a.sum) && a.ldr % EPV == 0 && a.lds % EPV == 0;
  if (!vec) {
    const int64_t grid = a.M < 148 * 8 ? a.M : 148 * 8;
    return launch_overlapped(rmsnorm_any<DT>, dim3((unsigned)grid), dim3(kBlock), 0, s, a);
  }
  // Few rows: as many threads to a row as have a vector (latency); many: four vectors to a thread.  bf16 rows of
  // 4096, a vector / four: 1 row 2.1 / 2.9 us, 148 rows 2.3 / 3.4, 296 3.1 / 3.5, 1000 7.8 / 5.7; fp32 rows of
  // 4096: 2.4 / 2.7, 2.5 / 3.0, 3.7 / 3.3, 10.8 / 6.6.
  if (a.M <= 148 && nv > 64) {
    if (nv <= 256) return launch_regs<DT, 256, 1>(a, s);
    if (nv <= 512) return launch_regs<DT, 512, 1>(a, s);
    if (nv <= 1024) return launch_regs<DT, 1024, 1>(a, s);
  }
  if (nv <= 32) return launch_regs<DT, 32, 1>(a, s);
  if (nv <= 64) return launch_regs<DT, 32, 2>(a, s);
  if (nv <= 128) return launch_regs<DT, 32, 4>(a, s);
  if (nv <= 256) return launch_regs<DT, 64, 4>(a, s);
  if (nv <= 512) return launch_regs<DT, 128, 4>(a, s);
  if (nv <= 1024) return launch_regs<DT, 256, 4>(a, s);
  if (nv <= 2048) return launch_regs<DT, 512, 4>(a, s);
  return launch_regs<DT, 1024, 4>(a, s);
}

}  // namespace

cudaError_t launch_rmsnorm_quant(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr, int64_t M,
                                 int64_t K, const float* weight, float eps, void* sum, int64_t lds, int8_t* aq,
                                 float* a_scale, void* h, cudaStream_t s) {
  NormArgs a;
  a.x = x; a.residual = residual; a.sum = sum; a.weight = weight; a.aq = aq; a.a_scale = a_scale; a.h = h;
  a.M = M; a.K = K; a.ldx = ldx; a.ldr = ldr; a.lds = lds; a.eps = eps;
  count_launch();
  if (dtype == SDQ_F32) return launch_typed<SDQ_F32>(a, s);
  if (dtype == SDQ_BF16) return launch_typed<SDQ_BF16>(a, s);
  return launch_typed<SDQ_F16>(a, s);
}

}  // namespace sdq
