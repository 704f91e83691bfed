// Element loads and the int8 rounding shared by the quantizing kernels.
//
// Every fp32 operation that decides an output bit uses an explicit round-to-nearest intrinsic, so
// that the compiler can neither fuse nor approximate it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstdint>

#include "sdq.h"

namespace sdq {

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// |x| folded into a running max the way std::max(mx, fabs(x)) does: a NaN is skipped.
__device__ __forceinline__ float fold_abs(float mx, float x) { return fmaxf(mx, fabsf(x)); }

// The reference rounds with cvtss2si (src/core/qgemm.cpp:62-69): nearest-even, and
// INT_MIN for NaN or anything outside 32 bits, then clamps to [-127,127].
__device__ __forceinline__ int act_round(float p) {
  int v = (fabsf(p) < 2147483648.0f) ? __float2int_rn(p) : INT_MIN;
  return max(-127, min(127, v));
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 0xff) | ((uint32_t)(b & 0xff) << 8) | ((uint32_t)(c & 0xff) << 16) |
         ((uint32_t)(d & 0xff) << 24);
}

// Programmatic dependent launch: lets the GEMM that follows in the stream (launched with
// the programmatic-serialization attribute) start its prologue -- barrier set-up, tensor
// memory allocation, descriptor prefetch -- while this kernel is still running.  The GEMM
// waits (griddepcontrol.wait) for this whole grid and its writes before it reads anything.
__device__ __forceinline__ void allow_dependent_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The other side, for a kernel launched with the programmatic-serialization attribute: returns once
// every kernel before it in the stream has completed and its writes are visible.
__device__ __forceinline__ void wait_prior_grids() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Scale of a row quantized by the few-bit kernels: max|x| * (1 / 127), and 1 where that is not a
// normal number (a row of zeros, or of values below 2^-119), so that its reciprocal stays finite and
// such a row becomes zeros.
__device__ __forceinline__ float int8_row_scale(float mx) {
  const float sc = __fmul_rn(mx, 1.0f / 127.0f);
  return sc < 1.17549435e-38f ? 1.0f : sc;
}

template <int DT>
__device__ __forceinline__ float load_src(const void* p, int64_t i);
template <>
__device__ __forceinline__ float load_src<SDQ_F32>(const void* p, int64_t i) {
  return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float load_src<SDQ_BF16>(const void* p, int64_t i) {
  // bits << 16, exactly the packer's widening (tools/quantize/pack_sdcpp.py:40-41)
  return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
template <>
__device__ __forceinline__ float load_src<SDQ_F16>(const void* p, int64_t i) {
  return __half2float(static_cast<const __half*>(p)[i]);  // exact widening
}

// One element of type DT, rounded to nearest even.
template <int DT>
__device__ __forceinline__ void store_dst(void* p, int64_t i, float v) {
  if constexpr (DT == SDQ_F32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == SDQ_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
template <int DT>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (DT == SDQ_F32) return v;
  else if constexpr (DT == SDQ_BF16) return __bfloat162float(__float2bfloat16_rn(v));
  else return __half2float(__float2half_rn(v));
}

// One 16-byte vector of a row: 8 bf16 / f16 or 4 fp32 elements.
template <int DT>
struct Vec {
  static constexpr int EPV = DT == SDQ_F32 ? 4 : 8;  // elements per 16-byte vector
  __device__ static void load(const void* row, int idx, float (&v)[EPV]) {
    unpack(__ldcs(reinterpret_cast<const uint4*>(row) + idx), v);
  }
  __device__ static void unpack(uint4 u, float (&v)[EPV]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (DT == SDQ_F32) {
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == SDQ_BF16) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v[2 * i] = __half2float(__ushort_as_half((unsigned short)(w[i] & 0xffffu)));
        v[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
      }
    }
  }
  __device__ static uint4 pack(const float (&v)[EPV]) {  // rounded to nearest even
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (DT == SDQ_F32) {
        w[i] = __float_as_uint(v[i]);
      } else if constexpr (DT == SDQ_BF16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Launch with the programmatic-serialization attribute: the kernel may start while the one before
// it in the stream is still running, and calls wait_prior_grids() before it touches memory that
// kernel may write (or writes memory that kernel may read).
template <typename... Params, typename... Args>
inline cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                                     Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace sdq
