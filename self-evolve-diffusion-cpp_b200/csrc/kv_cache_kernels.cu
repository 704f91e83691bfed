// Quantising keys and values as they enter the paged int8 cache, and reading them back.
//
// A row of D values of one token and head becomes D bytes and one fp32 scale: scale = max|x| * (1/127)
// (1 if that is 0), q = clamp(rne(x * (1 / scale)), -127, 127); reading gives q * scale, rounded once
// to the type asked for.
//
// Bound by HBM (a row of 16-bit values: 2 D bytes one way, D + 4 the other); single tokens by latency.
#include "kv_common.cuh"

namespace sdq {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxTokens = 64;  // tokens of a block: as many as give each lane group a row

struct IoArgs {
  void* k;       // [rows, heads, D], `ld` elements from row to row
  void* v;
  int64_t ld;
  int tokens;    // of one block
  int vec;       // the dense rows are 16-byte aligned
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t at, int vec, float (&x)[8]) {
  constexpr int EPV = Vec<DT>::EPV;
  if (vec) {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + at * (16 / EPV));
#pragma unroll
    for (int j = 0; j < 8 / EPV; j++) {
      float y[EPV];
      Vec<DT>::unpack(__ldcs(src + j), y);
#pragma unroll
      for (int e = 0; e < EPV; e++) x[j * EPV + e] = y[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = load_src<DT>(p, at + e);
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, int vec, const float (&x)[8]) {
  constexpr int EPV = Vec<DT>::EPV;
  if (vec) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(p) + at * (16 / EPV));
#pragma unroll
    for (int j = 0; j < 8 / EPV; j++) {
      float y[EPV];
#pragma unroll
      for (int e = 0; e < EPV; e++) y[e] = x[j * EPV + e];
      __stcs(dst + j, Vec<DT>::pack(y));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) store_dst<DT>(p, at + e, x[e]);
  }
}

// Pool row (head 0) of each of the block's tokens.
__device__ __forceinline__ void find_slots(const KvArgs& a, const IoArgs& io, int* slot) {
  if ((int)threadIdx.x < io.tokens) {
    const int64_t row = (int64_t)blockIdx.x * io.tokens + threadIdx.x;
    slot[threadIdx.x] = row < a.rows ? pool_row_of(a, (int)row) : -1;
  }
  __syncthreads();
}

// LPR lanes share a row of D <= 8 * LPR values; a block does all heads of k and v of its tokens.
template <int DT, int LPR>
__global__ void __launch_bounds__(kBlock) kv_append_kernel(const KvArgs a, const IoArgs io) {
  __shared__ int slot[kMaxTokens];
  allow_dependent_launch();
  wait_prior_grids();
  find_slots(a, io, slot);
  const int part = threadIdx.x % LPR;
  const bool mine = part * 8 < a.D;
  const int items = io.tokens * 2 * a.heads;
  for (int i0 = 0; i0 < items; i0 += kBlock / LPR) {   // whole warps go round together
    const int i = i0 + threadIdx.x / LPR;
    const int token = i / (2 * a.heads), rest = i - token * 2 * a.heads;
    const int is_v = rest >= a.heads, head = rest - is_v * a.heads;
    const int s = i < items ? slot[token] : -1;
    float x[8] = {};
    if (s >= 0 && mine) {
      const int64_t row = (int64_t)blockIdx.x * io.tokens + token;
      load8<DT>(is_v ? io.v : io.k, row * io.ld + head * a.D + part * 8, io.vec, x);
    }
    float mx = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) mx = fold_abs(mx, x[e]);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float sc = int8_row_scale(mx);
    const float inv = __fdiv_rn(1.0f, sc);
    if (s >= 0) {
      const int64_t at = (int64_t)s + (int64_t)head * a.page_size;
      if (part == 0) (is_v ? a.v_scale : a.k_scale)[at] = sc;
      if (mine) {
        int q[8];
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = act_round(__fmul_rn(x[e], inv));
        *reinterpret_cast<uint2*>((is_v ? a.v : a.k) + at * a.D + part * 8) =
            make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
      }
    }
  }
}

// The way back.  A row without a place in the table reads as zeros; rows behind the last sequence
// are left as they were.
template <int DT, int LPR>
__global__ void __launch_bounds__(kBlock) kv_read_kernel(const KvArgs a, const IoArgs io) {
  __shared__ int slot[kMaxTokens];
  allow_dependent_launch();
  wait_prior_grids();
  find_slots(a, io, slot);
  const int part = threadIdx.x % LPR;
  if (part * 8 >= a.D) return;
  const int first = __ldg(a.row_start), last = __ldg(a.row_start + a.batch);
  const int items = io.tokens * 2 * a.heads;
  for (int i = threadIdx.x / LPR; i < items; i += kBlock / LPR) {
    const int token = i / (2 * a.heads), rest = i - token * 2 * a.heads;
    const int is_v = rest >= a.heads, head = rest - is_v * a.heads;
    const int64_t row = (int64_t)blockIdx.x * io.tokens + token;
    if (row >= a.rows || row < first || row >= last) continue;
    const int s = slot[token];
    float x[8] = {};
    if (s >= 0) {
      const int64_t at = (int64_t)s + (int64_t)head * a.page_size;
      const float sc = __ldg((is_v ? a.v_scale : a.k_scale) + at);
      const uint2 w = __ldg(reinterpret_cast<const uint2*>((is_v ? a.v : a.k) + at * a.D + part * 8));
#pragma unroll
      for (int e = 0; e < 8; e++)
        x[e] = __fmul_rn((float)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3))), sc);
    }
    store8<DT>(is_v ? io.v : io.k, row * io.ld + head * a.D + part * 8, io.vec, x);
  }
}

template <int DT, int LPR>
cudaError_t launch_io(const KvArgs& a, IoArgs io, bool append, cudaStream_t s) {
  const int lanes = 2 * a.heads * LPR;   // lane groups that one token fills
  io.tokens = lanes >= kBlock ? 1 : kBlock / lanes;
  if (io.tokens > kMaxTokens) io.tokens = kMaxTokens;
  const unsigned grid = (unsigned)(((int64_t)a.rows + io.tokens - 1) / io.tokens);
  return append ? launch_overlapped(kv_append_kernel<DT, LPR>, dim3(grid), dim3(kBlock), 0, s, a, io)
                : launch_overlapped(kv_read_kernel<DT, LPR>, dim3(grid), dim3(kBlock), 0, s, a, io);
}

template <int DT>
cudaError_t launch_typed(const KvArgs& a, const IoArgs& io, bool append, cudaStream_t s) {
  if (a.D <= 16) return launch_io<DT, 2>(a, io, append, s);
  if (a.D <= 32) return launch_io<DT, 4>(a, io, append, s);
  if (a.D <= 64) return launch_io<DT, 8>(a, io, append, s);
  return launch_io<DT, 16>(a, io, append, s);
}

}  // namespace

cudaError_t launch_kv_io(const KvArgs& a, void* k, void* v, int dtype, int64_t ld, bool append, cudaStream_t s) {
  IoArgs io;
  io.k = k; io.v = v; io.ld = ld; io.tokens = 1;
  const int64_t per = dtype == SDQ_F32 ? 4 : 8;
  io.vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 && ld % per == 0;
  count_launch();
  if (dtype == SDQ_F32) return launch_typed<SDQ_F32>(a, io, append, s);
  if (dtype == SDQ_BF16) return launch_typed<SDQ_BF16>(a, io, append, s);
  return launch_typed<SDQ_F16>(a, io, append, s);
}

}  // namespace sdq
