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
constexpr int kMaxTokens = 64;
// Rows of D values that a group of lanes has under way, and how many times it goes round.  Appending and
// reading fp32 are carried by the number of warps; reading into 16 bits, a third of the bytes to write, by
// loads under way.  8001 rows of 24 x 64 fp32: append 27.5 us with one, 30.5 with four; read 28.3 and 35.9.
// 100003 rows of 8 x 128 bf16: read 139 us with one, 117 with four (208 with a block for each token).
template <int DT, bool APPEND>
constexpr int kAtOnce = APPEND || DT == SDQ_F32 ? 1 : 4;
template <int DT, bool APPEND>
constexpr int kRounds = kAtOnce<DT, APPEND> == 1 ? 4 : 2;

struct IoArgs {
  void* k;       // [rows, heads, D], `ld` elements from row to row
  void* v;
  int64_t ld;
  PageDiv per_token;   // 2 * heads rows of D values make a token
  int tokens;    // of one block
  int vec;       // the dense rows are 16-byte aligned
};
// The i-th row of D values of a block: its token, whether it is of v, and its head.
struct Item {
  int token, is_v, head;
  __device__ __forceinline__ Item(const KvArgs& a, const IoArgs& io, int i) {
    token = (int)io.per_token.page((uint32_t)i);
    const int rest = i - token * 2 * a.heads;
    is_v = rest >= a.heads;
    head = rest - (is_v ? a.heads : 0);
  }
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
  constexpr int kGroups = kBlock / LPR, U = kAtOnce<DT, true>;
  allow_dependent_launch();
  wait_prior_grids();
  find_slots(a, io, slot);
  const int part = threadIdx.x % LPR;
  const bool mine = part * 8 < a.D;
  const int items = io.tokens * 2 * a.heads;
  for (int i0 = threadIdx.x / LPR; i0 - (int)(threadIdx.x / LPR) < items; i0 += kGroups * U) {   // whole warps go round together
    float x[U][8];
    int64_t at[U];
    bool is_v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * kGroups;
#pragma unroll
      for (int e = 0; e < 8; e++) x[u][e] = 0.0f;
      at[u] = -1;
      if (i < items) {
        const Item it(a, io, i);
        const int s = slot[it.token];
        if (s >= 0) {
          at[u] = (int64_t)s + (int64_t)it.head * a.page_size;
          is_v[u] = it.is_v;
          const int64_t row = (int64_t)blockIdx.x * io.tokens + it.token;
          if (mine) load8<DT>(it.is_v ? io.v : io.k, row * io.ld + it.head * a.D + part * 8, io.vec, x[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      float mx = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) mx = fold_abs(mx, x[u][e]);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float sc = int8_row_scale(mx);
      const float inv = __fdiv_rn(1.0f, sc);
      if (at[u] >= 0) {
        if (part == 0) (is_v[u] ? a.v_scale : a.k_scale)[at[u]] = sc;
        if (mine) {
          int q[8];
#pragma unroll
          for (int e = 0; e < 8; e++) q[e] = act_round(__fmul_rn(x[u][e], inv));
          *reinterpret_cast<uint2*>((is_v[u] ? a.v : a.k) + at[u] * a.D + part * 8) =
              make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        }
      }
    }
  }
}

// The way back.  A row without a place in the table reads as zeros; rows behind the last sequence
// are left as they were.
template <int DT, int LPR>
__global__ void __launch_bounds__(kBlock) kv_read_kernel(const KvArgs a, const IoArgs io) {
  __shared__ int slot[kMaxTokens];
  constexpr int kGroups = kBlock / LPR, U = kAtOnce<DT, false>;
  allow_dependent_launch();
  wait_prior_grids();
  find_slots(a, io, slot);
  const int part = threadIdx.x % LPR;
  if (part * 8 >= a.D) return;
  const int first = __ldg(a.row_start), last = __ldg(a.row_start + a.batch);
  const int items = io.tokens * 2 * a.heads;
  for (int i0 = threadIdx.x / LPR; i0 < items; i0 += kGroups * U) {
    uint2 w[U];
    float sc[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * kGroups;
      w[u] = make_uint2(0, 0);
      sc[u] = 0.0f;
      if (i < items) {
        const Item it(a, io, i);
        const int s = slot[it.token];
        if (s >= 0) {
          const int64_t at = (int64_t)s + (int64_t)it.head * a.page_size;
          sc[u] = __ldg((it.is_v ? a.v_scale : a.k_scale) + at);
          w[u] = __ldcs(reinterpret_cast<const uint2*>((it.is_v ? a.v : a.k) + at * a.D + part * 8));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * kGroups;
      if (i >= items) break;
      const Item it(a, io, i);
      const int64_t row = (int64_t)blockIdx.x * io.tokens + it.token;
      if (row >= a.rows || row < first || row >= last) continue;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = __fmul_rn((float)(int8_t)((e < 4 ? w[u].x : w[u].y) >> (8 * (e & 3))), sc[u]);
      store8<DT>(it.is_v ? io.v : io.k, row * io.ld + it.head * a.D + part * 8, io.vec, x);
    }
  }
}

template <int DT, int LPR>
cudaError_t launch_io(const KvArgs& a, IoArgs io, bool append, cudaStream_t s) {
  // the rounds it takes, but no fewer than four blocks to an SM
  const int rows = (append ? kRounds<DT, true> * kAtOnce<DT, true> : kRounds<DT, false> * kAtOnce<DT, false>) * (kBlock / LPR);
  const int full = (rows + 2 * a.heads - 1) / (2 * a.heads);
  const int spread = a.rows / (148 * 4);
  io.tokens = full < spread ? full : spread;
  if (io.tokens > kMaxTokens) io.tokens = kMaxTokens;
  if (io.tokens < 1) io.tokens = 1;
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
  const int64_t per = dtype == SDQ_F32 ? 4 : 8;
  const IoArgs io{k, v, ld, PageDiv(2u * (uint32_t)a.heads), 1,
                  ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 && ld % per == 0};
  count_launch();
  if (dtype == SDQ_F32) return launch_typed<SDQ_F32>(a, io, append, s);
  if (dtype == SDQ_BF16) return launch_typed<SDQ_BF16>(a, io, append, s);
  return launch_typed<SDQ_F16>(a, io, append, s);
}

}  // namespace sdq
