// Attention of new tokens over the paged int8 cache: a warp per (row, head), one key at a time.
//   out = sum_j p_j v_j,  p = softmax(scale * q . k_j),  k_j = k_scale_j * kq_j,  v_j = v_scale_j * vq_j
#include "kv_common.cuh"

namespace sdq {
namespace {

template <int DT>
__global__ void __launch_bounds__(128) kv_attend_rows(const KvArgs a, const AttendArgs t) {
  wait_prior_grids();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int row = (int)(w / t.heads), head = (int)(w % t.heads);
  if (row >= a.rows) return;
  const int b = seq_of_row(a, row);
  if (b < 0) return;
  const int last = __ldg(a.row_start + b + 1), len = __ldg(a.kv_len + b);
  const int pos = len - last + row;
  const int keys = t.causal ? min(len, pos + 1) : len;
  const int kh = head / (t.heads / a.heads);
  float q[4], o[4] = {}, m = -INFINITY, l = 0.0f;
  for (int i = 0; i < 4; i++) {
    const int d = lane + 32 * i;
    q[i] = d < a.D ? load_src<DT>(t.q, (int64_t)row * t.ldq + (int64_t)head * a.D + d) * t.scale : 0.0f;
  }
  for (int j = 0; j < keys; j++) {
    const int s = pool_row(a, b, j);
    if (s < 0) continue;
    const int64_t at = (int64_t)s + (int64_t)kh * a.page_size;
    float dot = 0.0f;
    for (int i = 0; i < 4; i++) {
      const int d = lane + 32 * i;
      if (d < a.D) dot += q[i] * (float)a.k[at * a.D + d];
    }
    for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
    dot *= a.k_scale[at];
    const float mn = fmaxf(m, dot), f = expf(m - mn), p = expf(dot - mn);
    m = mn;
    l = l * f + p;
    for (int i = 0; i < 4; i++) {
      const int d = lane + 32 * i;
      if (d < a.D) o[i] = o[i] * f + p * a.v_scale[at] * (float)a.v[at * a.D + d];
    }
  }
  for (int i = 0; i < 4; i++) {
    const int d = lane + 32 * i;
    if (d < a.D) store_dst<DT>(t.out, (int64_t)row * t.ldo + (int64_t)head * a.D + d, l != 0.0f ? o[i] / l : 0.0f);
  }
}

}  // namespace

cudaError_t launch_kv_attention(const KvArgs& a, const AttendArgs& t, int dtype, cudaStream_t s) {
  const unsigned grid = (unsigned)(((int64_t)a.rows * t.heads + 3) / 4);
  count_launch();
  if (dtype == SDQ_F32) return launch_overlapped(kv_attend_rows<SDQ_F32>, dim3(grid), dim3(128), 0, s, a, t);
  if (dtype == SDQ_BF16) return launch_overlapped(kv_attend_rows<SDQ_BF16>, dim3(grid), dim3(128), 0, s, a, t);
  return launch_overlapped(kv_attend_rows<SDQ_F16>, dim3(grid), dim3(128), 0, s, a, t);
}

}  // namespace sdq
