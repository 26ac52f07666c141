// The multi-view scan for one new token of each sequence:
//   S <- exp(log_alpha) S + k^T [v | 1], read q S, for each view,
// with the state f32 [batch, heads, views, dk, width] updated in place.
//
// The state's bytes bound it, each read and written once.  A CTA goes over rows
// of one state, which lie back to back: its threads take whole rows side by side
// (a thread keeps its column), so that a step of the CTA is one run of memory
// whatever the width, and the reads need no sums between threads but one at the
// end.  With few sequences the rows of a state are split among the CTAs of a
// cluster, which join their reads through shared memory, in order.
#include "capi_internal.h"
#include "cluster.cuh"

namespace ts {

namespace {

constexpr int kScanStepThreads = 256;
constexpr int kScanStepAhead = 8;   // rows that a thread has on their way

struct ScanStepParams {
  int batch, heads, views, dk, dv, width;
  const void *q, *k, *v;
  long long q_strides[2], k_strides[2], v_strides[2];   // batch, head
  const float* log_alpha[TS_MAX_RETENTIONS];            // null: none
  long long log_alpha_batch[TS_MAX_RETENTIONS];         // elements between sequences (0: one for all)
  float* state;
  void* out;                                            // [views, batch, heads, width]
};

template <bool kBf16>
__device__ __forceinline__ float stream_value(const void* p, long long at) {
  return kBf16 ? bf2f(static_cast<const __nv_bfloat16*>(p)[at]) : static_cast<const float*>(p)[at];
}

template <bool kBf16>
__global__ void __launch_bounds__(kScanStepThreads) scan_step_kernel(const __grid_constant__ ScanStepParams p) {
  __shared__ float q[256], k[256], part[kScanStepThreads], total[256];
  const uint32_t rank = cluster_rank_of(), ranks = cluster_size_of();
  const int unit = blockIdx.x / ranks, view = unit % p.views, h = unit / p.views % p.heads, b = unit / p.views / p.heads;
  const int low = static_cast<int>(p.dk * rank / ranks), high = static_cast<int>(p.dk * (rank + 1) / ranks);
  for (int i = low + threadIdx.x; i < high; i += kScanStepThreads) {
    q[i] = stream_value<kBf16>(p.q, b * p.q_strides[0] + h * p.q_strides[1] + i);
    k[i] = stream_value<kBf16>(p.k, b * p.k_strides[0] + h * p.k_strides[1] + i);
  }
  const int groups = kScanStepThreads / p.width, group = threadIdx.x / p.width, column = threadIdx.x - group * p.width;
  const bool works = group < groups;
  const float* la = view < TS_MAX_RETENTIONS ? p.log_alpha[view] : nullptr;
  const float keep = la ? expf(__ldg(la + b * p.log_alpha_batch[view] + h)) : 1.f;
  const float v = !works ? 0.f : column < p.dv ? stream_value<kBf16>(p.v, b * p.v_strides[0] + h * p.v_strides[1] + column) : 1.f;
  float* state = p.state + static_cast<size_t>(unit) * p.dk * p.width + column;
  __syncthreads();
  float read = 0.f;
  if (works) {
    for (int row = low + group; row < high; row += groups * kScanStepAhead) {
      float s[kScanStepAhead];
#pragma unroll
      for (int i = 0; i < kScanStepAhead; ++i) {
        const int r = row + i * groups;
        s[i] = r < high ? __ldcs(state + static_cast<size_t>(r) * p.width) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kScanStepAhead; ++i) {
        const int r = row + i * groups;
        if (r < high) {
          s[i] = fmaf(s[i], keep, k[r] * v);
          read = fmaf(q[r], s[i], read);
          __stcs(state + static_cast<size_t>(r) * p.width, s[i]);
        }
      }
    }
  }
  part[threadIdx.x] = read;
  __syncthreads();
  if (threadIdx.x < p.width) {
    float sum = 0.f;
    for (int i = 0; i < groups; ++i) sum += part[i * p.width + threadIdx.x];
    total[threadIdx.x] = sum;
  }
  if (ranks > 1) cluster_barrier();
  if (rank == 0 && threadIdx.x < p.width) {
    float sum = total[threadIdx.x];
    for (uint32_t r = 1; r < ranks; ++r) sum += cluster_read(&total[threadIdx.x], r);
    const size_t at = ((static_cast<size_t>(view) * p.batch + b) * p.heads + h) * p.width + threadIdx.x;
    if (kBf16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(sum);
    else static_cast<float*>(p.out)[at] = sum;
  }
  if (ranks > 1) cluster_barrier();   // no CTA leaves while another reads its memory
}

}  // namespace

}  // namespace ts

using namespace ts;

extern "C" int ts_b200_scan_step(const ts_scan_step_args* a, ts_stream_t stream) {
  if (!a) return set_error(TS_ERR_VALUE, "scan_step: null arguments");
  if (a->batch < 1 || a->heads < 1) return set_error(TS_ERR_VALUE, "scan_step: batch and heads must be >= 1");
  if (a->dk < 1 || a->dk > 256) return set_error(TS_ERR_NOT_IMPLEMENTED, "scan_step: key width %d outside 1..256", a->dk);
  if (a->v_append_unit < 0 || a->v_append_unit > 1) return set_error(TS_ERR_VALUE, "scan_step: v_append_unit must be 0 or 1");
  if (a->dv < 1 + a->v_append_unit || a->dv > 256)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "scan_step: payload width %d outside 1..256", a->dv);
  if (a->n_retentions < 1 || a->n_retentions > TS_MAX_RETENTIONS)
    return set_error(TS_ERR_VALUE, "scan_step: n_retentions must be in 1..%d", TS_MAX_RETENTIONS);
  if (!a->q || !a->k || !a->v || !a->state || !a->out) return set_error(TS_ERR_VALUE, "scan_step: null tensor");
  if (a->dtype != TS_DTYPE_F32 && a->dtype != TS_DTYPE_BF16)
    return set_error(TS_ERR_VALUE, "scan_step: dtype must be TS_DTYPE_F32 or TS_DTYPE_BF16");
  const long long units = static_cast<long long>(a->batch) * a->heads * a->n_retentions;
  if (units > (1ll << 27)) return set_error(TS_ERR_NOT_IMPLEMENTED, "scan_step: too many heads and sequences");
  ScanStepParams p = {};
  p.batch = a->batch;
  p.heads = a->heads;
  p.views = a->n_retentions;
  p.dk = a->dk;
  p.width = a->dv;
  p.dv = a->dv - a->v_append_unit;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  for (int i = 0; i < 2; ++i) {
    p.q_strides[i] = a->q_strides[i];
    p.k_strides[i] = a->k_strides[i];
    p.v_strides[i] = a->v_strides[i];
  }
  for (int i = 0; i < a->n_retentions; ++i) {
    p.log_alpha[i] = a->log_alpha[i];
    p.log_alpha_batch[i] = a->log_alpha_batch[i];
  }
  p.state = a->state;
  p.out = a->out;
  // CTAs to a state: as many as bring all SMs to work, while each has 16 rows
  int cluster = 1;
  while (cluster < 8 && units * cluster < 592 && p.dk > 16 * cluster) cluster *= 2;
  const dim3 grid(static_cast<unsigned>(units * cluster));
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == TS_DTYPE_BF16
                            ? launch_cluster(scan_step_kernel<true>, grid, kScanStepThreads, 0, s, cluster, p)
                            : launch_cluster(scan_step_kernel<false>, grid, kScanStepThreads, 0, s, cluster, p);
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "scan_step: %s", cudaGetErrorString(e));
  return check_launch("scan_step");
}
