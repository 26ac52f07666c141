// The multi-view scan for one new token of each sequence:
//   S <- exp(log_alpha) S + k^T [v | 1], read q S, for each view,
// with the state f32 [batch, heads, views, dk, width] updated in place.
//
// The state's bytes bound it, each read and written once.  The rows of a state lie
// back to back, and a CTA goes over them as one run of memory: a thread takes 16
// bytes at a time, whatever the width, and the threads that take part are chosen so
// that a step of them is whole rows.  So a thread's four columns stay the same, and
// the reads need no sums between threads but one at the end.  Widths of 64 and 65
// leave 0 and 28 of 288 threads idle.  Five CTAs to an SM (192 sequences x 16 heads x
// 2 views of 256 x 65: 137 us, 6.0 TB/s; four bytes at a time 208, three CTAs 168).
// With few sequences the rows of a state are split among the CTAs of a cluster,
// which join their reads through shared memory, in order.
#include "capi_internal.h"
#include "cluster.cuh"

namespace ts {

namespace {

constexpr int kScanStepThreads = 288;   // at most

struct ScanStepParams {
  int batch, heads, views, dk, dv, width;
  int active;                                           // threads of a CTA that take part
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

// kVec: elements of the state that a thread takes at once, back to back (4: 16 bytes).
template <bool kBf16, int kVec>
__global__ void __launch_bounds__(kScanStepThreads, 5) scan_step_kernel(const __grid_constant__ ScanStepParams p) {
  constexpr int kAhead = 16 / kVec;   // loads that a thread has on their way
  __shared__ float2 kq[256];
  __shared__ float part[kScanStepThreads * kVec], total[256];
  const uint32_t rank = cluster_rank_of(), ranks = cluster_size_of();
  const int unit = blockIdx.x / ranks, view = unit % p.views, h = unit / p.views % p.heads, b = unit / p.views / p.heads;
  // this CTA's rows, from a multiple of 4 on
  const int rows = (p.dk / static_cast<int>(ranks) + 3) / 4 * 4;
  const int low = min(p.dk, rows * static_cast<int>(rank)), high = rank + 1 == ranks ? p.dk : min(p.dk, low + rows);
  // thread i starts at element kVec * i of the rows and goes on by p.active * kVec elements, which are whole rows
  const int at = kVec * static_cast<int>(threadIdx.x), count = static_cast<int>(threadIdx.x) < p.active ? (high - low) * p.width : 0;
  const int step = p.active * kVec, step_rows = step / p.width;
  float* state = p.state + (static_cast<size_t>(unit) * p.dk + low) * p.width;
  float s[kAhead][kVec];
  const auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (from + i * step < count) {
        if constexpr (kVec == 4) {
          const float4 x = *reinterpret_cast<const float4*>(state + from + i * step);
          s[i][0] = x.x; s[i][1] = x.y; s[i][2] = x.z; s[i][3] = x.w;
        } else {
          s[i][0] = state[from + i * step];
        }
      }
  };
  load(at);
  for (int i = threadIdx.x; i < high - low; i += blockDim.x)
    kq[i] = make_float2(stream_value<kBf16>(p.k, b * p.k_strides[0] + h * p.k_strides[1] + low + i),
                        stream_value<kBf16>(p.q, b * p.q_strides[0] + h * p.q_strides[1] + low + i));
  const float* la = view < TS_MAX_RETENTIONS ? p.log_alpha[view] : nullptr;
  const float keep = la ? expf(__ldg(la + b * p.log_alpha_batch[view] + h)) : 1.f;
  float v[kVec], read[kVec];
  int row[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int column = (at + j) % p.width;
    row[j] = (at + j) / p.width;
    v[j] = column < p.dv ? stream_value<kBf16>(p.v, b * p.v_strides[0] + h * p.v_strides[1] + column) : 1.f;
    read[j] = 0.f;
  }
  __syncthreads();
  for (int from = at; from < count; from += kAhead * step) {
    if (from != at) load(from);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (from + i * step < count) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float2 r = kq[row[j]];
          s[i][j] = fmaf(s[i][j], keep, r.x * v[j]);
          read[j] = fmaf(r.y, s[i][j], read[j]);
          row[j] += step_rows;
        }
        if constexpr (kVec == 4) *reinterpret_cast<float4*>(state + from + i * step) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        else state[from + i * step] = s[i][0];
      }
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) part[at + j] = read[j];
  __syncthreads();
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    float sum = 0.f;
    for (int i = c; i < step; i += p.width) sum += part[i];
    total[c] = sum;
  }
  if (ranks > 1) cluster_barrier();
  else __syncthreads();
  if (rank == 0) {
    for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
      float sum = total[c];
      for (uint32_t r = 1; r < ranks; ++r) sum += cluster_read(&total[c], r);
      const size_t to = ((static_cast<size_t>(view) * p.batch + b) * p.heads + h) * p.width + c;
      if (kBf16) static_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(sum);
      else static_cast<float*>(p.out)[to] = sum;
    }
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
  // 16 bytes at once where every state starts on a multiple of them
  const bool wide = reinterpret_cast<uintptr_t>(a->state) % 16 == 0 && (static_cast<long long>(p.dk) * p.width) % 4 == 0;
  int period = p.width;   // threads whose elements are whole rows
  if (wide) period = p.width % 4 == 0 ? p.width / 4 : p.width % 2 == 0 ? p.width / 2 : p.width;
  p.active = kScanStepThreads / period * period;
  const int threads = ceil_div(p.active, 32) * 32;
  const bool bf16 = a->dtype == TS_DTYPE_BF16;
  const auto kernel = wide ? (bf16 ? scan_step_kernel<true, 4> : scan_step_kernel<false, 4>)
                           : (bf16 ? scan_step_kernel<true, 1> : scan_step_kernel<false, 1>);
  const cudaError_t e = launch_cluster(kernel, grid, threads, 0, s, cluster, p);
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "scan_step: %s", cudaGetErrorString(e));
  return check_launch("scan_step");
}
