// Windowed attention for one new token of each sequence over a ring cache, and
// the copying of new tokens into such a cache.
//
// The cache of a key head has sinks + window slots: position j lies in slot j
// below `sinks`, in slot sinks + (j - sinks) mod window above.  The filled slots
// are then exactly the positions that the newest token sees (in no order, which
// the softmax does not need), so the token's attention has no mask but their number.
//
// The bytes of the cache bound it, each read once.  A warp takes 16 slots at a
// time straight from memory into the operands of mma.sync (16 query heads by 8
// slots, or by 8 channels): the score's inner index and the output's columns may
// come in any order, so each lane's 16-byte loads already are the fragments (the
// values' pairs of slots take one byte permutation each).  tcgen05 would want the
// tiles in shared memory and 128 rows where there are at most 16.  The warps of a
// CTA and the CTAs of a cluster go over different slots; their sums, with each
// one's largest score, are joined through shared memory, in order.
#include <cmath>

#include "capi_internal.h"
#include "cluster.cuh"
#include "window.cuh"

namespace ts {

namespace {

constexpr int kStepWarps = 8;
constexpr int kStepThreads = 32 * kStepWarps;

struct WinStepParams {
  int batch, heads, kv_heads, share, dim;
  int sinks, window;
  int groups;                // of 16 query heads that share a key head
  float scale2;              // scale * log2(e)
  const __nv_bfloat16 *q, *k, *v;
  long long q_strides[2], k_strides[2], v_strides[2];   // batch, head
  __nv_bfloat16 *keys, *values;
  long long keys_strides[3], values_strides[3];         // batch, head, slot
  const int* lengths;
  __nv_bfloat16* y;          // [batch, heads, dim] contiguous
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load16(const __nv_bfloat16* p, bool there) {
  return there ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

// kD: channels, padded to 64 or 128.  kRows: query heads of a group, padded to 8 or 16.
template <int kD, int kRows>
__global__ void __launch_bounds__(kStepThreads, 2) window_step_kernel(const __grid_constant__ WinStepParams p) {
  constexpr int kPad = kD + 4;   // floats of a row of sums: rows start in different banks
  extern __shared__ float sums[];                       // [warp][row][kPad]
  __shared__ float tops[kStepWarps][kRows], weights[kStepWarps][kRows], top[kRows], weight[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t rank = cluster_rank_of(), ranks = cluster_size_of();
  const int unit = blockIdx.x / ranks;
  const int group = unit % p.groups, kv_head = unit / p.groups % p.kv_heads, b = unit / p.groups / p.kv_heads;
  const long long length = __ldg(p.lengths + b);
  const int head0 = kv_head * p.share + 16 * group, rows = min(16, p.share - 16 * group);
  const bool here = length >= 0;
  const int slot = length < p.sinks ? static_cast<int>(length) : p.sinks + static_cast<int>((length - p.sinks) % p.window);
  const int filled = here ? static_cast<int>(min(length + 1, static_cast<long long>(p.sinks) + p.window)) : 0;
  const __nv_bfloat16* k_new = p.k + b * p.k_strides[0] + kv_head * p.k_strides[1];
  const __nv_bfloat16* v_new = p.v + b * p.v_strides[0] + kv_head * p.v_strides[1];
  __nv_bfloat16* keys = p.keys + b * p.keys_strides[0] + kv_head * p.keys_strides[1];
  __nv_bfloat16* values = p.values + b * p.values_strides[0] + kv_head * p.values_strides[1];
  // the new token's slot: written by one CTA, read by none (they take the token itself)
  if (here && rank == 0 && group == 0 && threadIdx.x < kD / 4) {
    const int c = 8 * (threadIdx.x % (kD / 8));
    const bool is_key = threadIdx.x < kD / 8;
    if (c < p.dim) {
      if (is_key) *reinterpret_cast<uint4*>(keys + slot * p.keys_strides[2] + c) = load16(k_new + c, true);
      else *reinterpret_cast<uint4*>(values + slot * p.values_strides[2] + c) = load16(v_new + c, true);
    }
  }
  // queries: this lane's rows g and g + 8, channels 32 c + 8 t .. + 7 as two inner steps' fragments
  uint32_t q[kD / 32][2][4];
#pragma unroll
  for (int c = 0; c < kD / 32; ++c) {
    const __nv_bfloat16* from = p.q + b * p.q_strides[0] + (head0 + g) * p.q_strides[1] + 32 * c + 8 * t;
    const bool inside = 32 * c + 8 * t < p.dim;
    const uint4 a = load16(from, inside && g < rows);
    uint4 z = make_uint4(0, 0, 0, 0);
    if (kRows > 8) z = load16(from + 8 * p.q_strides[1], inside && g + 8 < rows);
    q[c][0][0] = a.x; q[c][0][1] = z.x; q[c][0][2] = a.y; q[c][0][3] = z.y;
    q[c][1][0] = a.z; q[c][1][1] = z.z; q[c][1][2] = a.w; q[c][1][3] = z.w;
  }
  float o[kD / 8][4];   // of 64 channels c, mma j: channels 64 c + 16 t + j and + 8 of rows g, g + 8
#pragma unroll
  for (int i = 0; i < kD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  const int blocks = (filled + 15) >> 4, stride = kStepWarps * static_cast<int>(ranks);
  uint4 kk[kD / 32][2];
  auto load_keys = [&](int block) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int s = 16 * block + 8 * h + g;
      const __nv_bfloat16* from = s == slot ? k_new : keys + s * p.keys_strides[2];
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) kk[c][h] = load16(from + 32 * c + 8 * t, s < filled && 32 * c + 8 * t < p.dim);
    }
  };
  int block = static_cast<int>(rank) * kStepWarps + warp;
  if (block < blocks) load_keys(block);
  for (; block < blocks; block += stride) {
    uint4 vv[kD / 64][4];   // slots 2t, 2t + 1, 2t + 8, 2t + 9, channels 64 c + 8 g .. + 7
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = 16 * block + 2 * t + (i & 1) + 8 * (i >> 1);
      const __nv_bfloat16* from = s == slot ? v_new : values + s * p.values_strides[2];
#pragma unroll
      for (int c = 0; c < kD / 64; ++c) vv[c][i] = load16(from + 64 * c + 8 * g, s < filled && 64 * c + 8 * g < p.dim);
    }
    float s[2][4] = {};
#pragma unroll
    for (int c = 0; c < kD / 32; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mma_16816(s[h], q[c][0], kk[c][h].x, kk[c][h].y);
        mma_16816(s[h], q[c][1], kk[c][h].z, kk[c][h].w);
      }
    if (block + stride < blocks) load_keys(block + stride);
    // rows g (i = 0) and g + 8 (i = 1); columns 2t, 2t + 1 of each 8 slots
    uint32_t weight_pair[4];
#pragma unroll
    for (int i = 0; i < kRows / 8; ++i) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = 16 * block + 8 * (e >> 1) + 2 * t + (e & 1) < filled ? s[e >> 1][2 * i + (e & 1)] * p.scale2 : -INFINITY;
      float best = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
      if (__any_sync(0xffffffffu, best > m[i])) {
        const float next = fmaxf(best, m[i]);
        const float factor = m[i] == next ? 1.f : exp2_fast(m[i] - next);
        m[i] = next;
        l[i] *= factor;
#pragma unroll
        for (int j = 0; j < kD / 8; ++j) {
          o[j][2 * i] *= factor;
          o[j][2 * i + 1] *= factor;
        }
      }
      const float origin = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = exp2_fast(x[e] - origin);
        l[i] += x[e];
      }
      weight_pair[i] = pack_bf16(x[0], x[1]);
      weight_pair[2 + i] = pack_bf16(x[2], x[3]);
    }
    if (kRows <= 8) weight_pair[1] = weight_pair[3] = 0;
#pragma unroll
    for (int c = 0; c < kD / 64; ++c) {
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vv[c][0]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vv[c][1]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vv[c][2]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vv[c][3]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t pick = j & 1 ? 0x7632 : 0x5410;
        mma_16816(o[8 * c + j], weight_pair, __byte_perm(v0[j / 2], v1[j / 2], pick), __byte_perm(v2[j / 2], v3[j / 2], pick));
      }
    }
  }
  // each warp's sums, then the CTA's in warp order, then the cluster's in rank order
#pragma unroll
  for (int i = 0; i < kRows / 8; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int row = g + 8 * i;
    if (t == 0) {
      tops[warp][row] = m[i];
      weights[warp][row] = l[i];
    }
#pragma unroll
    for (int c = 0; c < kD / 64; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float* to = sums + (warp * kRows + row) * kPad + 64 * c + 16 * t + j;
        to[0] = o[8 * c + j][2 * i];
        to[8] = o[8 * c + j][2 * i + 1];
      }
  }
  __syncthreads();
  if (threadIdx.x < kRows) {
    const int row = threadIdx.x;
    float best = -INFINITY, sum = 0.f;
    for (int i = 0; i < kStepWarps; ++i) best = fmaxf(best, tops[i][row]);
    for (int i = 0; i < kStepWarps; ++i) {
      // a part without a score carries nothing; NaN goes on
      const float factor = tops[i][row] == -INFINITY && weights[i][row] == 0.f ? 0.f : exp2_fast(tops[i][row] - best);
      sum += weights[i][row] * factor;
      tops[i][row] = factor;
    }
    top[row] = best;
    weight[row] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kD; i += kStepThreads) {
    const int row = i / kD, c = i % kD;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kStepWarps; ++j) sum += tops[j][row] != 0.f ? sums[(j * kRows + row) * kPad + c] * tops[j][row] : 0.f;
    sums[row * kPad + c] = sum;   // the place of warp 0's own value, which this thread alone reads
  }
  if (ranks > 1) cluster_barrier();
  else __syncthreads();
  for (int i = static_cast<int>(rank) * kStepThreads + threadIdx.x; i < rows * kD; i += static_cast<int>(ranks) * kStepThreads) {
    const int row = i / kD, c = i % kD;
    float best = -INFINITY, value = 0.f, sum = 0.f;
    for (uint32_t r = 0; r < ranks; ++r) best = fmaxf(best, cluster_read(&top[row], r));
    for (uint32_t r = 0; r < ranks; ++r) {
      const float mine = cluster_read(&top[row], r), share = cluster_read(&weight[row], r);
      if (mine == -INFINITY && share == 0.f) continue;
      const float factor = exp2_fast(mine - best);
      sum += share * factor;
      value += cluster_read(&sums[row * kPad + c], r) * factor;
    }
    if (c < p.dim)
      p.y[(static_cast<size_t>(b) * p.heads + head0 + row) * p.dim + c] = __float2bfloat16_rn(here ? value / sum : 0.f);
  }
  if (ranks > 1) cluster_barrier();   // no CTA leaves while others read its memory
}

struct WinExtendParams {
  int kv_heads, dim, tokens, sinks, window;
  const __nv_bfloat16 *k, *v;
  long long k_strides[3], v_strides[3];                  // batch, head, token
  __nv_bfloat16 *keys, *values;
  long long keys_strides[3], values_strides[3];
  const int *lengths, *fresh;                            // fresh: new tokens of each sequence, or null
};

// A thread for 16 bytes of a slot: its newest position, where that is one of the new tokens.
__global__ void __launch_bounds__(256) window_extend_kernel(const __grid_constant__ WinExtendParams p) {
  const int b = blockIdx.z, head = blockIdx.y, chunks = p.dim / 8;
  const long long before = __ldg(p.lengths + b);
  const long long count = p.fresh ? max(0, min(__ldg(p.fresh + b), p.tokens)) : p.tokens;
  const long long at = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long slot = at / chunks, last = before + count - 1;
  const int c = 8 * static_cast<int>(at % chunks);
  if (before < 0 || slot >= static_cast<long long>(p.sinks) + p.window || slot > last) return;
  const long long position = slot < p.sinks ? slot : slot + (last - slot) / p.window * p.window;
  const long long token = position - before;
  if (token < 0) return;
  const uint4 key = load16(p.k + b * p.k_strides[0] + head * p.k_strides[1] + token * p.k_strides[2] + c, true);
  const uint4 value = load16(p.v + b * p.v_strides[0] + head * p.v_strides[1] + token * p.v_strides[2] + c, true);
  *reinterpret_cast<uint4*>(p.keys + b * p.keys_strides[0] + head * p.keys_strides[1] + slot * p.keys_strides[2] + c) = key;
  *reinterpret_cast<uint4*>(p.values + b * p.values_strides[0] + head * p.values_strides[1] + slot * p.values_strides[2] + c) = value;
}

bool aligned16(const void* p, const long long* strides, int count) {
  for (int i = 0; i < count; ++i)
    if (strides[i] % 8) return false;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

int check_cache(const ts_window_cache* c, const char* what) {
  if (!c) return set_error(TS_ERR_VALUE, "%s: null arguments", what);
  if (c->batch < 1 || c->kv_heads < 1) return set_error(TS_ERR_VALUE, "%s: sizes must be positive", what);
  if (c->dim < 8 || c->dim > 128 || c->dim % 8)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "%s: head width %d is not a multiple of 8 up to 128", what, c->dim);
  if (c->window < 1 || c->sinks < 0) return set_error(TS_ERR_VALUE, "%s: window must be >= 1 and sinks >= 0", what);
  if (c->window > (1 << 30) || c->sinks > (1 << 30) || c->batch > 65535 || c->kv_heads > 65535)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "%s: more than 2^30 slots, 65535 sequences or 65535 heads", what);
  if (!c->keys || !c->values || !c->lengths) return set_error(TS_ERR_VALUE, "%s: null tensor", what);
  if (!aligned16(c->keys, c->keys_strides, 3) || !aligned16(c->values, c->values_strides, 3))
    return set_error(TS_ERR_VALUE, "%s: the cache's bases and strides must be multiples of 16 bytes", what);
  return TS_OK;
}

template <int kD, int kRows>
int window_step_launch(const WinStepParams& p, int cluster, cudaStream_t s) {
  constexpr size_t smem = sizeof(float) * kStepWarps * kRows * (kD + 4);
  const auto kernel = window_step_kernel<kD, kRows>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e == cudaSuccess)
    e = launch_cluster(kernel, dim3(static_cast<unsigned>(p.batch * p.kv_heads * p.groups * cluster)), kStepThreads, smem, s,
                       cluster, p);
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "window_step: %s", cudaGetErrorString(e));
  return check_launch("window_step");
}

}  // namespace

}  // namespace ts

using namespace ts;

extern "C" {

int ts_b200_window_step(const ts_window_step_args* a, ts_stream_t stream) {
  if (!a) return set_error(TS_ERR_VALUE, "window_step: null arguments");
  const ts_window_cache& c = a->cache;
  if (const int rc = check_cache(&c, "window_step")) return rc;
  if (a->heads < 1 || a->heads % c.kv_heads)
    return set_error(TS_ERR_VALUE, "window_step: %d heads do not share %d key heads", a->heads, c.kv_heads);
  if (a->heads > 65535) return set_error(TS_ERR_NOT_IMPLEMENTED, "window_step: more than 65535 heads");
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return set_error(TS_ERR_VALUE, "window_step: scale must be positive and finite");
  if (!a->q || !a->k || !a->v || !a->y) return set_error(TS_ERR_VALUE, "window_step: null tensor");
  if (!aligned16(a->q, a->q_strides, 2) || !aligned16(a->k, a->k_strides, 2) || !aligned16(a->v, a->v_strides, 2))
    return set_error(TS_ERR_VALUE, "window_step: bases and strides must be multiples of 16 bytes");
  WinStepParams p = {};
  p.batch = c.batch;
  p.heads = a->heads;
  p.kv_heads = c.kv_heads;
  p.share = a->heads / c.kv_heads;
  p.dim = c.dim;
  p.sinks = c.sinks;
  p.window = c.window;
  p.groups = ceil_div(p.share, 16);
  p.scale2 = a->scale * kLog2e;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.keys = static_cast<__nv_bfloat16*>(c.keys);
  p.values = static_cast<__nv_bfloat16*>(c.values);
  p.lengths = c.lengths;
  p.y = static_cast<__nv_bfloat16*>(a->y);
  for (int i = 0; i < 3; ++i) {
    p.keys_strides[i] = c.keys_strides[i];
    p.values_strides[i] = c.values_strides[i];
    if (i == 2) break;
    p.q_strides[i] = a->q_strides[i];
    p.k_strides[i] = a->k_strides[i];
    p.v_strides[i] = a->v_strides[i];
  }
  // CTAs of a cluster: as many as bring all SMs to work, while each has 128 slots (16 to a warp)
  const long long units = static_cast<long long>(p.batch) * p.kv_heads * p.groups, slots = static_cast<long long>(p.sinks) + p.window;
  if (units > (1ll << 27)) return set_error(TS_ERR_NOT_IMPLEMENTED, "window_step: too many heads and sequences");
  int cluster = 1;
  while (cluster < 8 && units * cluster < 296 && slots > 128 * cluster) cluster *= 2;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool narrow = p.dim <= 64, few = p.share <= 8;
  if (narrow) return few ? window_step_launch<64, 8>(p, cluster, s) : window_step_launch<64, 16>(p, cluster, s);
  return few ? window_step_launch<128, 8>(p, cluster, s) : window_step_launch<128, 16>(p, cluster, s);
}

int ts_b200_window_extend(const ts_window_extend_args* a, ts_stream_t stream) {
  if (!a) return set_error(TS_ERR_VALUE, "window_extend: null arguments");
  const ts_window_cache& c = a->cache;
  if (const int rc = check_cache(&c, "window_extend")) return rc;
  if (a->tokens < 1 || !a->k || !a->v) return set_error(TS_ERR_VALUE, "window_extend: no new tokens");
  if (!aligned16(a->k, a->k_strides, 3) || !aligned16(a->v, a->v_strides, 3))
    return set_error(TS_ERR_VALUE, "window_extend: bases and strides must be multiples of 16 bytes");
  WinExtendParams p = {};
  p.kv_heads = c.kv_heads;
  p.dim = c.dim;
  p.tokens = a->tokens;
  p.sinks = c.sinks;
  p.window = c.window;
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.keys = static_cast<__nv_bfloat16*>(c.keys);
  p.values = static_cast<__nv_bfloat16*>(c.values);
  for (int i = 0; i < 3; ++i) {
    p.k_strides[i] = a->k_strides[i];
    p.v_strides[i] = a->v_strides[i];
    p.keys_strides[i] = c.keys_strides[i];
    p.values_strides[i] = c.values_strides[i];
  }
  p.lengths = c.lengths;
  p.fresh = a->fresh;
  const long long items = (static_cast<long long>(p.sinks) + p.window) * (p.dim / 8);
  const dim3 grid(static_cast<unsigned>((items + 255) / 256), static_cast<unsigned>(c.kv_heads), static_cast<unsigned>(c.batch));
  window_extend_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("window_extend");
}

}  // extern "C"
