// Windowed attention for one new token of each sequence over a ring cache, and
// the copying of new tokens into such a cache.
//
// The cache of a key head has sinks + window slots: position j lies in slot j
// below `sinks`, in slot sinks + (j - sinks) mod window above.  The filled slots
// are then exactly the positions that the newest token sees (in no order, which
// the softmax does not need), so the token's attention has no mask but their number.
//
// The bytes of the cache bound it, each read once.  A warp takes 16 slots at a
// time straight from memory into the operands of mma.sync (16 slots, then 16
// channels, by 8 query heads): the score's inner index and the output's rows may
// come in any order, so each lane's 16-byte loads already are the fragments (the
// values' pairs of slots take one byte permutation each, the weights one
// transposition).  tcgen05 would want the tiles in shared memory and 128 rows where
// there are at most 16.  The warps of a CTA and the CTAs of a cluster go over
// different slots; their sums, with each one's largest score, are joined through
// shared memory, in order.  The heads are the products' columns because 8 of them
// then cost no padding: with the heads as 16 rows the accumulators did not fit into
// registers (64 sequences x 32 heads of 128 channels, 4160 slots: 332 us; now 176,
// 5.4 TB/s, and 6.2 where the sequences fill the SMs evenly).
#include <cmath>

#include "capi_internal.h"
#include "cluster.cuh"
#include "window.cuh"

namespace ts {

namespace {

constexpr int kStepWarps = 8;   // at most

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

// 8 x 8 values of 16 bits: the lane's two of row g become its two of column g.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ uint4 load16(const __nv_bfloat16* p, bool there) {
  return there ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}

// kD: channels, padded to 64 or 128.  kHeads: query heads of a group, padded to 8 or 16.
template <int kD, int kHeads>
__global__ void __launch_bounds__(32 * kStepWarps, kD == 64 ? 2 : 1)
    window_step_kernel(const __grid_constant__ WinStepParams p) {
  constexpr int kPad = kD + 4;       // floats of a head's sums: heads start in different banks
  constexpr int kSets = kHeads / 8;  // of 8 query heads: the columns of a product
  constexpr int kTiles = kD / 16;    // of 16 channels: the rows of a product with the values
  extern __shared__ float sums[];    // [warp][head][kPad]
  __shared__ float tops[kStepWarps][kHeads], weights[kStepWarps][kHeads], top[kHeads], weight[kHeads];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t rank = cluster_rank_of(), ranks = cluster_size_of();
  const int unit = blockIdx.x / ranks;
  const int group = unit % p.groups, kv_head = unit / p.groups % p.kv_heads, b = unit / p.groups / p.kv_heads;
  const long long length = __ldg(p.lengths + b);
  const int head0 = kv_head * p.share + 16 * group, heads = min(16, p.share - 16 * group);
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
  const int blocks = (filled + 15) >> 4, stride = warps * static_cast<int>(ranks);
  // Whole blocks of old slots are read from one base each, with no test but that of the channels.
  bool key_there[kD / 32], value_there[kD / 64];
#pragma unroll
  for (int c = 0; c < kD / 32; ++c) key_there[c] = 32 * c + 8 * t < p.dim;
#pragma unroll
  for (int c = 0; c < kD / 64; ++c) value_there[c] = 64 * c + 8 * g < p.dim;
  const auto is_whole = [&](int block) { return 16 * block + 16 <= filled && slot >> 4 != block; };
  uint4 kk[kD / 32][2];   // slots g, g + 8, channels 32 c + 8 t .. + 7: two inner steps' fragments
  const auto load_keys = [&](int block) {
    const __nv_bfloat16* from = keys + (16 * block + g) * p.keys_strides[2] + 8 * t;
    if (is_whole(block)) {
#pragma unroll
      for (int h = 0; h < 2; ++h, from += 8 * p.keys_strides[2])
#pragma unroll
        for (int c = 0; c < kD / 32; ++c) kk[c][h] = load16(from + 32 * c, key_there[c]);
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h, from += 8 * p.keys_strides[2]) {
      const int s = 16 * block + 8 * h + g;
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) kk[c][h] = load16((s == slot ? k_new + 8 * t : from) + 32 * c, s < filled && key_there[c]);
    }
  };
  int block = static_cast<int>(rank) * warps + warp;
  if (block < blocks) load_keys(block);
  uint4 q[kSets][kD / 32];   // query heads g + 8 n, the same channels
#pragma unroll
  for (int n = 0; n < kSets; ++n)
#pragma unroll
    for (int c = 0; c < kD / 32; ++c)
      q[n][c] = load16(p.q + b * p.q_strides[0] + (head0 + g + 8 * n) * p.q_strides[1] + 32 * c + 8 * t,
                       32 * c + 8 * t < p.dim && g + 8 * n < heads);
  // rows g and g + 8 of tile j: channels 8 g + j and, at 128 channels, 64 + 8 g + j, at 64, 8 g + 4 + j
  // (the lane's own 16-byte loads of the values); columns: heads 2 t, 2 t + 1
  float o[kSets][kTiles][4];
  float m[kSets][2], l[kSets][2];   // of heads 2 t, 2 t + 1: largest score (all lanes of t alike), sum (this lane's slots)
#pragma unroll
  for (int n = 0; n < kSets; ++n) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
  }
  for (; block < blocks; block += stride) {
    uint4 vv[kD / 64][4];   // slots 2t, 2t + 1, 2t + 8, 2t + 9, channels 64 c + 8 g .. + 7
    const __nv_bfloat16* from = values + (16 * block + 2 * t) * p.values_strides[2] + 8 * g;
    const bool whole = is_whole(block);
    if (whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i, from += (i == 2 ? 7 : 1) * p.values_strides[2])
#pragma unroll
        for (int c = 0; c < kD / 64; ++c) vv[c][i] = load16(from + 64 * c, value_there[c]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i, from += (i == 2 ? 7 : 1) * p.values_strides[2]) {
        const int s = 16 * block + 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
        for (int c = 0; c < kD / 64; ++c) vv[c][i] = load16((s == slot ? v_new + 8 * g : from) + 64 * c, s < filled && value_there[c]);
      }
    }
    float s[kSets][4] = {};   // slots g (0, 1) and g + 8 (2, 3), heads 2 t, 2 t + 1
#pragma unroll
    for (int c = 0; c < kD / 32; ++c) {
      const uint32_t low[4] = {kk[c][0].x, kk[c][1].x, kk[c][0].y, kk[c][1].y};
      const uint32_t high[4] = {kk[c][0].z, kk[c][1].z, kk[c][0].w, kk[c][1].w};
#pragma unroll
      for (int n = 0; n < kSets; ++n) {
        mma_16816(s[n], low, q[n][c].x, q[n][c].y);
        mma_16816(s[n], high, q[n][c].z, q[n][c].w);
      }
    }
    if (block + stride < blocks) load_keys(block + stride);
    const bool first = whole || 16 * block + g < filled, second = whole || 16 * block + 8 + g < filled;
    uint32_t pair[kSets][2];   // weights of slots 2 t, 2 t + 1 (and + 8) for head g
#pragma unroll
    for (int n = 0; n < kSets; ++n) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (e < 2 ? first : second) ? s[n][e] * p.scale2 : -INFINITY;
      float best[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
      if (__any_sync(0xffffffffu, best[0] > m[n][0] || best[1] > m[n][1])) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 4; d <= 16; d *= 2) best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], d));
          const float next = fmaxf(best[e], m[n][e]);
          const float factor = m[n][e] == next ? 1.f : exp2_fast(m[n][e] - next);
          m[n][e] = next;
          l[n][e] *= factor;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            o[n][j][e] *= factor;
            o[n][j][2 + e] *= factor;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = exp2_fast(x[e] - (m[n][e & 1] == -INFINITY ? 0.f : m[n][e & 1]));
        l[n][e & 1] += x[e];
      }
      pair[n][0] = transpose_8x8(pack_bf16(x[0], x[1]));
      pair[n][1] = transpose_8x8(pack_bf16(x[2], x[3]));
    }
    const auto word = [&](int c, int i, int w) { return w == 0 ? vv[c][i].x : w == 1 ? vv[c][i].y : w == 2 ? vv[c][i].z : vv[c][i].w; };
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const uint32_t pick = j & 1 ? 0x7632 : 0x5410;
      const int far = kD / 64 - 1, w = j / 2, w_far = kD == 128 ? w : w + 2;
      const uint32_t a[4] = {__byte_perm(word(0, 0, w), word(0, 1, w), pick), __byte_perm(word(far, 0, w_far), word(far, 1, w_far), pick),
                             __byte_perm(word(0, 2, w), word(0, 3, w), pick), __byte_perm(word(far, 2, w_far), word(far, 3, w_far), pick)};
#pragma unroll
      for (int n = 0; n < kSets; ++n) mma_16816(o[n][j], a, pair[n][0], pair[n][1]);
    }
  }
  // each warp's sums, then the CTA's in warp order, then the cluster's in rank order
#pragma unroll
  for (int n = 0; n < kSets; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d <= 16; d *= 2) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
      const int head = 8 * n + 2 * t + e;
      if (g == 0) {
        tops[warp][head] = m[n][e];
        weights[warp][head] = l[n][e];
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        float* to = sums + (warp * kHeads + head) * kPad + 8 * g + j;
        to[0] = o[n][j][e];
        to[kD == 128 ? 64 : 4] = o[n][j][2 + e];
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < heads) {
    const int head = threadIdx.x;
    float best = -INFINITY, sum = 0.f;
    for (int i = 0; i < warps; ++i) best = fmaxf(best, tops[i][head]);
    for (int i = 0; i < warps; ++i) {
      // a part without a score carries nothing; NaN goes on
      const float factor = tops[i][head] == -INFINITY && weights[i][head] == 0.f ? 0.f : exp2_fast(tops[i][head] - best);
      sum += weights[i][head] * factor;
      tops[i][head] = factor;
    }
    top[head] = best;
    weight[head] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * kD; i += blockDim.x) {
    const int head = i / kD, c = i % kD;
    float sum = 0.f;
    for (int j = 0; j < warps; ++j) sum += tops[j][head] != 0.f ? sums[(j * kHeads + head) * kPad + c] * tops[j][head] : 0.f;
    sums[head * kPad + c] = sum;   // the place of warp 0's own value, which this thread alone reads
  }
  if (ranks > 1) cluster_barrier();
  else __syncthreads();
  for (int i = static_cast<int>(rank * blockDim.x + threadIdx.x); i < heads * kD; i += static_cast<int>(ranks * blockDim.x)) {
    const int head = i / kD, c = i % kD;
    float its_top[8], its_weight[8], its_sum[8], best = -INFINITY, value = 0.f, sum = 0.f;
#pragma unroll
    for (uint32_t r = 0; r < 8; ++r)
      if (r < ranks) {
        its_top[r] = cluster_read(&top[head], r);
        its_weight[r] = cluster_read(&weight[head], r);
        its_sum[r] = cluster_read(&sums[head * kPad + c], r);
        best = fmaxf(best, its_top[r]);
      }
#pragma unroll
    for (uint32_t r = 0; r < 8; ++r)
      if (r < ranks && !(its_top[r] == -INFINITY && its_weight[r] == 0.f)) {
        const float factor = exp2_fast(its_top[r] - best);
        sum += its_weight[r] * factor;
        value += its_sum[r] * factor;
      }
    if (c < p.dim)
      p.y[(static_cast<size_t>(b) * p.heads + head0 + head) * p.dim + c] = __float2bfloat16_rn(here ? value / sum : 0.f);
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

template <int kD, int kHeads>
int window_step_launch(const WinStepParams& p, int cluster, int warps, cudaStream_t s) {
  const size_t smem = sizeof(float) * warps * kHeads * (kD + 4);
  const auto kernel = window_step_kernel<kD, kHeads>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(sizeof(float) * kStepWarps * kHeads * (kD + 4)));
  if (e == cudaSuccess)
    e = launch_cluster(kernel, dim3(static_cast<unsigned>(p.batch * p.kv_heads * p.groups * cluster)), 32 * warps, smem, s,
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
  // CTAs of a cluster: as many as bring all SMs to work, while each has 64 slots (16 to a warp)
  const long long units = static_cast<long long>(p.batch) * p.kv_heads * p.groups, slots = static_cast<long long>(p.sinks) + p.window;
  if (units > (1ll << 27)) return set_error(TS_ERR_NOT_IMPLEMENTED, "window_step: too many heads and sequences");
  int cluster = 1;
  while (cluster < 8 && units * cluster < 592 && slots > 64 * cluster) cluster *= 2;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // 4 warps to a CTA, so that the last ones end together; 8 where there are too few CTAs for the SMs
  const int warps = units * cluster < 296 && slots > 64 * cluster ? 8 : 4;
  const bool narrow = p.dim <= 64, few = p.share <= 8;
  if (narrow) return few ? window_step_launch<64, 8>(p, cluster, warps, s) : window_step_launch<64, 16>(p, cluster, warps, s);
  return few ? window_step_launch<128, 8>(p, cluster, warps, s) : window_step_launch<128, 16>(p, cluster, warps, s);
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
