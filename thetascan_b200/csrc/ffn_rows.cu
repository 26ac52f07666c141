// The gated feed-forward block for few rows (decoding steps): the forward,
// which keeps g and u where a backward pass follows (ffn.cu).
//
// With up to kRowsMost rows the weights are read once for almost no
// arithmetic (6 D H bytes against 6 M D H operations), so what counts is to
// have their loads in flight on every SM at once.  A tile of the tensor-core
// path spends 128 rows of tensor memory and a pipeline's start on them; here a
// warp multiplies 16 rows of weights, which go from memory straight into the
// registers of mma.sync's A operand, by 8 rows of x at a time (the B operand).
//
//   gate: A = 8 rows of Wg and the 8 rows of Wu of the same hidden columns, so
//         that a thread ends with g and u of the same place: h = act(g) u
//   down: A = 16 rows of Wd
//
// h passes between the two as two bf16 values, its upper half and the rest
// (2^-16 together): the result then carries its own rounding alone (1.66e-3 of
// its norm, with h in bf16 2.35e-3), for a second load and instruction beside
// the weights' traffic (one row of 1024 x 4096: 7.8 -> 8.8 us, of 2048 x 5632:
// 16.6 -> 21.7 us).
//
// The order of the inner dimension is free as long as A and B agree, so a lane
// takes 8 neighbouring elements (16 bytes) of its row for two steps of
// m16n8k16.  The inner dimension is dealt in blocks of 32 to the CTA's eight
// warps (neighbouring warps read neighbouring 64 bytes) and, in the down
// product, to the CTAs of a cluster; sums meet in shared memory in a fixed
// order.  The down product is launched to overlap the gate (programmatic
// dependent launch): its first weights are on their way before it waits for h.
// The gate is launched in full order, so that weights which the launch before
// it wrote are there for both.
#include <cuda_bf16.h>

#include "capi_internal.h"
#include "common.cuh"
#include "ffn.cuh"

namespace ts {

namespace {

constexpr int kRowsWarps = 8;
constexpr int kRowsBatch = 4;        // blocks of 32 a warp has in flight

struct FfnRowsParams {
  const __nv_bfloat16 *x, *wg, *wu, *wd;
  long long xs, wgs, wus, wds;
  __nv_bfloat16 *h, *y;      // h: [2][rows][hidden]
  uint8_t* kept;             // g and u (keep_at), or null
  int rows, width, hidden, out;
};

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_weights(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// One warp's sums over its blocks of the inner dimension: kSets sets of 16 rows
// of the weights, `a[i]` and `b[i]` this lane's two of each (null: zeros), by the
// rows of `x`, 8 kTiles of them (kTwo: and by those of a second matrix behind
// it).  `first` and `stride` count blocks of 32.  ready() is called between the first weights' loads and the first of x.
template <int kSets, int kTiles, bool kTwo, class F>
__device__ __forceinline__ void rows_product(float (&c)[kSets * kTiles][4], const __nv_bfloat16* const (&a)[kSets],
                                             const __nv_bfloat16* const (&b)[kSets], const __nv_bfloat16* x,
                                             long long xs, int rows, int inner, int first, int stride, F ready) {
  constexpr int kBatch = kRowsBatch / kSets;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < kSets * kTiles; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
  const int blocks = (inner + 31) / 32;
  bool waited = false;
  for (int base = first; base < blocks || !waited; base += stride * kBatch) {
    uint4 wa[kBatch][kSets], wb[kBatch][kSets];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int k = (base + i * stride) * 32 + 8 * t;
#pragma unroll
      for (int m = 0; m < kSets; ++m) {
        wa[i][m] = a[m] && k < inner ? load_weights(a[m] + k) : zero;
        wb[i][m] = b[m] && k < inner ? load_weights(b[m] + k) : zero;
      }
    }
    if (!waited) {
      ready();
      waited = true;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int k = (base + i * stride) * 32 + 8 * t;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int row = 8 * n + g;
        const bool there = row < rows && k < inner;
        uint4 v[kTwo ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (kTwo ? 2 : 1); ++h)
          v[h] = there ? *reinterpret_cast<const uint4*>(x + (static_cast<long long>(h) * rows + row) * xs + k) : zero;
#pragma unroll
        for (int h = 0; h < (kTwo ? 2 : 1); ++h)
#pragma unroll
          for (int m = 0; m < kSets; ++m) {
            mma_16x8x16(c[m * kTiles + n], wa[i][m].x, wb[i][m].x, wa[i][m].y, wb[i][m].y, v[h].x, v[h].y);
            mma_16x8x16(c[m * kTiles + n], wa[i][m].z, wb[i][m].z, wa[i][m].w, wb[i][m].w, v[h].z, v[h].w);
          }
      }
    }
  }
}

// Sum of the CTA's warps, in their order, by the first 32 kTiles threads: thread 32 n + lane gets sum n's four values.
template <int kTiles>
__device__ __forceinline__ float4 rows_sum(const float (&c)[kTiles][4], float4* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < kTiles; ++n) part[(warp * kTiles + n) * 32 + lane] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
  __syncthreads();
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (threadIdx.x < 32 * kTiles) {
#pragma unroll
    for (int i = 0; i < kRowsWarps; ++i) {
      const float4 v = part[i * kTiles * 32 + threadIdx.x];
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
  }
  return sum;
}

// kKeep: g and u are kept.  An instance of its own: with both in one the compiler holds fewer loads in flight (86
// registers for 108; 2048 x 5632, 32 rows: 49 us for 32).
template <int kSets, int kTiles, int kAct, bool kKeep>
__global__ void __launch_bounds__(32 * kRowsWarps) ffn_rows_gate_kernel(const FfnRowsParams p) {
  constexpr int kAll = kSets * kTiles;
  __shared__ float4 part[kRowsWarps * kAll * 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const __nv_bfloat16 *wg[kSets], *wu[kSets];
#pragma unroll
  for (int m = 0; m < kSets; ++m) {
    const int j = (blockIdx.x * kSets + m) * 8 + g;   // hidden is a multiple of 8: a set of 8 columns is in it or not
    wg[m] = j < p.hidden ? p.wg + j * p.wgs : nullptr;
    wu[m] = j < p.hidden ? p.wu + j * p.wus : nullptr;
  }
  float c[kAll][4];
  rows_product<kSets, kTiles, false>(c, wg, wu, p.x, p.xs, p.rows, p.width, threadIdx.x >> 5, kRowsWarps, [] {});
  const float4 s = rows_sum<kAll>(c, part);
  const int m = (threadIdx.x >> 5) / kTiles, n = (threadIdx.x >> 5) % kTiles;
  const int j = (blockIdx.x * kSets + m) * 8 + g;
  if (threadIdx.x < 32 * kAll && j < p.hidden) {
    const int row = 8 * n + 2 * t;
    float slope;
    const float h[2] = {ffn_act<kAct>(s.x, slope) * s.z, ffn_act<kAct>(s.y, slope) * s.w};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (row + i >= p.rows) continue;
      __nv_bfloat16* to = p.h + static_cast<long long>(row + i) * p.hidden + j;
      *to = __float2bfloat16_rn(ffn_high(h[i]));
      to[static_cast<long long>(p.rows) * p.hidden] = __float2bfloat16_rn(ffn_rest(h[i]));
      if (kKeep) keep_one(p.kept, p.hidden, row + i, j, i ? s.y : s.x, i ? s.w : s.z);
    }
  }
}

// CTAs that share a down tile's inner length: at most 8, and 4 where their sums would outgrow static shared memory.
constexpr int rows_ranks(int all) { return all > 4 ? 4 : 8; }

template <int kSets, int kTiles>
__global__ void __launch_bounds__(32 * kRowsWarps) ffn_rows_down_kernel(const FfnRowsParams p) {
  constexpr int kAll = kSets * kTiles;
  __shared__ float4 part[kRowsWarps * kAll * 32];
  __shared__ float4 sums[rows_ranks(kAll) * kAll * 32];   // the cluster's, in its first CTA
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs: its memory may be written
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int first = blockIdx.x / ranks * 16 * kSets;
  const __nv_bfloat16 *wa[kSets], *wb[kSets];
#pragma unroll
  for (int m = 0; m < kSets; ++m) {
    const int o = first + 16 * m + g;   // out is a multiple of 8: rows o and o + 8 are whole groups
    wa[m] = o < p.out ? p.wd + o * p.wds : nullptr;
    wb[m] = o + 8 < p.out ? p.wd + (o + 8) * p.wds : nullptr;
  }
  float c[kAll][4];
  rows_product<kSets, kTiles, true>(c, wa, wb, p.h, p.hidden, p.rows, p.hidden,
                                    static_cast<int>(rank) * kRowsWarps + (threadIdx.x >> 5),
                                    static_cast<int>(ranks) * kRowsWarps,
                                    [] { asm volatile("griddepcontrol.wait;" ::: "memory"); });
  float4 s = rows_sum<kAll>(c, part);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < 32 * kAll) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;"
                 : "=r"(at)
                 : "r"(smem_u32(&sums[rank * kAll * 32 + threadIdx.x])));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(at), "f"(s.x), "f"(s.y), "f"(s.z), "f"(s.w)
                 : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank != 0 || threadIdx.x >= 32 * kAll) return;
  s = sums[threadIdx.x];
  for (uint32_t i = 1; i < ranks; ++i) {
    const float4 v = sums[i * kAll * 32 + threadIdx.x];
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  const int o = first + 16 * ((threadIdx.x >> 5) / kTiles) + g, row = 8 * ((threadIdx.x >> 5) % kTiles) + 2 * t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (row + i >= p.rows || o >= p.out) continue;
    __nv_bfloat16* y = p.y + static_cast<long long>(row + i) * p.out + o;
    y[0] = __float2bfloat16_rn(i ? s.y : s.x);
    if (o + 8 < p.out) y[8] = __float2bfloat16_rn(i ? s.w : s.z);
  }
}

template <int kSets, int kTiles, bool kKeep>
int ffn_rows_gate(const FfnRowsParams& p, int activation, cudaStream_t s) {
  const int grid = (p.hidden + 8 * kSets - 1) / (8 * kSets), threads = 32 * kRowsWarps;
  if (activation == TS_FFN_SILU) {
    ffn_rows_gate_kernel<kSets, kTiles, TS_FFN_SILU, kKeep><<<grid, threads, 0, s>>>(p);
  } else if (activation == TS_FFN_GELU) {
    ffn_rows_gate_kernel<kSets, kTiles, TS_FFN_GELU, kKeep><<<grid, threads, 0, s>>>(p);
  } else {
    ffn_rows_gate_kernel<kSets, kTiles, TS_FFN_RELU2, kKeep><<<grid, threads, 0, s>>>(p);
  }
  return check_launch("ffn_rows_gate");
}

template <int kSets, int kTiles>
int ffn_rows_down(const FfnRowsParams& p, cudaStream_t s) {
  // CTAs of a cluster share a tile's inner length: until two CTAs are there for each SM, or a warp has one batch
  const int tiles = (p.out + 16 * kSets - 1) / (16 * kSets), blocks = (p.hidden + 31) / 32;
  int ranks = 1;
  while (ranks < rows_ranks(kSets * kTiles) && tiles * ranks < 2 * 148 && blocks > ranks * kRowsWarps * kRowsBatch / kSets) ranks *= 2;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles * ranks));
  config.blockDim = dim3(32 * kRowsWarps);
  config.stream = s;
  config.attrs = attr;
  config.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, ffn_rows_down_kernel<kSets, kTiles>, p);
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "ffn_rows_down: %s", cudaGetErrorString(e));
  return check_launch("ffn_rows_down");
}

// Two sets of weight rows to a warp read x half as often, one set has twice the
// CTAs: two where there are several tiles of rows and CTAs enough all the same
// (2048 x 5632, 9 / 16 / 32 rows: 25.9 / 25.9 / 31.7 us with two, 27.3 / 29.7 /
// 37.6 with one; 1024 x 4096: 13.1 / 13.3 / 13.9 and 12.1 / 12.9 / 17.8).
constexpr int kRowsCtas = 148;

template <int kTiles>
int ffn_rows_launch(const FfnRowsParams& p, int activation, cudaStream_t s) {
  constexpr int kSets = kTiles > 1 ? 2 : 1;
  const bool wide = p.hidden / (8 * kSets) >= kRowsCtas;
  const int rc = p.kept ? (wide ? ffn_rows_gate<kSets, kTiles, true>(p, activation, s)
                                : ffn_rows_gate<1, kTiles, true>(p, activation, s))
                        : (wide ? ffn_rows_gate<kSets, kTiles, false>(p, activation, s)
                                : ffn_rows_gate<1, kTiles, false>(p, activation, s));
  if (rc) return rc;
  return p.out / (16 * kSets) * rows_ranks(kSets * kTiles) >= kRowsCtas ? ffn_rows_down<kSets, kTiles>(p, s)
                                                        : ffn_rows_down<1, kTiles>(p, s);
}

}  // namespace

int ffn_rows_fwd(const ts_ffn_args* a, void* h, cudaStream_t s) {
  FfnRowsParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(a->x);
  p.wg = static_cast<const __nv_bfloat16*>(a->w_gate);
  p.wu = static_cast<const __nv_bfloat16*>(a->w_up);
  p.wd = static_cast<const __nv_bfloat16*>(a->w_down);
  p.xs = a->x_stride;
  p.wgs = a->w_gate_stride;
  p.wus = a->w_up_stride;
  p.wds = a->w_down_stride;
  p.h = static_cast<__nv_bfloat16*>(h);
  p.y = static_cast<__nv_bfloat16*>(a->y);
  p.kept = static_cast<uint8_t*>(a->kept);
  p.rows = static_cast<int>(a->rows);
  p.width = a->width;
  p.hidden = a->hidden;
  p.out = a->width_out;
  if (a->rows <= 8) return ffn_rows_launch<1>(p, a->activation, s);
  if (a->rows <= 16) return ffn_rows_launch<2>(p, a->activation, s);
  return ffn_rows_launch<4>(p, a->activation, s);
}

}  // namespace ts
