// The gated feed-forward block and its backward pass on the tensor cores.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// bf16 operands, f32 accumulators in tensor memory; every stored value (h, y,
// dg, du and the gradients) is rounded once, from f32.  Four launches:
//
//   kGateFwd   both projections, the activation and the product: h
//   kProduct   y = h Wd^T
//   kGateBwd   dh, and g and u AGAIN, in one tile: dg, du and h.  Keeping g and
//              u from the forward would either round them (their error then
//              enters dg and du on top of dg's own rounding) or cost 16 bytes
//              of traffic per hidden element in f32; the two products cost
//              4 D operations per hidden element, which is as long as that
//              traffic at D = 900 and buys that nothing of the block is kept
//              for the backward but its input.
//   kProduct   dx, dWg, dWu and dWd: one launch over all their tiles
//
// A pair of CTAs (cta_group::2) computes a tile of 256 x 256: each loads its
// own 128 rows of A and its half of B's 256 rows, so an SM reads each operand
// byte for twice the arithmetic of a single CTA's tile.  Gate tiles are 256 x
// 128 hidden columns: one CTA of the pair loads rows of Wg, the other of Wu,
// and one N = 256 instruction forms g and u side by side, in the same lanes,
// where the epilogue needs them.  Warp 0 feeds a ring of kStages stages by
// TMA, a thread of warp 1 (of the leading CTA) issues the instructions, warps
// 4-11 take accumulators out of tensor memory while the next tile's are formed
// in the other half of it.  In kGateBwd three accumulators of 128 columns do
// not fit twice; the next tile's dh (two columns blocks in turn) is formed
// while this tile's epilogue still reads g and u.
//
// A product of few tiles and a long inner length (the weight gradients: the
// inner length is the number of tokens) is split along it; partial tiles go to
// a workspace in f32 and the CTA that finishes a tile last adds them in the
// order of the splits, so the result does not depend on timing.
#include <cmath>
#include <cstring>

#include "capi_internal.h"
#include "common.cuh"
#include "tma.cuh"

namespace ts {

namespace {

constexpr int kFfnThreads = 384;             // warps: 0 loads, 1 issues, 2 tensor memory, 4-11 epilogue
constexpr int kStages = 5;
constexpr uint32_t kStageBytes = 32768;      // a CTA's part: 16 KB of A, 16 KB of B
constexpr uint32_t kOutBlock = 4096;         // 32 rows x 64 bf16 columns
constexpr uint32_t kFfnSmem = kStages * kStageBytes + 8 * 2 * kOutBlock + 1024;
constexpr int kPairs = 74;
constexpr int kMinSplitSteps = 8;

enum FfnMode { kGateFwd = 0, kGateBwd = 1, kProduct = 2 };

// One product of a launch: C[M, N] = sum over segments A_i B_i^T.
struct FfnProblem {
  CUtensorMap a[2], b[2];    // per segment; gate modes: a = {x, dy}, b = {Wg, Wu}
  CUtensorMap out[3];        // product: {C}; gate modes: {h, dg, du}
  CUtensorMap b_down;        // kGateBwd: Wd
  int rows, cols;            // of C
  int tiles_n;
  int steps[2];              // 64-wide inner steps of each segment (kGateBwd: of x, of dy)
  int splits;
  int units;                 // tiles * splits
  int a_mn, b_mn;            // operands stored with M (N) contiguous
  float* partial;
  int* counters;
};

template <int kCount>
struct FfnParams {
  FfnProblem p[kCount];
  int count;
  int units;
};

// ---- pair-of-CTAs forms of the tensor-core instructions

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Cluster address of `bar` in the pair's leading CTA.
__device__ __forceinline__ uint32_t leader_addr(const void* bar) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
  return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// mbar_wait() at cluster scope: bounded by about a second, after which the error is recorded.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int code) {
  if (try_wait_cluster(bar, parity)) return true;
  const uint64_t start = globaltimer_ns();
  for (uint32_t i = 0; i < (1u << 24); ++i) {
    if (try_wait_cluster(bar, parity)) return true;
    if ((i & 255u) == 255u) {
      if (globaltimer_ns() - start > 1000000000ull) break;
      if (device_failed()) return false;
    }
  }
  record_error(code);
  return false;
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` (the same offset) in both CTAs when the instructions issued so far are done.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// Load a box into this CTA's shared memory, its bytes counted on the leading CTA's barrier.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Wait until at most kLeft of this thread's newest stores still read shared memory.
template <int kLeft>
__device__ __forceinline__ void tma_store_read_wait() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory");
}

// 16 columns of this lane's row at each of two (three) column addresses, one wait for all.
__device__ __forceinline__ void tmem_ld16x2(uint32_t a, uint32_t b, float (&x)[16], float (&y)[16]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a), "r"(b)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = __uint_as_float(r[i]);
    y[i] = __uint_as_float(r[16 + i]);
  }
}
__device__ __forceinline__ void tmem_ld16x3(uint32_t a, uint32_t b, uint32_t c, float (&x)[16], float (&y)[16],
                                            float (&z)[16]) {
  uint32_t r[48];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%48];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%49];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47}, [%50];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47])
      : "r"(a), "r"(b), "r"(c)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = __uint_as_float(r[i]);
    y[i] = __uint_as_float(r[16 + i]);
    z[i] = __uint_as_float(r[32 + i]);
  }
}

// ---- activations: value and slope

constexpr int kSilu = TS_FFN_SILU, kGelu = TS_FFN_GELU, kRelu2 = TS_FFN_RELU2;

template <int kAct>
__device__ __forceinline__ float ffn_act(float g, float& slope) {
  if (kAct == kSilu) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    slope = s * fmaf(g, 1.f - s, 1.f);
    return g * s;
  }
  if (kAct == kGelu) {
    // by erfc: 1 + erf would cancel where g is negative
    const float s = 0.5f * erfcf(g * -0.70710678118654752f);
    slope = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), s);
    return g * s;
  }
  const float s = fmaxf(g, 0.f);
  slope = 2.f * s;
  return s * s;
}

// ---- one unit of work

struct FfnUnit {
  const FfnProblem* p;
  int m, n;             // first row and column of the pair's tile
  int begin, end;       // inner steps
  int split, tile;
};

template <int kMode, int kCount>
__device__ __forceinline__ FfnUnit ffn_unit(const FfnParams<kCount>& q, int unit) {
  int i = 0;
  while (i + 1 < q.count && unit >= q.p[i].units) {
    unit -= q.p[i].units;
    ++i;
  }
  FfnUnit u;
  u.p = &q.p[i];
  const int splits = u.p->splits;
  u.tile = unit / splits;
  u.split = unit - u.tile * splits;
  u.m = u.tile / u.p->tiles_n * 256;
  u.n = u.tile % u.p->tiles_n * (kMode == kProduct ? 256 : 128);
  const int steps = u.p->steps[0] + u.p->steps[1];
  u.begin = static_cast<int>(static_cast<long long>(steps) * u.split / splits);
  u.end = static_cast<int>(static_cast<long long>(steps) * (u.split + 1) / splits);
  return u;
}

// Whether `ok` holds in all of the CTA's 256 epilogue threads (a barrier among them).
__device__ __forceinline__ bool epilogue_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, r;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred r, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, r;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return all != 0;
}

// 16 bf16 columns of a lane's row into its staging block (128-byte rows, swizzled as the store expects).
__device__ __forceinline__ void stage16(uint32_t block, int lane, int c16, const float (&v)[16]) {
  st_shared_v4(block + sw128_offset(lane, 2 * c16), pack8(v));
  st_shared_v4(block + sw128_offset(lane, 2 * c16 + 1), pack8(v + 8));
}

template <int kMode, int kAct, int kCount>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFfnThreads, 1)
    ffn_kernel(const __grid_constant__ FfnParams<kCount> q) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int is_last;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 16);   // the epilogue warps of both CTAs
    }
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc_pair(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0 && lane == 0) {
    // ---- loads
    int it = 0;
    bool ok = true;
    for (int w = pair; w < q.units && ok; w += pairs) {
      const FfnUnit u = ffn_unit<kMode>(q, w);
      const FfnProblem& p = *u.p;
      const int row = u.m + 128 * static_cast<int>(rank);
      for (int k = u.begin; k < u.end; ++k, ++it) {
        const int s = it % kStages;
        if (!(ok = wait_cluster(&empty[s], ((it / kStages) & 1) ^ 1, kErrMmaTimeout))) break;
        const uint32_t a = base + s * kStageBytes, b = a + 16384;
        const uint32_t bar = leader_addr(&full[s]);
        if (kMode == kProduct) {
          const int seg = k < p.steps[0] ? 0 : 1;
          const int x = 64 * (k - (seg ? p.steps[0] : 0));
          const int col = u.n + 128 * static_cast<int>(rank);
          if (rank == 0) mbar_expect_tx(&full[s], 2 * kStageBytes);
          if (p.a_mn) {
            tma_load_pair(a, &p.a[seg], row, x, bar);
            tma_load_pair(a + 8192, &p.a[seg], row + 64, x, bar);
          } else {
            tma_load_pair(a, &p.a[seg], x, row, bar);
          }
          if (p.b_mn) {
            tma_load_pair(b, &p.b[seg], col, x, bar);
            tma_load_pair(b + 8192, &p.b[seg], col + 64, x, bar);
          } else {
            tma_load_pair(b, &p.b[seg], x, col, bar);
          }
        } else if (kMode == kGateBwd && k < p.steps[1]) {
          if (rank == 0) mbar_expect_tx(&full[s], 2 * 24576);
          tma_load_pair(a, &p.a[1], 64 * k, row, bar);
          tma_load_pair(b, &p.b_down, u.n + 64 * static_cast<int>(rank), 64 * k, bar);
        } else {
          const int x = 64 * (kMode == kGateBwd ? k - p.steps[1] : k);
          if (rank == 0) mbar_expect_tx(&full[s], 2 * kStageBytes);
          tma_load_pair(a, &p.a[0], x, row, bar);
          tma_load_pair(b, &p.b[rank], x, u.n, bar);
        }
      }
    }
    if (!ok && rank == 0) {
      // given up: let the pair's copies in flight land before its memory goes (for a bounded time too)
      for (int i = it > kStages ? it - kStages : 0; i < it; ++i)
        for (int poll = 0; poll < (1 << 16) && !try_wait_cluster(&full[i % kStages], (i / kStages) & 1); ++poll) {
        }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- instructions
    int it = 0, n_unit = 0;
    bool ok = true;
    for (int w = pair; w < q.units && ok; w += pairs, ++n_unit) {
      const FfnUnit u = ffn_unit<kMode>(q, w);
      const FfnProblem& p = *u.p;
      const bool a_mn = kMode == kProduct && p.a_mn, b_mn = kMode == kProduct && p.b_mn;
      const int buf = kMode == kGateBwd ? 0 : n_unit & 1;
      const uint32_t free_parity = ((kMode == kGateBwd ? n_unit : n_unit >> 1) & 1) ^ 1;
      uint32_t acc = tmem + (kMode == kGateBwd ? 256u : 256u * buf);
      bool waited = false;
      for (int k = u.begin; k < u.end; ++k, ++it) {
        const int s = it % kStages;
        const bool down = kMode == kGateBwd && k < p.steps[1];
        if (!down && !waited) {
          // dh's own columns were free before: the epilogue that read them had
          // ended when the tile in between could form its g and u
          waited = true;
          if (!(ok = wait_cluster(&acc_empty[buf], free_parity, kErrMmaTimeout))) break;
        }
        if (!(ok = wait_cluster(&full[s], (it / kStages) & 1, kErrCopyTimeout))) break;
        tc_fence_after();
        const uint32_t a = base + s * kStageBytes, b = a + 16384;
        if (down) {
          const uint32_t id = idesc_bf16(256, 128, false, true);
          const uint32_t d = tmem + 128u * (n_unit & 1);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_pair(d, smem_desc_sw128(a + 32 * j, 16, 1024), smem_desc_sw128(b + 2048 * j, 8192, 1024), id,
                     k > u.begin || j > 0);
        } else {
          const uint32_t id = idesc_bf16(256, 256, a_mn, b_mn);
          const int first = kMode == kGateBwd ? p.steps[1] : u.begin;
          const uint32_t a_step = a_mn ? 2048 : 32, b_step = b_mn ? 2048 : 32;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_pair(acc, smem_desc_sw128(a + a_step * j, a_mn ? 8192 : 16, 1024),
                     smem_desc_sw128(b + b_step * j, b_mn ? 8192 : 16, 1024), id, k > first || j > 0);
        }
        mma_commit_pair(&empty[s]);
      }
      if (ok) mma_commit_pair(&acc_full[buf]);
    }
  } else if (warp >= 4) {
    // ---- accumulators out
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t stage = base + kStages * kStageBytes + (warp - 4) * 2 * kOutBlock;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    uint32_t turn = 0;
    int n_unit = 0;
    // the next staging block, once its store of two before has been read
    auto next_block = [&]() {
      if (lane == 0) tma_store_read_wait<1>();
      __syncwarp();
      return stage + (turn++ & 1) * kOutBlock;
    };
    auto store_block = [&](const CUtensorMap* map, uint32_t block, int x, int y, const FfnProblem& p) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        // a group for every block, empty where it lies outside: next_block() counts them
        if (x < p.cols && y < p.rows) tma_store_2d(map, x, y, block);
        tma_store_commit();
      }
    };
    for (int w = pair; w < q.units; w += pairs, ++n_unit) {
      const FfnUnit u = ffn_unit<kMode>(q, w);
      const FfnProblem& p = *u.p;
      const int buf = kMode == kGateBwd ? 0 : n_unit & 1;
      bool ok = wait_cluster(&acc_full[buf], (kMode == kGateBwd ? n_unit : n_unit >> 1) & 1, kErrMmaTimeout);
      // the warps of a product meet in barriers below: they go on, or give up, together
      if (kMode == kProduct) ok = epilogue_all(ok);
      if (!ok) break;
      tc_fence_after();
      const int row0 = u.m + 128 * static_cast<int>(rank) + 32 * quad;
      if (kMode == kProduct) {
        const uint32_t acc = tmem + 256u * buf + lanes;
        float* part = p.partial + (static_cast<size_t>(u.tile) * p.splits * 2 + rank) * 32768;
        if (p.splits > 1) {
          float* mine = part + static_cast<size_t>(u.split) * 65536 + 32 * quad + lane;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float v[16];
            tmem_ld16(acc + 128 * half + 16 * c, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) __stcg(mine + (128 * half + 16 * c + e) * 128, v[e]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(leader_addr(&acc_empty[buf]));
          __threadfence();
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (threadIdx.x == 128) is_last = atomicAdd(&p.counters[u.tile * 2 + rank], 1) == p.splits - 1;
          asm volatile("bar.sync 1, 256;" ::: "memory");
          const bool last = is_last != 0;
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (!last) continue;
          __threadfence();
        }
#pragma unroll
        for (int half64 = 0; half64 < 2; ++half64) {
          const uint32_t block = next_block();
          const int c0 = 128 * half + 64 * half64;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[16];
            if (p.splits > 1) {
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = 0.f;
              for (int i = 0; i < p.splits; ++i) {
                const float* from = part + static_cast<size_t>(i) * 65536 + (c0 + 16 * c) * 128 + 32 * quad + lane;
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] += __ldcg(from + e * 128);
              }
            } else {
              tmem_ld16(acc + c0 + 16 * c, v);
            }
            stage16(block, lane, c, v);
          }
          if (p.splits == 1 && half64 == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(leader_addr(&acc_empty[buf]));
          }
          store_block(&p.out[0], block, u.n + c0, row0, p);
        }
      } else if (kMode == kGateFwd) {
        const uint32_t acc = tmem + 256u * buf + lanes + 64 * half;
        const uint32_t block = next_block();
        // rolled: the unrolled code of the activations outgrows the instruction cache
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float g[16], v[16], slope;
          tmem_ld16x2(acc + 16 * c, acc + 128 + 16 * c, g, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= ffn_act<kAct>(g[e], slope);
          stage16(block, lane, c, v);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(leader_addr(&acc_empty[buf]));
        store_block(&p.out[0], block, u.n + 64 * half, row0, p);
      } else {
        const uint32_t dh_at = tmem + 128u * (n_unit & 1) + lanes + 64 * half, acc = tmem + 256u + lanes + 64 * half;
        uint32_t du[4][8], h[4][8];
        uint32_t block = next_block();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float dh[16], g[16], v[16];
          tmem_ld16x3(dh_at + 16 * c, acc + 16 * c, acc + 128 + 16 * c, dh, g, v);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float s0, s1;
            const float a0 = ffn_act<kAct>(g[e], s0), a1 = ffn_act<kAct>(g[e + 1], s1);
            h[c][e / 2] = pack_bf16(a0 * v[e], a1 * v[e + 1]);
            du[c][e / 2] = pack_bf16(dh[e] * a0, dh[e + 1] * a1);
            g[e] = dh[e] * v[e] * s0;
            g[e + 1] = dh[e + 1] * v[e + 1] * s1;
          }
          stage16(block, lane, c, g);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(leader_addr(&acc_empty[buf]));
        store_block(&p.out[1], block, u.n + 64 * half, row0, p);
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          block = next_block();
          const uint32_t(&x)[4][8] = o ? h : du;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            st_shared_v4(block + sw128_offset(lane, 2 * c), make_uint4(x[c][0], x[c][1], x[c][2], x[c][3]));
            st_shared_v4(block + sw128_offset(lane, 2 * c + 1), make_uint4(x[c][4], x[c][5], x[c][6], x[c][7]));
          }
          store_block(&p.out[o ? 0 : 2], block, u.n + 64 * half, row0, p);
        }
      }
    }
    if (lane == 0) tma_store_read_wait<0>();
  }
  // both CTAs stay until neither's memory is needed
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 2) tmem_dealloc_pair(tmem, 512);
}

// ---- host side

struct FfnShape {
  long long rows;
  int width, hidden, width_out;
};

int ffn_steps(long long k) { return static_cast<int>((k + 63) / 64); }
long long ffn_tiles(long long n, int size) { return (n + size - 1) / size; }

// Make the current device's context current in this thread: encoding a tensor
// map needs one, and a thread that has made no runtime call yet (an autograd
// worker's) has none.
bool ffn_bind_context() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess;
}

// Matrix [outer, inner] of bf16, inner contiguous: a map with boxes of 64 x `box`.
bool ffn_map(CUtensorMap* map, const void* base, long long outer, int inner, long long stride, uint32_t box) {
  const uint64_t dims[2] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(outer)};
  const int64_t strides[1] = {stride};
  const uint32_t boxes[2] = {64, box};
  return make_tmap_bf16_sw128(map, base, 2, dims, strides, boxes);
}

// Splits of a product's inner length: enough units for every pair of SMs where
// the tiles alone leave some without work, each at least kMinSplitSteps long.
int ffn_splits(long long tiles, int steps) {
  if (tiles >= kPairs) return 1;
  long long s = kPairs / tiles;
  if (s > steps / kMinSplitSteps) s = steps / kMinSplitSteps;
  return s < 1 ? 1 : static_cast<int>(s);
}

struct FfnSpace {
  size_t partial = 0, counters = 0;   // floats, ints
};

// Shape part of a product (no pointers): its tiles, steps and splits; its needs are added to `space`.
void ffn_product(FfnProblem* p, long long rows, int cols, long long k0, long long k1, FfnSpace* space) {
  p->rows = static_cast<int>(rows);
  p->cols = cols;
  p->tiles_n = static_cast<int>(ffn_tiles(cols, 256));
  p->steps[0] = ffn_steps(k0);
  p->steps[1] = k1 ? ffn_steps(k1) : 0;
  const long long tiles = ffn_tiles(rows, 256) * p->tiles_n;
  p->splits = ffn_splits(tiles, p->steps[0] + p->steps[1]);
  p->units = static_cast<int>(tiles * p->splits);
  if (p->splits > 1) {
    space->partial += static_cast<size_t>(p->units) * 65536;
    space->counters += static_cast<size_t>(tiles) * 2;
  }
}

void ffn_place(FfnProblem* p, float*& partial, int*& counters) {
  if (p->splits <= 1) return;
  p->partial = partial;
  p->counters = counters;
  partial += static_cast<size_t>(p->units) * 65536;
  counters += p->units / p->splits * 2;
}

template <int kMode, int kAct, int kCount>
int ffn_launch(FfnParams<kCount>& q, cudaStream_t s, const char* what) {
  q.units = 0;
  for (int i = 0; i < q.count; ++i) q.units += q.p[i].units;
  if (q.units == 0) return TS_OK;
  // an attribute of the function on the current device
  const cudaError_t set = cudaFuncSetAttribute(ffn_kernel<kMode, kAct, kCount>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kFfnSmem);
  if (set != cudaSuccess) return set_error(TS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(set));
  const int pairs = q.units < kPairs ? q.units : kPairs;
  ffn_kernel<kMode, kAct, kCount><<<2 * pairs, kFfnThreads, kFfnSmem, s>>>(q);
  return check_launch(what);
}

template <int kMode>
int ffn_launch_gate(FfnParams<1>& q, int activation, cudaStream_t s, const char* what) {
  if (activation == kSilu) return ffn_launch<kMode, kSilu>(q, s, what);
  if (activation == kGelu) return ffn_launch<kMode, kGelu>(q, s, what);
  return ffn_launch<kMode, kRelu2>(q, s, what);
}

size_t ffn_align(size_t x) { return (x + 1023) & ~static_cast<size_t>(1023); }

int ffn_check(const ts_ffn_args* a) {
  if (!a) return set_error(TS_ERR_VALUE, "ffn: null arguments");
  if (a->rows < 1 || a->rows > (1ll << 30)) return set_error(TS_ERR_VALUE, "ffn: rows must lie in 1..2^30");
  for (int d : {a->width, a->hidden, a->width_out})
    if (d < 8 || d % 8 || d > (1 << 20))
      return set_error(TS_ERR_NOT_IMPLEMENTED, "ffn: width %d must be a multiple of 8 in 8..2^20", d);
  if (a->activation < kSilu || a->activation > kRelu2)
    return set_error(TS_ERR_VALUE, "ffn: unknown activation %d", a->activation);
  // tiles of the largest product, split or not, count in 32 bits
  if (ffn_tiles(a->rows, 256) * ffn_tiles(a->hidden, 128) > (1 << 28) ||
      ffn_tiles(a->rows, 256) * ffn_tiles(a->width, 256) > (1 << 28) ||
      ffn_tiles(a->rows, 256) * ffn_tiles(a->width_out, 256) > (1 << 28))
    return set_error(TS_ERR_NOT_IMPLEMENTED, "ffn: too many tiles");
  return TS_OK;
}

const char* const kFfnLayout = "ffn: every matrix needs a 16-byte aligned base and a row stride that is a multiple of 8";

struct FfnForward {
  FfnProblem down = {};
  FfnSpace space;
  size_t h = 0, partial = 0, counters = 0, total = 0;
};

FfnForward ffn_forward(const ts_ffn_args* a) {
  FfnForward f;
  ffn_product(&f.down, a->rows, a->width_out, a->hidden, 0, &f.space);
  f.partial = ffn_align(static_cast<size_t>(a->rows) * a->hidden * 2);
  f.counters = f.partial + ffn_align(f.space.partial * 4);
  f.total = f.counters + ffn_align(f.space.counters * 4);
  return f;
}

struct FfnBackward {
  FfnProblem p[4] = {};   // dWg, dWu, dWd, dx
  FfnSpace space;
  size_t dg = 0, du = 0, h = 0, partial = 0, counters = 0, total = 0;
};

FfnBackward ffn_backward(const ts_ffn_args* a) {
  FfnBackward b;
  ffn_product(&b.p[0], a->hidden, a->width, a->rows, 0, &b.space);
  ffn_product(&b.p[1], a->hidden, a->width, a->rows, 0, &b.space);
  ffn_product(&b.p[2], a->width_out, a->hidden, a->rows, 0, &b.space);
  ffn_product(&b.p[3], a->rows, a->width, a->hidden, a->hidden, &b.space);
  const size_t one = ffn_align(static_cast<size_t>(a->rows) * a->hidden * 2);
  b.du = one;
  b.h = 2 * one;
  b.partial = 3 * one;
  b.counters = b.partial + ffn_align(b.space.partial * 4);
  b.total = b.counters + ffn_align(b.space.counters * 4);
  return b;
}

}  // namespace

}  // namespace ts

extern "C" {

size_t ts_b200_ffn_fwd_workspace_bytes(const ts_ffn_args* a) {
  return ts::ffn_check(a) ? 0 : ts::ffn_forward(a).total;
}

int ts_b200_ffn_fwd(const ts_ffn_args* a, ts_stream_t stream) {
  using namespace ts;
  if (const int rc = ffn_check(a)) return rc;
  if (!a->x || !a->w_gate || !a->w_up || !a->w_down || !a->y) return set_error(TS_ERR_VALUE, "ffn_fwd: null pointer");
  FfnForward f = ffn_forward(a);
  if (!a->workspace || a->workspace_bytes < f.total) return set_error(TS_ERR_VALUE, "ffn_fwd: workspace too small");
  if (!ffn_bind_context()) return set_error(TS_ERR_CUDA, "ffn_fwd: no context on the current device");
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  void* h = ws;
  FfnParams<1> gate = {};
  gate.count = 1;
  FfnProblem& p = gate.p[0];
  p.rows = static_cast<int>(a->rows);
  p.cols = a->hidden;
  p.tiles_n = static_cast<int>(ffn_tiles(a->hidden, 128));
  p.steps[0] = ffn_steps(a->width);
  p.splits = 1;
  p.units = static_cast<int>(ffn_tiles(a->rows, 256)) * p.tiles_n;
  if (!ffn_map(&p.a[0], a->x, a->rows, a->width, a->x_stride, 128) ||
      !ffn_map(&p.b[0], a->w_gate, a->hidden, a->width, a->w_gate_stride, 128) ||
      !ffn_map(&p.b[1], a->w_up, a->hidden, a->width, a->w_up_stride, 128) ||
      !ffn_map(&p.out[0], h, a->rows, a->hidden, a->hidden, 32))
    return set_error(TS_ERR_VALUE, kFfnLayout);
  FfnParams<1> down = {};
  down.count = 1;
  down.p[0] = f.down;
  float* partial = reinterpret_cast<float*>(ws + f.partial);
  int* counters = reinterpret_cast<int*>(ws + f.counters);
  if (f.space.counters) {
    const cudaError_t e = cudaMemsetAsync(counters, 0, f.space.counters * sizeof(int), stream);
    if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "ffn_fwd: %s", cudaGetErrorString(e));
  }
  ffn_place(&down.p[0], partial, counters);
  if (!ffn_map(&down.p[0].a[0], h, a->rows, a->hidden, a->hidden, 128) ||
      !ffn_map(&down.p[0].b[0], a->w_down, a->width_out, a->hidden, a->w_down_stride, 128) ||
      !ffn_map(&down.p[0].out[0], a->y, a->rows, a->width_out, a->width_out, 32))
    return set_error(TS_ERR_VALUE, kFfnLayout);
  if (const int rc = ffn_launch_gate<kGateFwd>(gate, a->activation, stream, "ffn_gate_fwd")) return rc;
  return ffn_launch<kProduct, 0>(down, stream, "ffn_down");
}

size_t ts_b200_ffn_bwd_workspace_bytes(const ts_ffn_args* a) {
  return ts::ffn_check(a) ? 0 : ts::ffn_backward(a).total;
}

int ts_b200_ffn_bwd(const ts_ffn_args* a, const ts_ffn_grad_args* g, ts_stream_t stream) {
  using namespace ts;
  if (const int rc = ffn_check(a)) return rc;
  if (!g || !a->x || !a->w_gate || !a->w_up || !a->w_down || !g->dy)
    return set_error(TS_ERR_VALUE, "ffn_bwd: null pointer");
  FfnBackward b = ffn_backward(a);
  if (!a->workspace || a->workspace_bytes < b.total) return set_error(TS_ERR_VALUE, "ffn_bwd: workspace too small");
  if (!ffn_bind_context()) return set_error(TS_ERR_CUDA, "ffn_bwd: no context on the current device");
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  void *dg = ws + b.dg, *du = ws + b.du, *h = ws + b.h;
  const long long M = a->rows;
  const int D = a->width, H = a->hidden, O = a->width_out;
  FfnParams<1> gate = {};
  gate.count = 1;
  FfnProblem& p = gate.p[0];
  p.rows = static_cast<int>(M);
  p.cols = H;
  p.tiles_n = static_cast<int>(ffn_tiles(H, 128));
  p.steps[0] = ffn_steps(D);
  p.steps[1] = ffn_steps(O);
  p.splits = 1;
  p.units = static_cast<int>(ffn_tiles(M, 256)) * p.tiles_n;
  bool ok = ffn_map(&p.a[0], a->x, M, D, a->x_stride, 128) && ffn_map(&p.a[1], g->dy, M, O, g->dy_stride, 128) &&
            ffn_map(&p.b[0], a->w_gate, H, D, a->w_gate_stride, 128) &&
            ffn_map(&p.b[1], a->w_up, H, D, a->w_up_stride, 128) &&
            ffn_map(&p.b_down, a->w_down, O, H, a->w_down_stride, 64) && ffn_map(&p.out[0], h, M, H, H, 32) &&
            ffn_map(&p.out[1], dg, M, H, H, 32) && ffn_map(&p.out[2], du, M, H, H, 32);
  if (!ok) return set_error(TS_ERR_VALUE, kFfnLayout);
  FfnParams<4> grads = {};
  float* partial = reinterpret_cast<float*>(ws + b.partial);
  int* counters = reinterpret_cast<int*>(ws + b.counters);
  if (b.space.counters) {
    const cudaError_t e = cudaMemsetAsync(counters, 0, b.space.counters * sizeof(int), stream);
    if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "ffn_bwd: %s", cudaGetErrorString(e));
  }
  // dWg = dg^T x, dWu = du^T x, dWd = dy^T h: the inner dimension is the tokens, outside in every operand
  auto weight = [&](FfnProblem& w, const void* left, long long left_cols, long long left_stride, const void* right,
                    int right_cols, long long right_stride, void* out) {
    if (!out) return true;
    w.a_mn = w.b_mn = 1;
    ffn_place(&w, partial, counters);
    const bool mapped = ffn_map(&w.a[0], left, M, static_cast<int>(left_cols), left_stride, 64) &&
                        ffn_map(&w.b[0], right, M, right_cols, right_stride, 64) &&
                        ffn_map(&w.out[0], out, left_cols, right_cols, right_cols, 32);
    grads.p[grads.count++] = w;
    return mapped;
  };
  ok = weight(b.p[0], dg, H, H, a->x, D, a->x_stride, g->dw_gate) &&
       weight(b.p[1], du, H, H, a->x, D, a->x_stride, g->dw_up) &&
       weight(b.p[2], g->dy, O, g->dy_stride, h, H, H, g->dw_down);
  if (ok && g->dx) {
    FfnProblem& x = b.p[3];
    x.b_mn = 1;
    ffn_place(&x, partial, counters);
    ok = ffn_map(&x.a[0], dg, M, H, H, 128) && ffn_map(&x.a[1], du, M, H, H, 128) &&
         ffn_map(&x.b[0], a->w_gate, H, D, a->w_gate_stride, 64) &&
         ffn_map(&x.b[1], a->w_up, H, D, a->w_up_stride, 64) && ffn_map(&x.out[0], g->dx, M, D, D, 32);
    grads.p[grads.count++] = x;
  }
  if (!ok) return set_error(TS_ERR_VALUE, kFfnLayout);
  if (grads.count == 0) return TS_OK;
  if (const int rc = ffn_launch_gate<kGateBwd>(gate, a->activation, stream, "ffn_gate_bwd")) return rc;
  return ffn_launch<kProduct, 0>(grads, stream, "ffn_grads");
}

}  // extern "C"
