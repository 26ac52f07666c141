// The gated feed-forward block and its backward pass on the tensor cores.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// bf16 operands, f32 accumulators in tensor memory; every stored value (h, y,
// dg, du and the gradients) is rounded once, from f32.  Launches:
//
//   kGateFwd   both projections, the activation and the product: h; for a
//              backward pass also g and u, in 24 bits (the f32 without its last
//              byte, within 2^-15: a bf16 copy would double the error of dg
//              and du, an f32 copy costs a third more traffic)
//   kProduct   y = h Wd^T
//   kGateGrad  dh = dy Wd and, from g and u, dg and du
//   kProduct   dx, dWg, dWu and dWd: one launch over all their tiles
//
// Up to kRowsMost rows the forward is ffn_rows.cu's, with gradients too, and h,
// dg and du pass in two bf16 parts each (kGateGradTwo, and products over twice
// the segments): with few rows the errors of a few large hidden values do not
// average out (2.6e-3 of dx's norm now and then, 1.66e-3 so).
//
// Forming g and u again in the backward instead of keeping them was built
// first and measured slower: dh, g and u then share a tile of 128 hidden
// columns, and the N = 128 instructions of dh run at half the rate of N = 256
// ones (65536 x 512 x 1024: 261 us; 8192 x 2048 x 5632: 632 us).
//
// A pair of CTAs (cta_group::2) computes a tile of 256 x 256: each loads its
// own 128 rows of A and its half of B's 256 rows, so an SM reads each operand
// byte for twice the arithmetic of a single CTA's tile.  kGateFwd's tiles are
// 256 x 128 hidden columns: one CTA of the pair loads rows of Wg, the other of
// Wu, and one N = 256 instruction forms g and u side by side, in the same
// lanes, where the epilogue needs them.  Warp 0 feeds a ring of kStages stages
// by TMA, a thread of warp 1 (of the leading CTA) issues the instructions,
// sixteen more warps take accumulators out of tensor memory while the next
// tile's are formed in the other half of it.
//
// What bounds it.  At 8192 x 2048 x 5632 a forward and backward pass takes
// 1460 to 1590 us from box to box, 1.17 to 1.07 PFLOP/s, where cuBLAS holds 1.37
// in a loop of a large product under the power limit; kGateFwd takes 350 us there (290 without keeping g and
// u), its instructions alone, loads left out, 248, its loads alone 174 (63
// bytes a cycle into each SM): both near their limits at once.  At 65536 x 512
// x 1024 (630 to 740 us) the inner length is eight steps, and the traffic of what is
// kept and exchanged counts: kGateFwd 153 us (134 with the instructions left
// out), kGateGrad 139 (737 MB), the gradients 262, the down product 73.
// An operand whose tile is 64 rows of the inner dimension comes as one copy of
// two column blocks (a map of three dimensions) where its columns are a
// multiple of 64, else as two copies: at 8192 x 2048 x 5632 the loads of the
// weight gradients alone take 571 us one way and 648 the other.  Two groups of
// epilogue warps on alternate tiles, a sixth stage and other orders of the
// tiles measured no faster.
//
// A product of few tiles and a long inner length (the weight gradients: the
// inner length is the number of tokens) is split along it; partial tiles go to
// a workspace in f32 and the CTA that finishes a tile last adds them in the
// order of the splits, so the result does not depend on timing.  That takes
// some 10 us, which the launch of the gradients has other tiles to spend on.
// The down product of few rows has not: there the pairs that share a tile are
// one cluster, and each sends its sums of the columns that another pair
// finishes into that pair's shared memory (24 tiles of 44 steps: 19 us with the
// workspace).
#include <cmath>
#include <cstring>

#include "capi_internal.h"
#include "common.cuh"
#include "ffn.cuh"
#include "tma.cuh"

namespace ts {

namespace {

constexpr int kEpiWarps = 16;
constexpr int kFfnThreads = 128 + 32 * kEpiWarps;  // warps: 0 loads, 1 issues, 2 tensor memory, 4.. epilogue
constexpr int kStages = 5;
constexpr uint32_t kStageBytes = 32768;      // a CTA's part: 16 KB of A, 16 KB of B
constexpr uint32_t kOutBlock = 2048;         // 32 rows x 32 bf16 columns
constexpr uint32_t kFfnSmem = kStages * kStageBytes + kEpiWarps * 2 * kOutBlock + 1024;
constexpr int kPairs = 74;
constexpr int kMinSplitSteps = 8;

// kProductCluster: a product whose few tiles are each split among the pairs of a cluster.
// kGateGradTwo: kGateGrad with dg and du in two parts; kProductTwo: kProduct over such parts.
enum FfnMode { kGateFwd = 0, kGateGrad = 1, kProduct = 2, kProductCluster = 3, kGateGradTwo = 4, kProductTwo = 5 };
// Maps of each kind that a problem has: the launches of the two-part forms alone have to carry more than 4 KB.
constexpr int ffn_maps(int mode) { return mode == kGateGradTwo || mode == kProductTwo ? 4 : 2; }

// How an operand lies in memory: inner dimension contiguous; or M (N)
// contiguous, loaded as two boxes of 64 columns or as one of 2 x 64.
enum FfnLayout { kInner = 0, kOuter = 1, kOuterBlocks = 2 };

// One product of a launch: C[M, N] = sum over segments A_i B_i^T, all of one inner length.
struct FfnSizes {
  int rows, cols;            // of C
  int tiles_n;
  int segments, steps;       // 64-wide inner steps of each segment
  int splits;
  int units;                 // tiles * splits
  int a_layout, b_layout;
  float* partial;
  int* counters;
  uint8_t* kept;             // g and u (see keep_at), or null
};

template <int kMaps>
struct FfnProblemOf : FfnSizes {
  CUtensorMap a[kMaps], b[kMaps];   // per segment; kGateFwd: a[0] = x, b = {Wg, Wu}
  CUtensorMap out[kMaps];           // {C}; kGateGrad: {dg, du}; kGateGradTwo: and the rests of both
};
using FfnProblem = FfnProblemOf<4>;

template <int kCount, int kMaps = 4>
struct FfnParams {
  FfnProblemOf<kMaps> p[kCount];
  int count;
  int units;
  int* clear;        // counters of the launch after this one, set to zero (or null)
  int clear_count;
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
// Cluster address of `at` (a shared address of this CTA) in the CTA of that rank.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t at, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
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
// Arrive on `bar` (the same offset) in both CTAs of the pair led by `lead` when the instructions issued so far are done.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3u << lead))
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
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// This CTA's 128 rows (from `row`, a multiple of 64) of an operand at inner step `k`.
__device__ __forceinline__ void ffn_load(uint32_t dst, const CUtensorMap* map, int layout, int row, int k, uint32_t bar) {
  if (layout == kInner) {
    tma_load_pair(dst, map, 64 * k, row, bar);
  } else if (layout == kOuterBlocks) {
    tma_load_pair(dst, map, 0, 64 * k, row >> 6, bar);
  } else {
    tma_load_pair(dst, map, row, 64 * k, bar);
    tma_load_pair(dst + 8192, map, row + 64, 64 * k, bar);
  }
}
// ---- g and u between the passes (keep_at)

// 16 values from r[c] on, as three vectors.
__device__ __forceinline__ void keep16(uint8_t* to, const uint32_t (&r)[32], int c) {
  uint32_t high[8], low[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) high[i] = __byte_perm(r[c + 2 * i], r[c + 2 * i + 1], 0x7632);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    low[i] = __byte_perm(__byte_perm(r[c + 4 * i], r[c + 4 * i + 1], 0x0051),
                         __byte_perm(r[c + 4 * i + 2], r[c + 4 * i + 3], 0x0051), 0x5410);
  uint4* q = reinterpret_cast<uint4*>(to);
  __stcs(q, make_uint4(high[0], high[1], high[2], high[3]));
  __stcs(q + 32, make_uint4(high[4], high[5], high[6], high[7]));
  __stcs(q + 64, make_uint4(low[0], low[1], low[2], low[3]));
}

// g and u of 16 columns of a lane's row.
struct KeptHalf {
  uint32_t high[2][8], low[2][4];
  __device__ __forceinline__ void load(const uint8_t* from) {
    const uint4* q = reinterpret_cast<const uint4*>(from);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 a = __ldcs(q + 96 * i), b = __ldcs(q + 96 * i + 32), c = __ldcs(q + 96 * i + 64);
      high[i][0] = a.x; high[i][1] = a.y; high[i][2] = a.z; high[i][3] = a.w;
      high[i][4] = b.x; high[i][5] = b.y; high[i][6] = b.z; high[i][7] = b.w;
      low[i][0] = c.x; low[i][1] = c.y; low[i][2] = c.z; low[i][3] = c.w;
    }
  }
  // The word again, with its third byte in the place of the lost fourth too:
  // nearer to the middle of what was cut off than zero on average (255 units of
  // 2^-23 at most), and zero and infinity stay what they are.
  __device__ __forceinline__ float value(int i, int e) const {
    const uint32_t byte = 4 + (e & 3), half = e & 1 ? 0x3200 : 0x1000;
    return __uint_as_float(__byte_perm(high[i][e >> 1], low[i][e >> 2], half | byte << 4 | byte));
  }
  __device__ __forceinline__ float gate(int e) const { return value(0, e); }
  __device__ __forceinline__ float up(int e) const { return value(1, e); }
};

// ---- one unit of work

template <int kMaps>
struct FfnUnit {
  const FfnProblemOf<kMaps>* p;
  int m, n;             // first row and column of the pair's tile
  int begin, end;       // inner steps
  int split, tile;
};

template <int kMode, int kCount, int kMaps>
__device__ __forceinline__ FfnUnit<kMaps> ffn_unit(const FfnParams<kCount, kMaps>& q, int unit) {
  int i = 0;
  while (i + 1 < q.count && unit >= q.p[i].units) {
    unit -= q.p[i].units;
    ++i;
  }
  FfnUnit<kMaps> u;
  u.p = &q.p[i];
  const int splits = u.p->splits;
  u.tile = unit / splits;
  u.split = unit - u.tile * splits;
  u.m = u.tile / u.p->tiles_n * 256;
  u.n = u.tile % u.p->tiles_n * (kMode == kGateFwd ? 128 : 256);
  const int steps = u.p->segments * u.p->steps;
  u.begin = static_cast<int>(static_cast<long long>(steps) * u.split / splits);
  u.end = static_cast<int>(static_cast<long long>(steps) * (u.split + 1) / splits);
  return u;
}

// Whether `ok` holds in all of the CTA's 512 epilogue threads (a barrier among them).
__device__ __forceinline__ bool epilogue_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, r;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred r, 1, 512, p;\n\t"
      "selp.u32 %0, 1, 0, r;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return all != 0;
}

// 16 bytes (8 bf16 columns) of a lane's row into its warp's staging block: 64-byte rows, swizzled as the store
// expects (the 16-byte chunk's index XORed with bits 1-2 of the row).
__device__ __forceinline__ void stage8(uint32_t block, int lane, int chunk, uint4 v) {
  st_shared_v4(block + 64 * lane + ((chunk ^ ((lane >> 1) & 3)) << 4), v);
}

template <int kMode, int kAct, int kCount>
__global__ void __launch_bounds__(kFfnThreads, 1)
    ffn_kernel(const __grid_constant__ FfnParams<kCount, ffn_maps(kMode)> q) {
  constexpr bool kGrad = kMode == kGateGrad || kMode == kGateGradTwo;
  constexpr bool kJoin = kMode == kProduct || kMode == kProductTwo;
  constexpr int kPasses = kMode == kGateGradTwo ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int is_last;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the CTA's place in its pair, and the rank in the cluster of the pair's leading CTA
  const uint32_t rank = cluster_rank() & 1, lead = cluster_rank() & ~1u;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpiWarps);   // the epilogue warps of both CTAs
    }
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc_pair(&tmem_slot, 512);
  if (warp == 3 && lane < q.count) {
    const auto& p = q.p[lane];
    tma_prefetch_map(&p.a[0]);
    tma_prefetch_map(&p.b[0]);
    tma_prefetch_map(&p.out[0]);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // up to here nothing of the launch before is read or written: this much overlaps its end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 3 && blockIdx.x == 0)
    for (int i = lane; i < q.clear_count; i += 32) q.clear[i] = 0;

  if (warp == 0 && lane == 0) {
    // ---- loads
    int it = 0;
    bool ok = true;
    for (int w = pair; w < q.units && ok; w += pairs) {
      const auto u = ffn_unit<kMode>(q, w);
      const auto& p = *u.p;
      const int row = u.m + 128 * static_cast<int>(rank);
      for (int k = u.begin; k < u.end; ++k, ++it) {
        const int s = it % kStages;
        if (!(ok = wait_cluster(&empty[s], ((it / kStages) & 1) ^ 1, kErrMmaTimeout))) break;
        const uint32_t a = base + s * kStageBytes, b = a + 16384;
        const uint32_t bar = cluster_addr(smem_u32(&full[s]), lead);
        if (rank == 0) mbar_expect_tx(&full[s], 2 * kStageBytes);
        if (kMode == kGateFwd) {
          ffn_load(a, &p.a[0], kInner, row, k, bar);
          ffn_load(b, &p.b[rank], kInner, u.n, k, bar);
        } else {
          // two segments at most, but for the products over two parts
          const int seg = kMode == kProductTwo ? k / p.steps : (k < p.steps ? 0 : 1);
          const int step = k - seg * p.steps;
          ffn_load(a, &p.a[seg], p.a_layout, row, step, bar);
          ffn_load(b, &p.b[seg], p.b_layout, u.n + 128 * static_cast<int>(rank), step, bar);
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
      const auto u = ffn_unit<kMode>(q, w);
      const auto& p = *u.p;
      const bool a_mn = p.a_layout != kInner, b_mn = p.b_layout != kInner;
      const int buf = n_unit & 1;
      const uint32_t acc = tmem + 256u * buf, id = idesc_bf16(256, 256, a_mn, b_mn);
      const uint32_t a_step = a_mn ? 2048 : 32, b_step = b_mn ? 2048 : 32;
      const uint32_t a_lbo = a_mn ? 8192 : 16, b_lbo = b_mn ? 8192 : 16;
      if (!(ok = wait_cluster(&acc_empty[buf], ((n_unit >> 1) & 1) ^ 1, kErrMmaTimeout))) break;
      for (int k = u.begin; k < u.end; ++k, ++it) {
        const int s = it % kStages;
        if (!(ok = wait_cluster(&full[s], (it / kStages) & 1, kErrCopyTimeout))) break;
        tc_fence_after();
        const uint32_t a = base + s * kStageBytes, b = a + 16384;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_pair(acc, smem_desc_sw128(a + a_step * j, a_lbo, 1024), smem_desc_sw128(b + b_step * j, b_lbo, 1024), id,
                   k > u.begin || j > 0);
        mma_commit_pair(&empty[s], lead);
      }
      if (ok) mma_commit_pair(&acc_full[buf], lead);
    }
  } else if (warp >= 4) {
    // ---- accumulators out: a warp takes the 32 rows of its quarter of tensor memory (warp % 4) and a quarter of
    // the columns
    const int quad = warp & 3, part = (warp - 4) >> 2;
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
    auto store_block = [&](const CUtensorMap* map, uint32_t block, int x, int y, const FfnSizes& p) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        // a group for every block, empty where it lies outside: next_block() counts them
        if (x < p.cols && y < p.rows) tma_store_2d(map, x, y, block);
        tma_store_commit();
      }
    };
    for (int w = pair; w < q.units; w += pairs, ++n_unit) {
      const auto u = ffn_unit<kMode>(q, w);
      const auto& p = *u.p;
      const int buf = n_unit & 1;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(cluster_addr(smem_u32(&acc_empty[buf]), lead));
      };
      const int row0 = u.m + 128 * static_cast<int>(rank) + 32 * quad;
      KeptHalf kept;
      const uint8_t* from = nullptr;
      if (kGrad) {
        // 64 columns of g and u: two blocks, the first half-block ahead of the wait
        from = keep_at(p.kept, p.cols, row0, u.n + 64 * part, lane);
        if (row0 < p.rows && u.n + 64 * part < p.cols) kept.load(from);
      }
      bool ok = wait_cluster(&acc_full[buf], (n_unit >> 1) & 1, kErrMmaTimeout);
      // the warps of a product meet in barriers below: they go on, or give up, together
      if (kJoin) ok = epilogue_all(ok);
      if (!ok) break;
      tc_fence_after();
      if (kMode == kProductCluster) break;   // its one tile goes on below
      if (kJoin) {
        const uint32_t acc = tmem + 256u * buf + lanes + 64 * part;
        float* sums = p.partial + (static_cast<size_t>(u.tile) * p.splits * 2 + rank) * 32768 + 64 * part * 128 +
                      32 * quad + lane;   // [split][rank][column][row]
        if (p.splits > 1) {
          float* mine = sums + static_cast<size_t>(u.split) * 65536;
#pragma unroll 1
          for (int c = 0; c < 64 && row0 < p.rows; c += 32) {
            uint32_t v[32];
            tmem_ld(acc + c, v);
            tmem_wait();
            tie(v);
#pragma unroll
            for (int e = 0; e < 32; ++e) __stcg(mine + (c + e) * 128, __uint_as_float(v[e]));
          }
          release();
          __threadfence();
          asm volatile("bar.sync 1, 512;" ::: "memory");
          if (threadIdx.x == 128) is_last = atomicAdd(&p.counters[u.tile * 2 + rank], 1) == p.splits - 1;
          asm volatile("bar.sync 1, 512;" ::: "memory");
          const bool last = is_last != 0;
          asm volatile("bar.sync 1, 512;" ::: "memory");
          if (!last) continue;
          __threadfence();
        }
        if (p.splits > 1 && row0 >= p.rows) continue;
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          const uint32_t block = next_block();
          float v[32];
          if (p.splits > 1) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.f;
            for (int i = 0; i < p.splits; ++i) {
              const float* from = sums + static_cast<size_t>(i) * 65536 + c * 128;
              float a[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) a[e] = __ldcg(from + e * 128);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] += a[e];
            }
          } else {
            uint32_t r[32];
            tmem_ld(acc + c, r);
            tmem_wait();
            tie(r);
            if (c == 32) release();
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) stage8(block, lane, i, pack8(v + 8 * i));
          store_block(&p.out[0], block, u.n + 64 * part + c, row0, p);
        }
      } else if (kMode == kGateFwd) {
        const uint32_t acc = tmem + 256u * buf + lanes + 32 * part;
        uint32_t g[32], v[32];
        tmem_ld(acc, g);
        tmem_ld(acc + 128, v);
        tmem_wait();
        tie(g);
        tie(v);
        release();
        const int col = u.n + 32 * part;
        if (p.kept && row0 < p.rows && col < p.cols) {
          uint8_t* to = keep_at(p.kept, p.cols, row0, col, lane);
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
            keep16(to + 6 * 512 * (c / 16), g, c);
            keep16(to + 6 * 512 * (c / 16) + 3 * 512, v, c);
          }
        }
        const uint32_t block = next_block();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float h[8], slope;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            h[e] = ffn_act<kAct>(__uint_as_float(g[8 * i + e]), slope) * __uint_as_float(v[8 * i + e]);
          stage8(block, lane, i, pack8(h));
        }
        store_block(&p.out[0], block, col, row0, p);
      } else {
        const uint32_t acc = tmem + 256u * buf + lanes + 64 * part;
        // blocks of 32 columns, in halves of 16; the next half's g and u are on their way meanwhile.  The second pass,
        // where there is one, stores what the first left.
#pragma unroll 1
        for (int turn_c = 0; turn_c < 64 * kPasses; turn_c += 32) {
          const int c = turn_c & 63, pass = kPasses > 1 ? turn_c >> 6 : 0;
          const int col = u.n + 64 * part + c;
          if (lane == 0) tma_store_read_wait<0>();
          __syncwarp();
#pragma unroll
          for (int o = 0; o < 32; o += 16) {
            uint32_t d[16];
            tmem_ld(acc + c + o, d);
            tmem_wait();
            tie(d);
            if (turn_c + o == 64 * kPasses - 16) release();
            KeptHalf next;
            // the columns after this half (or the first again), where they are this tile's and inside
            const int ahead = kPasses > 1 ? (c + o + 16) & 63 : c + o + 16;
            if (ahead < 64 && row0 < p.rows && u.n + 64 * part + (ahead & 32) < p.cols)
              next.load(from + (ahead >> 5) * TS_FFN_KEPT_BLOCK + ((ahead >> 4) & 1) * (6 * 512));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x[8], y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float dh = __uint_as_float(d[8 * i + e]);
                float slope;
                const float act = ffn_act<kAct>(kept.gate(8 * i + e), slope);
                x[e] = dh * kept.up(8 * i + e) * slope;
                y[e] = dh * act;
                if (kPasses > 1) {
                  x[e] = pass ? ffn_rest(x[e]) : ffn_high(x[e]);
                  y[e] = pass ? ffn_rest(y[e]) : ffn_high(y[e]);
                }
              }
              stage8(stage, lane, o / 8 + i, pack8(x));
              stage8(stage + kOutBlock, lane, o / 8 + i, pack8(y));
            }
            kept = next;
          }
          store_block(&p.out[2 * pass], stage, col, row0, p);
          store_block(&p.out[2 * pass + 1], stage + kOutBlock, col, row0, p);
        }
      }
    }
    if (lane == 0) tma_store_read_wait<0>();
  }
  if (kMode == kProductCluster) {
    // The pairs of the cluster hold sums of the same tile over their parts of the inner length.  Quarter p of its
    // columns is finished by pair p splits / 4; the others send it theirs: [sender][column][row], in the stages'
    // memory, which no instruction reads any more after the first barrier.
    const auto u = ffn_unit<kMode>(q, pair);
    const auto& p = *u.p;
    const int quad = warp & 3, part = (warp - 4) >> 2, owner = part * p.splits / 4;
    const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + 64 * part;
    const int row0 = u.m + 128 * static_cast<int>(rank) + 32 * quad;
    const bool inside = warp >= 4 && row0 < p.rows;
    // quarters of the owner before this one, and all of them
    const int first = (4 * owner + p.splits - 1) / p.splits, mine = (4 * (owner + 1) + p.splits - 1) / p.splits - first;
    auto slot = [&](int sender) {   // this thread's word of column 0
      const int place = sender < owner ? sender : sender - 1;
      return base + 4 * (((place * mine + part - first) * 64) * 128 + 32 * quad + lane);
    };
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    if (inside && owner != u.split) {
      const uint32_t to = cluster_addr(slot(u.split), 2 * owner + rank);
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) {
        uint32_t v[32];
        tmem_ld(acc + c, v);
        tmem_wait();
        tie(v);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + 512 * (c + e)), "r"(v[e]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync();
    if (inside && owner == u.split) {
      const uint32_t stage = base + kStages * kStageBytes + (warp - 4) * 2 * kOutBlock;
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) {
        uint32_t own[32];
        tmem_ld(acc + c, own);
        tmem_wait();
        tie(own);
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.f;
        for (int i = 0; i < p.splits; ++i) {   // in the order of the splits
          if (i == u.split) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += __uint_as_float(own[e]);
          } else {
            const uint32_t from = slot(i) + 512 * c;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              float x;
              asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(from + 512 * e));
              v[e] += x;
            }
          }
        }
        const uint32_t block = stage + (c >> 5) * kOutBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) stage8(block, lane, i, pack8(v + 8 * i));
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && u.n + 64 * part + c < p.cols) tma_store_2d(&p.out[0], u.n + 64 * part + c, row0, block);
      }
      if (lane == 0) {
        tma_store_commit();
        tma_store_read_wait<0>();
      }
    }
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

// Operand of a product whose inner dimension is its rows: [inner, cols], columns contiguous.
bool ffn_outer_map(CUtensorMap* map, int* layout, const void* base, long long inner, int cols, long long stride) {
  *layout = cols % 64 ? kOuter : kOuterBlocks;
  if (*layout == kOuter) return ffn_map(map, base, inner, cols, stride, 64);
  const uint64_t dims[3] = {64, static_cast<uint64_t>(inner), static_cast<uint64_t>(cols / 64)};
  const int64_t strides[2] = {stride, 64};
  const uint32_t boxes[3] = {64, 64, 2};
  return make_tmap_bf16_sw128(map, base, 3, dims, strides, boxes);
}

// Output [rows, cols], contiguous: boxes of 32 x 32.
bool ffn_out_map(CUtensorMap* map, const void* base, long long rows, int cols) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const int64_t strides[1] = {cols};
  const uint32_t boxes[2] = {32, 32};
  return make_tmap_bf16(map, base, 2, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_64B);
}

// Splits of a product's inner length: enough units for every pair of SMs where
// the launch's `tiles` alone leave some without work, each at least
// kMinSplitSteps long.
int ffn_splits(long long tiles, int steps) {
  if (tiles >= kPairs) return 1;
  long long s = kPairs / tiles;
  if (s > steps / kMinSplitSteps) s = steps / kMinSplitSteps;
  return s < 1 ? 1 : static_cast<int>(s);
}

struct FfnSpace {
  size_t partial = 0, counters = 0;   // floats, ints
};

// Shape part of a product (no pointers).
FfnProblem ffn_product(long long rows, int cols, long long inner, int segments) {
  FfnProblem p = {};
  p.rows = static_cast<int>(rows);
  p.cols = cols;
  p.tiles_n = static_cast<int>(ffn_tiles(cols, 256));
  p.segments = segments;
  p.steps = ffn_steps(inner);
  p.units = static_cast<int>(ffn_tiles(rows, 256) * p.tiles_n);
  p.splits = 1;
  return p;
}

// Splits it as one of `tiles` of its launch; what it needs is added to `space`.
void ffn_split(FfnProblem* p, long long tiles, FfnSpace* space) {
  p->splits = ffn_splits(tiles, p->segments * p->steps);
  if (p->splits == 1) return;
  space->counters += static_cast<size_t>(p->units) * 2;
  p->units *= p->splits;
  space->partial += static_cast<size_t>(p->units) * 65536;
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
  FfnParams<kCount, ffn_maps(kMode)> r;
  for (int i = 0; i < q.count; ++i) {
    static_cast<FfnSizes&>(r.p[i]) = q.p[i];
    std::memcpy(r.p[i].a, q.p[i].a, sizeof(r.p[i].a));
    std::memcpy(r.p[i].b, q.p[i].b, sizeof(r.p[i].b));
    std::memcpy(r.p[i].out, q.p[i].out, sizeof(r.p[i].out));
  }
  r.count = q.count;
  r.units = q.units;
  r.clear = q.clear;
  r.clear_count = q.clear_count;
  const int pairs = kMode == kProductCluster || q.units < kPairs ? q.units : kPairs;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(kMode == kProductCluster ? 2 * q.p[0].splits : 2);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  config.blockDim = dim3(kFfnThreads);
  config.dynamicSmemBytes = kFfnSmem;
  config.stream = s;
  config.attrs = attr;
  config.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, ffn_kernel<kMode, kAct, kCount>, r);
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

template <int kMode>
int ffn_launch_gate(FfnParams<1>& q, int activation, cudaStream_t s, const char* what) {
  if (activation == TS_FFN_SILU) return ffn_launch<kMode, TS_FFN_SILU>(q, s, what);
  if (activation == TS_FFN_GELU) return ffn_launch<kMode, TS_FFN_GELU>(q, s, what);
  return ffn_launch<kMode, TS_FFN_RELU2>(q, s, what);
}

size_t ffn_align(size_t x) { return (x + 1023) & ~static_cast<size_t>(1023); }

int ffn_check(const ts_ffn_args* a) {
  if (!a) return set_error(TS_ERR_VALUE, "ffn: null arguments");
  if (a->rows < 1 || a->rows > (1ll << 30)) return set_error(TS_ERR_VALUE, "ffn: rows must lie in 1..2^30");
  for (int d : {a->width, a->hidden, a->width_out})
    if (d < 8 || d % 8 || d > (1 << 20))
      return set_error(TS_ERR_NOT_IMPLEMENTED, "ffn: width %d must be a multiple of 8 in 8..2^20", d);
  if (a->activation < TS_FFN_SILU || a->activation > TS_FFN_RELU2)
    return set_error(TS_ERR_VALUE, "ffn: unknown activation %d", a->activation);
  // tiles of the largest product, split or not, count in 32 bits
  if (ffn_tiles(a->rows, 256) * ffn_tiles(a->hidden, 128) > (1 << 28) ||
      ffn_tiles(a->rows, 256) * ffn_tiles(a->width, 256) > (1 << 28) ||
      ffn_tiles(a->rows, 256) * ffn_tiles(a->width_out, 256) > (1 << 28))
    return set_error(TS_ERR_NOT_IMPLEMENTED, "ffn: too many tiles");
  return TS_OK;
}

const char* const kFfnLayout = "ffn: every matrix needs a 16-byte aligned base and a row stride that is a multiple of 8";

size_t ffn_hidden_bytes(const ts_ffn_args* a) { return static_cast<size_t>(a->rows) * a->hidden * 2; }

// Pairs of a cluster that share each of a product's tiles: as many as leave all
// clusters resident at once (33, 22 and 15 clusters of 2, 3 and 4 pairs on a
// B200), each with kMinSplitSteps steps at least.
int ffn_cluster_splits(int tiles, int steps) {
  constexpr int kResident[] = {kPairs, 33, 22, 15};
  int s = 1;
  while (s < 4 && tiles <= kResident[s] && steps >= (s + 1) * kMinSplitSteps) ++s;
  return s;
}

struct FfnBackward {
  FfnProblem p[4] = {};   // dWg, dWu, dWd, dx
  FfnSpace space;
  size_t du = 0, partial = 0, counters = 0, total = 0;   // offsets; dg at 0
};

FfnBackward ffn_backward(const ts_ffn_args* a) {
  FfnBackward b;
  const int parts = ffn_parts(a->rows);   // of h, dg and du
  b.p[0] = ffn_product(a->hidden, a->width, a->rows, parts);
  b.p[1] = ffn_product(a->hidden, a->width, a->rows, parts);
  b.p[2] = ffn_product(a->width_out, a->hidden, a->rows, parts);
  b.p[3] = ffn_product(a->rows, a->width, a->hidden, 2 * parts);
  // the weights' gradients, whose inner length is the tokens, come first and are split as one; dx takes what they
  // leave, but for few rows is split as if alone: its few tiles, each the whole length of both parts, would end long
  // after the others' (one row of 2048 x 5632, forward and backward: 196 us, split 106)
  const long long tiles = static_cast<long long>(b.p[0].units) + b.p[1].units + b.p[2].units;
  for (int i = 0; i < 3; ++i) ffn_split(&b.p[i], tiles, &b.space);
  const long long before = static_cast<long long>(b.p[0].units) + b.p[1].units + b.p[2].units;
  ffn_split(&b.p[3], (parts > 1 ? 0 : before) + b.p[3].units, &b.space);
  const size_t one = ffn_align(ffn_hidden_bytes(a) * parts);
  b.du = one;
  b.partial = 2 * one;
  b.counters = b.partial + ffn_align(b.space.partial * 4);
  b.total = b.counters + ffn_align(b.space.counters * 4);
  return b;
}

// A gate launch: tiles of 256 rows x `tile` hidden columns, not split.
FfnParams<1> ffn_gate(const ts_ffn_args* a, int tile, int inner) {
  FfnParams<1> q = {};
  q.count = 1;
  FfnProblem& p = q.p[0];
  p.rows = static_cast<int>(a->rows);
  p.cols = a->hidden;
  p.tiles_n = static_cast<int>(ffn_tiles(a->hidden, tile));
  p.segments = 1;
  p.steps = ffn_steps(inner);
  p.splits = 1;
  p.units = static_cast<int>(ffn_tiles(a->rows, 256)) * p.tiles_n;
  p.kept = static_cast<uint8_t*>(a->kept);
  return q;
}

}  // namespace

}  // namespace ts

extern "C" {

size_t ts_b200_ffn_kept_bytes(const ts_ffn_args* a) {
  if (ts::ffn_check(a)) return 0;
  return static_cast<size_t>((a->rows + 31) / 32) * ((a->hidden + 31) / 32) * TS_FFN_KEPT_BLOCK;
}

size_t ts_b200_ffn_fwd_workspace_bytes(const ts_ffn_args* a) {
  if (ts::ffn_check(a)) return 0;
  // h, where the caller keeps none; for few rows in two parts
  return ts::ffn_align(ts::ffn_hidden_bytes(a) * ts::ffn_parts(a->rows));
}

int ts_b200_ffn_fwd(const ts_ffn_args* a, ts_stream_t stream) {
  using namespace ts;
  if (const int rc = ffn_check(a)) return rc;
  if (!a->x || !a->w_gate || !a->w_up || !a->w_down || !a->y) return set_error(TS_ERR_VALUE, "ffn_fwd: null pointer");
  if (!a->kept != !a->h) return set_error(TS_ERR_VALUE, "ffn_fwd: h and kept belong together");
  if (reinterpret_cast<uintptr_t>(a->kept) & 15) return set_error(TS_ERR_VALUE, "ffn_fwd: kept must be 16-byte aligned");
  if (!a->workspace || a->workspace_bytes < ts_b200_ffn_fwd_workspace_bytes(a))
    return set_error(TS_ERR_VALUE, "ffn_fwd: workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  void* h = a->h ? a->h : ws;
  if (a->rows <= kRowsMost) {
    const auto bad = [](const void* base, long long stride) {
      return (reinterpret_cast<uintptr_t>(base) & 15) || stride % 8;
    };
    if (bad(a->x, a->x_stride) || bad(a->w_gate, a->w_gate_stride) || bad(a->w_up, a->w_up_stride) ||
        bad(a->w_down, a->w_down_stride) || bad(a->y, 0) || bad(h, 0))
      return set_error(TS_ERR_VALUE, kFfnLayout);
    return ffn_rows_fwd(a, h, stream);
  }
  if (!ffn_bind_context()) return set_error(TS_ERR_CUDA, "ffn_fwd: no context on the current device");
  FfnParams<1> gate = ffn_gate(a, 128, a->width);
  FfnProblem& p = gate.p[0];
  FfnParams<1> down = {};
  down.count = 1;
  FfnProblem& d = down.p[0];
  d = ffn_product(a->rows, a->width_out, a->hidden, 1);
  d.splits = ffn_cluster_splits(d.units, d.steps);
  d.units *= d.splits;
  if (!ffn_map(&p.a[0], a->x, a->rows, a->width, a->x_stride, 128) ||
      !ffn_map(&p.b[0], a->w_gate, a->hidden, a->width, a->w_gate_stride, 128) ||
      !ffn_map(&p.b[1], a->w_up, a->hidden, a->width, a->w_up_stride, 128) ||
      !ffn_out_map(&p.out[0], h, a->rows, a->hidden) || !ffn_map(&d.a[0], h, a->rows, a->hidden, a->hidden, 128) ||
      !ffn_map(&d.b[0], a->w_down, a->width_out, a->hidden, a->w_down_stride, 128) ||
      !ffn_out_map(&d.out[0], a->y, a->rows, a->width_out))
    return set_error(TS_ERR_VALUE, kFfnLayout);
  if (const int rc = ffn_launch_gate<kGateFwd>(gate, a->activation, stream, "ffn_gate_fwd")) return rc;
  return d.splits > 1 ? ffn_launch<kProductCluster, 0>(down, stream, "ffn_down")
                      : ffn_launch<kProduct, 0>(down, stream, "ffn_down");
}

size_t ts_b200_ffn_bwd_workspace_bytes(const ts_ffn_args* a) {
  return ts::ffn_check(a) ? 0 : ts::ffn_backward(a).total;
}

int ts_b200_ffn_bwd(const ts_ffn_args* a, const ts_ffn_grad_args* g, ts_stream_t stream) {
  using namespace ts;
  if (const int rc = ffn_check(a)) return rc;
  if (!g || !a->x || !a->w_gate || !a->w_up || !a->w_down || !a->h || !a->kept || !g->dy)
    return set_error(TS_ERR_VALUE, "ffn_bwd: null pointer");
  if (reinterpret_cast<uintptr_t>(a->kept) & 15) return set_error(TS_ERR_VALUE, "ffn_bwd: kept must be 16-byte aligned");
  FfnBackward b = ffn_backward(a);
  if (!a->workspace || a->workspace_bytes < b.total) return set_error(TS_ERR_VALUE, "ffn_bwd: workspace too small");
  if (!ffn_bind_context()) return set_error(TS_ERR_CUDA, "ffn_bwd: no context on the current device");
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  void *dg = ws, *du = ws + b.du;
  const long long M = a->rows;
  const int D = a->width, H = a->hidden, O = a->width_out;
  FfnParams<1> gate = ffn_gate(a, 256, O);
  FfnProblem& p = gate.p[0];
  const int parts = ffn_parts(M);
  // a part of a [parts, rows, hidden] matrix
  auto part_of = [&](const void* base, int part) {
    return static_cast<const uint8_t*>(base) + part * ffn_hidden_bytes(a);
  };
  bool ok = ffn_map(&p.a[0], g->dy, M, O, g->dy_stride, 128) &&
            ffn_outer_map(&p.b[0], &p.b_layout, a->w_down, O, H, a->w_down_stride);
  for (int i = 0; i < parts && ok; ++i)
    ok = ffn_out_map(&p.out[2 * i], part_of(dg, i), M, H) && ffn_out_map(&p.out[2 * i + 1], part_of(du, i), M, H);
  FfnParams<4> grads = {};
  float* partial = reinterpret_cast<float*>(ws + b.partial);
  int* counters = reinterpret_cast<int*>(ws + b.counters);
  gate.clear = counters;
  gate.clear_count = static_cast<int>(b.space.counters);
  // dWg = dg^T x, dWu = du^T x, dWd = dy^T h: the inner dimension is the tokens, outside in every operand
  // (`two_left`, `two_right`: the operand that is in parts)
  auto weight = [&](FfnProblem& w, const void* left, int left_cols, long long left_stride, bool two_left,
                    const void* right, int right_cols, long long right_stride, bool two_right, void* out) {
    if (!out) return true;
    ffn_place(&w, partial, counters);
    bool mapped = ffn_out_map(&w.out[0], out, left_cols, right_cols);
    for (int i = 0; i < parts && mapped; ++i)
      mapped = ffn_outer_map(&w.a[i], &w.a_layout, two_left ? part_of(left, i) : left, M, left_cols, left_stride) &&
               ffn_outer_map(&w.b[i], &w.b_layout, two_right ? part_of(right, i) : right, M, right_cols, right_stride);
    grads.p[grads.count++] = w;
    return mapped;
  };
  ok = ok && weight(b.p[0], dg, H, H, true, a->x, D, a->x_stride, false, g->dw_gate) &&
       weight(b.p[1], du, H, H, true, a->x, D, a->x_stride, false, g->dw_up) &&
       weight(b.p[2], g->dy, O, g->dy_stride, false, a->h, H, H, true, g->dw_down);
  if (ok && g->dx) {
    FfnProblem& x = b.p[3];
    ffn_place(&x, partial, counters);
    ok = ffn_out_map(&x.out[0], g->dx, M, D);
    for (int i = 0; i < parts && ok; ++i)
      ok = ffn_map(&x.a[2 * i], part_of(dg, i), M, H, H, 128) && ffn_map(&x.a[2 * i + 1], part_of(du, i), M, H, H, 128) &&
           ffn_outer_map(&x.b[2 * i], &x.b_layout, a->w_gate, H, D, a->w_gate_stride) &&
           ffn_outer_map(&x.b[2 * i + 1], &x.b_layout, a->w_up, H, D, a->w_up_stride);
    grads.p[grads.count++] = x;
  }
  if (!ok) return set_error(TS_ERR_VALUE, kFfnLayout);
  if (grads.count == 0) return TS_OK;
  if (const int rc = parts > 1 ? ffn_launch_gate<kGateGradTwo>(gate, a->activation, stream, "ffn_gate_grad")
                               : ffn_launch_gate<kGateGrad>(gate, a->activation, stream, "ffn_gate_grad"))
    return rc;
  return parts > 1 ? ffn_launch<kProductTwo, 0>(grads, stream, "ffn_grads")
                   : ffn_launch<kProduct, 0>(grads, stream, "ffn_grads");
}

}  // extern "C"
