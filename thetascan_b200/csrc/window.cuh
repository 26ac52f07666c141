// What the kernels of the windowed attention share: sizes, the tensor-memory
// operand form of the matrix instruction, masks of a row's columns.
//
// The query at position i sees the key at position j when j <= i and
// i - j < window or j < sinks, both below the sequence's length.  Queries are the
// last q_tokens of kv_tokens positions.  Tiles are 128 queries and 128 keys; the
// grid of the window's key tiles starts at the first query, so that a window that
// is a multiple of 128 is covered by window / 128 + 1 tiles whatever comes before.
#pragma once

#include "../../include/thetascan_b200.h"
#include "common.cuh"
#include "tma.cuh"

namespace ts {

constexpr float kLog2e = 1.4426950408889634f;

// A division by a constant of the launch.
struct Divisor {
  unsigned by, factor;   // factor: 2^32 / by, rounded up
  static Divisor of(int by) {
    return Divisor{static_cast<unsigned>(by), by > 1 ? static_cast<unsigned>(((1ull << 32) + by - 1) / by) : 0u};
  }
  // n below 2^31: the product is the quotient, or one more
  __device__ __forceinline__ int operator()(int n) const {
    if (by == 1) return n;
    const unsigned q = __umulhi(static_cast<unsigned>(n), factor);
    return static_cast<int>(q * by > static_cast<unsigned>(n) ? q - 1 : q);
  }
};

struct WinSizes {
  int batch, heads, kv_heads, share;   // share: query heads to a key head
  int dim;
  int q_tokens, kv_tokens, past;       // past: kv_tokens - q_tokens
  int window, sinks;                   // both at most kv_tokens
  int q_tiles;
  Divisor by_share, by_kv_heads;
  float scale;
  const int* lengths;                  // or null
};

__device__ __forceinline__ int win_length(const WinSizes& w, int b) {
  return w.lengths ? max(0, min(__ldg(w.lengths + b), w.kv_tokens)) : w.kv_tokens;
}

// The order in which the units (query or key tiles, or pairs) of the key heads are taken.  CTAs take every 148th, and units
// differ: by the window's start, by a sequence's end.  One key head after another would leave some CTAs up to twice the
// work of others, so units of one index come together, through all key heads, the ones with most work first (64 x 8 heads x
// 1024, width 64, window 256, forward and backward: 635 us one after another, 544 so).
enum WinHow {
  kWinApart,   // one key head after another
  kWinLevel,   // all key heads alike
  kWinTable    // sequences of different lengths: by a WinOrder
};
struct WinUnits {
  int units;
  Divisor by_each, by_rows;   // units of a key head; key heads of all sequences
  WinHow how;
};

// For a padded batch, in shared memory.  Of each key head of sequence b the units 0 .. live(b) - 1 have work: they come by
// falling index (or rising: backwards), those of all sequences that have one together, and what has no work at the end.
struct WinOrder {
  static constexpr int kMost = 64;   // sequences; more are taken one after another
  int begin[kMost + 1];              // first unit of those that the sequences 0 .. j, by falling length, have together
  uint16_t live[kMost];
  uint8_t sequence[kMost];
};

inline WinUnits win_units(const WinSizes& w, int each) {
  const int rows = w.batch * w.kv_heads;
  WinUnits n = {rows * each, Divisor::of(each), Divisor::of(rows), kWinLevel};
  if (w.lengths) n.how = w.batch <= WinOrder::kMost && each <= 0xffff ? kWinTable : kWinApart;
  if (n.units <= 148) n.how = kWinApart;   // each has an SM of its own
  return n;
}

// By one warp, before a barrier.
template <class F>
__device__ __forceinline__ void win_order(WinOrder& o, const WinSizes& w, F live) {
  const int lane = threadIdx.x & 31;
  int n[2], rank[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) n[h] = lane + 32 * h < w.batch ? live(lane + 32 * h) : 0;
  for (int i = 0; i < 32; ++i) {
    const int x[2] = {__shfl_sync(0xffffffffu, n[0], i), __shfl_sync(0xffffffffu, n[1], i)};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < 2; ++g) rank[h] += x[g] > n[h] || (x[g] == n[h] && i + 32 * g < lane + 32 * h);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    o.live[rank[h]] = static_cast<uint16_t>(n[h]);
    o.sequence[rank[h]] = static_cast<uint8_t>(lane + 32 * h);
  }
  __syncwarp();
  int before = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = lane + 32 * h;
    int upto = (o.live[j] - (j + 1 < WinOrder::kMost ? o.live[j + 1] : 0)) * (j + 1) * w.kv_heads;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    o.begin[j + 1] = before + upto;
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) o.begin[0] = 0;
}

// A unit's sequence, key head and index among the units of a key head.  kRising: the first ones have most work.
template <bool kRising>
__device__ __forceinline__ void win_place(const WinOrder& o, const WinUnits& n, const WinSizes& w, int unit, int& b, int& kv_head,
                                          int& at) {
  const int each = static_cast<int>(n.by_each.by);
  if (n.how != kWinTable) {
    int row;
    if (n.how == kWinApart) {
      row = n.by_each(unit);
      at = unit - row * each;
    } else {
      at = n.by_rows(unit);
      row = unit - at * static_cast<int>(n.by_rows.by);
      if (!kRising) at = each - 1 - at;
    }
    b = w.by_kv_heads(row);
    kv_head = row - b * w.kv_heads;
    return;
  }
  const int working = o.begin[WinOrder::kMost];
  int j = 0, rest = unit - working;
  if (rest < 0) {
    if (kRising) unit = working - 1 - unit;
#pragma unroll
    for (int s = WinOrder::kMost / 2; s > 0; s >>= 1) j += o.begin[j + s] <= unit ? s : 0;
    rest = unit - o.begin[j];
    const int row = rest / ((j + 1) * w.kv_heads);
    rest -= row * (j + 1) * w.kv_heads;
    at = o.live[j] - 1 - row;
    j = w.by_kv_heads(rest);
    kv_head = rest - j * w.kv_heads;
  } else {
    for (; j < WinOrder::kMost - 1; ++j) {
      const int none = (each - o.live[j]) * w.kv_heads;
      if (rest < none) break;
      rest -= none;
    }
    const int row = w.by_kv_heads(rest);
    at = o.live[j] + row;
    kv_head = rest - row * w.kv_heads;
  }
  b = o.sequence[j];
}

// ---- instructions

// D (+)= A B with A [128 x 16 per step] in tensor memory (bf16, two to a column) and B in shared memory.
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 columns of this lane's row (visible after tmem_store_wait()).
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The K-major operand (rows = M or N) and the MN-major one (rows = inner) of a 128-byte-swizzled tile of 128 rows
// in 64-column boxes, at inner step 0, and at step s of 16 from there: the descriptor's address counts 16 bytes and has
// room for all of shared memory, so that a step is an addition.
__device__ __forceinline__ uint64_t win_rows(uint32_t tile) { return smem_desc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t win_inner(uint32_t tile) { return smem_desc_sw128(tile, kSwBox, 1024); }
__device__ __forceinline__ uint64_t win_rows_step(uint64_t first, int s) {
  return first + ((s >> 2) * (kSwBox >> 4) + (s & 3) * 2);
}
__device__ __forceinline__ uint64_t win_inner_step(uint64_t first, int s) { return first + 128 * s; }

// One lane of a converged warp.  The warps that feed the tensor cores run with all lanes and let one issue, so that
// addresses stay in uniform registers (a single lane's loop took 120 cycles for each instruction of 64).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

// Whether `ok` holds in all of the kThreads threads that meet at the barrier `id`.
template <int kThreads>
__device__ __forceinline__ bool threads_agree(int id, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, r;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred r, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, r;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok)), "r"(id), "n"(kThreads)
      : "memory");
  return all != 0;
}

// Zeros in the rows of a tile from `from` on, by the warp that issues the products, before the ones in which they would meet
// weights of zero: what lies behind a sequence may be anything, and zero times infinity or NaN is not zero.
template <int kBoxes>
__device__ __forceinline__ void win_clear_rows(uint32_t tile, int from) {
#pragma unroll 1
  for (int at = 128 * max(from, 0) + 16 * static_cast<int>(threadIdx.x & 31); at < static_cast<int>(kSwBox); at += 512)
#pragma unroll
    for (int c = 0; c < kBoxes; ++c) st_shared_v4(tile + c * kSwBox + at, make_uint4(0, 0, 0, 0));
  fence_async_smem();
  __syncwarp();
}

// Give up registers of a warpgroup, or take more.
template <int kRegs>
__device__ __forceinline__ void win_fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void win_more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// ---- rows

// Bits [low, high] of a word (either may lie outside it; none where low > high).
__device__ __forceinline__ uint32_t bit_range(int low, int high) {
  if (high < 0 || low > 31 || low > high) return 0;
  const uint32_t up = high >= 31 ? 0xffffffffu : (2u << high) - 1;
  return low <= 0 ? up : up & ~((1u << low) - 1);
}
// Scores outside the columns [from, until] become minus infinity.
__device__ __forceinline__ void hide(uint32_t (&s)[32], int from, int until) {
  const uint32_t bits = bit_range(from, until);
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (!(bits >> e & 1)) s[e] = 0xff800000u;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Of numbers; a NaN is left out.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two f32 side by side: one instruction for both.
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

// ---- host

// A [batch, heads, tokens, dim] tensor as boxes of 64 columns x `rows` tokens.
bool win_map(CUtensorMap* map, const void* base, const long long* strides, int batch, int heads, int tokens, int dim,
             int rows);
// Checked arguments as sizes, or an error code.
int win_sizes(const ts_window_args* a, WinSizes* w, const char* what);

}  // namespace ts
