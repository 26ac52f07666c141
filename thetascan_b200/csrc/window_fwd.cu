// Causal attention over a sliding window with first tokens that stay visible:
// the forward pass over many queries.
//
//   y_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(scale q_i.k_j - m_i), j visible to i
//
// One pass over the keys with a running reference m_i and sum.  A CTA takes two
// tiles of 128 queries at a time, A and B: of two heads that share a key head, or
// neighbours of one head, so that both read the same keys.  One warp feeds a ring of
// key and value tiles by TMA, another or two issue the matrix instructions, eight
// own the rows of each query tile, two threads to a row.  S = Q K^T lies in tensor
// memory, 128 columns for each of A and B; P goes back there in bf16, in S's place
// or (heads of up to 64) beside it, and is the operand of O += P V from where it
// lies.  While one group forms its P the tensor cores work for the other: forming
// P and issuing instructions bound it, not the products (16 heads x 16384, width
// 128, window 2048, sinks 16: 284 us, 1.0 PFLOP/s of whole tiles; 64 x 8 heads x
// 1024, width 64, window 256, sinks 4: 115 us, 1.2 TB/s).
//
// A row's reference moves only when a score exceeds it by 2^8 (P is then at most
// 256, and bf16 keeps its relative error): O is seldom rescaled, and the row's own
// thread does that, before it hands P over.
//
// First tokens are tiles of their own, as narrow as 16 columns, so that four sinks
// cost a sixteenth of a tile; the window's tiles leave those keys out.
#include <cmath>
#include <cstring>

#include "capi_internal.h"
#include "window.cuh"

namespace ts {

namespace {

// Warps 0-15: rows, 16: loads, 17 and 19: instructions, 18: tensor memory.  Of the 61440 registers that 640 threads of 96
// are launched with, the row warps take 104 each, the others 64.
constexpr int kFwdRowWarps = 16;
constexpr int kFwdThreads = 32 * (kFwdRowWarps + 4);
constexpr int kFwdRowRegs = 104, kFwdOtherRegs = 64;
static_assert(32 * (kFwdRowWarps * kFwdRowRegs + 4 * kFwdOtherRegs) <= kFwdThreads * 96, "registers");

template <int kD>
struct WinFwdLayout {
  static constexpr int kBoxes = kD / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kSwBox;
  static constexpr int kSlots = kD == 64 ? 8 : 4;
  static constexpr uint32_t kOutBytes = 2048;          // a warp's 32 rows x 32 columns
  static constexpr uint32_t kQ = 0, kRing = 2 * kTileBytes, kOut = kRing + kSlots * kTileBytes;
  static constexpr uint32_t kSmem = kOut + kFwdRowWarps * kOutBytes + 1024;
};

struct WinFwdParams {
  CUtensorMap q, k, v, k_sink, v_sink, y;
  WinSizes w;
  int each;              // query tiles of a unit: 1 or 2
  WinUnits n;
  int sink_rows;         // rows of a sink box
  float* lse;            // or null
};

// One of the two query tiles of a unit.
struct WinFwdTile {
  int tile, head;
  bool exists, live;    // a tile of the tensor; a tile with rows below the length
  int low, last;        // its first window tile; its last index in the list of tiles
};

// What a CTA works on: two query tiles of one key head, and the key tiles that either sees.
struct WinFwdUnit {
  int b, kv_head, length;
  WinFwdTile a, z;
  int sinks;                 // keys below this come in sink tiles, not in the window's
  int sink_tiles, first;     // window tiles run from `first` (in tiles from the first query)
  int count;                 // tiles to go over

  __device__ __forceinline__ WinFwdTile place(const WinSizes& w, int at) const {
    WinFwdTile t;
    t.tile = w.by_share(at);
    t.head = kv_head * w.share + at - t.tile * w.share;
    t.exists = t.tile < w.q_tiles;
    t.live = t.exists && w.past + 128 * t.tile < length;
    return t;
  }
  __device__ __forceinline__ WinFwdUnit(const WinFwdParams& p, const WinOrder& order, int unit) {
    const WinSizes& w = p.w;
    int pair;
    win_place<false>(order, p.n, w, unit, b, kv_head, pair);
    length = win_length(w, b);
    a = place(w, p.each * pair);
    z = place(w, p.each == 2 ? 2 * pair + 1 : w.q_tiles * w.share);   // or none
    const int top = z.live ? z.tile : a.live ? a.tile : -1;
    const int end = min(w.past + 128 * top + 127, length - 1);   // the last position
    // rows that all see everything before them need no sinks
    sinks = end < w.window ? 0 : min(w.sinks, end + 1);
    sink_tiles = (sinks + 127) >> 7;
    const int reach = (w.window + 126) >> 7, least = (sinks - w.past) >> 7;
    first = a.low = max(a.tile - reach, least);
    z.low = max(z.tile - reach, least);
    a.last = sink_tiles - 1 + (a.tile >= a.low ? a.tile - first + 1 : 0);
    z.last = sink_tiles - 1 + (z.tile >= z.low ? z.tile - first + 1 : 0);
    count = top < 0 ? 0 : sink_tiles + top - first + 1;
  }
  __device__ __forceinline__ WinFwdTile of(int x) const {
    WinFwdTile t;
    t.tile = x ? z.tile : a.tile;
    t.head = x ? z.head : a.head;
    t.exists = x ? z.exists : a.exists;
    t.live = x ? z.live : a.live;
    t.low = x ? z.low : a.low;
    t.last = x ? z.last : a.last;
    return t;
  }
  __device__ __forceinline__ bool active(const WinFwdTile& x, int n) const {
    const int t = first + n - sink_tiles;
    return x.live && n < count && (n < sink_tiles || (t >= x.low && t <= x.tile));
  }
  __device__ __forceinline__ int columns(int n) const {
    return n < sink_tiles ? min(128, (sinks - 128 * n + 15) & ~15) : 128;
  }
  __device__ __forceinline__ int key(const WinSizes& w, int n) const {
    return n < sink_tiles ? 128 * n : w.past + 128 * (first + n - sink_tiles);
  }
};

__device__ __forceinline__ void st_shared_f32(uint32_t at, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ float ld_shared_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// 32 scores to weights in bf16, their sum to `part`.
__device__ __forceinline__ void row_exp(const uint32_t (&s)[32], uint32_t to, Pair scale2, Pair origin, Pair (&part)[2]) {
  uint32_t packed[16];
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const Pair x = fma2(Pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, origin);
    float a, b;
    x.get(a, b);
    a = exp2_fast(a);
    b = exp2_fast(b);
    part[e >> 1 & 1] = add2(part[e >> 1 & 1], Pair(a, b));
    packed[e / 2] = pack_bf16(a, b);
  }
  tmem_st(to, packed);
}

template <int kD>
__global__ void __launch_bounds__(kFwdThreads, 1) window_fwd_kernel(const __grid_constant__ WinFwdParams p) {
  using L = WinFwdLayout<kD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t full[L::kSlots], empty[L::kSlots], q_full[2], q_empty[2], s_full[2], s_free[2], p_full[2],
      p_free[2], o_full[2];
  __shared__ uint32_t tmem_slot;
  __shared__ WinOrder order;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinSizes& w = p.w;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kD == 64 ? 2 : 1);   // the warps that issue instructions
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 8);
      mbar_init(&p_full[i], 8);
      mbar_init(&p_free[i], 1);
      mbar_init(&o_full[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 18) tmem_alloc(&tmem_slot, 512);
  if (warp == 1 && p.n.how == kWinTable)
    win_order(order, w, [&](int b) {
      return (((max(0, win_length(w, b) - w.past) + 127) >> 7) * w.share + p.each - 1) / p.each;
    });
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all of tensor memory: its addresses start at 0.  Columns: S of A and B, then O of A and B.  P lies in S's place, or,
  // where O is narrow, behind O: the next S then need not wait for the product with P.
  constexpr bool kApart = kD == 64;
  constexpr uint32_t kScores = 128, kO = 256, kP = kApart ? 384 : 0, kPStride = kApart ? 64 : kScores;

  if (warp >= kFwdRowWarps) {
    win_fewer_registers<kFwdOtherRegs>();
    if (warp == 16) {
      // ---- loads
      uint32_t it = 0, q_turn[2] = {0, 0};
      bool ok = true;
      auto load = [&](const CUtensorMap* map, const CUtensorMap* sink_map, const WinFwdUnit& u, int n) {
        const uint32_t s = it % L::kSlots;
        if (!(ok = ok && mbar_wait_warp(&empty[s], ((it / L::kSlots) & 1) ^ 1, kErrMmaTimeout))) return;
        const bool sink = n < u.sink_tiles;
        const uint32_t rows = sink ? p.sink_rows : 128, to = base + L::kRing + s * L::kTileBytes;
        if (elect_one()) {
          mbar_expect_tx(&full[s], L::kBoxes * rows * 128);
#pragma unroll
          for (int c = 0; c < L::kBoxes; ++c)
            tma_load_4d(to + c * kSwBox, sink ? sink_map : map, 64 * c, u.key(w, n), u.kv_head, u.b, &full[s]);
        }
        ++it;
      };
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinFwdUnit u(p, order, unit);
        auto queries = [&](int x) {
          if (!u.of(x).live || !(ok = ok && mbar_wait_warp(&q_empty[x], (q_turn[x]++ & 1) ^ 1, kErrMmaTimeout))) return;
          if (elect_one()) {
            mbar_expect_tx(&q_full[x], L::kTileBytes);
#pragma unroll
            for (int c = 0; c < L::kBoxes; ++c)
              tma_load_4d(base + L::kQ + x * L::kTileBytes + c * kSwBox, &p.q, 64 * c, 128 * u.of(x).tile, u.of(x).head, u.b,
                          &q_full[x]);
          }
        };
        for (int n = 0; n < u.count && ok; ++n) {
          // (tile B's last product comes after A's: what A needs to begin comes before B's queries)
          if (n == 0) queries(0);
          load(&p.k, &p.k_sink, u, n);
          if (n > 0) load(&p.v, &p.v_sink, u, n);
          if (n == 0) {
            queries(1);
            load(&p.v, &p.v_sink, u, n);
          }
        }
      }
      if (!ok) {
        // given up: let the copies in flight land before the memory goes (for a bounded time too)
        for (uint32_t i = it > L::kSlots ? it - L::kSlots : 0; i < it; ++i)
          for (int poll = 0; poll < (1 << 16) && !mbar_try_wait(&full[i % L::kSlots], (i / L::kSlots) & 1); ++poll) {
          }
#pragma unroll
        for (int x = 0; x < 2; ++x)
          for (int poll = 0; poll < (1 << 16) && q_turn[x] > 0 && !mbar_try_wait(&q_full[x], (q_turn[x] - 1) & 1); ++poll) {
          }
      }
    } else if (!kApart && warp == 17) {
      // ---- instructions, where P takes S's place: one warp, each tile's products with P and then with the next keys,
      // in turn, so that a product has the tensor cores to itself.  This warp's own steps come between the tensor
      // cores': little is worked out here.
      constexpr uint32_t id_o = idesc_bf16(128, kD, false, true), id_s = idesc_bf16(128, 128, false, false);
      constexpr uint32_t kSlotStep = L::kTileBytes >> 4;
      const uint64_t q0 = win_rows(base + L::kQ), k0 = win_rows(base + L::kRing), v0 = win_inner(base + L::kRing);
      // the ring's next key tile and its next value tile: their slots and parities
      uint32_t k_slot = 0, k_parity = 0, v_slot = 1, v_parity = 0;
      uint32_t q_parity[2] = {0, 0}, p_parity[2] = {0, 0};
      bool ok = true;
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinFwdUnit u(p, order, unit);
        // tile x takes part in the first tokens' (n < sink_tiles) and from `low` to `last`
        const int low[2] = {0, u.sink_tiles + u.z.low - u.first}, last[2] = {u.a.live ? u.a.last : -1, u.z.live ? u.z.last : -1};
        auto active = [&](int x, int n) { return n <= last[x] && (x == 0 || n < u.sink_tiles || n >= low[x]); };
        auto keys_landed = [&] { return ok = ok && mbar_wait_warp(&full[k_slot], k_parity, kErrCopyTimeout); };
        auto keys_done = [&] {
          if (ok && elect_one()) mma_commit(&empty[k_slot]);
          k_slot += 2;
          if (k_slot >= L::kSlots) {
            k_slot -= L::kSlots;
            k_parity ^= 1;
          }
        };
        // Q of tile x, before its first product
        auto queries_landed = [&](int x, int n) {
          if (n == 0 || (x == 1 && u.sink_tiles == 0 && n == low[1])) {
            ok = ok && mbar_wait_warp(&q_full[x], q_parity[x], kErrCopyTimeout);
            q_parity[x] ^= 1;
          }
        };
        // S of query tile x against the next key tile, n in the list; by one lane
        auto scores = [&](int x, int n) {
          const uint32_t id = n < u.sink_tiles ? idesc_bf16(128, u.columns(n), false, false) : id_s;
          const uint64_t q = q0 + x * kSlotStep, k = k0 + k_slot * kSlotStep;
#pragma unroll
          for (int s = 0; s < kD / 16; ++s) mma_bf16(kScores * x, win_rows_step(q, s), win_rows_step(k, s), id, s > 0);
          mma_commit(&s_full[x]);
          if (n == last[x]) mma_commit(&q_empty[x]);
        };
        // O += P V with the next value tile, and then the next S, without a pause between them
        auto step = [&](int x, int n, bool more) {
          const bool now = active(x, n), then = more && active(x, n + 1);
          if (then) queries_landed(x, n + 1);
          if (now) {
            ok = ok && mbar_wait_warp(&p_full[x], p_parity[x], kErrMmaTimeout);
            p_parity[x] ^= 1;
          }
          if (!ok) return;
          tc_fence_after();
          const bool summed = x == 0 || u.sink_tiles > 0 ? n > 0 : n > low[1];
          const uint64_t v = v0 + v_slot * kSlotStep;
          const int steps = u.columns(n) >> 4;
          if (elect_one()) {
            if (now) {
#pragma unroll
              for (int s = 0; s < 8; ++s)
                if (s < steps)   // the columns of each half of the rows' warps lie in that half
                  mma_bf16_ts(kO + kD * x, kScores * x + 64 * (s >> 2) + 8 * (s & 3), win_inner_step(v, s), id_o, summed || s > 0);
              if (n == last[x]) mma_commit(&o_full[x]);
            }
            if (then) scores(x, n + 1);
          }
        };
        if (u.count > 0) {
          if (!keys_landed()) break;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!active(x, 0)) continue;
            queries_landed(x, 0);
            tc_fence_after();
            if (ok && elect_one()) scores(x, 0);
          }
          keys_done();
        }
        for (int n = 0; n < u.count && ok; ++n) {
          const bool more = n + 1 < u.count;
          if (!(ok = ok && mbar_wait_warp(&full[v_slot], v_parity, kErrCopyTimeout))) break;
          if (more && !keys_landed()) break;
          if (w.lengths && u.key(w, n) + 128 > u.length)
            win_clear_rows<L::kBoxes>(base + L::kRing + v_slot * L::kTileBytes, u.length - u.key(w, n));
          step(0, n, more);
          step(1, n, more);
          if (ok && elect_one()) mma_commit(&empty[v_slot]);
          if (more) keys_done();
          v_slot += 2;
          if (v_slot >= L::kSlots) {
            v_slot -= L::kSlots;
            v_parity ^= 1;
          }
        }
      }
    } else if (kApart && warp != 18) {
      // ---- instructions: warp 17 for tile A, warp 19 for B, so that neither waits for the other's rows.  These warps' own
      // steps come between the tensor cores': little is worked out here.
      const int x = warp == 17 ? 0 : 1;
      constexpr uint32_t id_o = idesc_bf16(128, kD, false, true), id_s = idesc_bf16(128, 128, false, false);
      constexpr uint32_t kSlotStep = L::kTileBytes >> 4;
      const uint64_t q0 = win_rows(base + L::kQ) + x * kSlotStep;
      const uint64_t k0 = win_rows(base + L::kRing), v0 = win_inner(base + L::kRing);
      const uint32_t s_to = kScores * x, p_at = kP + kPStride * x, o_to = kO + kD * x;
      uint64_t* const done_s = &s_full[x];
      // the ring's next key tile and its next value tile: their slots and parities
      uint32_t k_slot = 0, k_parity = 0, v_slot = 1, v_parity = 0;
      uint32_t q_parity = 0, s_parity = 1, p_parity = 0;
      bool ok = true;
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinFwdUnit u(p, order, unit);
        const WinFwdTile mine = u.of(x);
        // this tile takes part in the first tokens' (n < sink_tiles) and from `low` to `last`
        const int low = u.sink_tiles + mine.low - u.first, last = mine.live ? mine.last : -1;
        const int begin = u.sink_tiles > 0 ? 0 : low;
        auto active = [&](int n) { return n <= last && (n < u.sink_tiles || n >= low); };
        // S against the next key tile, n in the list
        auto scores = [&](int n) {
          if (!(ok = ok && mbar_wait_warp(&full[k_slot], k_parity, kErrCopyTimeout))) return;
          if (active(n)) {
            if (n == begin) {
              ok = ok && mbar_wait_warp(&q_full[x], q_parity, kErrCopyTimeout);
              q_parity ^= 1;
            }
            ok = ok && mbar_wait_warp(&s_free[x], s_parity, kErrMmaTimeout);
            s_parity ^= 1;
            if (!ok) return;
            tc_fence_after();
            const uint32_t id = n < u.sink_tiles ? idesc_bf16(128, u.columns(n), false, false) : id_s;
            const uint64_t k = k0 + k_slot * kSlotStep;
            if (elect_one()) {
#pragma unroll
              for (int s = 0; s < kD / 16; ++s) mma_bf16(s_to, win_rows_step(q0, s), win_rows_step(k, s), id, s > 0);
              mma_commit(done_s);
              mma_commit(&empty[k_slot]);
              if (n == last) mma_commit(&q_empty[x]);
            }
          } else if (elect_one()) {
            mbar_arrive(&empty[k_slot]);
          }
          k_slot += 2;
          if (k_slot >= L::kSlots) {
            k_slot -= L::kSlots;
            k_parity ^= 1;
          }
        };
        // O += P V with the next value tile
        auto sums = [&](int n) {
          if (!(ok = ok && mbar_wait_warp(&full[v_slot], v_parity, kErrCopyTimeout))) return;
          if (active(n)) {
            if (w.lengths && u.key(w, n) + 128 > u.length)
              win_clear_rows<L::kBoxes>(base + L::kRing + v_slot * L::kTileBytes, u.length - u.key(w, n));
            ok = mbar_wait_warp(&p_full[x], p_parity, kErrMmaTimeout);
            p_parity ^= 1;
            if (!ok) return;
            tc_fence_after();
            const uint64_t v = v0 + v_slot * kSlotStep;
            if (elect_one()) {
              if (n >= u.sink_tiles) {
#pragma unroll
                for (int s = 0; s < 8; ++s) mma_bf16_ts(o_to, p_at + 8 * s, win_inner_step(v, s), id_o, n > begin || s > 0);
              } else {
                const int steps = u.columns(n) >> 4;
                for (int s = 0; s < steps; ++s)
                  mma_bf16_ts(o_to, p_at + 8 * s, win_inner_step(v, s), id_o, n > begin || s > 0);
              }
              mma_commit(&p_free[x]);
              mma_commit(&empty[v_slot]);
              if (n == last) mma_commit(&o_full[x]);
            }
          } else if (elect_one()) {
            mbar_arrive(&empty[v_slot]);
          }
          v_slot += 2;
          if (v_slot >= L::kSlots) {
            v_slot -= L::kSlots;
            v_parity ^= 1;
          }
        };
        for (int n = 0; n <= u.count && u.count > 0 && ok; ++n) {
          if (n < u.count) scores(n);
          if (n > 0) sums(n - 1);
        }
      }
    }
  } else {
    // ---- rows: two threads for a row of tile x, each with half of the columns.  (One thread to a row leaves a scheduler
    // two warps, whose steps wait for one another: 64 x 8 heads x 1024, width 64, window 256 took 135 us.)
    win_more_registers<kFwdRowRegs>();
    const int x = warp >> 3, half = warp >> 2 & 1, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_at = kScores * x + lanes + 64 * half, p_at = kP + kPStride * x + lanes + (kApart ? 32 : 64) * half;
    const uint32_t o_at = kO + kD * x + lanes + kD / 2 * half;
    const uint32_t stage = base + L::kOut + warp * L::kOutBytes, partner = base + L::kOut + (warp ^ 4) * L::kOutBytes;
    const float scale2 = w.scale * kLog2e;
    uint32_t turn = 0, o_turn = 0, exchanges = 0;
    bool ok = true;
    auto signal = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // the two warps of these rows
    auto pair_meets = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * x + quad) : "memory"); };
    // the value of the other thread of the row, by two places in turn: one is written again once both warps have met
    // over the other, and so have read this one
    auto exchange = [&](float v) {
      const uint32_t slot = exchanges++ & 1;
      st_shared_f32(stage + 128 * slot + 4 * lane, v);
      pair_meets();
      return ld_shared_f32(partner + 128 * slot + 4 * lane);
    };
    WinFwdUnit next(p, order, blockIdx.x);
    for (int unit = blockIdx.x; unit < p.n.units; unit += gridDim.x) {
      const WinFwdUnit u = next;
      const WinFwdTile mine = u.of(x);
      if (unit + gridDim.x < p.n.units) next = WinFwdUnit(p, order, unit + gridDim.x);
      if (!mine.exists) continue;
      if (lane == 0) tma_store_read_wait<0>();   // the last store has read the stage, which carries exchanges now
      __syncwarp();
      const int q_row = 128 * mine.tile + row, at = w.past + q_row;
      const int near = max(at - w.window + 1, u.sinks), to = at < u.length ? at : -1;   // visible: first ones, near..to
      float ref = -INFINITY, sum = 0.f;
      bool first = true;
      // first tokens, then the window's own
      for (int n = 0; mine.live && n <= mine.last; ++n, ++turn) {
        if (n == u.sink_tiles) n += mine.low - u.first;
        const int cols = u.columns(n) - 64 * half, key = u.key(w, n) + 64 * half;
        const bool sink = n < u.sink_tiles;
        // this row's first and last visible column; a tile within reach of all rows is not masked
        const int from = sink ? 0 : near - key, until = min(to, sink ? u.sinks - 1 : to) - key;
        const bool masked = !__all_sync(0xffffffffu, from <= 0 && until >= 63);
        ok = ok && mbar_wait(&s_full[x], turn & 1, kErrMmaTimeout);
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld(s_at, s[0]);
        tmem_ld(s_at + 32, s[1]);
        tmem_wait();
        tie(s[0]);
        tie(s[1]);
        if (kApart) signal(&s_free[x]);
        // whether the warp's rows see anything of each 32 columns
        const bool some[2] = {!masked || __any_sync(0xffffffffu, until >= 0 && from <= 31),
                              !masked || __any_sync(0xffffffffu, until >= 32 && from <= 63)};
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (some[c]) hide(s[c], from - 32 * c, until - 32 * c);
        }
        float best = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!some[c]) continue;
          // chains side by side: each step waits for the one before
          float top[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 4]), __uint_as_float(s[c][i + 8]));
#pragma unroll
          for (int e = 12; e < 28; e += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = max3(top[i], __uint_as_float(s[c][e + i]), __uint_as_float(s[c][e + i + 4]));
          best = max3(best, max3(top[0], top[1], max3(top[2], top[3], __uint_as_float(s[c][28]))),
                      max3(__uint_as_float(s[c][29]), __uint_as_float(s[c][30]), __uint_as_float(s[c][31])));
        }
        best = fmaxf(best, exchange(best)) * scale2;
        if (kApart) {
          ok = ok && mbar_wait(&p_free[x], (turn & 1) ^ 1, kErrMmaTimeout);
          tc_fence_after();
        }
        // The row's reference: the largest score of its first tile, and later one that exceeds it by 2^8.  (A NaN leaves
        // the reference alone, and reaches the row by its weight.)
        if (first) {
          ref = best;
          first = false;
        } else if (__any_sync(0xffffffffu, best > ref + 8.f)) {
          const float moved = best > ref + 8.f ? best : ref;
          const float factor = moved == ref ? 1.f : exp2_fast(ref - moved);
          ref = moved;
          sum *= factor;
#pragma unroll 1
          for (int c = 0; c < kD / 2; c += 16) {
            uint32_t o[16];
            tmem_ld(o_at + c, o);
            tmem_wait();
            tie(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st(o_at + c, o);
          }
        }
        const Pair scales(scale2), origin(ref == -INFINITY ? 0.f : -ref);
        Pair part[2] = {Pair(sum, 0.f), Pair(0.f)};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (some[c]) {
            row_exp(s[c], p_at + 16 * c, scales, origin, part);
          } else if (32 * c < cols) {
            const uint32_t zero[16] = {};
            tmem_st(p_at + 16 * c, zero);
          }
        }
        float even, odd;
        add2(part[0], part[1]).get(even, odd);
        sum = even + odd;
        tmem_store_wait();
        signal(&p_full[x]);
      }
      sum += exchange(sum);
      ok = ok && (!mine.live || mbar_wait(&o_full[x], o_turn++ & 1, kErrMmaTimeout));
      // Both have read the other's sum: the stage takes the results.  They go on, or give up, together: the next unit's
      // exchanges are waits for one another.
      if (!threads_agree<64>(1 + 4 * x + quad, ok)) break;
      tc_fence_after();
      // A row behind its sequence sees nothing: zero.  All others see themselves at least; scores of minus infinity alone
      // sum to zero there, and 0 / 0 is no number.
      const bool sees = to >= 0;
      const float inverse = 1.f / sum;
#pragma unroll 1
      for (int c = 0; c < kD / 2; c += 32) {
        const int channel = kD / 2 * half + c;
        if (channel >= w.dim) break;
        uint32_t o[32];
        tmem_ld(o_at + c, o);
        tmem_wait();
        tie(o);
        if (lane == 0) tma_store_read_wait<0>();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = sees ? __uint_as_float(o[8 * i + e]) * inverse : 0.f;
          // 64-byte rows, swizzled as the store expects: the 16-byte piece's index XORed with bits 1-2 of the row
          st_shared_v4(stage + 64 * lane + ((i ^ (lane >> 1 & 3)) << 4), pack8(f));
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int to_row = 128 * mine.tile + 32 * quad;
          if (to_row < w.q_tokens) tma_store_4d(&p.y, channel, to_row, mine.head, u.b, stage);
          tma_store_commit();
        }
      }
      tc_fence_before();
      if (p.lse && half == 0) {
        // of the scores in units of log 2; +infinity, which makes every weight zero, for a row that sees nothing
        const float l = sees ? (ref == -INFINITY ? 0.f : ref) + log2f(sum) : INFINITY;
        p.lse[(static_cast<size_t>(u.b) * w.heads + mine.head) * (128 * static_cast<size_t>(w.q_tiles)) + q_row] = l;
      }
    }
    if (lane == 0) tma_store_read_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 18) {
    tc_fence_after();
    tmem_dealloc(tmem_slot, 512);
  }
}

template <int kD>
int window_fwd_launch(const WinFwdParams& p, cudaStream_t s) {
  constexpr int smem = WinFwdLayout<kD>::kSmem;
  const cudaError_t set = cudaFuncSetAttribute(window_fwd_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (set != cudaSuccess) return set_error(TS_ERR_CUDA, "window_fwd: %s", cudaGetErrorString(set));
  window_fwd_kernel<kD><<<p.n.units < 148 ? p.n.units : 148, kFwdThreads, smem, s>>>(p);
  return check_launch("window_fwd");
}

}  // namespace

bool win_map(CUtensorMap* map, const void* base, const long long* strides, int batch, int heads, int tokens, int dim,
             int rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(tokens), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(batch)};
  // a dimension of one has no stride of its own
  const int64_t any = (static_cast<int64_t>(dim) + 7) & ~7;
  const int64_t steps[3] = {tokens > 1 ? strides[2] : any, heads > 1 ? strides[1] : any, batch > 1 ? strides[0] : any};
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  return make_tmap_bf16_sw128(map, base, 4, dims, steps, box);
}

// The output in blocks of 32 rows and columns.
static bool win_out_map(CUtensorMap* map, const void* base, const long long* strides, const WinSizes& w) {
  const uint64_t dims[4] = {static_cast<uint64_t>(w.dim), static_cast<uint64_t>(w.q_tokens), static_cast<uint64_t>(w.heads),
                            static_cast<uint64_t>(w.batch)};
  const int64_t any = (static_cast<int64_t>(w.dim) + 7) & ~7;
  const int64_t steps[3] = {w.q_tokens > 1 ? strides[2] : any, w.heads > 1 ? strides[1] : any, w.batch > 1 ? strides[0] : any};
  const uint32_t box[4] = {32, 32, 1, 1};
  return make_tmap_bf16(map, base, 4, dims, steps, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

int win_sizes(const ts_window_args* a, WinSizes* w, const char* what) {
  if (!a) return set_error(TS_ERR_VALUE, "%s: null arguments", what);
  if (a->batch < 1 || a->heads < 1 || a->kv_heads < 1 || a->q_tokens < 1 || a->kv_tokens < a->q_tokens)
    return set_error(TS_ERR_VALUE, "%s: sizes must be positive and kv_tokens at least q_tokens", what);
  if (a->heads % a->kv_heads) return set_error(TS_ERR_VALUE, "%s: %d heads do not share %d key heads", what, a->heads, a->kv_heads);
  if (a->dim < 8 || a->dim > 128 || a->dim % 8)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "%s: head width %d is not a multiple of 8 up to 128", what, a->dim);
  if (a->kv_tokens > (1 << 30) || a->batch > 65535 || a->heads > 65535)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "%s: more than 2^30 tokens, 65535 sequences or 65535 heads", what);
  if (a->window < 1 || a->sinks < 0) return set_error(TS_ERR_VALUE, "%s: window must be >= 1 and sinks >= 0", what);
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return set_error(TS_ERR_VALUE, "%s: scale must be positive and finite", what);
  if (!a->q || !a->k || !a->v) return set_error(TS_ERR_VALUE, "%s: null tensor", what);
  w->batch = a->batch;
  w->heads = a->heads;
  w->kv_heads = a->kv_heads;
  w->share = a->heads / a->kv_heads;
  w->dim = a->dim;
  w->q_tokens = a->q_tokens;
  w->kv_tokens = a->kv_tokens;
  w->past = a->kv_tokens - a->q_tokens;
  w->window = a->window < a->kv_tokens ? a->window : a->kv_tokens;
  w->sinks = a->sinks < a->kv_tokens ? a->sinks : a->kv_tokens;
  w->q_tiles = ceil_div(a->q_tokens, 128);
  w->by_share = Divisor::of(w->share);
  w->by_kv_heads = Divisor::of(w->kv_heads);
  w->scale = a->scale;
  w->lengths = a->lengths;
  const long long units = static_cast<long long>(w->batch) * w->heads * (w->q_tiles + 1);
  if (units > 0x3fffffffll) return set_error(TS_ERR_NOT_IMPLEMENTED, "%s: too many query tiles", what);
  return TS_OK;
}

}  // namespace ts

using namespace ts;

extern "C" {

int ts_b200_window_fwd(const ts_window_args* a, ts_stream_t stream) {
  WinFwdParams p = {};
  if (const int rc = win_sizes(a, &p.w, "window_fwd")) return rc;
  if (!a->y) return set_error(TS_ERR_VALUE, "window_fwd: null output");
  const WinSizes& w = p.w;
  // two tiles to a CTA, which then seldom waits; one where all of them find an SM of their own (2 x 8 heads, 1000 queries:
  // 27 us, 34 in pairs)
  const int tiles = w.q_tiles * w.share;
  p.each = static_cast<long long>(w.batch) * w.kv_heads * tiles <= 148 ? 1 : 2;
  p.n = win_units(w, (tiles + p.each - 1) / p.each);
  p.sink_rows = w.sinks >= 128 ? 128 : round_up(w.sinks > 0 ? w.sinks : 1, 16);
  p.lse = a->lse;
  const bool ok = win_map(&p.q, a->q, a->q_strides, w.batch, w.heads, w.q_tokens, w.dim, 128) &&
                  win_map(&p.k, a->k, a->k_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, 128) &&
                  win_map(&p.v, a->v, a->v_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, 128) &&
                  win_map(&p.k_sink, a->k, a->k_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, p.sink_rows) &&
                  win_map(&p.v_sink, a->v, a->v_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, p.sink_rows) &&
                  win_out_map(&p.y, a->y, a->y_strides, w);
  if (!ok) return set_error(TS_ERR_VALUE, "window_fwd: bases and strides must be multiples of 16 bytes");
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return w.dim <= 64 ? window_fwd_launch<64>(p, s) : window_fwd_launch<128>(p, s);
}

}  // extern "C"
