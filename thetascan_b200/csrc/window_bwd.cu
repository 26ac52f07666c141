// Causal attention over a sliding window with first tokens that stay visible:
// the backward pass.
//
//   p_ij = exp(scale q_i.k_j - lse_i), delta_i = dy_i.y_i, ds_ij = p_ij (dy_i.v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij dy_i
//
// Two kernels, each with a tile's sums in tensor memory from first to last, so
// that no gradient is added up in an order that depends on timing: the first goes
// over the keys of a query tile (dq, and delta for the second), the other over the
// queries of a key tile, through all heads that share it (dk, dv).  Scores are
// formed in both: seven products instead of five, in exchange for no atomics and
// no f32 copy of dq.  The keys of first tokens meet all queries: their tiles are
// split among CTAs, whose sums go to a workspace in f32 and are joined in order.
//
// delta is formed of y as the forward stored it, in bf16: with the rounding of ds
// and the result's own a gradient is off by 2.6e-3 of its norm (1.7e-3 is its own
// rounding's), and no second copy of y is kept.
//
// Two or four threads share a row of a tile, with a part of the columns each; p
// and ds go back to tensor memory in bf16 and are the operand of the next
// product from there.  S^T = K Q^T and dP^T = V dY^T have
// keys in the rows, which is how dv and dk need them.
//
// The rows and the products of a tile wait for one another: narrow tiles are mostly
// forming p and ds, wide ones mostly products: 64 x 8 heads x 1024, width 64, window
// 256, sinks 4: 188 us for dq, 215 for dk and dv, 45 % of the issue slots, tensor
// cores at work for 18 and 25 %; 16 heads x 16384, width 128, window 2048, sinks 16:
// 489 and 576 us, 42 and 38 % of the issue slots, tensor cores 40 and 55 %.
#include "capi_internal.h"
#include "window.cuh"

namespace ts {

namespace {

// Warps 0-15: rows, 16: loads, 17: instructions, 18: tensor memory.  Of the 61440 registers that 640 threads of 96 are
// launched with, the row warps take 104 each, the others 64.  (With eight row warps each tile waited for them: 16 heads x
// 16384, width 128, window 2048 took 540 us for dq and 527 for dk and dv.)
constexpr int kBwdRowWarps = 16;
constexpr int kBwdThreads = 32 * (kBwdRowWarps + 4);
constexpr int kBwdRowRegs = 104, kBwdOtherRegs = 64;
static_assert(32 * (kBwdRowWarps * kBwdRowRegs + 4 * kBwdOtherRegs) <= kBwdThreads * 96, "registers");

template <int kD>
struct WinBwdLayout {
  static constexpr int kBoxes = kD / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kSwBox;
  // dq: q and dy, y where there is room, rings of keys (which wait for ds) and of values
  static constexpr bool kKeepsY = kD == 64;
  static constexpr int kKeySlots = kD == 64 ? 4 : 3, kValueSlots = kD == 64 ? 4 : 2;
  static constexpr uint32_t kSmemQ = (2 + (kKeepsY ? 1 : 0) + kKeySlots + kValueSlots) * kTileBytes + 1024;
  // dk and dv: k and v, a ring of q with dy, lse and delta
  static constexpr int kPairSlots = kD == 64 ? 4 : 2;
  static constexpr uint32_t kSmemKV = (2 + 2 * kPairSlots) * kTileBytes + kPairSlots * 1024 + 1024;
};

struct WinBwdParams {
  CUtensorMap q, k, v, k_sink, v_sink, y, dy;
  WinSizes w;
  WinUnits n;
  int sink_rows;
  // dk and dv: key tiles, the ones with first tokens, and the chunks (of `chunk` query tiles) that those are split in
  int key_tiles, sink_tiles, chunks, chunk;
  const float* lse;
  float* delta;
  float* partial;           // [batch, kv_heads, sink_tiles, chunks, dk and dv, dim padded, 128]
  const __nv_bfloat16* y_at;   // where the kernel reads y itself
  long long y_strides[3];
  __nv_bfloat16 *dq, *dk, *dv;
  long long dq_strides[3], dk_strides[3], dv_strides[3];
};

// 32 f32 columns of a row, scaled, to a bf16 row from channel c on (channels past dim left out).
__device__ __forceinline__ void store_row(__nv_bfloat16* row, const uint32_t (&r)[32], float scale, int c, int dim) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(r[8 * i + e]) * scale;
    if (c + 8 * i < dim) *reinterpret_cast<uint4*>(row + c + 8 * i) = pack8(f);
  }
}

// 2^(scale s - origin) of a pair of scores.  (A part of them by a polynomial, beside the special function unit, took
// longer: 16 heads x 16384, width 128, window 2048 464 -> 490 us for dq with half.)
__device__ __forceinline__ void weight_pair(uint32_t s0, uint32_t s1, Pair scale2, Pair origin, float& a, float& b) {
  fma2(Pair(__uint_as_float(s0), __uint_as_float(s1)), scale2, origin).get(a, b);
  a = exp2_fast(a);
  b = exp2_fast(b);
}

// ------------------------------------------------------------------ dq

// A query tile and the key tiles that it sees (as in the forward pass, for one tile).
struct WinQueryUnit {
  int b, head, kv_head, tile, length;
  bool live;
  int sinks, sink_tiles, first, count;

  __device__ __forceinline__ WinQueryUnit(const WinBwdParams& p, const WinOrder& order, int unit) {
    const WinSizes& w = p.w;
    int at;
    win_place<false>(order, p.n, w, unit, b, kv_head, at);
    tile = w.by_share(at);
    head = kv_head * w.share + at - tile * w.share;
    length = win_length(w, b);
    live = w.past + 128 * tile < length;
    const int end = min(w.past + 128 * tile + 127, length - 1);
    sinks = end < w.window ? 0 : min(w.sinks, end + 1);
    sink_tiles = (sinks + 127) >> 7;
    first = max(tile - ((w.window + 126) >> 7), (sinks - w.past) >> 7);
    count = live ? sink_tiles + max(0, tile - first + 1) : 0;
  }
  __device__ __forceinline__ int columns(int n) const {
    return n < sink_tiles ? min(128, (sinks - 128 * n + 15) & ~15) : 128;
  }
  __device__ __forceinline__ int key(const WinSizes& w, int n) const {
    return n < sink_tiles ? 128 * n : w.past + 128 * (first + n - sink_tiles);
  }
};

// ds of 32 columns from their weights p and dp, in bf16.  A hidden pair has p = 0 and whatever dp.
__device__ __forceinline__ void score_gradients(const uint32_t (&p)[32], const uint32_t (&dp)[32], float delta,
                                                uint32_t (&out)[16]) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    float d[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float w = __uint_as_float(p[e + i]);
      d[i] = w != 0.f ? w * (__uint_as_float(dp[e + i]) - delta) : 0.f;
    }
    out[e / 2] = pack_bf16(d[0], d[1]);
  }
}

template <int kD>
__global__ void __launch_bounds__(kBwdThreads, 1) window_bwd_q_kernel(const __grid_constant__ WinBwdParams p) {
  using L = WinBwdLayout<kD>;
  constexpr uint32_t kSlotStep = L::kTileBytes >> 4;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t k_full[L::kKeySlots], k_empty[L::kKeySlots], v_full[L::kValueSlots], v_empty[L::kValueSlots],
      q_full, q_empty, y_full, y_empty, s_full, dp_full, s_free, ds_full, ds_free, dq_full;
  __shared__ uint32_t tmem_slot;
  __shared__ WinOrder order;
  __shared__ float halves[2][128];   // free again before the next q_full, which waits for every row warp
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_at = base, dy_at = base + L::kTileBytes, keys = base + 2 * L::kTileBytes,
                 values = keys + L::kKeySlots * L::kTileBytes, y_at = values + L::kValueSlots * L::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinSizes& w = p.w;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kKeySlots; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < L::kValueSlots; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1 + kBwdRowWarps);   // the instructions, and the rows' reading of dy
    mbar_init(&y_full, 1);
    mbar_init(&y_empty, kBwdRowWarps);
    mbar_init(&s_full, 1);
    mbar_init(&dp_full, 1);
    mbar_init(&s_free, kBwdRowWarps);
    mbar_init(&ds_full, kBwdRowWarps);
    mbar_init(&ds_free, 1);
    mbar_init(&dq_full, 1);
    fence_mbar_init();
  }
  if (warp == 18) tmem_alloc(&tmem_slot, 512);
  if (warp == 1 && p.n.how == kWinTable)
    win_order(order, w, [&](int b) { return ((max(0, win_length(w, b) - w.past) + 127) >> 7) * w.share; });
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all of tensor memory: its addresses start at 0.  Columns: S, dP, dq, ds (bf16)
  constexpr uint32_t kDp = 128, kDq = 256, kDs = 384;

  if (warp >= kBwdRowWarps) {
    win_fewer_registers<kBwdOtherRegs>();
    if (warp == 16) {
      // ---- loads
      uint32_t it = 0, q_turn = 0, y_turn = 0;
      bool ok = true;
      auto load = [&](uint32_t to, uint64_t* full, uint64_t* empty, uint32_t turn, const CUtensorMap* map,
                      const CUtensorMap* sink_map, const WinQueryUnit& u, int n) {
        if (!(ok = ok && mbar_wait_warp(empty, (turn & 1) ^ 1, kErrMmaTimeout))) return;
        const bool sink = n < u.sink_tiles;
        if (elect_one()) {
          mbar_expect_tx(full, L::kBoxes * (sink ? p.sink_rows : 128) * 128);
#pragma unroll
          for (int c = 0; c < L::kBoxes; ++c)
            tma_load_4d(to + c * kSwBox, sink ? sink_map : map, 64 * c, u.key(w, n), u.kv_head, u.b, full);
        }
      };
      auto load_key = [&](const WinQueryUnit& u, int n) {
        const uint32_t s = it % L::kKeySlots;
        load(keys + s * L::kTileBytes, &k_full[s], &k_empty[s], it / L::kKeySlots, &p.k, &p.k_sink, u, n);
      };
      auto load_value = [&](const WinQueryUnit& u, int n) {
        const uint32_t s = it % L::kValueSlots;
        load(values + s * L::kTileBytes, &v_full[s], &v_empty[s], it / L::kValueSlots, &p.v, &p.v_sink, u, n);
        ++it;
      };
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinQueryUnit u(p, order, unit);
        if (u.count == 0) continue;
        load_key(u, 0);
        if (!(ok = ok && mbar_wait_warp(&q_empty, (q_turn++ & 1) ^ 1, kErrMmaTimeout))) break;
        if (elect_one()) {
          mbar_expect_tx(&q_full, 2 * L::kTileBytes);
#pragma unroll
          for (int c = 0; c < L::kBoxes; ++c) {
            tma_load_4d(q_at + c * kSwBox, &p.q, 64 * c, 128 * u.tile, u.head, u.b, &q_full);
            tma_load_4d(dy_at + c * kSwBox, &p.dy, 64 * c, 128 * u.tile, u.head, u.b, &q_full);
          }
        }
        load_value(u, 0);
        if (L::kKeepsY) {
          if (!(ok = ok && mbar_wait_warp(&y_empty, (y_turn++ & 1) ^ 1, kErrMmaTimeout))) break;
          if (elect_one()) {
            mbar_expect_tx(&y_full, L::kTileBytes);
#pragma unroll
            for (int c = 0; c < L::kBoxes; ++c)
              tma_load_4d(y_at + c * kSwBox, &p.y, 64 * c, 128 * u.tile, u.head, u.b, &y_full);
          }
        }
        for (int n = 1; n < u.count && ok; ++n) {
          load_key(u, n);
          load_value(u, n);
        }
      }
      if (!ok) {
        // given up: let the copies in flight land before the memory goes (for a bounded time too)
        auto landed = [](uint64_t* bar, uint32_t turn) {
          for (int poll = 0; poll < (1 << 16) && !mbar_try_wait(bar, turn & 1); ++poll) {
          }
        };
        for (uint32_t i = it > L::kKeySlots ? it - L::kKeySlots : 0; i <= it; ++i) {
          landed(&k_full[i % L::kKeySlots], i / L::kKeySlots);
          if (i < it) landed(&v_full[i % L::kValueSlots], i / L::kValueSlots);
        }
        if (q_turn > 0) landed(&q_full, q_turn - 1);
        if (y_turn > 0) landed(&y_full, y_turn - 1);
      }
    } else if (warp == 17) {
      // ---- instructions: the next S once the rows have this one in registers, the next dP and dq once they have sent ds
      constexpr uint32_t id_dq = idesc_bf16(128, kD, false, true), id_s = idesc_bf16(128, 128, false, false);
      const uint64_t q0 = win_rows(q_at), dy0 = win_rows(dy_at), k0 = win_rows(keys), v0 = win_rows(values), kt0 = win_inner(keys);
      uint32_t k_slot = 0, k_parity = 0, v_slot = 0, v_parity = 0, dq_slot = 0, q_parity = 0, s_parity = 1, ds_parity = 0;
      bool ok = true;
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinQueryUnit u(p, order, unit);
        if (u.count == 0) continue;
        auto id_of = [&](int n) { return n < u.sink_tiles ? idesc_bf16(128, u.columns(n), false, false) : id_s; };
        auto scores = [&](int n) {
          const uint32_t id = id_of(n);
          ok = ok && mbar_wait_warp(&k_full[k_slot], k_parity, kErrCopyTimeout) && mbar_wait_warp(&s_free, s_parity, kErrMmaTimeout);
          s_parity ^= 1;
          if (!ok) return;
          tc_fence_after();
          if (w.lengths && u.key(w, n) + 128 > u.length) win_clear_rows<L::kBoxes>(keys + k_slot * L::kTileBytes, u.length - u.key(w, n));
          const uint64_t k = k0 + k_slot * kSlotStep;
          if (elect_one()) {
#pragma unroll
            for (int s = 0; s < kD / 16; ++s) mma_bf16(0, win_rows_step(q0, s), win_rows_step(k, s), id, s > 0);
            mma_commit(&s_full);
          }
          if (++k_slot == L::kKeySlots) {
            k_slot = 0;
            k_parity ^= 1;
          }
        };
        // dP of tile n; by one lane
        auto weights = [&](int n, uint32_t id) {
          const uint64_t v = v0 + v_slot * kSlotStep;
#pragma unroll
          for (int s = 0; s < kD / 16; ++s) mma_bf16(kDp, win_rows_step(dy0, s), win_rows_step(v, s), id, s > 0);
          mma_commit(&dp_full);
          mma_commit(&v_empty[v_slot]);
          if (n == u.count - 1) mma_commit(&q_empty);
        };
        auto next_value = [&] {
          if (++v_slot == L::kValueSlots) {
            v_slot = 0;
            v_parity ^= 1;
          }
        };
        ok = ok && mbar_wait_warp(&q_full, q_parity, kErrCopyTimeout);
        q_parity ^= 1;
        scores(0);
        ok = ok && mbar_wait_warp(&v_full[v_slot], v_parity, kErrCopyTimeout);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) weights(0, id_of(0));
        next_value();
        for (int n = 0; n < u.count && ok; ++n) {
          const bool more = n + 1 < u.count;
          if (more) {
            scores(n + 1);
            ok = ok && mbar_wait_warp(&v_full[v_slot], v_parity, kErrCopyTimeout);
          }
          const uint32_t id = id_of(n + 1);
          const uint64_t k = kt0 + dq_slot * kSlotStep;
          const int steps = u.columns(n) >> 4;
          ok = ok && mbar_wait_warp(&ds_full, ds_parity, kErrMmaTimeout);
          ds_parity ^= 1;
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            if (more) weights(n + 1, id);
#pragma unroll
            for (int s = 0; s < 8; ++s)
              if (s < steps) mma_bf16_ts(kDq, kDs + 8 * s, win_inner_step(k, s), id_dq, n > 0 || s > 0);
            mma_commit(&ds_free);
            mma_commit(&k_empty[dq_slot]);
            if (!more) mma_commit(&dq_full);
          }
          if (more) next_value();
          if (++dq_slot == L::kKeySlots) dq_slot = 0;
        }
      }
    }
  } else {
    // ---- rows: part `part` of the columns of row `row`
    win_more_registers<kBwdRowRegs>();
    const int part = warp >> 2, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_at = lanes + 32 * part, dp_at = kDp + lanes + 32 * part, ds_at = kDs + lanes + 16 * part;
    const Pair scale2(w.scale * kLog2e);
    uint32_t turn = 0, it = 0, dq_turn = 0;
    bool ok = true;
    auto signal = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int unit = blockIdx.x; unit < p.n.units; unit += gridDim.x) {
      const WinQueryUnit u(p, order, unit);
      const int q_row = 128 * u.tile + row, at = w.past + q_row;
      const size_t stat = (static_cast<size_t>(u.b) * w.heads + u.head) * (128 * static_cast<size_t>(w.q_tiles)) + q_row;
      __nv_bfloat16* to = p.dq + u.b * p.dq_strides[0] + u.head * p.dq_strides[1] + q_row * p.dq_strides[2];
      if (u.count == 0) {
        // rows behind the sequence
        const uint32_t none[32] = {};
        if (q_row < w.q_tokens) store_row(to, none, 0.f, 32 * part, w.dim);
        if (part == 0) p.delta[stat] = 0.f;
        continue;
      }
      const Pair origin(-p.lse[stat]);
      // delta: half of the channels to each of two threads
      uint4 y[kD / 16];
      if (!L::kKeepsY && part < 2) {
        const __nv_bfloat16* from = p.y_at + u.b * p.y_strides[0] + u.head * p.y_strides[1] + q_row * p.y_strides[2];
#pragma unroll
        for (int i = 0; i < kD / 16; ++i) {
          const int c = 8 * (part * (kD / 16) + i);
          y[i] = q_row < w.q_tokens && c < w.dim ? __ldg(reinterpret_cast<const uint4*>(from + c)) : make_uint4(0, 0, 0, 0);
        }
      }
      ok = ok && mbar_wait(&q_full, turn & 1, kErrCopyTimeout) && (!L::kKeepsY || mbar_wait(&y_full, turn & 1, kErrCopyTimeout));
      ++turn;
      if (ok && part < 2) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kD / 16; ++i) {
          const int c8 = part * (kD / 16) + i;
          const uint32_t off = (c8 >> 3) * kSwBox + sw128_offset(row, c8 & 7);
          if (L::kKeepsY) y[i] = ld_shared_v4(y_at + off);
          float a[8], b[8];
          unpack8(ld_shared_v4(dy_at + off), a);
          unpack8(y[i], b);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(a[e], b[e], sum);
        }
        halves[part][row] = sum;
      }
      // The row warps meet here, and only here: they go on, or give up, together.  (All have read the dq of the unit
      // before, which this one's first ds lets be overwritten.)
      if (!threads_agree<32 * kBwdRowWarps>(1, ok)) break;
      const float delta = halves[0][row] + halves[1][row];
      if (part == 0) p.delta[stat] = delta;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&y_empty);
        mbar_arrive(&q_empty);
      }
      const int near = max(at - w.window + 1, u.sinks), upto = at < u.length ? at : -1;   // visible: first ones, near..upto
      // (a wait that has given up does not end this: lanes leave together, at the barrier above)
      for (int n = 0; n < u.count; ++n, ++it) {
        const int key = u.key(w, n) + 32 * part;
        const bool sink = n < u.sink_tiles;
        const int from = sink ? 0 : near - key, until = min(upto, sink ? u.sinks - 1 : upto) - key;
        // whether all, or any, of the warp's rows see all, or any, of its columns
        const bool all = __all_sync(0xffffffffu, from <= 0 && until >= 31);
        const bool some = all || __any_sync(0xffffffffu, from <= 31 && until >= 0 && from <= until);
        ok = ok && mbar_wait(&s_full, it & 1, kErrMmaTimeout);
        tc_fence_after();
        uint32_t s[32], d[32], out[16];
        tmem_ld(s_at, s);
        tmem_wait();
        tie(s);
        signal(&s_free);
        if (some) {
          if (!all) hide(s, from, until);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float a, b;
            weight_pair(s[e], s[e + 1], scale2, origin, a, b);
            s[e] = __float_as_uint(a);
            s[e + 1] = __float_as_uint(b);
          }
        }
        ok = ok && mbar_wait(&dp_full, it & 1, kErrMmaTimeout) && mbar_wait(&ds_free, (it & 1) ^ 1, kErrMmaTimeout);
        tc_fence_after();
        tmem_ld(dp_at, d);
        tmem_wait();
        tie(d);
        if (some) {
          score_gradients(s, d, delta, out);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) out[e] = 0;
        }
        tmem_st(ds_at, out);
        tmem_store_wait();
        signal(&ds_full);
      }
      ok = ok && mbar_wait(&dq_full, dq_turn++ & 1, kErrMmaTimeout);
      tc_fence_after();
      if (32 * part < w.dim) {
        uint32_t r[32];
        tmem_ld(kDq + lanes + 32 * part, r);
        tmem_wait();
        tie(r);
        if (ok && q_row < w.q_tokens) store_row(to, r, w.scale, 32 * part, w.dim);
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 18) {
    tc_fence_after();
    tmem_dealloc(tmem_slot, 512);
  }
}

// ------------------------------------------------------------------ dk, dv

// A key tile (or one chunk of the queries of one that holds first tokens) and the query tiles that see it.
struct WinKeyUnit {
  int b, kv_head, tile, chunk, length;
  int first, tiles, count;   // query tiles first .. first + tiles - 1 of each head that shares the keys
  bool split;

  __device__ __forceinline__ WinKeyUnit(const WinBwdParams& p, const WinOrder& order, int unit) {
    const WinSizes& w = p.w;
    int at;
    win_place<true>(order, p.n, w, unit, b, kv_head, at);
    const bool sink = at < p.sink_tiles * p.chunks;
    tile = sink ? at / p.chunks : at - p.sink_tiles * p.chunks + p.sink_tiles;
    chunk = sink ? at - tile * p.chunks : 0;
    split = sink && p.chunks > 1;
    length = win_length(w, b);
    const int key = 128 * tile, end = min(key + 127, length - 1);
    const int last = sink ? length - 1 : min(length - 1, end + w.window - 1);   // the last position that sees any
    int low = max(0, (key - w.past) >> 7), high = min(w.q_tiles - 1, (last - w.past) >> 7);
    if (sink) {
      low = max(low, chunk * p.chunk);
      high = min(high, (chunk + 1) * p.chunk - 1);
    }
    first = low;
    tiles = key < length ? max(0, high - low + 1) : 0;
    count = tiles * w.share;
  }
  __device__ __forceinline__ void query(const WinSizes& w, int n, int& head, int& q_tile) const {
    const int g = n / tiles;
    head = kv_head * w.share + g;
    q_tile = first + n - g * tiles;
  }
};

// Threads that share a row.  (Four at width 64, where tiles are short work: 64 x 8 heads x 1024, window 256 took 310 us so
// and 337 with two, one key head after another; two at width 128: 16 heads x 16384, window 2048 582 us with four.)
constexpr int kv_parts(int d) { return d == 64 ? 4 : 2; }
constexpr int kv_row_warps(int d) { return 4 * kv_parts(d); }
constexpr int kv_threads(int d) { return 32 * (kv_row_warps(d) + 4); }

template <int kD>
__global__ void __launch_bounds__(kv_threads(kD), 1) window_bwd_kv_kernel(const __grid_constant__ WinBwdParams p) {
  using L = WinBwdLayout<kD>;
  constexpr int kSlots = L::kPairSlots, kParts = kv_parts(kD), kRowWarps = kv_row_warps(kD), kCols = 128 / kParts;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t full[kSlots], empty[kSlots], kv_full, kv_empty, s_full, dp_full, p_full, ds_full, done;
  __shared__ uint32_t tmem_slot;
  __shared__ WinOrder order;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t k_at = base, v_at = base + L::kTileBytes, ring = base + 2 * L::kTileBytes;
  const uint32_t stats = ring + 2 * kSlots * L::kTileBytes;   // of each slot: 128 lse, 128 delta
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinSizes& w = p.w;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&kv_full, 1);
    mbar_init(&kv_empty, 1);
    mbar_init(&s_full, 1);
    mbar_init(&dp_full, 1);
    mbar_init(&p_full, kRowWarps);
    mbar_init(&ds_full, kRowWarps);
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == kRowWarps + 2) tmem_alloc(&tmem_slot, 512);
  if (warp == 1 && p.n.how == kWinTable)
    win_order(order, w, [&](int b) {   // first tokens' chunks, and the tiles behind them that hold keys
      const int length = win_length(w, b);
      return length > 0 ? p.sink_tiles * p.chunks + max(0, ((length + 127) >> 7) - p.sink_tiles) : 0;
    });
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all of tensor memory: its addresses start at 0.  Columns: S^T and P^T in its place (each group of warps within its
  // columns), dP^T and dS^T in its place, dv, dk
  constexpr uint32_t kDp = 128, kDv = 256, kDk = 384;

  if (warp >= kRowWarps) {
    if constexpr (kParts == 4) win_fewer_registers<kBwdOtherRegs>();
    if (warp == kRowWarps) {
      // ---- loads
      uint32_t it = 0, turn = 0;
      bool ok = true;
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinKeyUnit u(p, order, unit);
        if (u.count == 0) continue;
        if (!(ok = mbar_wait_warp(&kv_empty, (turn++ & 1) ^ 1, kErrMmaTimeout))) break;
        if (elect_one()) {
          mbar_expect_tx(&kv_full, 2 * L::kTileBytes);
#pragma unroll
          for (int c = 0; c < L::kBoxes; ++c) {
            tma_load_4d(k_at + c * kSwBox, &p.k, 64 * c, 128 * u.tile, u.kv_head, u.b, &kv_full);
            tma_load_4d(v_at + c * kSwBox, &p.v, 64 * c, 128 * u.tile, u.kv_head, u.b, &kv_full);
          }
        }
        for (int n = 0; n < u.count; ++n, ++it) {
          const uint32_t s = it % kSlots;
          if (!(ok = mbar_wait_warp(&empty[s], ((it / kSlots) & 1) ^ 1, kErrMmaTimeout))) break;
          int head, tile;
          u.query(w, n, head, tile);
          const size_t stat = (static_cast<size_t>(u.b) * w.heads + head) * (128 * static_cast<size_t>(w.q_tiles)) + 128 * tile;
          if (elect_one()) {
            const uint32_t to = ring + s * 2 * L::kTileBytes;
            mbar_expect_tx(&full[s], 2 * L::kTileBytes + 1024);
#pragma unroll
            for (int c = 0; c < L::kBoxes; ++c) {
              tma_load_4d(to + c * kSwBox, &p.q, 64 * c, 128 * tile, head, u.b, &full[s]);
              tma_load_4d(to + L::kTileBytes + c * kSwBox, &p.dy, 64 * c, 128 * tile, head, u.b, &full[s]);
            }
            bulk_load(stats + 1024 * s, p.lse + stat, 512, &full[s]);
            bulk_load(stats + 1024 * s + 512, p.delta + stat, 512, &full[s]);
          }
        }
      }
      if (!ok) {
        // given up: let the copies in flight land before the memory goes (for a bounded time too)
        for (uint32_t i = it > kSlots ? it - kSlots : 0; i < it; ++i)
          for (int poll = 0; poll < (1 << 16) && !mbar_try_wait(&full[i % kSlots], (i / kSlots) & 1); ++poll) {
          }
        for (int poll = 0; poll < (1 << 16) && turn > 0 && !mbar_try_wait(&kv_full, (turn - 1) & 1); ++poll) {
        }
      }
    } else if (warp == kRowWarps + 1) {
      // ---- instructions: while the rows form ds of this query tile, dv and the next S; while they form the next p, dk
      // and the next dP
      constexpr uint32_t id_s = idesc_bf16(128, 128, false, false), id_d = idesc_bf16(128, kD, false, true);
      constexpr uint32_t kStep = 2 * L::kTileBytes >> 4, kHalf = L::kTileBytes >> 4;   // a slot's queries, its gradients
      const uint64_t k0 = win_rows(k_at), v0 = win_rows(v_at), rows0 = win_rows(ring), inner0 = win_inner(ring);
      uint32_t slot = 0, parity = 0, kv_parity = 0, p_parity = 0;
      bool ok = true;
      // S^T or dP^T: rows of K or V with rows of a slot's queries or their gradients; by one lane
      auto product = [&](uint32_t to, uint64_t a, uint64_t b, uint64_t* finished) {
#pragma unroll
        for (int s = 0; s < kD / 16; ++s) mma_bf16(to, win_rows_step(a, s), win_rows_step(b, s), id_s, s > 0);
        mma_commit(finished);
      };
      // dv or dk: what lies at `a` in tensor memory, kCols queries in each part
      auto sum = [&](uint32_t to, uint32_t a, uint64_t b, bool more) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          mma_bf16_ts(to, a + kCols * (16 * s / kCols) + 16 * s % kCols / 2, win_inner_step(b, s), id_d, more || s > 0);
      };
      for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
        const WinKeyUnit u(p, order, unit);
        if (u.count == 0) continue;
        int tile = u.first;   // of the queries that come next
        auto queries_landed = [&] {
          const int limit = u.length - w.past - 128 * tile;
          if (w.lengths && limit < 128) {
            win_clear_rows<L::kBoxes>(ring + 2 * slot * L::kTileBytes, limit);
            win_clear_rows<L::kBoxes>(ring + (2 * slot + 1) * L::kTileBytes, limit);
          }
          tile = tile + 1 == u.first + u.tiles ? u.first : tile + 1;
        };
        ok = ok && mbar_wait_warp(&kv_full, kv_parity, kErrCopyTimeout) && mbar_wait_warp(&full[slot], parity, kErrCopyTimeout);
        kv_parity ^= 1;
        if (!ok) break;
        tc_fence_after();
        queries_landed();
        if (elect_one()) {
          product(0, k0, rows0 + slot * kStep, &s_full);
          product(kDp, v0, rows0 + slot * kStep + kHalf, &dp_full);
        }
        for (int n = 0; n < u.count && ok; ++n) {
          const bool more = n + 1 < u.count;
          const uint32_t now = slot;
          slot = slot + 1 == kSlots ? 0 : slot + 1;
          parity ^= slot == 0;
          if (more && (ok = mbar_wait_warp(&full[slot], parity, kErrCopyTimeout))) queries_landed();
          ok = ok && mbar_wait_warp(&p_full, p_parity, kErrMmaTimeout);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            sum(kDv, 0, inner0 + now * kStep + kHalf, n > 0);
            if (more) product(0, k0, rows0 + slot * kStep, &s_full);
          }
          ok = mbar_wait_warp(&ds_full, p_parity, kErrMmaTimeout);
          p_parity ^= 1;
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            sum(kDk, kDp, inner0 + now * kStep, n > 0);
            mma_commit(&empty[now]);
            if (more) product(kDp, v0, rows0 + slot * kStep + kHalf, &dp_full);
          }
        }
        if (ok && elect_one()) {
          mma_commit(&kv_empty);
          mma_commit(&done);
        }
      }
    }
  } else {
    // ---- rows: part `part` of the columns (queries) of row `row` (a key)
    if constexpr (kParts == 4) win_more_registers<kBwdRowRegs>();
    const int part = warp >> 2, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_at = lanes + kCols * part, dp_at = kDp + lanes + kCols * part;
    const Pair scale2(w.scale * kLog2e);
    uint32_t slot = 0, parity = 0, it = 0, turn = 0;
    bool ok = true;
    auto signal = [&](uint64_t* bar) {
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int unit = blockIdx.x; unit < p.n.units && ok; unit += gridDim.x) {
      const WinKeyUnit u(p, order, unit);
      const int key = 128 * u.tile + row;
      const bool is_key = key < u.length, everywhere = key < w.sinks;
      const int last = is_key ? (everywhere ? u.length - 1 : min(u.length - 1, key + w.window - 1)) : -1;
      int tile = u.first;
      // (a wait that has given up does not end this: the lanes of a warp leave together, below)
      for (int n = 0; n < u.count; ++n, ++it) {
        // the columns (queries) that see this row's key
        const int first = w.past + 128 * tile + kCols * part, from = key - first, until = last - first;
        tile = tile + 1 == u.first + u.tiles ? u.first : tile + 1;
        const bool all = __all_sync(0xffffffffu, from <= 0 && until >= kCols - 1);
        const bool some = all || __any_sync(0xffffffffu, from <= kCols - 1 && until >= 0 && from <= until);
        ok = ok && mbar_wait(&full[slot], parity, kErrCopyTimeout) && mbar_wait(&s_full, it & 1, kErrMmaTimeout);
        tc_fence_after();
        const uint32_t lse = stats + 1024 * slot + 4 * kCols * part, delta = lse + 512;
        slot = slot + 1 == kSlots ? 0 : slot + 1;
        parity ^= slot == 0;
        uint32_t s[kCols / 32][32];
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_ld(s_at + 32 * c, s[c]);
        tmem_wait();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t out[16];
          tie(s[c]);
          if (some) {
            if (!all) hide(s[c], from - 32 * c, until - 32 * c);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const uint4 l = ld_shared_v4(lse + 128 * c + 4 * e);
              const uint32_t of[4] = {l.x, l.y, l.z, l.w};
              float f[4];
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                weight_pair(s[c][e + i], s[c][e + i + 1], scale2, Pair(-__uint_as_float(of[i]), -__uint_as_float(of[i + 1])),
                            f[i], f[i + 1]);
                s[c][e + i] = __float_as_uint(f[i]);
                s[c][e + i + 1] = __float_as_uint(f[i + 1]);
              }
              out[e / 2] = pack_bf16(f[0], f[1]);
              out[e / 2 + 1] = pack_bf16(f[2], f[3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) out[e] = 0;
          }
          tmem_st(s_at + 16 * c, out);
        }
        signal(&p_full);
        ok = ok && mbar_wait(&dp_full, it & 1, kErrMmaTimeout);
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t d[32], out[16];
          tmem_ld(dp_at + 32 * c, d);
          tmem_wait();
          tie(d);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const uint4 l = ld_shared_v4(delta + 128 * c + 4 * e);
            const uint32_t of[4] = {l.x, l.y, l.z, l.w};
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float weight = some ? __uint_as_float(s[c][e + i]) : 0.f;
              f[i] = weight != 0.f ? weight * (__uint_as_float(d[e + i]) - __uint_as_float(of[i])) : 0.f;
            }
            out[e / 2] = pack_bf16(f[0], f[1]);
            out[e / 2 + 1] = pack_bf16(f[2], f[3]);
          }
          tmem_st(dp_at + 16 * c, out);
        }
        signal(&ds_full);
      }
      ok = ok && (u.count == 0 || mbar_wait(&done, turn++ & 1, kErrMmaTimeout));
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      // even parts: dv, odd ones: dk; with four, half of the channels each
      constexpr int kChannels = 2 * kD / kParts;
      const int what = part & 1;
      const uint32_t acc = (what ? kDk : kDv) + lanes;
      const long long* strides = what ? p.dk_strides : p.dv_strides;
      __nv_bfloat16* to = (what ? p.dk : p.dv) + u.b * strides[0] + u.kv_head * strides[1] + key * strides[2];
      const float scale = u.count == 0 ? 0.f : what ? w.scale : 1.f;
      const size_t item = ((static_cast<size_t>(u.b) * w.kv_heads + u.kv_head) * p.sink_tiles + u.tile) * p.chunks + u.chunk;
      float* sums = p.partial + (item * 2 + what) * (kD * 128) + row;
#pragma unroll 1
      for (int c = kChannels * (part >> 1); c < kChannels * ((part >> 1) + 1) && c < w.dim; c += 32) {
        uint32_t r[32];
        tmem_ld(acc + c, r);
        tmem_wait();
        tie(r);
        if (u.count == 0) {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0;
        }
        if (u.split) {
#pragma unroll
          for (int e = 0; e < 32; ++e) __stcg(sums + (c + e) * 128, __uint_as_float(r[e]) * scale);
        } else if (key < w.kv_tokens) {
          store_row(to, r, scale, c, w.dim);
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kRowWarps + 2) {
    tc_fence_after();
    tmem_dealloc(tmem_slot, 512);
  }
}

// The sums of first tokens' key tiles, chunk by chunk; a CTA for each 8 channels of a tile of dk or dv.
template <int kD>
__global__ void __launch_bounds__(128) window_bwd_join_kernel(const __grid_constant__ WinBwdParams p) {
  const WinSizes& w = p.w;
  const int part = blockIdx.y % (kD / 8), what = blockIdx.y / (kD / 8), tile = blockIdx.x % p.sink_tiles;
  const int row = blockIdx.x / p.sink_tiles, b = row / w.kv_heads, kv_head = row - b * w.kv_heads;
  const int key = 128 * tile + threadIdx.x, c = 8 * part;
  if (key >= w.kv_tokens || c >= w.dim) return;
  const float* from = p.partial + (static_cast<size_t>(blockIdx.x) * p.chunks * 2 + what) * (kD * 128) + c * 128 + threadIdx.x;
  float sum[8] = {};
#pragma unroll 4
  for (int i = 0; i < p.chunks; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += __ldcg(from + static_cast<size_t>(i) * (2 * kD * 128) + e * 128);
  }
  const long long* strides = what ? p.dk_strides : p.dv_strides;
  __nv_bfloat16* to = (what ? p.dk : p.dv) + b * strides[0] + kv_head * strides[1] + key * strides[2];
  *reinterpret_cast<uint4*>(to + c) = pack8(sum);
}

size_t win_stats_bytes(const WinSizes& w) {
  return static_cast<size_t>(w.batch) * w.heads * w.q_tiles * 128 * sizeof(float);
}
// Tiles of first tokens and how they are split: chunks as long as the other tiles' work, eight query tiles at least.
void win_split(const WinSizes& w, WinBwdParams* p) {
  p->key_tiles = ceil_div(w.kv_tokens, 128);
  // sinks that the window reaches from everywhere need no tiles of their own
  p->sink_tiles = w.window >= w.kv_tokens ? 0 : ceil_div(w.sinks, 128);
  const int usual = (w.window + 126) / 128 + 1;
  p->chunk = usual < 8 ? 8 : usual;
  p->chunks = ceil_div(w.q_tiles, p->chunk);
  // their sums are kept until they are joined: no more chunks than 16 for each SM, of all key tiles together (310 MB at
  // width 128; 64 sequences x 8 heads x 16384 with 4096 first tokens would take 34 GB)
  const long long rows = static_cast<long long>(w.batch) * w.kv_heads * p->sink_tiles;
  if (p->chunks > 1 && rows * p->chunks > 16 * 148) {
    const long long most = rows < 16 * 148 ? 16 * 148 / rows : 1;
    p->chunk = static_cast<int>((w.q_tiles + most - 1) / most);
    p->chunks = ceil_div(w.q_tiles, p->chunk);
  }
}
size_t win_partial_bytes(const WinSizes& w, const WinBwdParams& p) {
  if (p.chunks < 2) return 0;
  return static_cast<size_t>(w.batch) * w.kv_heads * p.sink_tiles * p.chunks * 2 * (w.dim <= 64 ? 64 : 128) * 128 * sizeof(float);
}

template <int kD>
int window_bwd_launch(WinBwdParams& p, cudaStream_t s) {
  using L = WinBwdLayout<kD>;
  const WinSizes& w = p.w;
  cudaError_t set = cudaFuncSetAttribute(window_bwd_q_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemQ);
  if (set == cudaSuccess)
    set = cudaFuncSetAttribute(window_bwd_kv_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemKV);
  if (set != cudaSuccess) return set_error(TS_ERR_CUDA, "window_bwd: %s", cudaGetErrorString(set));
  p.n = win_units(w, w.share * w.q_tiles);
  window_bwd_q_kernel<kD><<<p.n.units < 148 ? p.n.units : 148, kBwdThreads, L::kSmemQ, s>>>(p);
  if (const int rc = check_launch("window_bwd_q")) return rc;
  p.n = win_units(w, p.sink_tiles * p.chunks + p.key_tiles - p.sink_tiles);
  window_bwd_kv_kernel<kD><<<p.n.units < 148 ? p.n.units : 148, kv_threads(kD), L::kSmemKV, s>>>(p);
  if (const int rc = check_launch("window_bwd_kv")) return rc;
  if (p.sink_tiles == 0 || p.chunks < 2) return TS_OK;
  window_bwd_join_kernel<kD><<<dim3(w.batch * w.kv_heads * p.sink_tiles, kD / 8 * 2), 128, 0, s>>>(p);
  return check_launch("window_bwd_join");
}

}  // namespace

}  // namespace ts

using namespace ts;

extern "C" {

size_t ts_b200_window_bwd_workspace_bytes(const ts_window_args* a) {
  WinSizes w = {};
  if (win_sizes(a, &w, "window_bwd") != TS_OK) return 0;
  WinBwdParams p = {};
  win_split(w, &p);
  return win_stats_bytes(w) + win_partial_bytes(w, p);
}

int ts_b200_window_bwd(const ts_window_args* a, const ts_window_grad_args* g, ts_stream_t stream) {
  WinBwdParams p = {};
  if (const int rc = win_sizes(a, &p.w, "window_bwd")) return rc;
  const WinSizes& w = p.w;
  if (!g || !g->dy || !g->dq || !g->dk || !g->dv || !a->y || !a->lse)
    return set_error(TS_ERR_VALUE, "window_bwd: null tensor");
  win_split(w, &p);
  const size_t stats = win_stats_bytes(w);
  if (!g->workspace || g->workspace_bytes < stats + win_partial_bytes(w, p))
    return set_error(TS_ERR_VALUE, "window_bwd: workspace too small");
  // the kernel of dk and dv copies lse and delta in pieces of 16 bytes
  if (reinterpret_cast<uintptr_t>(a->lse) % 16 || reinterpret_cast<uintptr_t>(g->workspace) % 16)
    return set_error(TS_ERR_VALUE, "window_bwd: lse and workspace must be 16-byte aligned");
  if (static_cast<long long>(w.batch) * w.kv_heads * (static_cast<long long>(p.sink_tiles) * p.chunks + p.key_tiles) > 0x3fffffffll)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "window_bwd: too many key tiles");
  p.sink_rows = w.sinks >= 128 ? 128 : round_up(w.sinks > 0 ? w.sinks : 1, 16);
  p.lse = a->lse;
  p.delta = static_cast<float*>(g->workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(g->workspace) + stats);
  p.y_at = static_cast<const __nv_bfloat16*>(a->y);
  p.dq = static_cast<__nv_bfloat16*>(g->dq);
  p.dk = static_cast<__nv_bfloat16*>(g->dk);
  p.dv = static_cast<__nv_bfloat16*>(g->dv);
  for (int i = 0; i < 3; ++i) {
    p.y_strides[i] = a->y_strides[i];
    p.dq_strides[i] = g->dq_strides[i];
    p.dk_strides[i] = g->dk_strides[i];
    p.dv_strides[i] = g->dv_strides[i];
    for (long long s : {g->dq_strides[i], g->dk_strides[i], g->dv_strides[i]})
      if (s % 8) return set_error(TS_ERR_VALUE, "window_bwd: strides must be multiples of 8");
  }
  for (const void* t : {g->dq, g->dk, g->dv})
    if (reinterpret_cast<uintptr_t>(t) % 16) return set_error(TS_ERR_VALUE, "window_bwd: bases must be 16-byte aligned");
  const bool ok = win_map(&p.q, a->q, a->q_strides, w.batch, w.heads, w.q_tokens, w.dim, 128) &&
                  win_map(&p.k, a->k, a->k_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, 128) &&
                  win_map(&p.v, a->v, a->v_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, 128) &&
                  win_map(&p.k_sink, a->k, a->k_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, p.sink_rows) &&
                  win_map(&p.v_sink, a->v, a->v_strides, w.batch, w.kv_heads, w.kv_tokens, w.dim, p.sink_rows) &&
                  win_map(&p.y, a->y, a->y_strides, w.batch, w.heads, w.q_tokens, w.dim, 128) &&
                  win_map(&p.dy, g->dy, g->dy_strides, w.batch, w.heads, w.q_tokens, w.dim, 128);
  if (!ok) return set_error(TS_ERR_VALUE, "window_bwd: bases and strides must be multiples of 16 bytes");
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return w.dim <= 64 ? window_bwd_launch<64>(p, s) : window_bwd_launch<128>(p, s);
}

}  // extern "C"
