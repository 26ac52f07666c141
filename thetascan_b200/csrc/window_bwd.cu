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
// In both, thread t of warps 0-3 and its partner in warps 4-7 own a row of the
// tile and half of the columns; p and ds go back to tensor memory in bf16 and are
// the operand of the next product from there.  S^T = K Q^T and dP^T = V dY^T have
// keys in the rows, which is how dv and dk need them.
#include "capi_internal.h"
#include "window.cuh"

namespace ts {

namespace {

// Warps 0-7: rows, 8: loads, 9: instructions, 10: tensor memory.
constexpr int kBwdThreads = 384;

template <int kD>
struct WinBwdLayout {
  static constexpr int kBoxes = kD / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kSwBox;
  static constexpr int kSlots = kD == 64 ? 8 : 4;
  static constexpr int kPairSlots = kSlots / 2;                          // of queries and their gradients
  static constexpr uint32_t kRingBytes = kSlots * kTileBytes;
  static constexpr uint32_t kSmemQ = 3 * kTileBytes + kRingBytes + 1024;                      // q, dy, y; keys and values
  static constexpr uint32_t kSmemKV = 2 * kTileBytes + kRingBytes + kPairSlots * 1024 + 1024; // k, v; q, dy; lse, delta
};

struct WinBwdParams {
  CUtensorMap q, k, v, k_sink, v_sink, y, dy;
  WinSizes w;
  int units;
  int sink_rows;
  // dk and dv: key tiles, the ones with first tokens, and the chunks (of `chunk` query tiles) that those are split in
  int key_tiles, sink_tiles, chunks, chunk;
  const float* lse;
  float* delta;
  float* partial;           // [batch, kv_heads, sink_tiles, chunks, dk and dv, dim padded, 128]
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

// ------------------------------------------------------------------ dq

// A query tile and the key tiles that it sees (as in the forward pass, for one tile).
struct WinQueryUnit {
  int b, head, kv_head, tile, length;
  bool live;
  int sinks, sink_tiles, first, count;

  __device__ __forceinline__ WinQueryUnit(const WinSizes& w, int unit) {
    const int row = unit / (w.q_tiles * w.share), at = unit - row * (w.q_tiles * w.share);
    b = row / w.kv_heads;
    kv_head = row - b * w.kv_heads;
    tile = at / w.share;
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

// Whether `ok` holds in all of the 256 row threads (a barrier among them).
__device__ __forceinline__ bool rows_all(bool ok) {
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

template <int kD>
__global__ void __launch_bounds__(kBwdThreads, 1) window_bwd_q_kernel(const __grid_constant__ WinBwdParams p) {
  using L = WinBwdLayout<kD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t full[L::kSlots], empty[L::kSlots], q_full, q_empty, y_full, y_empty, s_full, dp_full,
      s_free, dp_free, ds_full, ds_free, dq_full;
  __shared__ uint32_t tmem_slot;
  __shared__ float halves[2][128];   // free again before the next q_full, which waits for every row warp
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_at = base, dy_at = base + L::kTileBytes, y_at = base + 2 * L::kTileBytes, ring = base + 3 * L::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WinSizes& w = p.w;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 9);   // the instructions, and the rows' reading of dy
    mbar_init(&y_full, 1);
    mbar_init(&y_empty, 8);
    mbar_init(&s_full, 1);
    mbar_init(&dp_full, 1);
    mbar_init(&s_free, 8);
    mbar_init(&dp_free, 8);
    mbar_init(&ds_full, 8);
    mbar_init(&ds_free, 1);
    mbar_init(&dq_full, 1);
    fence_mbar_init();
  }
  if (warp == 10) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all of tensor memory: its addresses start at 0.  Columns: S, dP, dq, ds (bf16)
  constexpr uint32_t kDp = 128, kDq = 256, kDs = 384;

  if (warp == 8) {
    // ---- loads
    uint32_t it = 0, q_turn = 0, y_turn = 0;
    bool ok = true;
    auto load = [&](const CUtensorMap* map, const CUtensorMap* sink_map, const WinQueryUnit& u, int n) {
      const uint32_t s = it % L::kSlots;
      if (!(ok = ok && mbar_wait_warp(&empty[s], ((it / L::kSlots) & 1) ^ 1, kErrMmaTimeout))) return;
      const bool sink = n < u.sink_tiles;
      if (elect_one()) {
        mbar_expect_tx(&full[s], L::kBoxes * (sink ? p.sink_rows : 128) * 128);
#pragma unroll
        for (int c = 0; c < L::kBoxes; ++c)
          tma_load_4d(ring + s * L::kTileBytes + c * kSwBox, sink ? sink_map : map, 64 * c, u.key(w, n), u.kv_head, u.b,
                      &full[s]);
      }
      ++it;
    };
    for (int unit = blockIdx.x; unit < p.units && ok; unit += gridDim.x) {
      const WinQueryUnit u(w, unit);
      if (u.count == 0) continue;
      if (!(ok = mbar_wait_warp(&q_empty, (q_turn++ & 1) ^ 1, kErrMmaTimeout))) break;
      if (elect_one()) {
        mbar_expect_tx(&q_full, 2 * L::kTileBytes);
#pragma unroll
        for (int c = 0; c < L::kBoxes; ++c) {
          tma_load_4d(q_at + c * kSwBox, &p.q, 64 * c, 128 * u.tile, u.head, u.b, &q_full);
          tma_load_4d(dy_at + c * kSwBox, &p.dy, 64 * c, 128 * u.tile, u.head, u.b, &q_full);
        }
      }
      load(&p.k, &p.k_sink, u, 0);
      load(&p.v, &p.v_sink, u, 0);
      if (!(ok = ok && mbar_wait_warp(&y_empty, (y_turn++ & 1) ^ 1, kErrMmaTimeout))) break;
      if (elect_one()) {
        mbar_expect_tx(&y_full, L::kTileBytes);
#pragma unroll
        for (int c = 0; c < L::kBoxes; ++c)
          tma_load_4d(y_at + c * kSwBox, &p.y, 64 * c, 128 * u.tile, u.head, u.b, &y_full);
      }
      for (int n = 1; n < u.count && ok; ++n) {
        load(&p.k, &p.k_sink, u, n);
        load(&p.v, &p.v_sink, u, n);
      }
    }
    if (!ok) {
      // given up: let the copies in flight land before the memory goes (for a bounded time too)
      for (uint32_t i = it > L::kSlots ? it - L::kSlots : 0; i < it; ++i)
        for (int poll = 0; poll < (1 << 16) && !mbar_try_wait(&full[i % L::kSlots], (i / L::kSlots) & 1); ++poll) {
        }
      for (int poll = 0; poll < (1 << 16) && q_turn > 0 && !mbar_try_wait(&q_full, (q_turn - 1) & 1); ++poll) {
      }
      for (int poll = 0; poll < (1 << 16) && y_turn > 0 && !mbar_try_wait(&y_full, (y_turn - 1) & 1); ++poll) {
      }
    }
  } else if (warp == 9) {
    // ---- instructions
    uint32_t it = 0, q_turn = 0, n_s = 0, n_ds = 0;
    bool ok = true;
    constexpr uint32_t id_dq = idesc_bf16(128, kD, false, true);
    const uint64_t q0 = win_rows(q_at), dy0 = win_rows(dy_at);
    for (int unit = blockIdx.x; unit < p.units && ok; unit += gridDim.x) {
      const WinQueryUnit u(w, unit);
      if (u.count == 0) continue;
      // a product of the query side (rows in shared memory) with ring item `item`, once its place is free
      auto product = [&](uint32_t to, uint64_t a, uint32_t item, int n, uint64_t* free, uint64_t* done) {
        ok = ok && mbar_wait_warp(free, (n_s & 1) ^ 1, kErrMmaTimeout) &&
             mbar_wait_warp(&full[item % L::kSlots], (item / L::kSlots) & 1, kErrCopyTimeout);
        if (!ok) return;
        tc_fence_after();
        const uint64_t b = win_rows(ring + item % L::kSlots * L::kTileBytes);
        const uint32_t id = idesc_bf16(128, u.columns(n), false, false);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < kD / 16; ++s) mma_bf16(to, win_rows_step(a, s), win_rows_step(b, s), id, s > 0);
          mma_commit(done);
        }
      };
      if (!(ok = mbar_wait_warp(&q_full, q_turn++ & 1, kErrCopyTimeout))) break;
      tc_fence_after();
      product(0, q0, it, 0, &s_free, &s_full);
      product(kDp, dy0, it + 1, 0, &dp_free, &dp_full);
      if (ok && elect_one()) {
        mma_commit(&empty[(it + 1) % L::kSlots]);
        if (u.count == 1) mma_commit(&q_empty);
      }
      ++n_s;
      for (int n = 0; n < u.count && ok; ++n, it += 2) {
        if (n + 1 < u.count) {
          product(0, q0, it + 2, n + 1, &s_free, &s_full);
          product(kDp, dy0, it + 3, n + 1, &dp_free, &dp_full);
          if (ok && elect_one()) {
            mma_commit(&empty[(it + 3) % L::kSlots]);
            if (n + 2 == u.count) mma_commit(&q_empty);
          }
          ++n_s;
        }
        if (!(ok = ok && mbar_wait_warp(&ds_full, n_ds++ & 1, kErrMmaTimeout))) break;
        tc_fence_after();
        const uint64_t k = win_inner(ring + it % L::kSlots * L::kTileBytes);
        const int steps = u.columns(n) >> 4;
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 8; ++s)
            if (s < steps) mma_bf16_ts(kDq, kDs + 8 * s, win_inner_step(k, s), id_dq, n > 0 || s > 0);
          mma_commit(&ds_free);
          mma_commit(&empty[it % L::kSlots]);
          if (n == u.count - 1) mma_commit(&dq_full);
        }
      }
    }
  } else if (warp < 8) {
    // ---- rows
    const int half = warp >> 2, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_at = lanes + 64 * half, dp_at = kDp + lanes + 64 * half, ds_at = kDs + lanes + 32 * half;
    const float scale2 = w.scale * kLog2e;
    uint32_t turn = 0, n_s = 0, dq_turn = 0;
    bool ok = true;
    auto signal = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
      const WinQueryUnit u(w, unit);
      const int q_row = 128 * u.tile + row, at = w.past + q_row;
      const size_t stat = (static_cast<size_t>(u.b) * w.heads + u.head) * (128 * static_cast<size_t>(w.q_tiles)) + q_row;
      __nv_bfloat16* to = p.dq + u.b * p.dq_strides[0] + u.head * p.dq_strides[1] + q_row * p.dq_strides[2];
      if (u.count == 0) {
        // rows behind the sequence
        const uint32_t none[32] = {};
        for (int c = 32 * half; c < w.dim; c += 64)
          if (q_row < w.q_tokens) store_row(to, none, 0.f, c, w.dim);
        if (half == 0) p.delta[stat] = 0.f;
        continue;
      }
      const float lse = p.lse[stat];
      // delta: this thread's half of the channels, and its partner's
      ok = ok && mbar_wait(&q_full, turn & 1, kErrCopyTimeout) && mbar_wait(&y_full, turn & 1, kErrCopyTimeout);
      ++turn;
      float part = 0.f;
      if (ok) {
#pragma unroll
        for (int i = 0; i < kD / 16; ++i) {
          const int c8 = half * (kD / 16) + i;
          const uint32_t off = (c8 >> 3) * kSwBox + sw128_offset(row, c8 & 7);
          float a[8], b[8];
          unpack8(ld_shared_v4(dy_at + off), a);
          unpack8(ld_shared_v4(y_at + off), b);
#pragma unroll
          for (int e = 0; e < 8; ++e) part = fmaf(a[e], b[e], part);
        }
      }
      // the row warps meet here, and only here: they go on, or give up, together
      halves[half][row] = part;
      if (!rows_all(ok)) break;
      const float delta = halves[0][row] + halves[1][row];
      if (half == 0) p.delta[stat] = delta;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&y_empty);
        mbar_arrive(&q_empty);
      }
      const int near = max(at - w.window + 1, u.sinks), upto = at < u.length ? at : -1;   // visible: first ones, near..upto
      for (int n = 0; n < u.count && ok; ++n, ++n_s) {
        const int cols = u.columns(n), key = u.key(w, n);
        const bool sink = n < u.sink_tiles;
        const int from = (sink ? 0 : near - key) - 64 * half;
        const int until = min(min(upto, sink ? u.sinks - 1 : upto) - key, cols - 1) - 64 * half;
        if (!(ok = mbar_wait(&s_full, n_s & 1, kErrMmaTimeout))) break;
        tc_fence_after();
        if (cols <= 64) {
          // a narrow tile: 32 columns at a time, all of them the first group's
          if (!(ok = mbar_wait(&dp_full, n_s & 1, kErrMmaTimeout) && mbar_wait(&ds_free, (n_s & 1) ^ 1, kErrMmaTimeout))) break;
          tc_fence_after();
          if (half == 0) {
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
              uint32_t s[32], d[32], out[16];
              tmem_ld(s_at + c, s);
              tmem_ld(dp_at + c, d);
              tmem_wait();
              tie(s);
              tie(d);
              hide(s, from - c, until - c);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                s[e] = __float_as_uint(exp2_fast(fmaf(__uint_as_float(s[e]), scale2, -lse)));
              score_gradients(s, d, delta, out);
              tmem_st(ds_at + c / 2, out);
            }
            tmem_store_wait();
          }
          signal(&s_free);
          signal(&dp_free);
          signal(&ds_full);
          continue;
        }
        uint32_t s[32], t[32];
        tmem_ld(s_at, s);
        tmem_ld(s_at + 32, t);
        tmem_wait();
        tie(s);
        tie(t);
        signal(&s_free);
        if (!__all_sync(0xffffffffu, from <= 0 && until >= 63)) {
          hide(s, from, until);
          hide(t, from - 32, until - 32);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(exp2_fast(fmaf(__uint_as_float(s[e]), scale2, -lse)));
#pragma unroll
        for (int e = 0; e < 32; ++e) t[e] = __float_as_uint(exp2_fast(fmaf(__uint_as_float(t[e]), scale2, -lse)));
        if (!(ok = mbar_wait(&dp_full, n_s & 1, kErrMmaTimeout))) break;
        tc_fence_after();
        uint32_t out[2][16];
        {
          uint32_t d[32];
          tmem_ld(dp_at, d);
          tmem_wait();
          tie(d);
          score_gradients(s, d, delta, out[0]);
        }
        {
          uint32_t d[32];
          tmem_ld(dp_at + 32, d);
          tmem_wait();
          tie(d);
          signal(&dp_free);
          score_gradients(t, d, delta, out[1]);
        }
        if (!(ok = mbar_wait(&ds_free, (n_s & 1) ^ 1, kErrMmaTimeout))) break;
        tc_fence_after();
        tmem_st(ds_at, out[0]);
        tmem_st(ds_at + 16, out[1]);
        tmem_store_wait();
        signal(&ds_full);
      }
      if (!(ok = ok && mbar_wait(&dq_full, dq_turn++ & 1, kErrMmaTimeout))) continue;
      tc_fence_after();
#pragma unroll 1
      for (int c = 32 * half; c < w.dim; c += 64) {
        uint32_t r[32];
        tmem_ld(kDq + lanes + c, r);
        tmem_wait();
        tie(r);
        if (q_row < w.q_tokens) store_row(to, r, w.scale, c, w.dim);
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 10) {
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

  __device__ __forceinline__ WinKeyUnit(const WinBwdParams& p, int unit) {
    const WinSizes& w = p.w;
    const int each = p.sink_tiles * p.chunks + p.key_tiles - p.sink_tiles;
    const int row = unit / each, at = unit - row * each;
    b = row / w.kv_heads;
    kv_head = row - b * w.kv_heads;
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

template <int kD>
__global__ void __launch_bounds__(kBwdThreads, 1) window_bwd_kv_kernel(const __grid_constant__ WinBwdParams p) {
  using L = WinBwdLayout<kD>;
  constexpr int kSlots = L::kPairSlots;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t full[kSlots], empty[kSlots], kv_full, kv_empty, s_full, dp_full, p_full, ds_full, done;
  __shared__ uint32_t tmem_slot;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t k_at = base, v_at = base + L::kTileBytes, ring = base + 2 * L::kTileBytes;
  const uint32_t stats = ring + L::kRingBytes;   // of each slot: 128 lse, 128 delta
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
    mbar_init(&p_full, 8);
    mbar_init(&ds_full, 8);
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 10) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all of tensor memory: its addresses start at 0.  Columns: S^T and P^T in its place (each group of warps within its
  // half), dP^T and dS^T in its place, dv, dk
  constexpr uint32_t kDp = 128, kDv = 256, kDk = 384;

  if (warp == 8) {
    // ---- loads
    uint32_t it = 0, turn = 0;
    bool ok = true;
    for (int unit = blockIdx.x; unit < p.units && ok; unit += gridDim.x) {
      const WinKeyUnit u(p, unit);
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
    }
  } else if (warp == 9) {
    // ---- instructions
    uint32_t it = 0, turn = 0, n_p = 0;
    bool ok = true;
    constexpr uint32_t id_s = idesc_bf16(128, 128, false, false), id_d = idesc_bf16(128, kD, false, true);
    const uint64_t k0 = win_rows(k_at), v0 = win_rows(v_at);
    // S^T or dP^T: rows of K or V with rows of the item's queries or their gradients
    auto product = [&](uint32_t to, uint64_t a, uint32_t tile, uint64_t* finished) {
      const uint64_t b = win_rows(tile);
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < kD / 16; ++s) mma_bf16(to, win_rows_step(a, s), win_rows_step(b, s), id_s, s > 0);
        mma_commit(finished);
      }
    };
    // dv or dk: what lies at `a` in tensor memory, 64 queries in each half of 64 columns
    auto sum = [&](uint32_t to, uint32_t a, uint32_t tile, bool more) {
      const uint64_t b = win_inner(tile);
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          mma_bf16_ts(to, a + 64 * (s >> 2) + 8 * (s & 3), win_inner_step(b, s), id_d, more || s > 0);
      }
    };
    for (int unit = blockIdx.x; unit < p.units && ok; unit += gridDim.x) {
      const WinKeyUnit u(p, unit);
      if (u.count == 0) continue;
      auto landed = [&](uint32_t item) {
        ok = ok && mbar_wait_warp(&full[item % kSlots], (item / kSlots) & 1, kErrCopyTimeout);
        tc_fence_after();
        return ok;
      };
      if (!(ok = mbar_wait_warp(&kv_full, turn++ & 1, kErrCopyTimeout)) || !landed(it)) break;
      product(0, k0, ring + it % kSlots * 2 * L::kTileBytes, &s_full);
      product(kDp, v0, ring + it % kSlots * 2 * L::kTileBytes + L::kTileBytes, &dp_full);
      for (int n = 0; n < u.count && ok; ++n, ++it) {
        const uint32_t q = ring + it % kSlots * 2 * L::kTileBytes, next = ring + (it + 1) % kSlots * 2 * L::kTileBytes;
        const bool more = n + 1 < u.count;
        if (!(ok = mbar_wait_warp(&p_full, n_p & 1, kErrMmaTimeout))) break;
        tc_fence_after();
        sum(kDv, 0, q + L::kTileBytes, n > 0);
        if (more) {
          if (!landed(it + 1)) break;
          product(0, k0, next, &s_full);
        }
        if (!(ok = mbar_wait_warp(&ds_full, n_p++ & 1, kErrMmaTimeout))) break;
        tc_fence_after();
        sum(kDk, kDp, q, n > 0);
        if (elect_one()) mma_commit(&empty[it % kSlots]);
        if (more) product(kDp, v0, next + L::kTileBytes, &dp_full);
      }
      if (ok && elect_one()) {
        mma_commit(&kv_empty);
        mma_commit(&done);
      }
    }
  } else if (warp < 8) {
    // ---- rows
    const int half = warp >> 2, quad = warp & 3, row = 32 * quad + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_at = lanes + 64 * half, dp_at = kDp + lanes + 64 * half;
    const float scale2 = w.scale * kLog2e;
    uint32_t it = 0, turn = 0;
    bool ok = true;
    auto signal = [&](uint64_t* bar) {
      tmem_store_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int unit = blockIdx.x; unit < p.units && ok; unit += gridDim.x) {
      const WinKeyUnit u(p, unit);
      const int key = 128 * u.tile + row;
      const bool is_key = key < u.length, everywhere = key < w.sinks;
      for (int n = 0; n < u.count && ok; ++n, ++it) {
        const uint32_t slot = it % kSlots;
        int head, tile;
        u.query(w, n, head, tile);
        // the columns (queries) that see this row's key
        const int first = w.past + 128 * tile + 64 * half;
        const int from = key - first;
        const int until = is_key ? (everywhere ? u.length - 1 : min(u.length - 1, key + w.window - 1)) - first : -1;
        const bool masked = !__all_sync(0xffffffffu, from <= 0 && until >= 63);
        if (!(ok = mbar_wait(&full[slot], (it / kSlots) & 1, kErrCopyTimeout) && mbar_wait(&s_full, it & 1, kErrMmaTimeout)))
          break;
        tc_fence_after();
        const uint32_t lse = stats + 1024 * slot + 256 * half, delta = lse + 512;
        uint32_t s[2][32];
        tmem_ld(s_at, s[0]);
        tmem_ld(s_at + 32, s[1]);
        tmem_wait();
        tie(s[0]);
        tie(s[1]);
        if (masked) {
          hide(s[0], from, until);
          hide(s[1], from - 32, until - 32);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t out[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const uint4 l = ld_shared_v4(lse + 128 * h + 4 * e);
            const uint32_t of[4] = {l.x, l.y, l.z, l.w};
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f[i] = exp2_fast(fmaf(__uint_as_float(s[h][e + i]), scale2, -__uint_as_float(of[i])));
              s[h][e + i] = __float_as_uint(f[i]);
            }
            out[e / 2] = pack_bf16(f[0], f[1]);
            out[e / 2 + 1] = pack_bf16(f[2], f[3]);
          }
          tmem_st(s_at + 16 * h, out);
        }
        signal(&p_full);
        if (!(ok = mbar_wait(&dp_full, it & 1, kErrMmaTimeout))) break;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t d[32], out[16];
          tmem_ld(dp_at + 32 * h, d);
          tmem_wait();
          tie(d);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const uint4 l = ld_shared_v4(delta + 128 * h + 4 * e);
            const uint32_t of[4] = {l.x, l.y, l.z, l.w};
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float weight = __uint_as_float(s[h][e + i]);
              f[i] = weight != 0.f ? weight * (__uint_as_float(d[e + i]) - __uint_as_float(of[i])) : 0.f;
            }
            out[e / 2] = pack_bf16(f[0], f[1]);
            out[e / 2 + 1] = pack_bf16(f[2], f[3]);
          }
          tmem_st(dp_at + 16 * h, out);
        }
        signal(&ds_full);
      }
      if (!ok || (u.count > 0 && !(ok = mbar_wait(&done, turn++ & 1, kErrMmaTimeout)))) break;
      tc_fence_after();
      // the first group's dv, the second's dk
      const uint32_t acc = (half ? kDk : kDv) + lanes;
      const long long* strides = half ? p.dk_strides : p.dv_strides;
      __nv_bfloat16* to = (half ? p.dk : p.dv) + u.b * strides[0] + u.kv_head * strides[1] + key * strides[2];
      const float scale = u.count == 0 ? 0.f : half ? w.scale : 1.f;
      const size_t item = ((static_cast<size_t>(u.b) * w.kv_heads + u.kv_head) * p.sink_tiles + u.tile) * p.chunks + u.chunk;
      float* sums = p.partial + (item * 2 + half) * (kD * 128) + row;
#pragma unroll 1
      for (int c = 0; c < w.dim; c += 32) {
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
  if (warp == 10) {
    tc_fence_after();
    tmem_dealloc(tmem_slot, 512);
  }
}

// The sums of first tokens' key tiles, chunk by chunk; a CTA for each 32 channels of a tile of dk or dv.
template <int kD>
__global__ void __launch_bounds__(128) window_bwd_join_kernel(const __grid_constant__ WinBwdParams p) {
  const WinSizes& w = p.w;
  const int part = blockIdx.x % (kD / 32), what = blockIdx.x / (kD / 32) & 1, tile = blockIdx.y % p.sink_tiles;
  const int row = blockIdx.y / p.sink_tiles, b = row / w.kv_heads, kv_head = row - b * w.kv_heads;
  const int key = 128 * tile + threadIdx.x, c = 32 * part;
  if (key >= w.kv_tokens || c >= w.dim) return;
  const float* from = p.partial + (static_cast<size_t>(blockIdx.y) * p.chunks * 2 + what) * (kD * 128) + c * 128 + threadIdx.x;
  float sum[32] = {};
  for (int i = 0; i < p.chunks; ++i) {
#pragma unroll
    for (int e = 0; e < 32; ++e) sum[e] += __ldcg(from + static_cast<size_t>(i) * (2 * kD * 128) + e * 128);
  }
  uint32_t r[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(sum[e]);
  const long long* strides = what ? p.dk_strides : p.dv_strides;
  store_row((what ? p.dk : p.dv) + b * strides[0] + kv_head * strides[1] + key * strides[2], r, 1.f, c, w.dim);
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
  p.units = w.batch * w.heads * w.q_tiles;
  window_bwd_q_kernel<kD><<<p.units < 148 ? p.units : 148, kBwdThreads, L::kSmemQ, s>>>(p);
  if (const int rc = check_launch("window_bwd_q")) return rc;
  p.units = w.batch * w.kv_heads * (p.sink_tiles * p.chunks + p.key_tiles - p.sink_tiles);
  window_bwd_kv_kernel<kD><<<p.units < 148 ? p.units : 148, kBwdThreads, L::kSmemKV, s>>>(p);
  if (const int rc = check_launch("window_bwd_kv")) return rc;
  if (p.sink_tiles == 0 || p.chunks < 2) return TS_OK;
  window_bwd_join_kernel<kD><<<dim3(kD / 32 * 2, w.batch * w.kv_heads * p.sink_tiles), 128, 0, s>>>(p);
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
  if (static_cast<long long>(w.batch) * w.kv_heads * p.sink_tiles > 65535)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "window_bwd: too many tiles of first tokens");
  if (static_cast<long long>(w.batch) * w.kv_heads * (static_cast<long long>(p.sink_tiles) * p.chunks + p.key_tiles) > 0x3fffffffll)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "window_bwd: too many key tiles");
  p.sink_rows = w.sinks >= 128 ? 128 : round_up(w.sinks > 0 ? w.sinks : 1, 16);
  p.lse = a->lse;
  p.delta = static_cast<float*>(g->workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(g->workspace) + stats);
  p.dq = static_cast<__nv_bfloat16*>(g->dq);
  p.dk = static_cast<__nv_bfloat16*>(g->dk);
  p.dv = static_cast<__nv_bfloat16*>(g->dv);
  for (int i = 0; i < 3; ++i) {
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
