// The choice of a token from each row of logits, by given uniform numbers.
//
// Tokens in the order of falling logits, the lower index first among equals; of
// these the first top_k; of those the shortest prefix with top_p of their mass;
// of those the ones with at least min_p times the largest probability.  The token
// is the first, by index, at which the running mass of what is left exceeds
// uniform times its total.
//
// A CTA, or the CTAs of a cluster, keep a row in shared memory and pass over it a
// few times (rows too long for that come from L2 again).  Masses are integers,
// exp((x - max) / temperature) in units of 2^-40: their sums do not depend on an
// order, and come out the same in every CTA, which therefore take the same turns
// without asking each other.  Nothing is sorted: a histogram over 32nds of the
// distance from the maximum, in powers of two (monotone in the logit, so its bins
// are stretches of the order), says in which bin a cut falls; the bin's tokens,
// usually under a hundred, are gathered and ranked against each other.  A bin of
// more is cut into parts by its logits' bits until it is not, or has one value
// left, whose tokens then count in the order of their index.
//
// What bounds it is the number of instructions: 104 for each logit with top-p (512
// rows x 50257: 140 us at 58 % of the issue slots), 120 with every filter, whose
// cluster of CTAs also waits at its barriers (64 rows x 128257: 62 us at 50 %).  The
// exponential is in 64 bits, which run at half the rate of 32 but need no
// compensation: the sum of 1.5 2^52 and the product of a logit's difference from
// the largest has the rounded distance, which is the bin too, in its low word.
// Only the pass that fills the histogram takes it of every logit: a cut's bin is
// found again by its first and last logit, and kept tokens are brought side by side
// in shared memory before their masses are summed (512 rows x 50257, top-p: 168 ->
// 140 us; 64 rows x 128257 bf16, every filter: 69 -> 62 us).  A mass is right to
// half a unit and 1e-13 of itself.
#include <cmath>
#include <type_traits>

#include "capi_internal.h"
#include "cluster.cuh"

namespace ts {

namespace {

using u64 = unsigned long long;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSteps = 32;                     // bins of a power of two
constexpr int kLastStep = 41 * kSteps;         // tokens further than 2^-41 have no mass
constexpr int kBins = 1536, kPerThread = kBins / kSampleThreads;
constexpr int kRanked = 512;                   // tokens that are ranked against each other
constexpr int kFew = 128;                      // kept tokens of a piece that are taken together
constexpr int kPieces = 2048;                  // of a CTA's tokens: stretches that one warp goes over
constexpr int kCacheMost = 66560;              // bytes of a CTA's tokens: two CTAs to an SM
constexpr u64 kOne = 1ull << 40;
static_assert(kLastStep < kBins && kBins % kSampleThreads == 0, "bins");

struct SampleParams {
  int rows, vocab, slice;                      // slice: tokens of a CTA
  bool cache;                                  // it fits into shared memory
  const void* logits;
  long long row_stride;
  const float* uniform;
  const float* temperature; double temperature_value;
  const int* top_k; int top_k_value;           // 0: off
  const float* top_p; double top_p_value;      // 1: off
  const float* min_p; double min_p_value;      // 0: off
  long long* tokens;
  float* logprobs;                             // or null
};

// Larger for larger logits, and back.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);   // minus zero is zero
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The histogram's masses are 64-bit sums in two words: most tokens have less than 2^32 and bring no carry, so one atomic
// each.  (Atomics on random bins bound the pass that fills it: 3.5 cycles of the SM for a warp's.)
struct SampleShared {
  union {
    struct {
      uint32_t count[kBins], low[kBins], high[kBins];
    };
    u64 piece[kPieces];                        // once no CTA reads the histogram any more
  };
  double power[kSteps];                        // 2^(k/32) in units of 2^-40
  uint32_t key[kRanked], index[kRanked];       // tokens of a bin: this CTA's
  union {
    struct {
      u64 all_place[kRanked], all_mass[kRanked];   // and the cluster's: key and index, falling in the order
    };
    float few[kSampleWarps][kFew];             // after the cuts: kept logits of the piece that a warp is at
  };
  u64 warp_sum[kSampleWarps], warp_sum_b[kSampleWarps];
  u64 total, total_b, smallest, largest;       // of this CTA, for the others
  float top;
  uint32_t listed, gathered, first;
  // for this CTA's threads
  double scale;                                // of the distance (see Sampler)
  float lowest, floor_at;
  float edge[2];                               // a bin's logits: from the first on, below the second
  u64 before, before_b, rest;
  uint32_t bin, cut_key, cut_index, found;
  int piece_at;
};

__device__ __forceinline__ u64 warp_max64(u64 v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Of every thread of the CTA, in every thread; `scratch` may be used again after the next barrier.
template <class F>
__device__ __forceinline__ u64 block_join(u64 v, u64* scratch, F join) {
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = scratch[0];
#pragma unroll
  for (int i = 1; i < kSampleWarps; ++i) r = join(r, scratch[i]);
  return r;
}
// Sum over the threads before this one.
__device__ __forceinline__ u64 block_before(u64 v, u64* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 upto = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  u64 r = upto - v;
#pragma unroll
  for (int i = 0; i < kSampleWarps - 1; ++i)
    if (i < warp) r += scratch[i];
  return r;
}

// kPer: tokens of a piece that a lane has.
template <bool kBf16, int kPer>
struct Sampler {
  static constexpr int kPiece = 32 * kPer;
  using Raw = std::conditional_t<kBf16, __nv_bfloat16, float>;

  const SampleParams& p;
  SampleShared& m;
  Raw* cache;
  const Raw* from;                             // this CTA's tokens
  uint32_t rank, ranks;
  int row, start, size, pieces;
  bool infinite;                               // the largest logit is infinite: its tokens are 0, and alone
  bool scaled;                                 // logits are taken times 2^-20: f32 has room below the ones with mass
  float lowest;                                // what lies below has no mass, and is this
  double scale, peak;                          // distance in 32nds of a power of two: scale (x - peak), 0 at the top

  __device__ __forceinline__ Sampler(const SampleParams& p_, SampleShared& m_, void* cache_)
      : p(p_), m(m_), cache(static_cast<Raw*>(cache_)) {
    rank = cluster_rank_of();
    ranks = cluster_size_of();
    row = blockIdx.x / ranks;
    start = min(p.vocab, static_cast<int>(rank) * p.slice);
    size = min(p.vocab, start + p.slice) - start;
    pieces = (size + kPiece - 1) / kPiece;
    from = static_cast<const Raw*>(p.logits) + row * p.row_stride + start;
  }
  __device__ __forceinline__ void barrier() const {
    if (ranks > 1) cluster_barrier();
    else __syncthreads();
  }
  template <class T>
  __device__ __forceinline__ T of(const T* at, uint32_t r) const {
    return ranks > 1 ? cluster_read(at, r) : *at;
  }

  static __device__ __forceinline__ float value(Raw r) {
    if constexpr (kBf16) return bf2f(r);
    else return r;
  }
  __device__ __forceinline__ float meant(float x) const {
    return infinite ? (x == INFINITY ? 0.f : -INFINITY) : scaled ? x * 0x1p-20f : x;
  }
  // A piece's logits as they are; behind the slice minus infinity.
  __device__ __forceinline__ void load(const Raw* at, int piece, float (&x)[kPer]) const {
    const int i0 = piece * kPiece + static_cast<int>(threadIdx.x & 31);
    if ((piece + 1) * kPiece <= size) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) x[j] = value(at[i0 + 32 * j]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) x[j] = i0 + 32 * j < size ? value(at[i0 + 32 * j]) : -INFINITY;
    }
  }
  // f(x, first place in the slice, piece) for this thread's tokens of each piece, which are 32 places apart.  A NaN, as
  // everything that has no mass, is `lowest` (not where f only asks what is above some logit that is not below `lowest`).  (The tokens of a piece are taken side by side: one after the other, with
  // what each of them may lead to between, the waits for their 64-bit operations add up.)
  template <bool kRaise = true, class F>
  __device__ __forceinline__ void each(F f) const {
    for (int piece = threadIdx.x >> 5; piece < pieces; piece += kSampleWarps) {
      float x[kPer];
      load(p.cache ? cache : from, piece, x);
      if (infinite || scaled) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[j] = meant(x[j]);
      }
      if constexpr (kRaise) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[j] = fmaxf(x[j], lowest);
      }
      f(x, piece * kPiece + static_cast<int>(threadIdx.x & 31), piece);
    }
  }
  using Tokens = float (&)[kPer];
  // Bits of the tokens for which f holds.
  template <class F>
  static __device__ __forceinline__ uint32_t which(Tokens x, F f) {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) bits |= f(x[j], 32 * j) ? 1u << j : 0u;
    return bits;
  }
  // f(x, place) for the tokens of `bits`: rare ones.
  template <class F>
  static __device__ __forceinline__ void few(Tokens x, int i0, uint32_t bits, F f) {
    if (!__any_sync(0xffffffffu, bits)) return;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (bits >> j & 1) f(x[j], i0 + 32 * j);
  }

  // 32 log2 of a token's mass, rounded, times -1: its bin.
  __device__ __forceinline__ uint32_t bin(float x) const {
    return static_cast<uint32_t>(-__double2loint(fma(x - peak, scale, 6755399441055744.)));
  }
  __device__ __forceinline__ u64 mass(float x, uint32_t& bin) const {
    const double d = x - peak, near = fma(d, scale, 6755399441055744.);
    const int i = __double2loint(near);
    bin = static_cast<uint32_t>(-i);
    // 2^(i/32) 2^(r/32), |r| <= 1/2: the second by a polynomial fitted there, within 1e-13
    const double r = fma(d, scale, 6755399441055744. - near);
    double e = fma(r, 9.172621781784e-9, 1.693863388074e-6);
    e = fma(e, r, 2.345961981964e-4);
    e = fma(e, r, 2.166084939172e-2);
    e = fma(e, r, 1.);
    e *= m.power[i & (kSteps - 1)];
    // times 2^(i >> 5), and the integer out of a sum with 2^52
    e = __hiloint2double(__double2hiint(e) + ((i >> 5) << 20), __double2loint(e)) + 4503599627370496.;
    const u64 w = static_cast<u64>(__double_as_longlong(e)) & 0xfffffffffffffull;   // the bits of 2^52 fall away
    return w;   // 0 below -kLastStep: it was less than 1/2
  }
  __device__ __forceinline__ u64 mass(float x) const {
    uint32_t b;
    return mass(x, b);
  }

  // The smallest logit in the bins up to `most` (0: the largest logit is in it), by a whole warp: one that lies behind the
  // largest logit for most < 0.
  __device__ __forceinline__ float edge(int most, float top) const {
    if (most < 0) return INFINITY;
    uint32_t out = order_key(lowest) - 1, in = order_key(top);   // 32 places between the two at a time
    while (in - out > 1) {
      const uint32_t step = (in - out + 31) / 32, at = out + (threadIdx.x & 31) * step + step;
      const bool past = at >= in || at < out;
      const uint32_t yes = __ballot_sync(0xffffffffu, past || static_cast<int>(bin(key_value(past ? in : at))) <= most);
      const int first = __ffs(yes) - 1;   // the last place is `in` or past it
      const uint32_t here = out + first * step;
      if (in - here > step) in = here + step;
      out = here;
    }
    return key_value(in);
  }

  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += kSampleThreads) m.count[i] = m.low[i] = m.high[i] = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add(uint32_t bin, u64 w) {
    const uint32_t part = static_cast<uint32_t>(w), was = atomicAdd(&m.low[bin], part);
    const uint32_t up = static_cast<uint32_t>(w >> 32) + (was + part < was ? 1u : 0u);
    if (up) atomicAdd(&m.high[bin], up);
  }
  // The same for a piece's tokens.
  __device__ __forceinline__ void add(const uint32_t (&bin)[kPer], const u64 (&w)[kPer]) {
    uint32_t up[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint32_t part = static_cast<uint32_t>(w[j]), was = w[j] ? atomicAdd(&m.low[bin[j]], part) : 0;
      up[j] = static_cast<uint32_t>(w[j] >> 32) + (was + part < was ? 1u : 0u);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (up[j]) atomicAdd(&m.high[bin[j]], up[j]);
  }

  // The cluster's histogram: this thread's bins and what comes before them.  After a barrier().
  struct Bins {
    uint32_t count[kPerThread];
    u64 mass[kPerThread], count_before, mass_before;
  };
  __device__ __forceinline__ Bins joined() {
    if (ranks > 1) {
      // each CTA joins its share of the bins, in place: nobody else reads these from it before the barrier
      const int share = kBins / ranks, first = rank * share;
      for (int i = first + threadIdx.x; i < first + share; i += kSampleThreads) {
        uint32_t count = 0;
        u64 mass = 0;
        for (uint32_t r = 0; r < ranks; ++r) {
          count += cluster_read(&m.count[i], r);
          mass += cluster_read(&m.low[i], r) | static_cast<u64>(cluster_read(&m.high[i], r)) << 32;
        }
        m.count[i] = count;
        m.low[i] = static_cast<uint32_t>(mass);
        m.high[i] = static_cast<uint32_t>(mass >> 32);
      }
      cluster_barrier();
    }
    Bins b;
    u64 counts = 0, masses = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int at = kPerThread * threadIdx.x + i;
      if (ranks > 1) {
        const uint32_t owner = at / (kBins / ranks);
        b.count[i] = cluster_read(&m.count[at], owner);
        b.mass[i] = cluster_read(&m.low[at], owner) | static_cast<u64>(cluster_read(&m.high[at], owner)) << 32;
      } else {
        b.count[i] = m.count[at];
        b.mass[i] = m.low[at] | static_cast<u64>(m.high[at]) << 32;
      }
      counts += b.count[i];
      masses += b.mass[i];
    }
    b.count_before = block_before(counts, m.warp_sum);
    b.mass_before = block_before(masses, m.warp_sum_b);
    return b;
  }
  // The bin in which the running count (mass) reaches `target`: into m.bin (kBins: in none), with what comes before it.
  __device__ __forceinline__ void locate(const Bins& b, bool by_mass, u64 target) {
    if (threadIdx.x == 0) m.bin = kBins;
    __syncthreads();
    u64 counts = b.count_before, masses = b.mass_before;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const u64 at = by_mass ? masses : counts, here = by_mass ? b.mass[i] : b.count[i];
      if (at < target && target <= at + here) {
        m.bin = kPerThread * threadIdx.x + i;
        m.before = counts;
        m.before_b = masses;
      }
      counts += b.count[i];
      masses += b.mass[i];
    }
    __syncthreads();
  }

  // Of a value for each piece in m.piece, summed to `mine` in this CTA and to `before` in those before it: the token, in
  // index order, at which the running sum exceeds `target`, into m.found of the CTA that holds it (returned: whether
  // this one does).  f is the value of a token.
  template <class F>
  __device__ __forceinline__ bool choose(F f, u64 target, u64 before, u64 mine) {
    if (!(before <= target && target < before + mine)) return false;
    target -= before;
    constexpr int kEach = kPieces / kSampleThreads;
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int piece = kEach * threadIdx.x + i;
      sum += piece < pieces ? m.piece[piece] : 0;
    }
    u64 at = block_before(sum, m.warp_sum_b);
    if (at <= target && target < at + sum) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int piece = kEach * threadIdx.x + i;
        const u64 here = piece < pieces ? m.piece[piece] : 0;
        if (at <= target && target < at + here) {
          m.piece_at = piece;
          m.rest = target - at;
        }
        at += here;
      }
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      // its 32 tokens at a time
      u64 ahead = 0;
      const u64 rest = m.rest;
      const Raw* tokens = p.cache ? cache : from;
#pragma unroll 1
      for (int j = 0; j < kPer; ++j) {
        const int i = m.piece_at * kPiece + 32 * j + static_cast<int>(threadIdx.x);
        float x = i < size ? value(tokens[i]) : -INFINITY;
        x = meant(x);
        const u64 w = f(fmaxf(x, lowest), i);
        u64 upto = w;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const u64 v = __shfl_up_sync(0xffffffffu, upto, d);
          if (threadIdx.x >= d) upto += v;
        }
        upto += ahead;
        if (upto - w <= rest && rest < upto) m.found = static_cast<uint32_t>(start + i);
        ahead = __shfl_sync(0xffffffffu, upto, 31);
        if (ahead > rest) break;
      }
    }
    __syncthreads();
    return true;
  }

  // The cluster's tokens of a bin with keys from `least` to `most`, in every CTA's m.all_place and m.all_mass, their count
  // in m.gathered; false where there are more than kRanked.
  template <class F>
  __device__ __forceinline__ bool gather(F in_bin, uint32_t least, uint32_t most) {
    if (threadIdx.x == 0) m.listed = 0;
    barrier();
    const bool whole = least == 0 && most == 0xffffffffu;
    each<false>([&](Tokens x, int i0, int) {
      few(x, i0, which(x, [&](float v, int) { return in_bin(v); }), [&](float v, int i) {
        const uint32_t k = order_key(v);
        if (!whole && (k < least || k > most)) return;
        const uint32_t at = atomicAdd(&m.listed, 1u);
        if (at < kRanked) {
          m.key[at] = k;
          m.index[at] = static_cast<uint32_t>(start + i);
        }
      });
    });
    barrier();
    uint32_t count = 0;
    for (uint32_t r = 0; r < ranks; ++r) {
      const uint32_t theirs = of(&m.listed, r);
      for (uint32_t i = threadIdx.x; i < theirs && count + i < kRanked; i += kSampleThreads) {
        const uint32_t k = of(&m.key[i], r);
        m.all_place[count + i] = static_cast<u64>(k) << 32 | (0xffffffffu - of(&m.index[i], r));
        m.all_mass[count + i] = mass(key_value(k));
      }
      count += theirs;
    }
    if (threadIdx.x == 0) m.gathered = count;
    barrier();   // the others have read this CTA's list
    return count <= kRanked;
  }

  // The last token that is kept when the order is cut where the count (mass) reaches `target` within the bin in m.bin:
  // m.cut_key and m.cut_index; returned: the mass of the bin's tokens up to it.  The target counts from the bin's start.
  __device__ __forceinline__ u64 cut(bool by_mass, u64 target, float top) {
    // the bin's logits; where a lane has two tokens the search for them would take longer than asking each for its bin
    const uint32_t cut_bin = m.bin;
    if (kPer > 2 && threadIdx.x < 64) {
      const float at = edge(static_cast<int>(m.bin) - (threadIdx.x < 32 ? 0 : 1), top);
      if ((threadIdx.x & 31) == 0) m.edge[threadIdx.x >> 5] = at;
    }
    __syncthreads();
    const float from_edge = m.edge[0], to_edge = m.edge[1];
    auto in_bin = [&](float v) { return kPer > 2 ? v >= from_edge && v < to_edge : bin(fmaxf(v, lowest)) == cut_bin; };
    uint32_t least = 0, most = 0xffffffffu;   // of the keys that are still in question
    u64 before = 0;
    auto in_question = [&](float v) {
      const uint32_t k = order_key(v);
      return in_bin(v) && k >= least && k <= most;
    };
#pragma unroll 1
    while (!gather(in_bin, least, most)) {
      // the largest and smallest key
      u64 low = ~0ull, high = 0;
      each([&](Tokens x, int i0, int) {
        few(x, i0, which(x, [&](float v, int) { return in_question(v); }), [&](float v, int) {
          low = min(low, static_cast<u64>(order_key(v)));
          high = max(high, static_cast<u64>(order_key(v)));
        });
      });
      low = block_join(~warp_max64(~low), m.warp_sum, [](u64 a, u64 b) { return min(a, b); });
      high = block_join(warp_max64(high), m.warp_sum_b, [](u64 a, u64 b) { return max(a, b); });
      if (threadIdx.x == 0) {
        m.smallest = low;
        m.largest = high;
      }
      barrier();
      for (uint32_t r = 0; r < ranks; ++r) {
        low = min(low, of(&m.smallest, r));
        high = max(high, of(&m.largest, r));
      }
      least = static_cast<uint32_t>(low);
      most = static_cast<uint32_t>(high);
      if (least == most) {
        // one value: its tokens in the order of their index
        const u64 w = mass(key_value(least));
        const u64 wanted = by_mass ? (target + w - 1) / w : target;
        auto one = [&](float v, int) -> u64 { return in_question(v) ? 1 : 0; };
        u64 all = 0;
        each([&](Tokens x, int, int piece) {
          const u64 s = warp_sum64(__popc(which(x, [&](float v, int) { return in_question(v); })));
          if ((threadIdx.x & 31) == 0) m.piece[piece] = s;
          all += s;
        });
        all = block_join(all, m.warp_sum, [](u64 a, u64 b) { return a + b; });
        if (threadIdx.x == 0) m.total = all;
        barrier();
        u64 sum = 0, ahead = 0;
        uint32_t owner = 0;
        for (uint32_t r = 0; r < ranks; ++r) {
          const u64 c = of(&m.total, r);
          if (sum <= wanted - 1 && wanted - 1 < sum + c) owner = r;
          if (r == rank) ahead = sum;
          sum += c;
        }
        choose(one, wanted - 1, ahead, all);
        barrier();
        const uint32_t token = of(&m.found, owner);
        __syncthreads();
        if (threadIdx.x == 0) {
          m.cut_key = least;
          m.cut_index = token;
        }
        barrier();
        return before + wanted * w;
      }
      int shift = 0;
      while (((most - least) >> shift) >= kBins) ++shift;
      barrier();   // the others have read this CTA's histogram
      clear();
      each([&](Tokens x, int i0, int) {
        few(x, i0, which(x, [&](float v, int) { return in_question(v); }), [&](float v, int) {
          const uint32_t part = (most - order_key(v)) >> shift;
          atomicAdd(&m.count[part], 1u);
          add(part, mass(v));
        });
      });
      barrier();
      const Bins b = joined();
      locate(b, by_mass, target);
      const uint32_t part = m.bin, high_was = most;
      target -= by_mass ? m.before_b : m.before;
      before += m.before_b;
      most -= part << shift;
      const uint32_t width = (1u << shift) - 1;
      least = most - least > width ? most - width : least;
      if (high_was < most) least = most;   // not reached: a bin that was located lies inside
    }
    const uint32_t count = m.gathered;
    // eight threads for a token, each against an eighth of the others
    const int part = threadIdx.x & 7;
    for (uint32_t i0 = 0; i0 < count; i0 += kSampleThreads / 8) {
      const uint32_t i = i0 + (threadIdx.x >> 3);
      const u64 place = i < count ? m.all_place[i] : 0;
      uint32_t counts = 0;
      u64 masses = 0;
#pragma unroll 2
      for (uint32_t j = part; j < count; j += 8) {
        const bool ahead = m.all_place[j] > place;
        counts += ahead ? 1 : 0;
        masses += ahead ? m.all_mass[j] : 0;
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) {
        counts += __shfl_xor_sync(0xffffffffu, counts, d);
        masses += __shfl_xor_sync(0xffffffffu, masses, d);
      }
      if (i < count && part == 0) {
        const u64 at = by_mass ? masses : counts, mine = by_mass ? m.all_mass[i] : 1;
        if (at < target && target <= at + mine) {
          m.cut_key = static_cast<uint32_t>(place >> 32);
          m.cut_index = 0xffffffffu - static_cast<uint32_t>(place);
          m.rest = masses + m.all_mass[i];
        }
      }
    }
    __syncthreads();
    return before + m.rest;
  }

  __device__ __forceinline__ void run() {
    const double given = p.temperature ? static_cast<double>(__ldg(p.temperature + row)) : p.temperature_value;
    const bool greedy = !(given > 0.);
    double temperature = greedy ? 1. : fmin(given, 3.4028234663852886e38);
    if (threadIdx.x < kSteps) m.power[threadIdx.x] = exp2(static_cast<int>(threadIdx.x) * (1. / kSteps) + 40.);
    // the largest logit; the slice into shared memory, where each thread reads again what it has put there
    float top = -INFINITY;
    for (int piece = threadIdx.x >> 5; piece < pieces; piece += kSampleWarps) {
      float x[kPer];
      load(from, piece, x);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (p.cache) cache[piece * kPiece + 32 * j + static_cast<int>(threadIdx.x & 31)] = Raw(x[j]);
        top = fmaxf(top, x[j]);
      }
    }
    top = key_value(static_cast<uint32_t>(block_join(warp_max64(order_key(top)), m.warp_sum, [](u64 a, u64 b) { return max(a, b); })));
    if (ranks > 1) {
      if (threadIdx.x == 0) m.top = top;
      cluster_barrier();
      for (uint32_t r = 0; r < ranks; ++r) top = fmaxf(top, cluster_read(&m.top, r));
    }
    const bool nothing = top == -INFINITY;
    infinite = top == INFINITY;
    if (infinite) {
      top = 0.f;
      temperature = 1.;
    }
    // What has no mass is a logit below the rest, which these leave no room for.  (Where two logits then become one, they
    // are less than a 2^100th of the temperature or of the largest apart.)
    scaled = top < -1e38f || temperature > 1e36;
    if (scaled) {
      top *= 0x1p-20f;
      temperature *= 0x1p-20;
    }
    int top_k = greedy ? 0 : p.top_k ? __ldg(p.top_k + row) : p.top_k_value;
    const double top_p = greedy ? 1. : p.top_p ? static_cast<double>(__ldg(p.top_p + row)) : p.top_p_value;
    if (threadIdx.x == 0) {
      const double min_p = greedy ? 0. : p.min_p ? static_cast<double>(__ldg(p.min_p + row)) : p.min_p_value;
      const float below = nextafterf(top, -INFINITY);
      // the next smaller logit is 4096 steps away at most: further is without mass too, and the low word holds it
      const double s = min(kSteps * 1.4426950408889634 / temperature, 4096. / (static_cast<double>(top) - below));
      m.scale = s;
      m.lowest = min(__double2float_rd(top - (kLastStep + kSteps) / s), below);
      m.floor_at = min_p > 0. ? __double2float_ru(top + temperature * log(min(min_p, 1.))) : -INFINITY;
    }
    __syncthreads();
    scale = m.scale;
    peak = top;
    lowest = m.lowest;
    const float floor_at = m.floor_at;

    if (top_k <= 0 || top_k >= p.vocab) top_k = 0;
    const bool by_mass = top_p < 1.;           // a NaN is no limit
    const bool want_total = p.logprobs || (by_mass && top_k == 0);
    u64 total = 0;                             // the mass of all tokens, where it is wanted
    float cut_at = -INFINITY;                  // kept: logits above, and those equal up to the index
    uint32_t cut_index = 0xffffffffu;
    if (!nothing && (top_k > 0 || by_mass || want_total)) {
      u64 sum = 0;
      if (by_mass || want_total) {
        if (top_k > 0 || by_mass) clear();
        each([&](Tokens x, int, int) {
          uint32_t b[kPer];
          u64 w[kPer];
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            w[j] = mass(x[j], b[j]);
            sum += w[j];
          }
          if (top_k > 0) {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
              if (b[j] <= kLastStep) atomicAdd(&m.count[b[j]], 1u);
          }
          if (by_mass) add(b, w);
        });
      } else {
        clear();
        each([&](Tokens x, int, int) {
          uint32_t b[kPer];
#pragma unroll
          for (int j = 0; j < kPer; ++j) b[j] = bin(x[j]);
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (b[j] <= kLastStep) atomicAdd(&m.count[b[j]], 1u);
        });
      }
      if (want_total) {
        sum = block_join(warp_sum64(sum), m.warp_sum, [](u64 a, u64 b) { return a + b; });
        if (threadIdx.x == 0) m.total_b = sum;
      }
      barrier();
      if (want_total)
        for (uint32_t r = 0; r < ranks; ++r) total += of(&m.total_b, r);
      if (top_k > 0 || by_mass) {
        const Bins b = joined();
        u64 kept = total;
        if (top_k > 0) {
          locate(b, false, static_cast<u64>(top_k));
          if (m.bin < kBins) {
            const u64 ahead = m.before_b;
            kept = ahead + cut(false, top_k - m.before, top);
            cut_at = key_value(m.cut_key);
            cut_index = m.cut_index;
          } else if (by_mass) {
            // the cut lies among tokens without mass
            __syncthreads();
            u64 s = 0;
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) s += b.mass[i];
            kept = block_join(warp_sum64(s), m.warp_sum, [](u64 x, u64 y) { return x + y; });
          }
        }
        if (by_mass) {
          const double wanted = ceil(top_p * static_cast<double>(kept));
          const u64 target = wanted >= 1. ? min(static_cast<u64>(wanted), kept) : 1;
          __syncthreads();
          locate(b, true, target);
          if (m.bin < kBins) {
            cut(true, target - m.before_b, top);
            cut_at = key_value(m.cut_key);
            cut_index = m.cut_index;
          }
        }
        barrier();   // the others have read this CTA's histogram
      }
    }
    if (nothing) {
      if (rank == 0 && threadIdx.x == 0) {
        p.tokens[row] = -1;
        if (p.logprobs) p.logprobs[row] = -INFINITY;
      }
    } else if (greedy) {
      first_of(top, total);
    } else {
      // kept: what is at least `least` up to the place `last` of the slice, what is above it behind that
      const float least = fmaxf(fmaxf(cut_at, floor_at), lowest), above = nextafterf(least, INFINITY);
      const int last = cut_at < least || cut_index - start > 0x7fffffffu
                           ? (cut_at < least || cut_index >= static_cast<uint32_t>(start) ? 0x7fffffff : -1)
                           : static_cast<int>(cut_index - start);
      auto kept = [&](float v, int i) { return v >= (i <= last ? least : above); };
      u64 mine = 0;
      each<false>([&](Tokens x, int i0, int piece) {
        uint32_t bits;
        if (last < (piece + 1) * kPiece && last >= piece * kPiece) {
          bits = which(x, [&](float v, int i) { return kept(v, i0 + i); });
        } else {
          const float from_here = last < piece * kPiece ? above : least;
          bits = which(x, [&](float v, int) { return v >= from_here; });
        }
        u64 sum = 0;
        if (__any_sync(0xffffffffu, bits)) {
          // the kept ones side by side, where they are few: their masses are what costs
          uint32_t upto = __popc(bits);
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const uint32_t before = __shfl_up_sync(0xffffffffu, upto, d);
            if ((threadIdx.x & 31) >= d) upto += before;
          }
          const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
          if (all <= kFew) {
            float* to = m.few[threadIdx.x >> 5];
            uint32_t at = upto - __popc(bits);
#pragma unroll
            for (int j = 0; j < kPer; ++j)
              if (bits >> j & 1) to[at++] = x[j];
            __syncwarp();
            for (uint32_t i = threadIdx.x & 31; i < all; i += 32) sum += mass(to[i]);
            __syncwarp();
          } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              const u64 w = mass(fmaxf(x[j], lowest));
              sum += bits >> j & 1 ? w : 0;
            }
          }
          // below 2^44 in a lane: its parts of 24 bits
          sum = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(sum) & 0xffffffu) +
                (static_cast<u64>(__reduce_add_sync(0xffffffffu, static_cast<uint32_t>(sum >> 24))) << 24);
          mine += sum;
        }
        if ((threadIdx.x & 31) == 0) m.piece[piece] = sum;
      });
      mine = block_join(mine, m.warp_sum, [](u64 a, u64 b) { return a + b; });
      if (threadIdx.x == 0) m.total = mine;
      barrier();
      u64 chosen_total = 0, ahead = 0;
      for (uint32_t r = 0; r < ranks; ++r) {
        if (r == rank) ahead = chosen_total;
        chosen_total += of(&m.total, r);
      }
      const double u = static_cast<double>(__ldg(p.uniform + row));
      const double at = u > 0. ? u * static_cast<double>(chosen_total) : 0.;   // a NaN is 0
      const u64 target = min(at < 9e18 ? static_cast<u64>(at) : ~0ull, chosen_total - 1);
      if (choose([&](float v, int i) -> u64 { return kept(v, i) ? mass(v) : 0; }, target, ahead, mine) && threadIdx.x == 0)
        finish(m.found, temperature, top, total);
    }
    if (ranks > 1) cluster_barrier();   // no CTA leaves while others read its memory
  }
  // The first token with the largest logit.
  __device__ __forceinline__ void first_of(float top, u64 total) {
    uint32_t first = 0xffffffffu;
    each([&](Tokens x, int i0, int) {
      few(x, i0, which(x, [&](float v, int) { return v == top; }),
          [&](float, int i) { first = min(first, static_cast<uint32_t>(start + i)); });
    });
    __syncthreads();
    first = ~static_cast<uint32_t>(block_join(warp_max64(~first), m.warp_sum, [](u64 a, u64 b) { return max(a, b); }));
    if (threadIdx.x == 0) m.first = first;
    barrier();
    if (rank == 0 && threadIdx.x == 0) {
      for (uint32_t r = 0; r < ranks; ++r) first = min(first, of(&m.first, r));
      finish(first, 1., top, total);
    }
  }
  __device__ __forceinline__ void finish(uint32_t token, double temperature, float top, u64 total) {
    p.tokens[row] = token;
    if (!p.logprobs) return;
    const float v = meant(value(static_cast<const Raw*>(p.logits)[row * p.row_stride + token]));
    const double distance = infinite || v == top ? 0. : (static_cast<double>(v) - top) / temperature;
    p.logprobs[row] = static_cast<float>(distance - log(static_cast<double>(total) / static_cast<double>(kOne)));
  }
};

template <bool kBf16, int kPer>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint8_t sample_cache[];
  __shared__ SampleShared m;
  Sampler<kBf16, kPer> s(p, m, sample_cache);
  s.run();
}

template <bool kBf16, int kPer>
cudaError_t sample_launch(const SampleParams& p, int cluster, int bytes, cudaStream_t s) {
  const auto kernel = sample_kernel<kBf16, kPer>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCacheMost);
  if (e != cudaSuccess) return e;
  return launch_cluster(kernel, dim3(static_cast<unsigned>(p.rows * cluster)), kSampleThreads, static_cast<size_t>(bytes), s, cluster, p);
}

}  // namespace

}  // namespace ts

using namespace ts;

extern "C" int ts_b200_sample(const ts_sample_args* a, ts_stream_t stream) {
  if (!a) return set_error(TS_ERR_VALUE, "sample: null arguments");
  if (a->rows < 1 || a->vocab < 1) return set_error(TS_ERR_VALUE, "sample: rows and vocab must be >= 1");
  if (a->vocab > (1 << 21) || a->rows > (1 << 27))
    return set_error(TS_ERR_NOT_IMPLEMENTED, "sample: more than 2^21 tokens or 2^27 rows");
  if (!a->logits || !a->uniform || !a->tokens) return set_error(TS_ERR_VALUE, "sample: null tensor");
  if (a->dtype != TS_DTYPE_F32 && a->dtype != TS_DTYPE_BF16)
    return set_error(TS_ERR_VALUE, "sample: dtype must be TS_DTYPE_F32 or TS_DTYPE_BF16");
  SampleParams p = {};
  p.rows = a->rows;
  p.vocab = a->vocab;
  p.logits = a->logits;
  p.row_stride = a->row_stride;
  p.uniform = a->uniform;
  p.temperature = a->temperature;
  p.temperature_value = a->temperature_value;
  p.top_k = a->top_k;
  p.top_k_value = a->top_k_value;
  p.top_p = a->top_p;
  p.top_p_value = a->top_p_value;
  p.min_p = a->min_p;
  p.min_p_value = a->min_p_value;
  p.tokens = a->tokens;
  p.logprobs = a->logprobs;
  // CTAs of a row: as many as bring one to each SM with 2048 tokens each.  (A row that is too long for the shared memory of
  // the one CTA that it has is read from L2 again: 512 x 50257 took 297 us with clusters of four that hold it, 184 so.)
  const int size = a->dtype == TS_DTYPE_BF16 ? 2 : 4;
  auto bytes = [&](int c) { return (ceil_div(p.vocab, c) + 255) / 256 * 256 * size; };
  int cluster = 1;
  while (cluster < 8 && ((p.rows * cluster < 148 && p.vocab > 2048 * cluster) || p.vocab > (1 << 18) * cluster)) cluster *= 2;
  p.slice = ceil_div(p.vocab, cluster);
  p.cache = bytes(cluster) <= kCacheMost;
  const int cache = p.cache ? bytes(cluster) : 0;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf16 = a->dtype == TS_DTYPE_BF16, few = p.slice <= 2 * kSampleThreads;
  const cudaError_t e = bf16 ? (few ? sample_launch<true, 2>(p, cluster, cache, s) : sample_launch<true, 8>(p, cluster, cache, s))
                             : (few ? sample_launch<false, 2>(p, cluster, cache, s) : sample_launch<false, 8>(p, cluster, cache, s));
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
  return check_launch("sample");
}
