// The choice of a token from each row of logits, by given uniform numbers.
//
// Tokens in the order of falling logits, the lower index first among equals; of
// these the first top_k; of those the shortest prefix with top_p of their mass;
// of those the ones with at least min_p times the largest probability.  The token
// is the first, by index, at which the running mass of what is left exceeds
// uniform times its total.
//
// A cluster of CTAs holds a row in registers: the logits are read once.  Masses
// are integers, exp((x - max) / temperature) in units of 2^-40, within 2^-29 of
// themselves: their sums do not depend on an order, and come out the same in every
// CTA, which therefore take the same turns without asking each other.  Nothing is
// sorted: a histogram over 64ths of the scaled distance from the maximum (monotone
// in the logit, so its bins are stretches of the order) says in which bin a cut
// falls; the bin's tokens, usually a few hundred, are gathered and ranked against
// each other.  A bin of more is cut into 2048 by its logits' bits until it is not,
// or has one value left, whose tokens then count in the order of their index.
#include <cmath>

#include "capi_internal.h"
#include "cluster.cuh"

namespace ts {

namespace {

using u64 = unsigned long long;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048, kPerThread = kBins / kSampleThreads;
constexpr int kRanked = 512;                   // tokens that are ranked against each other
constexpr u64 kOne = 1ull << 40;
constexpr uint32_t kNoKey = 0x007fffffu;       // of minus infinity: masked tokens

struct SampleParams {
  int rows, vocab, slice;                      // slice: tokens of a CTA
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

// Larger for larger logits.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SampleShared {
  uint32_t count[kBins], low[kBins], high[kBins];
  u64 fixed[33];                               // 2^(k/32), k = -16..16, in units of 2^-40
  float single[33];
  uint32_t key[kRanked], index[kRanked];       // tokens of a bin: this CTA's
  uint32_t all_key[kRanked], all_index[kRanked];
  u64 all_mass[kRanked];
  u64 warp_sum[kSampleWarps], warp_sum_b[kSampleWarps];
  u64 piece[kSampleThreads];
  u64 total, total_b, best, smallest, largest; // of this CTA, for the others
  uint32_t listed;
  // results, for this CTA's threads
  u64 before, before_b, within, rest;
  uint32_t bin, cut_key, cut_index, found;
  int piece_at;
};

// exp of a distance, as an integer mass.
struct Mass {
  float top, high, low, bins;                  // the largest logit; log2(e) / temperature in two parts; 64 / temperature

  __device__ __forceinline__ u64 of(const SampleShared& m, float x) const {
    if (x == top) return kOne;
    // the distance and what its rounding lost
    const float t = x - top, back = t - x, lost = (x - (t - back)) - (top + back);
    const float a = t * high;
    if (!(a > -41.5f)) return 0;
    const float rest = fmaf(t, high, -a) + fmaf(t, low, lost * high);
    // 2^a = 2^n 2^(k/32) 2^r, |r| <= 1/64: the last by its series, as what it adds to 1
    const float n = rintf(a), f = a - n, k = rintf(f * 32.f);
    const float r = fmaf(k, -0.03125f, f) + rest;
    const float q = r * fmaf(r, fmaf(r, fmaf(r, 0.0096181291f, 0.0555041087f), 0.2402265070f), 0.6931471806f);
    const int at = static_cast<int>(k) + 16, shift = -static_cast<int>(n);
    const long long more = static_cast<long long>(__float2int_rn(m.single[at] * q * 68719476736.f)) << 4;
    const u64 w = m.fixed[at] + static_cast<u64>(more);
    return shift > 0 ? (w + (1ull << (shift - 1))) >> shift : w;
  }
  __device__ __forceinline__ uint32_t bin(float x) const {
    if (x == top) return 0;
    const float d = (top - x) * bins;
    return d < kBins - 1 ? static_cast<uint32_t>(d) : kBins - 1;
  }
};

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
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
__device__ __forceinline__ u64 block_sum64(u64 v, u64* scratch) {
  return block_join(warp_sum(v), scratch, [](u64 a, u64 b) { return a + b; });
}
// Sum over the threads before this one; `all`: over all.
__device__ __forceinline__ u64 block_before(u64 v, u64* scratch, u64& all) {
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
  all = 0;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    if (i < warp) r += scratch[i];
    all += scratch[i];
  }
  return r;
}

template <bool kBf16, int kPer>
struct Sampler {
  const SampleParams& p;
  SampleShared& m;
  uint32_t rank, ranks;
  int row, start, end;                         // this CTA's tokens
  bool resident;                               // all of them are in x
  float x[kPer];
  Mass mass;

  __device__ __forceinline__ Sampler(const SampleParams& p_, SampleShared& m_) : p(p_), m(m_) {
    rank = cluster_rank_of();
    ranks = cluster_size_of();
    row = blockIdx.x / ranks;
    start = min(p.vocab, static_cast<int>(rank) * p.slice);
    end = min(p.vocab, start + p.slice);
    resident = p.slice <= kPer * kSampleThreads;
  }
  __device__ __forceinline__ void barrier() const {
    if (ranks > 1) cluster_barrier();
    else __syncthreads();
  }
  // NaN is a masked token, and so is what lies behind the slice; minus zero is zero.
  __device__ __forceinline__ void load(int from) {
    const long long at = row * p.row_stride;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = from + j * kSampleThreads + threadIdx.x;
      float v = -INFINITY;
      if (i < end)
        v = kBf16 ? bf2f(static_cast<const __nv_bfloat16*>(p.logits)[at + i]) : static_cast<const float*>(p.logits)[at + i];
      x[j] = v != v ? -INFINITY : v + 0.f;
    }
  }
  // f(j, x, token) for each of this thread's tokens that is not masked, in stretches of kPer * 512.
  template <class F>
  __device__ __forceinline__ void each(F f) {
    for (int from = start; from < end; from += kPer * kSampleThreads) {
      if (!resident) load(from);
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (x[j] != -INFINITY) f(j, x[j], from + j * kSampleThreads + static_cast<int>(threadIdx.x));
    }
  }
  // Sum of the CTAs' values at `at`.
  __device__ __forceinline__ u64 cluster_sum(const u64* at) const {
    u64 s = 0;
    for (uint32_t r = 0; r < ranks; ++r) s += ranks > 1 ? cluster_read(at, r) : *at;
    return s;
  }

  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += kSampleThreads) m.count[i] = m.low[i] = m.high[i] = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add(uint32_t bin, u64 w) {
    atomicAdd(&m.count[bin], 1u);
    if (w) {
      const uint32_t part = static_cast<uint32_t>(w);
      const uint32_t old = atomicAdd(&m.low[bin], part);
      const uint32_t up = static_cast<uint32_t>(w >> 32) + (old + part < old ? 1u : 0u);
      if (up) atomicAdd(&m.high[bin], up);
    }
  }

  // The cluster's histogram: this thread's bins and what comes before them.  After a barrier().
  struct Bins {
    u64 count[kPerThread], mass[kPerThread], count_before, mass_before;
  };
  __device__ __forceinline__ Bins joined() {
    Bins b;
    u64 counts = 0, masses = 0, all;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int at = kPerThread * threadIdx.x + i;
      b.count[i] = b.mass[i] = 0;
      for (uint32_t r = 0; r < ranks; ++r) {
        b.count[i] += ranks > 1 ? cluster_read(&m.count[at], r) : m.count[at];
        b.mass[i] += ranks > 1 ? cluster_read(&m.low[at], r) : m.low[at];
        b.mass[i] += static_cast<u64>(ranks > 1 ? cluster_read(&m.high[at], r) : m.high[at]) << 32;
      }
      counts += b.count[i];
      masses += b.mass[i];
    }
    b.count_before = block_before(counts, m.warp_sum, all);
    b.mass_before = block_before(masses, m.warp_sum_b, all);
    return b;
  }
  // The bin in which the running count (mass) reaches `target`: into m.bin, with what comes before it and its count.
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
        m.within = b.count[i];
      }
      counts += b.count[i];
      masses += b.mass[i];
    }
    __syncthreads();
  }

  // The token, in index order, at which the running sum of f exceeds `target`; in every thread of the CTA that holds it
  // (returned: whether this one does), `rank_of` in all.  `sums`: f summed over this thread's tokens.
  template <class F>
  __device__ __forceinline__ bool choose(F f, u64 target, u64 before, u64 mine) {
    if (!(before <= target && target < before + mine)) return false;
    target -= before;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int from = start; from < end; from += kPer * kSampleThreads) {
      if (!resident) load(from);
      // piece j * 16 + warp: 32 tokens; the pieces follow each other in index order
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = from + j * kSampleThreads + static_cast<int>(threadIdx.x);
        const u64 s = warp_sum(x[j] != -INFINITY ? f(x[j], i) : 0);
        if (lane == 0) m.piece[j * kSampleWarps + warp] = s;
      }
      if (threadIdx.x == 0) m.piece_at = -1;
      __syncthreads();
      const u64 own = threadIdx.x < kPer * kSampleWarps ? m.piece[threadIdx.x] : 0;
      u64 all;
      const u64 at = block_before(own, m.warp_sum, all);
      if (at <= target && target < at + own) {
        m.piece_at = threadIdx.x;
        m.rest = target - at;
      }
      __syncthreads();
      if (m.piece_at >= 0) {
        const int j0 = m.piece_at / kSampleWarps;
        if (warp == m.piece_at % kSampleWarps) {
          u64 w = 0;
          const int i = from + j0 * kSampleThreads + static_cast<int>(threadIdx.x);
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (j == j0 && x[j] != -INFINITY) w = f(x[j], i);
          u64 upto = w;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
          }
          if (upto - w <= m.rest && m.rest < upto) m.found = static_cast<uint32_t>(i);
        }
        __syncthreads();
        return true;
      }
      target -= all;
      __syncthreads();
    }
    return false;
  }

  // The last token that is kept when the order is cut where the count (mass) reaches `target` within the bin in m.bin:
  // m.cut_key and m.cut_index; returned: the mass of the bin's tokens up to it.  The target counts from the bin's start.
  __device__ __forceinline__ u64 cut(bool by_mass, u64 target) {
    const uint32_t bin = m.bin;
    uint32_t least = 0, most = 0xffffffffu;   // of the keys that are still in question
    u64 within = m.within, before = 0;
    auto in_question = [&](float v) {
      const uint32_t k = order_key(v);
      return k >= least && k <= most && mass.bin(v) == bin;
    };
    while (within > kRanked) {
      // the largest and smallest key
      u64 low = ~0ull, high = 0;
      each([&](int, float v, int) {
        if (in_question(v)) {
          low = min(low, static_cast<u64>(order_key(v)));
          high = max(high, static_cast<u64>(order_key(v)));
        }
      });
      low = ~warp_max(~low);
      high = warp_max(high);
      low = block_join(low, m.warp_sum, [](u64 a, u64 b) { return min(a, b); });
      high = block_join(high, m.warp_sum_b, [](u64 a, u64 b) { return max(a, b); });
      if (threadIdx.x == 0) {
        m.smallest = low;
        m.largest = high;
      }
      barrier();
      for (uint32_t r = 0; r < ranks && ranks > 1; ++r) {
        low = min(low, cluster_read(&m.smallest, r));
        high = max(high, cluster_read(&m.largest, r));
      }
      least = static_cast<uint32_t>(low);
      most = static_cast<uint32_t>(high);
      if (least == most) {
        // one value: its tokens in the order of their index
        const u64 w = mass.of(m, __uint_as_float(least & 0x80000000u ? least & 0x7fffffffu : ~least));
        const u64 wanted = by_mass ? (target + w - 1) / w : target;
        auto one = [&](float v, int) -> u64 { return in_question(v) ? 1 : 0; };
        u64 counted = 0;
        each([&](int, float v, int i) { counted += one(v, i); });
        counted = block_sum64(counted, m.warp_sum);
        if (threadIdx.x == 0) m.total = counted;
        barrier();
        u64 sum = 0, ahead = 0;
        uint32_t owner = 0;
        for (uint32_t r = 0; r < ranks; ++r) {
          const u64 c = ranks > 1 ? cluster_read(&m.total, r) : m.total;
          if (sum <= wanted - 1 && wanted - 1 < sum + c) owner = r;
          if (r == rank) ahead = sum;
          sum += c;
        }
        choose(one, wanted - 1, ahead, counted);
        barrier();
        const uint32_t token = ranks > 1 ? cluster_read(&m.found, owner) : m.found;
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
      each([&](int, float v, int) {
        if (in_question(v)) add((most - order_key(v)) >> shift, mass.of(m, v));
      });
      barrier();
      const Bins b = joined();
      locate(b, by_mass, target);
      const uint32_t part = m.bin;
      target -= by_mass ? m.before_b : m.before;
      before += m.before_b;
      within = m.within;
      const uint32_t old_least = least, old_most = most;
      most = old_most - (part << shift);
      least = max(old_least, most - ((1u << shift) - 1));
      if (least > most) least = old_least;   // the subtraction passed zero
    }
    // few: all CTAs gather them and rank them
    if (threadIdx.x == 0) m.listed = 0;
    barrier();
    each([&](int, float v, int i) {
      if (in_question(v)) {
        const uint32_t at = atomicAdd(&m.listed, 1u);
        if (at < kRanked) {
          m.key[at] = order_key(v);
          m.index[at] = static_cast<uint32_t>(i);
        }
      }
    });
    barrier();
    uint32_t count = 0;
    for (uint32_t r = 0; r < ranks; ++r) {
      const uint32_t theirs = min(ranks > 1 ? cluster_read(&m.listed, r) : m.listed, kRanked - count);
      for (uint32_t i = threadIdx.x; i < theirs; i += kSampleThreads) {
        const uint32_t k = ranks > 1 ? cluster_read(&m.key[i], r) : m.key[i];
        m.all_key[count + i] = k;
        m.all_index[count + i] = ranks > 1 ? cluster_read(&m.index[i], r) : m.index[i];
        m.all_mass[count + i] = mass.of(m, __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k));
      }
      count += theirs;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += kSampleThreads) {
      const uint32_t k = m.all_key[i], at = m.all_index[i];
      u64 counts = 0, masses = 0;
      for (uint32_t j = 0; j < count; ++j) {
        if (m.all_key[j] > k || (m.all_key[j] == k && m.all_index[j] < at)) {
          ++counts;
          masses += m.all_mass[j];
        }
      }
      const u64 from = by_mass ? masses : counts, mine = by_mass ? m.all_mass[i] : 1;
      if (from < target && target <= from + mine) {
        m.cut_key = k;
        m.cut_index = at;
        m.rest = masses + m.all_mass[i];
      }
    }
    __syncthreads();
    const u64 upto = m.rest;
    barrier();   // the others have read this CTA's list
    return before + upto;
  }

  __device__ __forceinline__ void run() {
    const double given = p.temperature ? static_cast<double>(__ldg(p.temperature + row)) : p.temperature_value;
    const bool greedy = !(given > 0.);
    const double temperature = greedy ? 1. : given;
    if (threadIdx.x < 33) {
      const double v = exp2((static_cast<int>(threadIdx.x) - 16) / 32.);
      m.fixed[threadIdx.x] = static_cast<u64>(llrint(v * kOne));
      m.single[threadIdx.x] = static_cast<float>(v);
    }
    if (resident) load(start);
    // the largest logit, and the first token that has it
    u64 best = 0;
    each([&](int, float v, int i) { best = max(best, static_cast<u64>(order_key(v)) << 32 | (0xffffffffu - i)); });
    best = block_join(warp_max(best), m.warp_sum, [](u64 a, u64 b) { return max(a, b); });
    if (threadIdx.x == 0) m.best = best;
    barrier();
    for (uint32_t r = 0; r < ranks && ranks > 1; ++r) best = max(best, cluster_read(&m.best, r));
    const bool nothing = best == 0;
    const uint32_t top_key = static_cast<uint32_t>(best >> 32), first = 0xffffffffu - static_cast<uint32_t>(best);
    mass.top = __uint_as_float(top_key & 0x80000000u ? top_key & 0x7fffffffu : ~top_key);
    const double scale = min(1.4426950408889634 / temperature, 1e30);
    mass.high = static_cast<float>(scale);
    mass.low = static_cast<float>(scale - mass.high);
    mass.bins = static_cast<float>(min(64. / temperature, 1e30));

    int top_k = greedy ? 0 : p.top_k ? __ldg(p.top_k + row) : p.top_k_value;
    double top_p = greedy ? 1. : p.top_p ? static_cast<double>(__ldg(p.top_p + row)) : p.top_p_value;
    const double min_p = greedy ? 0. : p.min_p ? static_cast<double>(__ldg(p.min_p + row)) : p.min_p_value;
    if (top_k <= 0 || top_k >= p.vocab) top_k = 0;
    const bool by_mass = top_p < 1.;           // a NaN is no limit
    const bool want_total = p.logprobs || (by_mass && top_k == 0);
    u64 total = 0;                              // the mass of all tokens, where it is wanted
    uint32_t cut_key = 0, cut_index = 0;        // kept: keys above, and this key's tokens up to the index
    if (!nothing && (top_k > 0 || by_mass || want_total)) {
      if (top_k > 0 || by_mass) clear();
      u64 sum = 0;
      each([&](int, float v, int) {
        const uint32_t bin = mass.bin(v);
        const u64 w = by_mass || want_total ? mass.of(m, v) : 0;
        sum += w;
        if ((top_k > 0 || by_mass) && bin < kBins - 1) add(bin, by_mass ? w : 0);
      });
      if (want_total) {
        sum = block_sum64(sum, m.warp_sum);
        if (threadIdx.x == 0) m.total_b = sum;
      }
      barrier();
      if (want_total) total = cluster_sum(&m.total_b);
      if (top_k > 0 || by_mass) {
        const Bins b = joined();
        u64 kept = total;
        if (top_k > 0) {
          locate(b, false, static_cast<u64>(top_k));
          if (m.bin < kBins) {
            const u64 ahead = m.before_b;
            kept = ahead + cut(false, top_k - m.before);
            cut_key = m.cut_key;
            cut_index = m.cut_index;
          } else if (by_mass) {
            // the cut lies among tokens without mass
            kept = block_mass(b);
          }
        }
        if (by_mass) {
          const double wanted = ceil(top_p * static_cast<double>(kept));
          const u64 target = wanted >= 1. ? min(static_cast<u64>(wanted), kept) : 1;
          __syncthreads();
          locate(b, true, target);
          if (m.bin < kBins) {
            cut(true, target - m.before_b);
            cut_key = m.cut_key;
            cut_index = m.cut_index;
          }
        }
      }
    }
    // a limit on the logit itself
    float floor_at = -INFINITY;
    if (min_p > 0. && mass.top < INFINITY) {
      const double at = static_cast<double>(mass.top) + temperature * log(min(min_p, 1.));
      floor_at = __double2float_ru(at);
    }
    u64 chosen_total = 0, mine = 0, ahead = 0;
    auto weight = [&](float v, int i) -> u64 {
      const uint32_t k = order_key(v);
      if (k < cut_key || (k == cut_key && static_cast<uint32_t>(i) > cut_index) || !(v >= floor_at)) return 0;
      return mass.of(m, v);
    };
    if (!nothing && !greedy) {
      each([&](int, float v, int i) { mine += weight(v, i); });
      __syncthreads();
      mine = block_sum64(mine, m.warp_sum);
      if (threadIdx.x == 0) m.total = mine;
      barrier();
      for (uint32_t r = 0; r < ranks; ++r) {
        const u64 c = ranks > 1 ? cluster_read(&m.total, r) : m.total;
        if (r == rank) ahead = chosen_total;
        chosen_total += c;
      }
      const double u = static_cast<double>(__ldg(p.uniform + row));
      const double at = u > 0. ? u * static_cast<double>(chosen_total) : 0.;   // a NaN is 0
      const u64 target = min(at < 9e18 ? static_cast<u64>(at) : ~0ull, chosen_total - 1);
      __syncthreads();
      if (choose(weight, target, ahead, mine) && threadIdx.x == 0) finish(static_cast<int>(m.found), temperature, total);
    } else if (rank == 0 && threadIdx.x == 0) {
      if (nothing) {
        p.tokens[row] = -1;
        if (p.logprobs) p.logprobs[row] = -INFINITY;
      } else {
        finish(static_cast<int>(first), temperature, total);
      }
    }
    if (ranks > 1) cluster_barrier();   // no CTA leaves while others read its memory
  }
  // The mass of all bins (each thread's and those before).
  __device__ __forceinline__ u64 block_mass(const Bins& b) {
    u64 s = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) s += b.mass[i];
    __syncthreads();
    return block_sum64(s, m.warp_sum);
  }
  __device__ __forceinline__ void finish(int token, double temperature, u64 total) {
    p.tokens[row] = token;
    if (!p.logprobs) return;
    const long long at = row * p.row_stride + token;
    const float v = kBf16 ? bf2f(static_cast<const __nv_bfloat16*>(p.logits)[at]) : static_cast<const float*>(p.logits)[at];
    const double distance = v == mass.top ? 0. : (static_cast<double>(v) - mass.top) / temperature;
    p.logprobs[row] = static_cast<float>(distance - log(static_cast<double>(total) / static_cast<double>(kOne)));
  }
};

template <bool kBf16, int kPer>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleParams p) {
  __shared__ SampleShared m;
  Sampler<kBf16, kPer> s(p, m);
  s.run();
}

template <bool kBf16>
cudaError_t sample_launch(const SampleParams& p, int cluster, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.rows * cluster));
  if (p.slice <= 4 * kSampleThreads) return launch_cluster(sample_kernel<kBf16, 4>, grid, kSampleThreads, 0, s, cluster, p);
  if (p.slice <= 16 * kSampleThreads) return launch_cluster(sample_kernel<kBf16, 16>, grid, kSampleThreads, 0, s, cluster, p);
  return launch_cluster(sample_kernel<kBf16, 32>, grid, kSampleThreads, 0, s, cluster, p);
}

}  // namespace

}  // namespace ts

extern "C" int ts_b200_sample(const ts_sample_args* a, ts_stream_t stream) {
  if (!a) return set_error(TS_ERR_VALUE, "sample: null arguments");
  if (a->rows < 1 || a->vocab < 1) return set_error(TS_ERR_VALUE, "sample: rows and vocab must be >= 1");
  if (a->vocab > (1 << 22) || a->rows > (1 << 27))
    return set_error(TS_ERR_NOT_IMPLEMENTED, "sample: more than 2^22 tokens or 2^27 rows");
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
  // CTAs of a row: as many as hold it in registers (32 a thread), or bring all SMs to work with 2048 tokens each
  int cluster = 1;
  while (cluster < 8 && (p.vocab > 32 * kSampleThreads * cluster || (p.rows * cluster < 148 && p.vocab > 2048 * cluster))) cluster *= 2;
  p.slice = ceil_div(p.vocab, cluster);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == TS_DTYPE_BF16 ? sample_launch<true>(p, cluster, s) : sample_launch<false>(p, cluster, s);
  if (e != cudaSuccess) return set_error(TS_ERR_CUDA, "sample: %s", cudaGetErrorString(e));
  return check_launch("sample");
}
