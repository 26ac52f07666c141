// Root-mean-square norm of rows, with the residual's addition, its backward
// pass, and an output in 8 bits.
//
//   s = round(x + r)                    the residual stream, as it is stored
//   y = s * rstd * w,  rstd = (mean_c s_c^2 + eps)^(-1/2)
//   8-bit output: scale = max(max|y|, 2^-100) / 448 over the row or over each
//   128 columns, code = e4m3(y / scale), y in f32 (no rounding in between); a
//   NaN makes its scale NaN, and with it the codes of that row or those columns
//   backward, u = s rstd:  dx = rstd (w dy - u mean_c(w dy u)) + dsum,
//                          dw = sum_rows dy u
//   (1 - mean u^2 = eps rstd^2, so that in a row of one column the difference
//   is w dy eps rstd^2: it is taken in that form there, where it would cancel)
//
// The norm is the norm of the STORED sum: the next block and the backward
// pass read that value, so both see the same function.  All sums are f32.
//
// Bound by HBM: every stream is read once and written once.  kTpr threads own
// a row and keep its values (in their own type) in registers between the
// reduction and the output, so nothing is read twice.  A thread has 16 values
// of each stream in the forward and 8 in the backward (twice as many above
// 8192 columns): at 65536 x 512 the forward takes 42 us with 16 and 54 with 8,
// the backward, which has four streams and the weight gradient's sums, 69 with
// 16 and 58 with 8.  That leaves registers for 1024 threads on an SM and 48 to
// 64 KB of loads in flight there (6.4 TB/s in the forward, 4.6 in the
// backward, whose instructions then count too).  CTAs have 128 threads where
// the rows allow it, so that a row's barrier holds up no other row (8-bit
// output of 16384 x 2048: 56 us, with 256 threads 62), and as many are launched
// as are resident.  They walk over rows, so a thread meets the same columns in
// every row and the weight gradient is a register sum; one partial row per CTA
// goes to a workspace, and a second kernel adds the partials in a fixed order
// (no atomics: the result does not depend on timing).  Rows that no 16-byte
// load divides are read value by value (4099 x 1537 f32: 17 and 19 us, half of
// the aligned rate).
#include <cuda_fp8.h>

#include "capi_internal.h"
#include "common.cuh"

namespace ts {

constexpr int kNormMaxWidth = 16384;
constexpr int kNormGroup = 128;      // columns that share a scale, where not the whole row
constexpr float kE4m3Max = 448.f;
constexpr float kScaleFloor = 7.8886090522101181e-31f;  // 2^-100

struct NormParams {
  long long rows;
  int width;
  int w_bf16;
  float eps;
  const void* x;
  const void* r;               // or null
  const void* w;
  long long xs, rs;            // row strides (elements) of x and r
  void* y;                     // y, or the 8-bit codes
  void* sum;                   // stored sum (with r), or null
  float* rstd;                 // [rows] or null
  float* scales;               // 8-bit: [rows, ceil(width / group)]
  int group;                   // 0: one scale per row
  // backward (x is the stored sum there)
  const void* dy;
  const void* dsum;            // or null
  long long dys, dss;
  void* dx;
  float* partial;              // [CTAs, width]
};

namespace {

// kVec values of one stream in their own type, 16 bytes where kVec > 1.
template <typename T, int kVec>
struct alignas(kVec * sizeof(T)) Pack {
  T v[kVec];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <int kVec>
__device__ __forceinline__ void load_weight(const void* w, bool bf16, int c, float (&out)[kVec]) {
  if (bf16) {
    const Pack<__nv_bfloat16, kVec> p =
        *reinterpret_cast<const Pack<__nv_bfloat16, kVec>*>(static_cast<const __nv_bfloat16*>(w) + c);
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = to_f(p.v[e]);
  } else {
    constexpr int kPart = kVec < 4 ? kVec : 4;
#pragma unroll
    for (int q = 0; q < kVec; q += kPart) {
      const Pack<float, kPart> p =
          *reinterpret_cast<const Pack<float, kPart>*>(static_cast<const float*>(w) + c + q);
#pragma unroll
      for (int e = 0; e < kPart; ++e) out[q + e] = p.v[e];
    }
  }
}

// The larger of two; NaN where one is (a scale has to show it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum (or, kMax, maximum) over the kTpr threads of this thread's row.  `red`
// holds two buffers of one float per warp; `turn` picks one, so that a
// reduction needs a single barrier.
template <int kTpr, bool kMax>
__device__ __forceinline__ float row_reduce(float v, float* red, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, v, o);
    v = kMax ? max_nan(v, other) : v + other;
  }
  if (kTpr > 32) {
    float* buf = red + turn * 32;
    turn ^= 1;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    constexpr int kWarps = kTpr / 32;
    const int first = warp / kWarps * kWarps;
    v = buf[first];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v = kMax ? max_nan(v, buf[first + i]) : v + buf[first + i];
  }
  return v;
}

template <int kTpr>
constexpr int norm_threads() { return kTpr < 128 ? 128 : kTpr; }

// CTAs of a kernel that an SM holds at once: threads that fit beside `regs`
// registers each.  The kernels are compiled to it and the grids made for it
// (a grid of more CTAs than are resident leaves a ragged last wave).
template <int kTpr>
constexpr int norm_resident(int regs) {
  return 65536 / regs / norm_threads<kTpr>() > 0 ? 65536 / regs / norm_threads<kTpr>() : 1;
}
template <int kTpr>
constexpr int norm_fwd_resident() { return norm_resident<kTpr>(64); }
template <int kTpr>
constexpr int norm_bwd_resident() { return norm_resident<kTpr>(64); }

__device__ __forceinline__ uint8_t to_e4m3(float x) {
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
}

template <typename T, int kVec, int kPacks, int kTpr, bool kCodes>
__global__ void __launch_bounds__(norm_threads<kTpr>(), (norm_fwd_resident<kTpr>()))
    norm_fwd_kernel(const NormParams p) {
  constexpr int kRows = norm_threads<kTpr>() / kTpr;
  __shared__ float red[64];
  __shared__ int group_max[kCodes && kVec == 1 ? kRows * (kNormMaxWidth / kNormGroup) : 1];
  const int t = threadIdx.x % kTpr, slot = threadIdx.x / kTpr;
  const float inv_width = 1.f / static_cast<float>(p.width);
  int turn = 0;
  for (long long base = static_cast<long long>(blockIdx.x) * kRows; base < p.rows;
       base += static_cast<long long>(gridDim.x) * kRows) {
    const long long row = base + slot;
    const bool active = row < p.rows;
    const T* x = static_cast<const T*>(p.x) + row * p.xs;
    const T* r = static_cast<const T*>(p.r) + row * p.rs;
    Pack<T, kVec> s[kPacks];
    float square = 0.f;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      if (active && c < p.width) s[k] = *reinterpret_cast<const Pack<T, kVec>*>(x + c);
    }
    if (p.r) {
      Pack<T, kVec> a[kPacks];
#pragma unroll
      for (int k = 0; k < kPacks; ++k) {
        const int c = (k * kTpr + t) * kVec;
        if (active && c < p.width) a[k] = *reinterpret_cast<const Pack<T, kVec>*>(r + c);
      }
#pragma unroll
      for (int k = 0; k < kPacks; ++k) {
        const int c = (k * kTpr + t) * kVec;
        if (active && c < p.width) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) s[k].v[e] = from_f<T>(to_f(s[k].v[e]) + to_f(a[k].v[e]));
          *reinterpret_cast<Pack<T, kVec>*>(static_cast<T*>(p.sum) + row * p.width + c) = s[k];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      if (active && c < p.width) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) square = fmaf(to_f(s[k].v[e]), to_f(s[k].v[e]), square);
      }
    }
    square = row_reduce<kTpr, false>(square, red, turn);
    const float rstd = rsqrtf(fmaf(square, inv_width, p.eps));
    if (active && t == 0 && p.rstd) p.rstd[row] = rstd;
    if (!kCodes) {
#pragma unroll
      for (int k = 0; k < kPacks; ++k) {
        const int c = (k * kTpr + t) * kVec;
        if (active && c < p.width) {
          float w[kVec];
          load_weight<kVec>(p.w, p.w_bf16, c, w);
#pragma unroll
          for (int e = 0; e < kVec; ++e) s[k].v[e] = from_f<T>(to_f(s[k].v[e]) * rstd * w[e]);
          *reinterpret_cast<Pack<T, kVec>*>(static_cast<T*>(p.y) + row * p.width + c) = s[k];
        }
      }
      continue;
    }
    // 8-bit codes.  A pack's columns lie in one group; with packs of 16 bytes a
    // group is 16 (bf16) or 32 (f32) neighbouring lanes, with single values it
    // is 128 / kTpr passes of this row's threads, whose maxima meet in shared
    // memory (as the bits of non-negative floats, which order like integers, NaN above all).
    constexpr int kLanes = kNormGroup / kVec < 32 ? kNormGroup / kVec : 32;
    const int n_groups = p.group ? (p.width + kNormGroup - 1) / kNormGroup : 1;
    int* gmax = group_max + slot * (kNormMaxWidth / kNormGroup);
    float top[kPacks], row_top = 0.f;
    if (kVec == 1 && p.group) {
      __syncthreads();
      for (int i = t; i < n_groups; i += kTpr) gmax[i] = 0;
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      top[k] = 0.f;
      if (active && c < p.width) {
        float w[kVec];
        load_weight<kVec>(p.w, p.w_bf16, c, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          top[k] = max_nan(top[k], fabsf(to_f(s[k].v[e]) * rstd * w[e]));
        }
      }
      row_top = max_nan(row_top, top[k]);
      if (p.group) {
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) top[k] = max_nan(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
        if (kVec == 1 && (t & 31) == 0 && c < p.width) atomicMax(&gmax[c / kNormGroup], __float_as_int(top[k]));
      }
    }
    if (p.group == 0) {
      row_top = row_reduce<kTpr, true>(row_top, red, turn);
    } else if (kVec == 1) {
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      if (!active || c >= p.width) continue;
      const int g = p.group ? c / kNormGroup : 0;
      float largest = p.group ? (kVec == 1 ? __int_as_float(gmax[g]) : top[k]) : row_top;
      // the scale, its reciprocal in two parts, and y / scale to half a unit in the last place, so that ties fall as
      // they should
      const float scale = max_nan(largest, kScaleFloor) * (1.f / kE4m3Max);
      if (c == g * kNormGroup) p.scales[row * n_groups + g] = scale;
      const float r = __fdividef(1.f, scale), inv = fmaf(fmaf(-scale, r, 1.f), r, r);
      const float rest = fmaf(-scale, inv, 1.f) * inv;
      Pack<uint8_t, kVec> code;
      float y[kVec];
      load_weight<kVec>(p.w, p.w_bf16, c, y);
#pragma unroll
      for (int e = 0; e < kVec; ++e) y[e] *= to_f(s[k].v[e]) * rstd;
      if (kVec == 1) {
        code.v[0] = to_e4m3(fmaf(y[0], inv, y[0] * rest));
      } else {
#pragma unroll
        for (int e = 0; e < kVec; e += 2) {
          const float2 q = make_float2(fmaf(y[e], inv, y[e] * rest), fmaf(y[e + 1], inv, y[e + 1] * rest));
          const uint16_t two = __nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3);
          code.v[e] = static_cast<uint8_t>(two);
          code.v[e + 1] = static_cast<uint8_t>(two >> 8);
        }
      }
      *reinterpret_cast<Pack<uint8_t, kVec>*>(static_cast<uint8_t*>(p.y) + row * p.width + c) = code;
    }
  }
}

template <typename T, int kVec, int kPacks, int kTpr>
__global__ void __launch_bounds__(norm_threads<kTpr>(), (norm_bwd_resident<kTpr>()))
    norm_bwd_kernel(const NormParams p) {
  constexpr int kThreads = norm_threads<kTpr>(), kRows = kThreads / kTpr;
  __shared__ float red[64];
  __shared__ float columns[kRows > 1 ? kThreads * kVec : 1];
  const int t = threadIdx.x % kTpr, slot = threadIdx.x / kTpr;
  const float inv_width = 1.f / static_cast<float>(p.width);
  float dw[kPacks][kVec];
#pragma unroll
  for (int k = 0; k < kPacks; ++k)
#pragma unroll
    for (int e = 0; e < kVec; ++e) dw[k][e] = 0.f;
  int turn = 0;
  for (long long base = static_cast<long long>(blockIdx.x) * kRows; base < p.rows;
       base += static_cast<long long>(gridDim.x) * kRows) {
    const long long row = base + slot;
    const bool active = row < p.rows;
    const T* x = static_cast<const T*>(p.x) + row * p.xs;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dys;
    const T* dsum = static_cast<const T*>(p.dsum) + row * p.dss;
    Pack<T, kVec> s[kPacks], g[kPacks], a[kPacks];
    const float rstd = active ? p.rstd[row] : 0.f;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      if (active && c < p.width) {
        s[k] = *reinterpret_cast<const Pack<T, kVec>*>(x + c);
        g[k] = *reinterpret_cast<const Pack<T, kVec>*>(dy + c);
        if (p.dsum) a[k] = *reinterpret_cast<const Pack<T, kVec>*>(dsum + c);
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      if (active && c < p.width) {
        float w[kVec];
        load_weight<kVec>(p.w, p.w_bf16, c, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float du = to_f(g[k].v[e]) * (to_f(s[k].v[e]) * rstd);
          dw[k][e] += du;
          dot = fmaf(du, w[e], dot);
        }
      }
    }
    dot = row_reduce<kTpr, false>(dot, red, turn) * inv_width;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int c = (k * kTpr + t) * kVec;
      if (active && c < p.width) {
        float w[kVec];
        load_weight<kVec>(p.w, p.w_bf16, c, w);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float u = to_f(s[k].v[e]) * rstd;
          const float dn = to_f(g[k].v[e]) * w[e];
          float d = rstd * (p.width > 1 ? fmaf(-u, dot, dn) : dn * (p.eps * rstd * rstd));
          if (p.dsum) d += to_f(a[k].v[e]);
          a[k].v[e] = from_f<T>(d);
        }
        *reinterpret_cast<Pack<T, kVec>*>(static_cast<T*>(p.dx) + row * p.width + c) = a[k];
      }
    }
  }
  // this CTA's partial of the weight gradient: its row slots added in order
#pragma unroll
  for (int k = 0; k < kPacks; ++k) {
    const int c = (k * kTpr + t) * kVec;
    if (kRows > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kVec; ++e) columns[e * kThreads + threadIdx.x] = dw[k][e];
      __syncthreads();
      if (slot == 0) {
        for (int i = 1; i < kRows; ++i)
#pragma unroll
          for (int e = 0; e < kVec; ++e) dw[k][e] += columns[e * kThreads + i * kTpr + t];
      }
    }
    if (slot == 0) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (c + e < p.width) p.partial[static_cast<long long>(blockIdx.x) * p.width + c + e] = dw[k][e];
    }
  }
}

// Sum of the partial rows: 32 columns a CTA, its 32 warps each over every
// 32nd row, then the warps in order.
constexpr int kDwWarps = 32;

__global__ void __launch_bounds__(32 * kDwWarps) norm_dweight_kernel(const float* __restrict__ partial, int n,
                                                                     int width, void* dw, int bf16) {
  __shared__ float part[kDwWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int i = warp; i < n; i += kDwWarps) sum += partial[static_cast<long long>(i) * width + c];
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < kDwWarps; ++i) sum += part[i][lane];
    if (bf16) {
      static_cast<__nv_bfloat16*>(dw)[c] = __float2bfloat16_rn(sum);
    } else {
      static_cast<float*>(dw)[c] = sum;
    }
  }
}

constexpr int kNormSms = 148;

// CTAs of a walk over `rows`: at most `resident` on each SM, and no more than there are rows to give.
int norm_grid(long long rows, int rows_per_cta, int resident) {
  const long long wanted = (rows + rows_per_cta - 1) / rows_per_cta;
  const long long most = static_cast<long long>(kNormSms) * resident;
  return static_cast<int>(wanted < most ? wanted : most);
}

template <typename T, int kVec, int kPacks, int kTpr, bool kCodes>
int norm_fwd_launch(const NormParams& p, cudaStream_t s) {
  constexpr int kThreads = norm_threads<kTpr>();
  const int grid = norm_grid(p.rows, kThreads / kTpr, norm_fwd_resident<kTpr>());
  norm_fwd_kernel<T, kVec, kPacks, kTpr, kCodes><<<grid, kThreads, 0, s>>>(p);
  return check_launch("norm_fwd");
}

template <int kTpr>
int norm_bwd_grid(long long rows) {
  return norm_grid(rows, norm_threads<kTpr>() / kTpr, norm_bwd_resident<kTpr>());
}

template <typename T, int kVec, int kPacks, int kTpr>
int norm_bwd_launch(const NormParams& p, void* dweight, cudaStream_t s) {
  const int grid = norm_bwd_grid<kTpr>(p.rows);
  norm_bwd_kernel<T, kVec, kPacks, kTpr><<<grid, norm_threads<kTpr>(), 0, s>>>(p);
  if (const int rc = check_launch("norm_bwd")) return rc;
  norm_dweight_kernel<<<ceil_div(p.width, 32), 32 * kDwWarps, 0, s>>>(p.partial, grid, p.width, dweight, p.w_bf16);
  return check_launch("norm_dweight");
}

// Threads per row: F::kEach values of a stream to a thread; twice as many in the widest rows.
template <typename T, int kVec, class F>
int norm_by_width(int width, F f) {
  constexpr int kEach = F::kEach, kPacks = kEach / kVec, kMost = 8192 / kEach;
  if (width <= 32 * kEach) return f.template operator()<T, kVec, kPacks, 32>();
  if (width <= 64 * kEach) return f.template operator()<T, kVec, kPacks, 64>();
  if (width <= 128 * kEach) return f.template operator()<T, kVec, kPacks, 128>();
  if (width <= 256 * kEach) return f.template operator()<T, kVec, kPacks, 256>();
  if (kMost > 512 && width <= 512 * kEach) return f.template operator()<T, kVec, kPacks, (kMost > 512 ? 512 : kMost)>();
  if (width <= kMost * kEach) return f.template operator()<T, kVec, kPacks, kMost>();
  return f.template operator()<T, kVec, 2 * kPacks, kMost>();
}

template <class F>
int norm_dispatch(int dtype, bool vector, int width, F f) {
  if (dtype == TS_DTYPE_BF16)
    return vector ? norm_by_width<__nv_bfloat16, 8>(width, f) : norm_by_width<__nv_bfloat16, 1>(width, f);
  return vector ? norm_by_width<float, 4>(width, f) : norm_by_width<float, 1>(width, f);
}

template <bool kCodes>
struct NormFwd {
  static constexpr int kEach = 16;
  const NormParams& p;
  cudaStream_t s;
  template <typename T, int kVec, int kPacks, int kTpr>
  int operator()() const { return norm_fwd_launch<T, kVec, kPacks, kTpr, kCodes>(p, s); }
};
struct NormBwd {
  static constexpr int kEach = 8;
  const NormParams& p;
  void* dweight;
  cudaStream_t s;
  template <typename T, int kVec, int kPacks, int kTpr>
  int operator()() const { return norm_bwd_launch<T, kVec, kPacks, kTpr>(p, dweight, s); }
};
struct NormBwdGrid {
  static constexpr int kEach = NormBwd::kEach;
  long long rows;
  template <typename T, int kVec, int kPacks, int kTpr>
  int operator()() const { return norm_bwd_grid<kTpr>(rows); }
};

int norm_check(const ts_norm_args* a) {
  if (!a) return set_error(TS_ERR_VALUE, "norm: null arguments");
  if (a->rows < 1) return set_error(TS_ERR_VALUE, "norm: rows must be >= 1");
  if (a->width < 1 || a->width > kNormMaxWidth)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "norm: width %d outside 1..%d", a->width, kNormMaxWidth);
  if (a->dtype != TS_DTYPE_F32 && a->dtype != TS_DTYPE_BF16)
    return set_error(TS_ERR_VALUE, "norm: dtype must be TS_DTYPE_F32 or TS_DTYPE_BF16");
  if (a->weight_dtype != TS_DTYPE_F32 && a->weight_dtype != TS_DTYPE_BF16)
    return set_error(TS_ERR_VALUE, "norm: weight_dtype must be TS_DTYPE_F32 or TS_DTYPE_BF16");
  if (!a->x || !a->weight) return set_error(TS_ERR_VALUE, "norm: null x or weight");
  if (!(a->eps >= 0.f)) return set_error(TS_ERR_VALUE, "norm: eps must be >= 0");
  if (a->group != 0 && a->group != kNormGroup)
    return set_error(TS_ERR_NOT_IMPLEMENTED, "norm: group must be 0 (whole rows) or %d", kNormGroup);
  return TS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

NormParams norm_params(const ts_norm_args* a) {
  NormParams p = {};
  p.rows = a->rows;
  p.width = a->width;
  p.w_bf16 = a->weight_dtype == TS_DTYPE_BF16;
  p.eps = a->eps;
  p.x = a->x;
  p.r = a->residual;
  p.w = a->weight;
  p.xs = a->x_stride;
  p.rs = a->residual_stride;
  p.y = a->y;
  p.sum = a->sum;
  p.rstd = a->rstd;
  p.scales = a->scales;
  p.group = a->group;
  return p;
}

// Whether every row of every stream starts at a multiple of 16 bytes and holds whole packs.
bool norm_vector(const ts_norm_args* a) {
  const int per = a->dtype == TS_DTYPE_BF16 ? 8 : 4;
  return a->width % per == 0 && a->x_stride % per == 0 && (!a->residual || a->residual_stride % per == 0) &&
         aligned16(a->x) && aligned16(a->residual) && aligned16(a->weight) && aligned16(a->y) && aligned16(a->sum);
}

}  // namespace

}  // namespace ts

extern "C" {

int ts_b200_norm_fwd(const ts_norm_args* a, ts_stream_t stream) {
  if (const int rc = ts::norm_check(a)) return rc;
  if (!a->y) return ts::set_error(TS_ERR_VALUE, "norm_fwd: null output");
  if (a->residual && !a->sum) return ts::set_error(TS_ERR_VALUE, "norm_fwd: a residual needs the sum's output");
  if (a->group && !a->scales) return ts::set_error(TS_ERR_VALUE, "norm_fwd: a group needs scales");
  const ts::NormParams p = ts::norm_params(a);
  const bool vector = ts::norm_vector(a);
  return a->scales ? ts::norm_dispatch(a->dtype, vector, a->width, ts::NormFwd<true>{p, stream})
                   : ts::norm_dispatch(a->dtype, vector, a->width, ts::NormFwd<false>{p, stream});
}

size_t ts_b200_norm_bwd_workspace_bytes(const ts_norm_args* a) {
  if (ts::norm_check(a)) return 0;
  // the grid does not depend on how the rows are aligned
  const int grid = ts::norm_dispatch(a->dtype, true, a->width, ts::NormBwdGrid{a->rows});
  return static_cast<size_t>(grid) * a->width * sizeof(float);
}

int ts_b200_norm_bwd(const ts_norm_args* a, const ts_norm_grad_args* g, ts_stream_t stream) {
  if (const int rc = ts::norm_check(a)) return rc;
  if (!g || !g->dy || !g->dx || !g->dweight || !a->rstd)
    return ts::set_error(TS_ERR_VALUE, "norm_bwd: null rstd, dy, dx or dweight");
  if (!g->workspace || g->workspace_bytes < ts_b200_norm_bwd_workspace_bytes(a))
    return ts::set_error(TS_ERR_VALUE, "norm_bwd: workspace too small");
  ts::NormParams p = ts::norm_params(a);
  p.dy = g->dy;
  p.dsum = g->dsum;
  p.dys = g->dy_stride;
  p.dss = g->dsum_stride;
  p.dx = g->dx;
  p.partial = static_cast<float*>(g->workspace);
  const int per = a->dtype == TS_DTYPE_BF16 ? 8 : 4;
  const bool vector = ts::norm_vector(a) && g->dy_stride % per == 0 && (!g->dsum || g->dsum_stride % per == 0) &&
                      ts::aligned16(g->dy) && ts::aligned16(g->dsum) && ts::aligned16(g->dx);
  return ts::norm_dispatch(a->dtype, vector, a->width, ts::NormBwd{p, g->dweight, stream});
}

}  // extern "C"
