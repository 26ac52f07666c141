// What the kernels of the gated feed-forward block share.
#pragma once

#include "../../include/thetascan_b200.h"
#include "common.cuh"

namespace ts {

// Rows up to which an inference call streams the weights past the rows
// (ffn_rows.cu) instead of forming tiles of 256 rows (ffn.cu).
// At 1024 x 4096 and 1 / 16 / 32 rows this takes 8.8 / 13.3 / 13.9 us, the
// tiles 26 / 25 / 25; at 2048 x 5632 21.7 / 25.9 / 31.7 us, the tiles 39 / 35 /
// 34, and 34 still at 48 and 64 rows, where this would read x and h once more.
constexpr int kRowsMost = TS_FFN_TWO_PART_ROWS;

// bf16 parts of h, dg and du of a call (ffn_high, ffn_rest).
constexpr int ffn_parts(long long rows) { return rows <= kRowsMost ? 2 : 1; }

// The forward for few rows; arguments checked, h holds [2, rows, hidden].
int ffn_rows_fwd(const ts_ffn_args* a, void* h, cudaStream_t s);

// g and u kept for a backward pass: blocks of 32 rows x 32 columns, a lane's
// row as twelve 16-byte vectors [vector][lane] (a warp's access is 512
// contiguous bytes); for each half of 16 columns: the upper halves of g's words,
// two vectors, their third bytes, one vector, and the same of u.
__device__ __forceinline__ uint8_t* keep_at(uint8_t* base, int cols, int row, int col, int lane) {
  const size_t blocks = static_cast<size_t>((cols + 31) >> 5);
  return base + ((row >> 5) * blocks + (col >> 5)) * TS_FFN_KEPT_BLOCK + 16 * lane;
}
// One place of them.
__device__ __forceinline__ void keep_one(uint8_t* base, int cols, int row, int col, float g, float u) {
  uint8_t* half = keep_at(base, cols, row, col, row & 31) + ((col >> 4) & 1) * (6 * 512);
  const int c = col & 15;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t word = __float_as_uint(i ? u : g);
    uint8_t* to = half + 3 * 512 * i;
    reinterpret_cast<uint16_t*>(to + 512 * (c >> 3))[c & 7] = static_cast<uint16_t>(word >> 16);
    to[2 * 512 + c] = static_cast<uint8_t>(word >> 8);
  }
}

// A value in two bf16 parts, within 2^-16 of it: its upper half, and what is
// left.  Cut off and not rounded, so that both parts have the value's sign, and
// the second is never zero beside a first that is not: a product with an
// infinity is then infinite in both, where the difference of two infinities, or
// 0 inf, would be NaN.  (2^-126 is nothing beside values over 2^-100.)
__device__ __forceinline__ float ffn_high(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ float ffn_rest(float x) {
  const float rest = x - ffn_high(x);   // NaN of an infinity
  return fabsf(x) > 7.8886090522101181e-31f && !(fabsf(rest) > 0.f) ? copysignf(1.1754943508222875e-38f, x) : rest;
}

// The activations: value and slope.
template <int kAct>
__device__ __forceinline__ float ffn_act(float g, float& slope) {
  if (kAct == TS_FFN_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    slope = s * fmaf(g, 1.f - s, 1.f);
    return g * s;
  }
  if (kAct == TS_FFN_GELU) {
    // The normal distribution's share below -|g| is erfc(z) / 2, z = |g| / sqrt 2
    // (1 + erf would cancel there).  With t = 1 / (1 + z / 2), erfc(z) = t exp(f(t)
    // - z^2) (the form of erfc in Numerical Recipes, Press et al.) and f is smooth
    // on (0, 1]: a least-squares polynomial of degree 7 on 64 Chebyshev points of
    // (0, 1], fitted here to log(exp(z^2) erfc(z) / t), is within 3e-6.  f32 keeps
    // gelu within 4e-6 of itself for g >= -5; below, the rounding of z^2 counts:
    // 8e-6 to -9 and 2.3e-5 to -13, where gelu is under 1e-17 itself.  CUDA's erfcf
    // took a forward pass of 1531 x 1024 x 2816 5 us more.
    const float z = fabsf(g) * 0.70710678118654752f, zz = z * z;
    const float t = __fdividef(1.f, fmaf(0.5f, z, 1.f));
    float f = fmaf(-0.16612210869789124f, t, 0.668515145778656f);
    f = fmaf(f, t, -0.8729041218757629f);
    f = fmaf(f, t, 0.24829064309597015f);
    f = fmaf(f, t, 0.004035713616758585f);
    f = fmaf(f, t, 0.384089857339859f);
    f = fmaf(f, t, 0.9996045827865601f);
    f = fmaf(f, t, -1.2655092477798462f);
    const float below = 0.5f * t * __expf(f - zz);
    const float s = g > 0.f ? 1.f - below : below;
    slope = fmaf(g * 0.39894228040143268f, __expf(-zz), s);
    return g * s;
  }
  float s;   // max(g, 0), and NaN for a NaN
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(s) : "f"(g));
  slope = 2.f * s;
  return s * s;
}

}  // namespace ts
