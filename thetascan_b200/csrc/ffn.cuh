// What the kernels of the gated feed-forward block share.
#pragma once

#include "../../include/thetascan_b200.h"
#include "common.cuh"

namespace ts {

// Rows up to which an inference call streams the weights past the rows
// (ffn_rows.cu) instead of forming tiles of 256 rows (ffn.cu).
// At 1024 x 4096 and 1 / 16 / 32 rows this takes 7.8 / 10.2 / 11.9 us, the
// tiles 26; at 2048 x 5632 and 32 rows 31 us, the tiles 34, and at 48 and 64
// rows 69 and 73 with the tiles still at 34.
constexpr int kRowsMost = 32;

// The forward for few rows; arguments checked, h holds [rows, hidden].
int ffn_rows_fwd(const ts_ffn_args* a, void* h, cudaStream_t s);

// The activations: value and slope.
template <int kAct>
__device__ __forceinline__ float ffn_act(float g, float& slope) {
  if (kAct == TS_FFN_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    slope = s * fmaf(g, 1.f - s, 1.f);
    return g * s;
  }
  if (kAct == TS_FFN_GELU) {
    // by erfc: 1 + erf would cancel where g is negative
    const float s = 0.5f * erfcf(g * -0.70710678118654752f);
    slope = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), s);
    return g * s;
  }
  const float s = fmaxf(g, 0.f);
  slope = 2.f * s;
  return s * s;
}

}  // namespace ts
