// scaled_epilogue.cuh -- what follows a product of block-scaled activations with packed weights.
#pragma once

#include "scaled_rows.cuh"

namespace b200 {
namespace scaled {

struct Epilogue {
  const void *bias;      // [experts][rows of a matrix], or null
  const void *residual;  // [rows][cols], or null
  void *y;               // [rows][cols]
  uint8_t *ys;           // [rows][cols / 32], 8-bit y
  int64_t cols, rstride;
  int bdt, rdt, ydt, activation, gated;
};

inline Epilogue epilogue_of(const b200_packed_desc *w, const b200_scaled_args *a) {
  const int64_t n = a->experts > 0 ? w->rows / a->experts : w->rows;
  return Epilogue{a->bias, a->residual, a->y, (uint8_t *)a->y_scales, a->gated ? n / 2 : n, a->residual_stride,
                  a->bias_dtype, a->residual_dtype, a->y_dtype, a->activation, a->gated};
}

// In fp32, with CUDA's own functions: an exponential's or an error function's rounding is 2 ulp, far below
// the output types'.
__device__ __forceinline__ float activate(float v, int activation) {
  switch (activation) {
    case B200_ACT_RELU: return v > 0.f ? v : v != v ? v : 0.f;
    case B200_ACT_SILU: return v / (1.f + expf(-v));
    // (1 + erf(z)) = erfc(-z) and (1 + tanh(z)) / 2 = 1 / (1 + e^(-2z)): nothing cancels for negative v
    case B200_ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678118654752f);
    case B200_ACT_GELU_TANH: return v / (1.f + expf(-1.5957691216057307f * fmaf(0.044715f * v, v * v, v)));
  }
  return v;
}

}  // namespace scaled
}  // namespace b200
