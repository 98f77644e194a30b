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

// v times the sigmoid of z, by t = e^-|z|: 1 / (1 + t) or t / (1 + t). The denominator lies in [1, 2], where the fast division
// is within 2 ulp, and t keeps its relative precision until it is subnormal, so a tail is exact to 6 ulp of itself. The
// exponential is the full one: __expf's error grows with |z| (20 ulp at 16), and its 1 + e^-z left nothing of z below -87.
__device__ __forceinline__ float times_sigmoid(float v, float z) {
  const float t = expf(-fabsf(z));
  return __fdividef(z < 0.f ? v * t : v, 1.f + t);
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == B200_ACT_RELU) return v > 0.f ? v : v != v ? v : 0.f;
  if constexpr (ACT == B200_ACT_SILU) return times_sigmoid(v, v);
  if constexpr (ACT == B200_ACT_GELU) {
    // erf by Abramowitz and Stegun's 7.1.26 (within 1.5e-7): without a branch, so that a warp's columns run side
    // by side (CUDA's erff does not: 4096 tokens x 14336 x 4096 456 us)
    const float z = fabsf(v) * 0.70710678118654752f, t = __fdividef(1.f, fmaf(0.3275911f, z, 1.f));
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    const float tail = q * t * __expf(-z * z);  // 1 - erf(z)
    return 0.5f * v * (v < 0.f ? tail : 2.f - tail);
  }
  // (1 + tanh(z)) / 2 is the sigmoid of 2z
  if constexpr (ACT == B200_ACT_GELU_TANH) return times_sigmoid(v, 1.5957691216057307f * fmaf(0.044715f * v, v * v, v));
  return v;
}
__device__ __forceinline__ float activate(float v, int activation) {
  switch (activation) {
    case B200_ACT_RELU: return activate<B200_ACT_RELU>(v);
    case B200_ACT_SILU: return activate<B200_ACT_SILU>(v);
    case B200_ACT_GELU: return activate<B200_ACT_GELU>(v);
    case B200_ACT_GELU_TANH: return activate<B200_ACT_GELU_TANH>(v);
  }
  return v;
}

}  // namespace scaled
}  // namespace b200
