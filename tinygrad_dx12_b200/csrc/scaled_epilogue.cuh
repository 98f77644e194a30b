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
// is within 2 ulp, and t keeps its relative precision, so a tail is exact to 6 + |z| / 8 ulp of itself down to t = 2^-126,
// where it becomes zero (z = -87.3). The power of two takes |z| log2(e) with what it rounds off; without that it is off by
// |z| ulp. 4096 tokens x 14336 x 4096, us: gated 241, FP6 with a bias 279; with CUDA's full exponential 248 and 302, with its
// fast one 236 and 270.
__device__ __forceinline__ float times_sigmoid(float v, float z) {
  const float a = fminf(fabsf(z), 128.f), h = a * -1.44269504f;
  float t;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(h));
  t = fmaf(t * 0.69314718f, fmaf(a, -1.44269504f, -h), t);
  return __fdividef(z < 0.f ? v * t : v, 1.f + t);
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == B200_ACT_RELU) return v > 0.f ? v : v != v ? v : 0.f;
  if constexpr (ACT == B200_ACT_SILU) return times_sigmoid(v, v);
  if constexpr (ACT == B200_ACT_GELU) {
    // v Phi(v) by the tail erfc(a / sqrt 2) = e^(-a^2 / 2) t P(t), a = |v|, t = 1 / (1 + 0.35 a): P fitted to within 3.3e-8 of
    // itself over a in [0, 15], its Chebyshev series weighted until the largest relative errors were level. The power of
    // two takes a^2 and its product with log2(e) / 2 with what they round off, so the tail is exact to 12 + a^2 / 16 ulp of
    // itself down to 2^-126, which is where it becomes zero (a = 13.1). Without a branch, so that a warp's columns run side by
    // side. 4096 tokens x 14336 x 4096 FP6, us: 287; with CUDA's exponential in place of the power 299, and what a^2 rounds
    // off put back 319; with the fast one, exact to 12 + a^2 ulp, 277; with erff 456.
    const float a = fminf(fabsf(v), 15.f), sq = a * a, y = sq * -0.72134752f;
    float tail;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(tail) : "f"(y));
    tail = fmaf(tail * 0.69314718f, fmaf(fmaf(a, a, -sq), -0.72134752f, fmaf(sq, -0.72134752f, -y)), tail);
    const float t = __fdividef(1.f, fmaf(0.35f, a, 1.f));
    float q = fmaf(-0.0583277047f, t, 0.288120955f);
    q = fmaf(q, t, -0.511802554f);
    q = fmaf(q, t, 0.318784654f);
    q = fmaf(q, t, -0.0465269908f);
    q = fmaf(q, t, 0.211149365f);
    q = fmaf(q, t, 0.239631042f);
    q = fmaf(q, t, 0.279728681f);
    q = fmaf(q, t, 0.279242516f);
    tail *= q * t;
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
