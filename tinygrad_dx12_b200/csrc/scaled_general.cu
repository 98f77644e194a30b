// scaled_general.cu -- products of block-scaled activations with packed weights on the CUDA cores, for what
// the tensor-core kernel (scaled_mma.cu) does not take: columns that are no multiple of 128, weights that
// do not begin on a 32-byte boundary.
//
// A warp computes one output: lane l takes the blocks of 32 columns l, l + 32, ..., decodes 32 codes of
// each side exactly, sums their products in fp32 and multiplies by the product of the two powers of two. Raw sums go to
// scratch; a second launch applies bias, activation, gate and residual, and rounds or quantises (a warp
// holds 32 neighbouring columns, a block). Bound by the decoding: some 0.1 TFLOP/s. It is there so that
// every call has an answer, not for speed.
#include "common.cuh"
#include "kernels.h"
#include "scaled_epilogue.cuh"

namespace b200 {
namespace scaled {

struct GeneralParams {
  const uint8_t *w, *ws, *x, *xs;
  float *raw;           // [rows][n]
  const int32_t *offsets, *order;
  int64_t rows, n, cols;  // rows of y, weight rows of one matrix
  int experts, fan, x_rows, y_rows;
};

// The pair at place i of the plan and its expert; -1 without one.
__device__ __forceinline__ int expert_at(const int32_t *offsets, int experts, int64_t i) {
  if (i >= offsets[experts]) return -1;
  int lo = 0, hi = experts;  // offsets[lo] <= i < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// part * 2^(a - 127) * 2^(b - 127), rounded once: by the exponents' sum, as the tensor cores have it. (One factor after the other
// overflows or loses bits on the way where the scales lie far apart.)
__device__ __forceinline__ float scaled_sum(float part, int a, int b) {
  return a == 255 || b == 255 ? __uint_as_float(0x7FC00000u) : ldexpf(part, a + b - 254);
}

template <int FMT>
__global__ void __launch_bounds__(256) product_kernel(const __grid_constant__ GeneralParams p) {
  constexpr int BITS = Fmt<FMT>::bits, BYTES = 4 * BITS;  // of a block of 32 codes
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= p.n) return;
  const int64_t nblk = p.cols >> 5;
  for (int64_t i = blockIdx.y; i < p.rows; i += gridDim.y) {
    int64_t xrow = i, yrow = i, wrow = n;
    if (p.experts > 0) {
      const int e = expert_at(p.offsets, p.experts, i);
      if (e < 0) break;  // the pairs without an expert are the last
      const int64_t pair = p.order[i];
      yrow = p.y_rows == B200_ROWS_PLAN ? i : pair;
      xrow = p.x_rows == B200_ROWS_PLAN ? i : p.x_rows == B200_ROWS_PAIRS ? pair : pair / p.fan;
      wrow = e * p.n + n;
    }
    const uint8_t *w = p.w + wrow * nblk * BYTES, *x = p.x + xrow * p.cols;
    float sum = 0.f;
    for (int64_t b = lane; b < nblk; b += 32) {
      float part = 0.f;
      for (int g = 0; g < 8; ++g) {  // four codes: two or three bytes
        const uint8_t *c = w + b * BYTES + g * (BITS / 2);
        uint32_t word = (uint32_t)c[0] | (uint32_t)c[1] << 8;
        if constexpr (BITS == 6) word |= (uint32_t)c[2] << 16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          part = fmaf(decode_fp<FMT>((word >> (j * BITS)) & ((1u << BITS) - 1)), rows8::code_value(x[b * 32 + g * 4 + j]), part);
      }
      sum += scaled_sum(part, p.ws[wrow * nblk + b], p.xs[xrow * nblk + b]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) p.raw[yrow * p.n + n] = sum;
  }
}

// A warp 32 columns of one row of y.
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ GeneralParams p, const Epilogue ep) {
  const int lane = threadIdx.x & 31;
  const int64_t c = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * 32 + lane;
  if (c - lane >= ep.cols) return;
  for (int64_t i = blockIdx.y; i < p.rows; i += gridDim.y) {
    int64_t yrow = i;
    int e = 0;
    if (p.experts > 0) {
      e = expert_at(p.offsets, p.experts, i);
      if (p.y_rows == B200_ROWS_PLAN && e < 0) break;  // not written: they are the last
      yrow = p.y_rows == B200_ROWS_PLAN ? i : p.order[i];
    }
    float v = 0.f;
    if (c < ep.cols && e >= 0) {
      const float *raw = p.raw + yrow * p.n;
      const int64_t brow = e * p.n;
      float g = raw[c];
      if (ep.bias != nullptr) g += load_as_f32(ep.bias, brow + c, ep.bdt);
      v = activate(g, ep.activation);
      if (ep.gated) {
        float u = raw[ep.cols + c];
        if (ep.bias != nullptr) u += load_as_f32(ep.bias, brow + ep.cols + c, ep.bdt);
        v = __fmul_rn(v, u);
      }
      if (ep.residual != nullptr) v += load_as_f32(ep.residual, yrow * ep.rstride + c, ep.rdt);
    }
    if (ep.ydt == B200_DT_F8E4M3) {
      const uint32_t byte = rows8::scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7FFFFFFFu));
      ((uint8_t *)ep.y)[yrow * ep.cols + c] = (uint8_t)rows8::codes2(v, 0.f, rows8::inverse(byte), byte == 255u);
      if (lane == 0) ep.ys[yrow * (ep.cols >> 5) + (c >> 5)] = (uint8_t)byte;
    } else if (c < ep.cols) {
      store_f32(ep.y, yrow * ep.cols + c, ep.ydt, v);
    }
  }
}

template <int FMT>
static int32_t products(const GeneralParams &p, cudaStream_t stream) {
  const unsigned gy = (unsigned)(p.rows < 65535 ? p.rows : 65535);
  product_kernel<FMT><<<dim3((unsigned)((p.n + 7) / 8), gy), 256, 0, stream>>>(p);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

static bool real(int dt) { return dt == B200_DT_F16 || dt == B200_DT_BF16 || dt == B200_DT_F32; }

}  // namespace scaled

int32_t launch_scaled_general(const b200_packed_desc *w, const b200_scaled_args *a, cudaStream_t stream) {
  using namespace scaled;
  GeneralParams p;
  p.w = (const uint8_t *)w->data, p.ws = (const uint8_t *)w->scales, p.x = (const uint8_t *)a->x, p.xs = (const uint8_t *)a->x_scales;
  p.raw = (float *)a->scratch;
  p.offsets = a->offsets, p.order = a->order;
  p.rows = a->rows, p.n = a->experts > 0 ? w->rows / a->experts : w->rows, p.cols = w->cols;
  p.experts = (int)a->experts, p.fan = a->fan, p.x_rows = a->x_rows, p.y_rows = a->y_rows;
  int32_t rc;
  switch (w->format) {
    case B200_FMT_FP4_E2M1: rc = products<B200_FMT_FP4_E2M1>(p, stream); break;
    case B200_FMT_FP6_E2M3: rc = products<B200_FMT_FP6_E2M3>(p, stream); break;
    default: rc = products<B200_FMT_FP6_E3M2>(p, stream); break;
  }
  if (rc != B200_OK) return rc;
  const Epilogue ep = epilogue_of(w, a);
  const unsigned gy = (unsigned)(p.rows < 65535 ? p.rows : 65535);
  finish_kernel<<<dim3((unsigned)((ep.cols + 255) / 256), gy), 256, 0, stream>>>(p, ep);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

}  // namespace b200

using namespace b200;
using namespace b200::scaled;

static int32_t check_scaled(const b200_packed_desc *w, const b200_scaled_args *a) {
  if (w == nullptr || a == nullptr) return b200_set_error(B200_ERR_INVALID, "scaled_linear: null arguments");
  if (int32_t rc = b200_validate(w)) return rc;
  if (w->format != B200_FMT_FP4_E2M1 && w->format != B200_FMT_FP6_E2M3 && w->format != B200_FMT_FP6_E3M2)
    return b200_set_error(B200_ERR_UNSUPPORTED, "scaled_linear: FP4 or FP6 weights");
  if (w->scale_dtype != B200_DT_E8M0 || w->block_size != 32 || w->cols < 1 || w->cols % 32 != 0)
    return b200_set_error(B200_ERR_UNSUPPORTED, "scaled_linear: weights with E8M0 scales in whole blocks of 32");
  if (a->rows < 0 || a->rows > 0x7FFFFFFF || a->experts < 0 || a->experts > 1024)
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: rows or experts out of range");
  if (a->experts > 0 && (w->rows % a->experts != 0 || a->fan < 1 || a->residual != nullptr))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: experts of equal rows, a fan, and no residual");
  if (a->experts > 0 && (a->x_rows < B200_ROWS_TOKENS || a->x_rows > B200_ROWS_PLAN || (a->y_rows != B200_ROWS_PAIRS && a->y_rows != B200_ROWS_PLAN)))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: unknown kind of rows");
  const int64_t n = a->experts > 0 ? w->rows / a->experts : w->rows;
  if (a->activation < B200_ACT_NONE || a->activation > B200_ACT_GELU_TANH || (a->gated && n % 2 != 0))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: unknown activation, or a gate over an odd number of rows");
  const bool eight = a->y_dtype == B200_DT_F8E4M3;
  if ((!eight && !real(a->y_dtype)) || (a->bias != nullptr && !real(a->bias_dtype)) || (a->residual != nullptr && !real(a->residual_dtype)))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: float16, bfloat16 or float32, and fp8e4m3 results");
  if (eight && (a->gated ? n / 2 : n) % 32 != 0)
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: 8-bit rows are whole blocks of 32");
  if (a->rows == 0 || n == 0) return B200_OK;
  if (a->x == nullptr || a->x_scales == nullptr || a->y == nullptr || (eight && a->y_scales == nullptr) || w->data == nullptr ||
      w->scales == nullptr || (a->experts > 0 && (a->offsets == nullptr || a->order == nullptr)))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: null pointer");
  auto off = [](const void *p, int size) { return p != nullptr && (uintptr_t)p % size != 0; };
  if (off(a->y, dt_size(a->y_dtype)) || off(a->bias, a->bias != nullptr ? dt_size(a->bias_dtype) : 1) ||
      off(a->residual, a->residual != nullptr ? dt_size(a->residual_dtype) : 1) || (a->experts > 0 && (off(a->offsets, 4) || off(a->order, 4))))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: a tensor off its elements' boundary");
  return B200_OK;
}

extern "C" {

int64_t b200_scaled_linear_scratch(const b200_packed_desc *w, const b200_scaled_args *a) {
  if (w == nullptr || a == nullptr || a->rows < 0 || a->experts < 0) return 0;
  if (!a->general && scaled_mma_takes(w, a)) return scaled_gathers(a) ? a->rows * w->cols : 0;
  return a->rows * (a->experts > 0 ? w->rows / a->experts : w->rows) * 4;
}

int32_t b200_scaled_linear(const b200_packed_desc *w, const b200_scaled_args *a, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (int32_t rc = check_scaled(w, a)) return rc;
  if (a->rows == 0 || w->rows == 0) return B200_OK;
  const bool mma = !a->general && scaled_mma_takes(w, a);
  if ((!mma || scaled_gathers(a)) && (a->scratch == nullptr || (uintptr_t)a->scratch % 16 != 0))
    return b200_set_error(B200_ERR_INVALID, "scaled_linear: this call needs scratch on a 16-byte boundary");
  if (mma) return launch_scaled_mma(w, a, (cudaStream_t)stream);
  return launch_scaled_general(w, a, (cudaStream_t)stream);
}

}  // extern "C"
