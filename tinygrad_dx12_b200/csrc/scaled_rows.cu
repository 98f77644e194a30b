// scaled_rows.cu -- RMS norm with the residual's addition, its output in 16 bits or block-scaled 8 bits;
// and the values of block-scaled rows.
//
//   total = x + residual (fp32, rounded to the residual's type and stored)       with a residual
//   y     = t * rsqrt(mean(t^2) + eps) * weight, t = total or x                  fp32, rounded once
//   codes = rne_e4m3(y / s), s a power of two for every 32 values                8-bit output
//
// One pass over memory: a CTA keeps its row in registers, 8 values a thread and vector (a block of 32 is
// four neighbouring lanes), so x and the residual are read once, total and y written once, and nothing is
// read again after the reduction. Bound by HBM for prompts and by the launch and one chain of load,
// reduction and store for a token.
#include "kernels.h"
#include "scaled_rows.cuh"

namespace b200 {
namespace rows8 {

// Launched behind a kernel that lets its followers start early: everything waits for it, and lets others start.
__device__ __forceinline__ void follow() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... KArgs, typename... Args>
static cudaError_t launch(void (*kernel)(KArgs...), int64_t ctas, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

struct NormParams {
  const void *x, *residual, *weight;
  void *total, *y;
  uint8_t *ys;
  int64_t cols, xs, rs, ts;
  int wdt;
  float eps;
};

template <typename T>
__device__ __forceinline__ void unpack8(const T *p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
  else return v;
}
__device__ __forceinline__ float widened(__half v) { return __half2float(v); }
__device__ __forceinline__ float widened(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widened(float v) { return v; }

template <typename T>
__device__ __forceinline__ void pack8(T *p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T a = rounded<T>(f[2 * i]), b = rounded<T>(f[2 * i + 1]);
      w[i] = (uint32_t)*reinterpret_cast<const uint16_t *>(&a) | (uint32_t)*reinterpret_cast<const uint16_t *>(&b) << 16;
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Sum over the CTA's threads, the same in all of them.
__device__ __forceinline__ float cta_sum(float v) {
  __shared__ float part[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if (lane == 0) part[warp] = v;
  __syncthreads();
  v = lane < warps ? part[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct E4M3 {};  // y in 8 bits

// Types: TX of x, TR of the residual and total (TX without one), TY of y. V vectors of 8 values a thread.
template <typename TX, typename TR, typename TY, int V, bool RESIDUAL, bool NORMALIZE>
__global__ void __launch_bounds__(1024) norm_kernel(const __grid_constant__ NormParams p) {
  follow();
  const int64_t row = blockIdx.x;
  const int nvec = (int)(p.cols >> 3);
  float v[V][8];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = i * blockDim.x + threadIdx.x;
    if (at < nvec) {
      unpack8((const TX *)p.x + row * p.xs + 8 * (int64_t)at, v[i]);
      if constexpr (RESIDUAL) {
        float r[8];
        unpack8((const TR *)p.residual + row * p.rs + 8 * (int64_t)at, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = widened(rounded<TR>(__fadd_rn(v[i][j], r[j])));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  if constexpr (RESIDUAL) {  // the stored total is what the norm is of
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = i * blockDim.x + threadIdx.x;
      if (at < nvec) pack8((TR *)p.total + row * p.ts + 8 * (int64_t)at, v[i]);
    }
  }
  float inv = 1.f;
  if constexpr (NORMALIZE) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(v[i][j], v[i][j], sum);
    inv = rsqrtf(cta_sum(sum) / (float)p.cols + p.eps);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = i * blockDim.x + threadIdx.x;
    const bool live = at < nvec;
    if constexpr (NORMALIZE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = __fmul_rn(v[i][j], inv);
      if (p.weight != nullptr && live) {
        float w[8];
        if (p.wdt == B200_DT_F32) unpack8((const float *)p.weight + 8 * at, w);
        else if (p.wdt == B200_DT_F16) unpack8((const __half *)p.weight + 8 * at, w);
        else unpack8((const __nv_bfloat16 *)p.weight + 8 * at, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = __fmul_rn(v[i][j], w[j]);
      }
    }
    if constexpr (std::is_same<TY, E4M3>::value) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t byte = scale_byte(top);
      const float s = inverse(byte);
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = codes2(v[i][2 * j], v[i][2 * j + 1], s, byte == 255u);
      if (live) {
        *reinterpret_cast<uint2 *>((uint8_t *)p.y + row * p.cols + 8 * (int64_t)at) =
            make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
        if ((threadIdx.x & 3) == 0) p.ys[row * (p.cols >> 5) + (at >> 2)] = (uint8_t)byte;
      }
    } else {
      if (live) pack8((TY *)p.y + row * p.cols + 8 * (int64_t)at, v[i]);
    }
  }
}

// Any width, alignment and mix of types: a CTA a row, the row read again after the reduction (from total
// where there is one). A warp holds 32 neighbouring values, so a block's largest is one warp's.
__global__ void __launch_bounds__(256) norm_general_kernel(const NormParams p, int xdt, int tdt, int ydt, int normalize) {
  follow();
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31;
  float sum = 0.f;
  if (p.residual != nullptr || normalize) {
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) {
      float t = load_as_f32(p.x, row * p.xs + c, xdt);
      if (p.residual != nullptr) {
        t += load_as_f32(p.residual, row * p.rs + c, tdt);
        store_f32(p.total, row * p.ts + c, tdt, t);
        t = load_as_f32(p.total, row * p.ts + c, tdt);
      }
      sum = fmaf(t, t, sum);
    }
  }
  const float inv = normalize ? rsqrtf(cta_sum(sum) / (float)p.cols + p.eps) : 1.f;
  for (int64_t first = threadIdx.x - lane; first < p.cols; first += 256) {
    const int64_t c = first + lane;
    float t = 0.f;
    if (c < p.cols) {
      t = p.residual != nullptr ? load_as_f32(p.total, row * p.ts + c, tdt) : load_as_f32(p.x, row * p.xs + c, xdt);
      if (normalize) {
        t = __fmul_rn(t, inv);
        if (p.weight != nullptr) t = __fmul_rn(t, load_as_f32(p.weight, c, p.wdt));
      }
    }
    if (ydt == B200_DT_F8E4M3) {
      const uint32_t byte = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(t) & 0x7FFFFFFFu));
      ((uint8_t *)p.y)[row * p.cols + c] = (uint8_t)codes2(t, 0.f, inverse(byte), byte == 255u);
      if (lane == 0) p.ys[row * (p.cols >> 5) + (c >> 5)] = (uint8_t)byte;
    } else if (c < p.cols) {
      store_f32(p.y, row * p.cols + c, ydt, t);
    }
  }
}

template <typename TX, typename TR, typename TY, int V, bool RESIDUAL>
static int32_t launch_norm(const NormParams &p, int64_t rows, int threads, bool normalize, cudaStream_t stream) {
  if (normalize) B200_CUDA_TRY(launch(norm_kernel<TX, TR, TY, V, RESIDUAL, true>, rows, threads, stream, p));
  else B200_CUDA_TRY(launch(norm_kernel<TX, TR, TY, V, RESIDUAL, false>, rows, threads, stream, p));
  return B200_OK;
}

// One vector a thread for few rows (a row's chain of loads is short then), up to four for many (fewer
// threads meet in the reduction).
template <typename TX, typename TR, typename TY, bool RESIDUAL>
static int32_t sized_norm(const NormParams &p, int64_t rows, bool normalize, cudaStream_t stream) {
  const int nvec = (int)(p.cols / 8);
  int sms = 0;
  B200_CUDA_TRY(device_sms(&sms));
  int v = nvec > 2048 ? 4 : nvec > 1024 ? 2 : 1;
  if (rows > 2 * (int64_t)sms) v = nvec > 256 ? 4 : nvec > 128 ? 2 : 1;
  const int threads = ((nvec + v - 1) / v + 31) / 32 * 32;
  if (v == 4) return launch_norm<TX, TR, TY, 4, RESIDUAL>(p, rows, threads, normalize, stream);
  if (v == 2) return launch_norm<TX, TR, TY, 2, RESIDUAL>(p, rows, threads, normalize, stream);
  return launch_norm<TX, TR, TY, 1, RESIDUAL>(p, rows, threads, normalize, stream);
}

template <typename T>
static int32_t typed_norm(const NormParams &p, int64_t rows, int ydt, bool normalize, cudaStream_t stream) {
  const bool res = p.residual != nullptr;
  if (ydt == B200_DT_F8E4M3)
    return res ? sized_norm<T, T, E4M3, true>(p, rows, normalize, stream) : sized_norm<T, T, E4M3, false>(p, rows, normalize, stream);
  return res ? sized_norm<T, T, T, true>(p, rows, normalize, stream) : sized_norm<T, T, T, false>(p, rows, normalize, stream);
}

// 16 codes a thread. The product of a code and a power of two is exact but for what `dtype` cannot hold.
__global__ void __launch_bounds__(256) values_kernel(const uint8_t *codes, const uint8_t *scales, void *out, int dt, int64_t n16) {
  follow();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256) {
    const uint4 u = reinterpret_cast<const uint4 *>(codes)[i];
    const float s = e8m0_to_f32(scales[i >> 1]);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float f[2][8];
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j >> 3][j & 7] = code_value((uint8_t)(w[j >> 2] >> (8 * (j & 3)))) * s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (dt == B200_DT_F32) pack8((float *)out + 16 * i + 8 * h, f[h]);
      else if (dt == B200_DT_F16) pack8((__half *)out + 16 * i + 8 * h, f[h]);
      else pack8((__nv_bfloat16 *)out + 16 * i + 8 * h, f[h]);
    }
  }
}

// fp32 x into a 16-bit residual: a projection's partial sums into the stream.
template <typename TR>
static int32_t mixed_norm(const NormParams &p, int64_t rows, int ydt, bool normalize, cudaStream_t stream) {
  return ydt == B200_DT_F8E4M3 ? sized_norm<float, TR, E4M3, true>(p, rows, normalize, stream)
                               : sized_norm<float, TR, TR, true>(p, rows, normalize, stream);
}

static bool real(int dt) { return dt == B200_DT_F16 || dt == B200_DT_BF16 || dt == B200_DT_F32; }
static bool aligned(const void *p, int64_t stride, int64_t rows, int dt) {
  return (uintptr_t)p % 16 == 0 && (rows <= 1 || stride * dt_size(dt) % 16 == 0);
}

}  // namespace rows8
}  // namespace b200

using namespace b200;
using namespace b200::rows8;

extern "C" {

int32_t b200_rms_norm(const b200_norm_args *a, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (a == nullptr || a->rows < 0 || a->cols < 0) return b200_set_error(B200_ERR_INVALID, "rms_norm: null or negative arguments");
  const bool eight = a->y_dtype == B200_DT_F8E4M3;
  if (!real(a->x_dtype) || (!eight && !real(a->y_dtype)) || (a->residual != nullptr && !real(a->total_dtype)) ||
      (a->weight != nullptr && !real(a->weight_dtype)))
    return b200_set_error(B200_ERR_INVALID, "rms_norm: float16, bfloat16 or float32 operands, and fp8e4m3 results");
  if (eight && a->cols % 32 != 0) return b200_set_error(B200_ERR_INVALID, "rms_norm: 8-bit rows are whole blocks of 32");
  if (a->rows == 0 || a->cols == 0) return B200_OK;
  if (a->x == nullptr || a->y == nullptr || (eight && a->y_scales == nullptr) || (a->residual != nullptr && a->total == nullptr))
    return b200_set_error(B200_ERR_INVALID, "rms_norm: null pointer");
  if (a->rows > 0x7FFFFFFF) return b200_set_error(B200_ERR_UNSUPPORTED, "rms_norm: more than 2^31 - 1 rows");
  NormParams p{a->x, a->residual, a->normalize ? a->weight : nullptr, a->total, a->y, (uint8_t *)a->y_scales,
               a->cols, a->x_stride, a->residual_stride, a->total_stride, a->weight_dtype, a->eps};
  const bool res = a->residual != nullptr;
  // rows in registers: one type throughout (or fp32 x beside a 16-bit stream), whole vectors, at most 32768 values
  const int tdt = res ? a->total_dtype : a->x_dtype;
  const bool mixed = tdt != a->x_dtype;
  const bool fits = a->cols % 8 == 0 && a->cols <= 32768 && aligned(a->x, a->x_stride, a->rows, a->x_dtype) &&
                    (!mixed || a->x_dtype == B200_DT_F32) &&
                    (!res || (aligned(a->residual, a->residual_stride, a->rows, tdt) && aligned(a->total, a->total_stride, a->rows, tdt))) &&
                    (p.weight == nullptr || (uintptr_t)p.weight % 16 == 0) &&
                    (eight ? (uintptr_t)a->y % 8 == 0 : a->y_dtype == tdt && (uintptr_t)a->y % 16 == 0);
  cudaStream_t s = (cudaStream_t)stream;
  if (fits) {
    if (mixed) return tdt == B200_DT_F16 ? mixed_norm<__half>(p, a->rows, a->y_dtype, a->normalize != 0, s)
                                         : mixed_norm<__nv_bfloat16>(p, a->rows, a->y_dtype, a->normalize != 0, s);
    if (a->x_dtype == B200_DT_F32) return typed_norm<float>(p, a->rows, a->y_dtype, a->normalize != 0, s);
    if (a->x_dtype == B200_DT_F16) return typed_norm<__half>(p, a->rows, a->y_dtype, a->normalize != 0, s);
    return typed_norm<__nv_bfloat16>(p, a->rows, a->y_dtype, a->normalize != 0, s);
  }
  B200_CUDA_TRY(launch(norm_general_kernel, a->rows, 256, s, p, (int)a->x_dtype, (int)a->total_dtype, (int)a->y_dtype, (int)a->normalize));
  return B200_OK;
}

int32_t b200_scaled_values(const void *codes, const void *scales, int64_t rows, int64_t cols, void *out, int32_t dtype,
                           void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (rows < 0 || cols < 0 || cols % 32 != 0 || !real(dtype))
    return b200_set_error(B200_ERR_INVALID, "scaled_values: rows of whole blocks of 32, as float16, bfloat16 or float32");
  if (rows == 0 || cols == 0) return B200_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr || (uintptr_t)codes % 16 != 0 || (uintptr_t)out % 16 != 0)
    return b200_set_error(B200_ERR_INVALID, "scaled_values: null or unaligned pointer");
  const int64_t n16 = rows * cols / 16;
  const int64_t ctas = (n16 + 255) / 256;
  int sms = 0;
  B200_CUDA_TRY(device_sms(&sms));
  B200_CUDA_TRY(launch(values_kernel, ctas < 64 * sms ? ctas : 64 * sms, 256, (cudaStream_t)stream, (const uint8_t *)codes,
                       (const uint8_t *)scales, out, (int)dtype, n16));
  return B200_OK;
}

}  // extern "C"
