// cache_ops.cu -- rotary positions, and the packed key/value cache's writing and reading back.
//
// All three move each value once and compute little: their floor is HBM bandwidth for prompts and
// the launch for single tokens. Rotary is at 90 % of it; writing and reading back wait for chains of
// loads (a token's slot, position, angles and rows, then its codes) that the warps of an SM do not cover.
// The reference has no attention; these feed cache_attn.cu. Measured (device time): rotary over 8192 x 64
// heads of 128 bf16 values 46 us = 5.9 TB/s, one token 2.1 us; 32768 tokens of 8 + 8 heads and 32 query
// heads turned and written as fp8 and read back, 209 us of a floor of 146; 1999 tokens of 64 query heads
// with FP4 blocks 26 us of 13; 16 tokens 5.2 us.
#include "cache.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace b200 {

int32_t cache_ops_device_error(unsigned int *v, bool clear) {
  B200_CUDA_TRY(tu_device_error(v, clear));
  return B200_OK;
}

namespace cache {

__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

__device__ __forceinline__ int64_t load_index(const void *p, int64_t i, bool wide) {
  return wide ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// N consecutive values as fp32; `vec` says that the address is a multiple of their size.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T *p, bool vec, float (&f)[N]) {
  T t[N];
  if (vec) {
    if constexpr (sizeof(T) * N >= 16) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * N / 16; ++i)
        reinterpret_cast<uint4 *>(t)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = p[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)t[i];
}
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <typename T, int N>
__device__ __forceinline__ void store_n(T *p, bool vec, const float (&f)[N]) {
  alignas(16) T t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = from_f32<T>(f[i]);
  if (vec) {
    if constexpr (sizeof(T) * N >= 16) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * N / 16; ++i)
        reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(t)[i];
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = t[i];
}

// 16 bytes of T as fp32, and back.
template <typename T, int N>
__device__ __forceinline__ void widen_raw(const uint4 &r, float (&f)[N]) {
  const T *t = reinterpret_cast<const T *>(&r);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)t[i];
}
template <typename T, int N>
__device__ __forceinline__ uint4 narrow_raw(const float (&f)[N]) {
  uint4 r;
  if constexpr (sizeof(T) == 4) {
    r = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    alignas(16) T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = from_f32<T>(f[i]);
    r = *reinterpret_cast<const uint4 *>(t);
  }
  return r;
}

// ---- rotary positions ----------------------------------------------------------------------------
// Pair (a, b) of a head becomes (a cos - b sin, b cos + a sin), the transposed map (the gradient)
// takes -sin. Products and sums are rounded one by one (no contraction): the same bits as the
// formula in fp32. HBM-bound: each value is read and written once, 16 bytes a lane, and a thread
// keeps its angles for HPT heads, so that the tables (L2) are read HPT times less often.
struct RotaryArgs {
  const void *x;
  void *y;
  int64_t xsb, xst, xsh, ysb, yst, ysh;
  uint32_t batch, tokens;
  int heads, dim, rot;
  const float *cos, *sin;
  int64_t rows;
  const void *pos;
  int pos_wide, interleaved;
  float sign;
  uint32_t hgroups, units, total;
};

__device__ __forceinline__ bool in_table(const RotaryArgs &a, int64_t p) {
  const bool ok = p >= 0 && p < a.rows;
  if (!ok) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
  return ok;
}

// A unit is two vectors of 16 bytes: the sides of VEC pairs (half layout), neighbours in the rotated
// part (interleaved), or two behind it, which pass unchanged: one path for all lanes of a warp.
template <typename T, bool INTER, int HPT>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  pdl_enter();
  constexpr int VEC = 16 / sizeof(T), NA = VEC;  // angles of a unit
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= a.total) return;
  const uint32_t hi = idx / a.units, u = idx - hi * a.units;
  const uint32_t tok = hi / a.hgroups, hg = hi - tok * a.hgroups;
  const uint32_t b = a.batch == 1 ? 0 : tok / a.tokens, t = tok - b * a.tokens;
  const int half = a.rot / 2, turned = half / VEC;
  const bool turn = (int)u < turned;
  const int rest = (a.dim - a.rot) / 2;
  const int d0 = INTER ? (int)u * 2 * VEC : turn ? (int)u * VEC : a.rot + ((int)u - turned) * VEC;
  const int d1 = INTER ? d0 + VEC : turn ? d0 + half : d0 + rest;
  const int h0 = (int)hg * HPT;
  const T *x = (const T *)a.x + b * a.xsb + t * a.xst + (int64_t)h0 * a.xsh;
  T *y = (T *)a.y + b * a.ysb + t * a.yst + (int64_t)h0 * a.ysh;
  uint4 r[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (h0 + i < a.heads) {
      r[i][0] = *reinterpret_cast<const uint4 *>(x + i * a.xsh + d0);
      r[i][1] = *reinterpret_cast<const uint4 *>(x + i * a.xsh + d1);
    }
  float c[NA], s[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) c[i] = s[i] = __uint_as_float(0x7FC00000u);
  if (turn) {
    const int64_t p = load_index(a.pos, tok, a.pos_wide);
    if (in_table(a, p)) {
      const float *ct = a.cos + p * half + (INTER ? d0 / 2 : d0), *st = a.sin + p * half + (INTER ? d0 / 2 : d0);
#pragma unroll
      for (int i = 0; i < NA / 4; ++i) {
        reinterpret_cast<float4 *>(c)[i] = __ldg(reinterpret_cast<const float4 *>(ct) + i);
        reinterpret_cast<float4 *>(s)[i] = __ldg(reinterpret_cast<const float4 *>(st) + i);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NA; ++i) s[i] *= a.sign;
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (h0 + i < a.heads) {
      if (turn) {
        float f[VEC], g[VEC], m[VEC], n[VEC];
        widen_raw<T, VEC>(r[i][0], f);
        widen_raw<T, VEC>(r[i][1], g);
        if constexpr (INTER) {
#pragma unroll
          for (int j = 0; j < VEC; j += 2) {
            const float c0 = c[j / 2], s0 = s[j / 2], c1 = c[VEC / 2 + j / 2], s1 = s[VEC / 2 + j / 2];
            m[j] = __fsub_rn(__fmul_rn(f[j], c0), __fmul_rn(f[j + 1], s0));
            m[j + 1] = __fadd_rn(__fmul_rn(f[j + 1], c0), __fmul_rn(f[j], s0));
            n[j] = __fsub_rn(__fmul_rn(g[j], c1), __fmul_rn(g[j + 1], s1));
            n[j + 1] = __fadd_rn(__fmul_rn(g[j + 1], c1), __fmul_rn(g[j], s1));
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            m[j] = __fsub_rn(__fmul_rn(f[j], c[j]), __fmul_rn(g[j], s[j]));
            n[j] = __fadd_rn(__fmul_rn(g[j], c[j]), __fmul_rn(f[j], s[j]));
          }
        }
        r[i][0] = narrow_raw<T, VEC>(m), r[i][1] = narrow_raw<T, VEC>(n);
      }
      *reinterpret_cast<uint4 *>(y + i * a.ysh + d0) = r[i][0];
      *reinterpret_cast<uint4 *>(y + i * a.ysh + d1) = r[i][1];
    }
}

// Any size and alignment: a thread a pair, or two values behind the rotated part.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const RotaryArgs a) {
  pdl_enter();
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= a.total) return;
  const uint32_t hi = idx / a.units, u = idx - hi * a.units;
  const uint32_t tok = hi / (uint32_t)a.heads, h = hi - tok * a.heads;
  const uint32_t b = tok / a.tokens, t = tok - b * a.tokens;
  const int half = a.rot / 2;
  const T *x = (const T *)a.x + b * a.xsb + t * a.xst + (int64_t)h * a.xsh;
  T *y = (T *)a.y + b * a.ysb + t * a.yst + (int64_t)h * a.ysh;
  if ((int)u >= half) {
    const int d = 2 * (int)u;
    y[d] = x[d];
    if (d + 1 < a.dim) y[d + 1] = x[d + 1];
    return;
  }
  const int d0 = a.interleaved ? 2 * (int)u : (int)u, d1 = a.interleaved ? d0 + 1 : d0 + half;
  const int64_t p = load_index(a.pos, tok, a.pos_wide);
  float c = __uint_as_float(0x7FC00000u), s = c;
  if (in_table(a, p)) c = a.cos[p * half + u], s = a.sin[p * half + u] * a.sign;
  const float f = (float)x[d0], g = (float)x[d1];
  y[d0] = from_f32<T>(__fsub_rn(__fmul_rn(f, c), __fmul_rn(g, s)));
  y[d1] = from_f32<T>(__fadd_rn(__fmul_rn(g, c), __fmul_rn(f, s)));
}

template <typename T>
static int32_t launch_rotary_dt(RotaryArgs a, int64_t batch, int64_t tokens, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  auto fits = [](const void *p, int64_t sb, int64_t st, int64_t sh) {
    return (uintptr_t)p % 16 == 0 && sb % VEC == 0 && st % VEC == 0 && sh % VEC == 0;
  };
  const bool vec = fits(a.x, a.xsb, a.xst, a.xsh) && fits(a.y, a.ysb, a.yst, a.ysh) && a.rot % (2 * VEC) == 0 &&
                   (a.dim - a.rot) % (2 * VEC) == 0 && (uintptr_t)a.cos % 16 == 0 && (uintptr_t)a.sin % 16 == 0 &&
                   (a.rot / 2) % 4 == 0;
  // Two heads a thread once that leaves every SM its 2048 threads. 64 heads, one and two a thread: 8192
  // tokens 51.3 and 45.4 us, 2048 15.2 and 14.5, 1200 8.6 and 8.2, 512 4.3 and 4.8.
  const bool wide = vec && batch * tokens * a.heads * (a.dim / (2 * VEC)) >= 148 * 2048 * 2;
  a.units = vec ? a.dim / (2 * VEC) : (a.dim + 1) / 2;
  a.hgroups = wide ? (a.heads + 1) / 2 : a.heads;
  const int64_t per_token = (int64_t)a.units * a.hgroups;
  if (per_token > (1 << 30)) return b200_set_error(B200_ERR_UNSUPPORTED, "rotary: a token of too many values");
  // launches of less than 2^31 threads: runs of whole batches, or of one batch's tokens
  const int64_t most = (1ll << 30) / per_token;
  const int64_t nt = tokens < most ? tokens : most, nb = tokens < most ? most / tokens : 1;
  const RotaryArgs all = a;
  const int64_t es = sizeof(T), ps = a.pos_wide ? 8 : 4;
  for (int64_t b = 0; b < batch; b += nb)
    for (int64_t t = 0; t < tokens; t += nt) {
      a.batch = (uint32_t)(batch - b < nb ? batch - b : nb);
      a.tokens = (uint32_t)(tokens - t < nt ? tokens - t : nt);
      a.x = (const uint8_t *)all.x + (b * a.xsb + t * a.xst) * es;
      a.y = (uint8_t *)all.y + (b * a.ysb + t * a.yst) * es;
      a.pos = (const uint8_t *)all.pos + (b * tokens + t) * ps;
      a.total = (uint32_t)(a.batch * (int64_t)a.tokens * per_token);
      const dim3 grid((a.total + 255) / 256), block(256);
      if (!vec) B200_CUDA_TRY(launch_pdl(rotary_any_kernel<T>, grid, block, stream, a));
      else if (a.interleaved && wide) B200_CUDA_TRY(launch_pdl(rotary_kernel<T, true, 2>, grid, block, stream, a));
      else if (a.interleaved) B200_CUDA_TRY(launch_pdl(rotary_kernel<T, true, 1>, grid, block, stream, a));
      else if (wide) B200_CUDA_TRY(launch_pdl(rotary_kernel<T, false, 2>, grid, block, stream, a));
      else B200_CUDA_TRY(launch_pdl(rotary_kernel<T, false, 1>, grid, block, stream, a));
    }
  return B200_OK;
}

// ---- writing -------------------------------------------------------------------------------------
// One lane holds 8 values of a row (a head of a token), dim / 8 lanes a row; block maxima travel by
// shuffles. A CTA works on one token: its lanes load their angles once and go over the token's
// query, key and value heads, four rows in flight.
struct WriteArgs {
  b200_cache_desc c;
  const void *q, *k, *v;
  void *q_out;
  int64_t qst, qsh, kst, ksh, vst, vsh;
  int64_t tokens;
  int q_heads;
  const void *slots;
  int slots_wide;
  const float *cos, *sin;
  int64_t rows;
  int rot, interleaved;
  const void *pos;
  int pos_wide;
  int qvec, kvec, vvec, tvec, page_shift;
};

template <int F>
__device__ __forceinline__ void encode8(const float (&x)[8], float inv, uint8_t *dst) {
  if constexpr (F == B200_CACHE_INT8) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = max(-127, min(127, __float2int_rn(__fmul_rn(x[i], inv))));
      w[i / 4] |= ((uint32_t)n & 0xFFu) << (8 * (i % 4));
    }
    *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
  } else if constexpr (F == B200_CACHE_FP8E4M3) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[4 * i], inv), __fmul_rn(x[4 * i + 1], inv)),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[4 * i + 2], inv), __fmul_rn(x[4 * i + 3], inv)),
                                                   __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
  } else if constexpr (F == B200_CACHE_INT4) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = max(-7, min(7, __float2int_rn(__fmul_rn(x[i], inv))));
      w |= ((uint32_t)n & 0xFu) << (4 * i);
    }
    *reinterpret_cast<uint32_t *>(dst) = w;
  } else {
    uint32_t w;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(x[i], inv);
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    *reinterpret_cast<uint32_t *>(dst) = w;
  }
}

// A block's scale from its largest magnitude, stored at `at` when `writes`.
template <int F>
__device__ __forceinline__ float block_scale(float top, bool e8m0, void *scales, int64_t at, bool writes) {
  constexpr float lo = 0x1p-100f, hi = 0x1p100f;
  const float r = __fmul_rn(top, (float)(1.0 / CFmt<F>::qmax));
  if (e8m0) {
    uint32_t e = (__float_as_uint(r) + 0x7FFFFFu) >> 23;
    e = r != r ? 255u : min(227u, max(27u, e));
    if (writes) ((uint8_t *)scales)[at] = (uint8_t)e;
    return e == 255u ? r : __uint_as_float(e << 23);
  }
  float sc = __bfloat162float(__float2bfloat16_rn(r));
  sc = sc < lo ? lo : sc > hi ? hi : sc;
  if (writes) ((__nv_bfloat16 *)scales)[at] = __float2bfloat16_rn(sc);
  return sc;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN above all
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
template <int F>
__device__ __forceinline__ void encode8_scaled(float (&y)[8], float sc, uint8_t *codes) {
  // under a NaN scale codes are zeros: in attention the NaN then reaches only rows that see the key
  if (sc != sc)
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = 0.f;
  encode8<F>(y, __frcp_rn(sc != sc ? 1.f : sc), codes);
}

// The usual shapes of 16-bit inputs: a lane holds the two vectors of 8 values that turn together (or
// two that pass), dim / 16 lanes a row, so that every value is read once; two rows in flight a lane and 8
// CTAs an SM (one CTA a token spends its time in the chain position -> angles -> store). INTER:
// interleaved pairs, or none to turn (cos null).
constexpr int PT = 128, PR = 2;
template <typename T, int F, int D, bool INTER>
__global__ void __launch_bounds__(PT, 8) cache_write_pairs_kernel(const WriteArgs a) {
  pdl_enter();
  constexpr int LPR = D / 16, RPC = PT / LPR;
  const int j = threadIdx.x % LPR, slot_row = threadIdx.x / LPR, step = RPC * gridDim.y;
  const int kvh = a.c.kv_heads, total = a.q_heads + 2 * kvh, half = a.rot / 2;
  const uint32_t t = blockIdx.x;
  const int turned = INTER ? LPR : half / 8;
  const bool mine = INTER || j < turned;
  const int d0 = INTER || j < turned ? j * 8 : a.rot + (j - turned) * 8;
  const int d1 = INTER ? d0 + D / 2 : mine ? d0 + half : d0 + (D - a.rot) / 2;
  const int64_t slot = load_index(a.slots, t, a.slots_wide);
  const int64_t cells = a.c.pages << a.page_shift;
  if (slot >= cells && threadIdx.x == 0) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
  const bool place = slot >= 0 && slot < cells;
  const int64_t page = place ? slot >> a.page_shift : 0, offset = place ? slot & ((1 << a.page_shift) - 1) : 0;
  const int64_t code0 = page * a.c.strides[0] + offset * a.c.strides[2];
  const int64_t scale0 = page * a.c.scale_strides[0] + offset * a.c.scale_strides[2];
  const bool e8 = a.c.scale_dtype == B200_DT_E8M0;
  const int blk = a.c.block_size, lanes = blk == D ? LPR : 4;
  float c[8], s[8];  // half layout: of the pairs; interleaved: 4 of the first vector, 4 of the second
  const bool turn0 = a.cos != nullptr && (INTER ? d0 < a.rot : mine), turn1 = a.cos != nullptr && (INTER ? d1 < a.rot : mine);
  const int r_first = slot_row + blockIdx.y * RPC;
  for (int r0 = r_first; r0 - slot_row % (32 / LPR) < total; r0 += PR * step) {  // uniform in a warp
    uint4 x[PR][2];
#pragma unroll
    for (int i = 0; i < PR; ++i) {
      const int r = r0 + i * step;
      if (r < total) {
        const T *src = r < a.q_heads ? (const T *)a.q + t * a.qst + r * a.qsh
                       : r < a.q_heads + kvh ? (const T *)a.k + t * a.kst + (r - a.q_heads) * a.ksh
                                             : (const T *)a.v + t * a.vst + (r - a.q_heads - kvh) * a.vsh;
        x[i][0] = *reinterpret_cast<const uint4 *>(src + d0);
        x[i][1] = *reinterpret_cast<const uint4 *>(src + d1);
      }
    }
    if (r0 == r_first && a.cos != nullptr) {  // once, behind the first rows' loads
      const int64_t p = load_index(a.pos, t, a.pos_wide);
      const bool ok = p >= 0 && p < a.rows;
      if (!ok && threadIdx.x == 0) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __uint_as_float(0x7FC00000u);
      const float *ct = a.cos + p * half, *st = a.sin + p * half;
      if (ok && turn0) {
        const int at = INTER ? d0 / 2 : d0;
        reinterpret_cast<float4 *>(c)[0] = __ldg((const float4 *)(ct + at));
        reinterpret_cast<float4 *>(s)[0] = __ldg((const float4 *)(st + at));
      }
      if (ok && turn1) {
        const int at = INTER ? d1 / 2 : d0 + 4;
        reinterpret_cast<float4 *>(c)[1] = __ldg((const float4 *)(ct + at));
        reinterpret_cast<float4 *>(s)[1] = __ldg((const float4 *)(st + at));
      }
    }
#pragma unroll
    for (int i = 0; i < PR; ++i) {
      const int r = r0 + i * step;
      if (r - slot_row % (32 / LPR) >= total) break;  // the whole warp is done
      const bool in = r < total, isq = r < a.q_heads, isk = r < a.q_heads + kvh;
      float f[8], g[8];
      widen_raw<T, 8>(x[i][0], f);
      widen_raw<T, 8>(x[i][1], g);
      if (isk) {
        if constexpr (INTER) {
          if (turn0)
#pragma unroll
            for (int y = 0; y < 8; y += 2) {
              const float m = f[y], n = f[y + 1];
              f[y] = __fsub_rn(__fmul_rn(m, c[y / 2]), __fmul_rn(n, s[y / 2]));
              f[y + 1] = __fadd_rn(__fmul_rn(n, c[y / 2]), __fmul_rn(m, s[y / 2]));
            }
          if (turn1)
#pragma unroll
            for (int y = 0; y < 8; y += 2) {
              const float m = g[y], n = g[y + 1];
              g[y] = __fsub_rn(__fmul_rn(m, c[4 + y / 2]), __fmul_rn(n, s[4 + y / 2]));
              g[y + 1] = __fadd_rn(__fmul_rn(n, c[4 + y / 2]), __fmul_rn(m, s[4 + y / 2]));
            }
        } else if (turn0) {
#pragma unroll
          for (int y = 0; y < 8; ++y) {
            const float m = f[y], n = g[y];
            f[y] = __fsub_rn(__fmul_rn(m, c[y]), __fmul_rn(n, s[y]));
            g[y] = __fadd_rn(__fmul_rn(n, c[y]), __fmul_rn(m, s[y]));
          }
        }
      }
      if (isq) {
        T *dst = (T *)a.q_out + ((int64_t)t * a.q_heads + r) * D;
        *reinterpret_cast<uint4 *>(dst + d0) = narrow_raw<T, 8>(f);
        *reinterpret_cast<uint4 *>(dst + d1) = narrow_raw<T, 8>(g);
      }
      if (__all_sync(0xFFFFFFFFu, isq)) continue;
      float tf = 0.f, tg = 0.f;
#pragma unroll
      for (int y = 0; y < 8; ++y) tf = max_nan(tf, fabsf(f[y])), tg = max_nan(tg, fabsf(g[y]));
      if (blk == D) tf = tg = max_nan(tf, tg);
      for (int m = 1; m < lanes; m <<= 1) {
        tf = max_nan(tf, __shfl_xor_sync(0xFFFFFFFFu, tf, m));
        if (blk != D) tg = max_nan(tg, __shfl_xor_sync(0xFFFFFFFFu, tg, m));
      }
      if (!in || isq || !place) continue;
      const int h = isk ? r - a.q_heads : r - a.q_heads - kvh;
      void *scales = isk ? a.c.k_scales : a.c.v_scales;
      uint8_t *codes = (uint8_t *)(isk ? a.c.k : a.c.v) + code0 + h * a.c.strides[1];
      const int64_t at = scale0 + h * a.c.scale_strides[1];
      const float sf = block_scale<F>(tf, e8, scales, at + d0 / blk, d0 % blk == 0);
      const float sg = blk == D ? sf : block_scale<F>(tg, e8, scales, at + d1 / blk, d1 % blk == 0);
      encode8_scaled<F>(f, sf, codes + d0 * CFmt<F>::bits / 8);
      encode8_scaled<F>(g, sg, codes + d1 * CFmt<F>::bits / 8);
    }
  }
}

constexpr int WT = 256, WR = 4;  // threads of a CTA, rows in flight per lane

template <typename T, int F, int D>
__global__ void __launch_bounds__(WT) cache_write_kernel(WriteArgs a) {
  pdl_enter();
  constexpr int LPR = D / 8, RPC = WT / LPR;  // lanes a row, rows of a CTA at a time
  const int lane_d = (threadIdx.x % LPR) * 8, row0 = threadIdx.x / LPR + blockIdx.y * RPC, step = RPC * gridDim.y;
  const int64_t t = blockIdx.x;
  const int kvh = a.c.kv_heads, total = a.q_heads + 2 * kvh;
  const int64_t slot = load_index(a.slots, t, a.slots_wide);
  const int64_t cells = a.c.pages * a.c.page_size;
  if (slot >= cells && threadIdx.x == 0) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
  const bool place = slot >= 0 && slot < cells;
  const int64_t page = place ? slot >> a.page_shift : 0, offset = place ? slot - (page << a.page_shift) : 0;
  const int half = a.rot / 2;
  const bool turns = a.cos != nullptr;
  // the angles of this lane's values, and which way the other of a pair lies: half layout
  float c[8], s[8];
  if (turns) {
    const int64_t p = load_index(a.pos, t, a.pos_wide);
    const bool ok = p >= 0 && p < a.rows;
    if (!ok && threadIdx.x == 0) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
    const float *ct = a.cos + p * half, *st = a.sin + p * half;
    if (!a.interleaved && a.tvec && ok && lane_d < a.rot) {
      const int i0 = lane_d < half ? lane_d : lane_d - half;
      load_n<float, 8>(ct + i0, true, c);
      load_n<float, 8>(st + i0, true, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = lane_d < half ? -s[i] : s[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane_d + i;
        const int at = a.interleaved ? d >> 1 : d < half ? d : d - half;
        const bool first = a.interleaved ? (d & 1) == 0 : d < half;
        c[i] = d < a.rot ? (ok ? ct[at] : __uint_as_float(0x7FC00000u)) : 1.f;
        s[i] = d < a.rot ? (ok ? (first ? -st[at] : st[at]) : __uint_as_float(0x7FC00000u)) : 0.f;
      }
    }
  }
  for (int r0 = row0 - (threadIdx.x / LPR) % (32 / LPR); r0 < total; r0 += WR * step) {  // uniform in a warp
    float x[WR][8], o[WR][8];
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const int r = r0 + (threadIdx.x / LPR) % (32 / LPR) + i * step;
      if (r < total) {
        const bool isq = r < a.q_heads, isk = r < a.q_heads + kvh;
        const int h = isq ? r : isk ? r - a.q_heads : r - a.q_heads - kvh;
        const T *src = isq ? (const T *)a.q + t * a.qst + h * a.qsh
                           : isk ? (const T *)a.k + t * a.kst + h * a.ksh : (const T *)a.v + t * a.vst + h * a.vsh;
        const bool vec = isq ? a.qvec : isk ? a.kvec : a.vvec;
        load_n<T, 8>(src + lane_d, vec, x[i]);
        if (turns && isk && !a.interleaved) {
          if (a.tvec) {
            if (lane_d < a.rot) load_n<T, 8>(src + (lane_d < half ? lane_d + half : lane_d - half), vec, o[i]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int d = lane_d + j;
              o[i][j] = d < a.rot ? (float)src[d < half ? d + half : d - half] : 0.f;
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const int r = r0 + (threadIdx.x / LPR) % (32 / LPR) + i * step;
      if (r0 + i * step >= total) break;  // the whole warp is done
      const bool in = r < total, isq = r < a.q_heads, isk = r < a.q_heads + kvh;
      float y[8];
      if (!in) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = 0.f;
      } else if (turns && isk) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = a.interleaved ? x[i][j ^ 1] : o[i][j];
          // x cos + other (+-sin), each operation rounded
          y[j] = lane_d + j < a.rot ? __fadd_rn(__fmul_rn(x[i][j], c[j]), __fmul_rn(other, s[j])) : x[i][j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[i][j];
      }
      if (in && isq) store_n<T, 8>((T *)a.q_out + (t * a.q_heads + r) * D + lane_d, true, y);
      uint32_t top = 0;  // magnitudes order as integers, NaN above all
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(y[j]) & 0x7FFFFFFFu);
      const int lanes = a.c.block_size / 8;
      for (int m = 1; m < lanes; m <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, m));
      if (in && !isq && place) {
        const int h = isk ? r - a.q_heads : r - a.q_heads - kvh;
        const int64_t at = scale_row(a.c, page, h, offset) + lane_d / a.c.block_size;
        const float sc = block_scale<F>(__uint_as_float(top), a.c.scale_dtype == B200_DT_E8M0,
                                        isk ? a.c.k_scales : a.c.v_scales, at, lane_d % a.c.block_size == 0);
        encode8_scaled<F>(y, sc, (uint8_t *)(isk ? a.c.k : a.c.v) + code_row(a.c, page, h, offset) +
                                     lane_d * CFmt<F>::bits / 8);
      }
    }
  }
}

template <typename T, int F, int D>
static int32_t launch_write_d(const WriteArgs &a, cudaStream_t stream) {
  const int rows = a.q_heads + 2 * a.c.kv_heads;
  // Few tokens: a CTA for every run of rows; many: one a token, its angles loaded once. Written and read
  // back, 64 query heads, FP4 blocks: 16 tokens 5.0 and 6.9 us, 592 11.6 and 12.2, 740 13.7 and 13.4, 1999
  // 30.3 and 25.5; 32 heads, fp8: 592 9.1 and 9.3, 740 10.0 and 9.9, 32768 305 and 209.
  const bool many = a.tokens >= 148 * 5;
  if constexpr (sizeof(T) == 2) {
    const int blk = a.c.block_size, rest = D - a.rot;
    const bool inter = a.cos == nullptr || a.interleaved;
    const bool pairs = (a.q_heads == 0 || a.qvec) && a.kvec && a.vvec &&
                       (a.cos == nullptr || (a.tvec && (inter ? a.rot % 8 == 0 : (rest / 2) % 8 == 0))) &&
                       (inter || blk == D || ((a.rot / 2) % 32 == 0 && (rest / 2) % 32 == 0));
    if (pairs) {
      const int rpc = PT / (D / 16);
      const dim3 grid((unsigned)a.tokens, (unsigned)(many ? 1 : (rows + rpc - 1) / rpc));
      if (inter) B200_CUDA_TRY(launch_pdl(cache_write_pairs_kernel<T, F, D, true>, grid, dim3(PT), stream, a));
      else B200_CUDA_TRY(launch_pdl(cache_write_pairs_kernel<T, F, D, false>, grid, dim3(PT), stream, a));
      return B200_OK;
    }
  }
  const int rpc = WT / (D / 8);
  const dim3 grid((unsigned)a.tokens, (unsigned)(many ? 1 : (rows + rpc - 1) / rpc));
  B200_CUDA_TRY(launch_pdl(cache_write_kernel<T, F, D>, grid, dim3(WT), stream, a));
  return B200_OK;
}
template <typename T, int F>
static int32_t launch_write_t(const WriteArgs &a, cudaStream_t stream) {
  return a.c.head_dim == 64 ? launch_write_d<T, F, 64>(a, stream)
         : a.c.head_dim == 128 ? launch_write_d<T, F, 128>(a, stream) : launch_write_d<T, F, 256>(a, stream);
}
template <typename T>
static int32_t launch_write_f(const WriteArgs &a, cudaStream_t stream) {
  switch (a.c.format) {
    case B200_CACHE_INT8: return launch_write_t<T, B200_CACHE_INT8>(a, stream);
    case B200_CACHE_FP8E4M3: return launch_write_t<T, B200_CACHE_FP8E4M3>(a, stream);
    case B200_CACHE_INT4: return launch_write_t<T, B200_CACHE_INT4>(a, stream);
    default: return launch_write_t<T, B200_CACHE_FP4_E2M1>(a, stream);
  }
}

// ---- reading back --------------------------------------------------------------------------------
// out[t, h, :] = codes * scale of slot t, one fp32 product rounded to the output type; a thread
// gives 16 values of the key and of the value. A negative slot reads zeros.
struct ReadArgs {
  b200_cache_desc c;
  const void *slots;
  int slots_wide, page_shift;
  uint32_t total;
  void *k_out, *v_out;
};

// 8 * W codes as fp32, W = 1 or 2 words of 4-bit codes, 2 of 8-bit.
template <int F>
__device__ __forceinline__ void decode16(const uint32_t (&w)[CFmt<F>::bits / 2], float (&f)[16]) {
  uint32_t p[8];
  if constexpr (CFmt<F>::bits == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) decode4_8bit<F>(w[i], p[2 * i], p[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) decode8_4<F>(w[i], reinterpret_cast<uint32_t(&)[4]>(p[4 * i]));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&p[i]));
    if constexpr (F == B200_CACHE_INT4) f[8 * (i / 4) + i % 4] = v.x, f[8 * (i / 4) + i % 4 + 4] = v.y;
    else f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}

template <typename T, int F, int D>
__global__ void __launch_bounds__(256) cache_read_kernel(const ReadArgs a) {
  pdl_enter();
  constexpr int LPR = D / 16, W = CFmt<F>::bits / 2;  // lanes of a row, words of 16 codes
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= a.total) return;
  const int d = (int)(idx % LPR) * 16;
  const uint32_t hi = idx / LPR, kvh = a.c.kv_heads, t = hi / kvh, h = hi - t * kvh;
  const int64_t slot = load_index(a.slots, t, a.slots_wide);
  const int64_t cells = a.c.pages << a.page_shift;
  if (slot >= cells) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
  float k[16], v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) k[i] = v[i] = 0.f;
  if (slot >= 0 && slot < cells) {
    const int64_t page = slot >> a.page_shift, offset = slot - (page << a.page_shift);
    const int64_t at = scale_row(a.c, page, h, offset) + d / a.c.block_size;
    const int64_t cd = code_row(a.c, page, h, offset) + d * CFmt<F>::bits / 8;
    uint32_t wk[W], wv[W];
    if constexpr (W == 4) {
      *reinterpret_cast<uint4 *>(wk) = *reinterpret_cast<const uint4 *>((const uint8_t *)a.c.k + cd);
      *reinterpret_cast<uint4 *>(wv) = *reinterpret_cast<const uint4 *>((const uint8_t *)a.c.v + cd);
    } else {
      *reinterpret_cast<uint2 *>(wk) = *reinterpret_cast<const uint2 *>((const uint8_t *)a.c.k + cd);
      *reinterpret_cast<uint2 *>(wv) = *reinterpret_cast<const uint2 *>((const uint8_t *)a.c.v + cd);
    }
    const bool e8 = a.c.scale_dtype == B200_DT_E8M0;
    const float ks = scale_f32(a.c.k_scales, at, e8), vs = scale_f32(a.c.v_scales, at, e8);
    decode16<F>(wk, k);
    decode16<F>(wv, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) k[i] *= ks, v[i] *= vs;
  }
  const int64_t to = (int64_t)hi * D + d;
  store_n<T, 16>((T *)a.k_out + to, true, k);
  store_n<T, 16>((T *)a.v_out + to, true, v);
}

template <typename T, int F>
static int32_t launch_read_f(ReadArgs a, int64_t tokens, cudaStream_t stream) {
  // launches of less than 2^31 threads
  const int64_t per_token = (int64_t)a.c.kv_heads * (a.c.head_dim / 16), most = (1ll << 30) / per_token;
  const ReadArgs all = a;
  for (int64_t t = 0; t < tokens; t += most) {
    const int64_t n = tokens - t < most ? tokens - t : most, out = t * a.c.kv_heads * a.c.head_dim;
    a.slots = (const uint8_t *)all.slots + t * (a.slots_wide ? 8 : 4);
    a.k_out = (T *)all.k_out + out, a.v_out = (T *)all.v_out + out;
    a.total = (uint32_t)(n * per_token);
    const dim3 grid((a.total + 255) / 256), block(256);
    if (a.c.head_dim == 64) B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, F, 64>, grid, block, stream, a));
    else if (a.c.head_dim == 128) B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, F, 128>, grid, block, stream, a));
    else B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, F, 256>, grid, block, stream, a));
  }
  return B200_OK;
}
template <typename T>
static int32_t launch_read_t(const ReadArgs &a, int64_t tokens, cudaStream_t stream) {
  switch (a.c.format) {
    case B200_CACHE_INT8: return launch_read_f<T, B200_CACHE_INT8>(a, tokens, stream);
    case B200_CACHE_FP8E4M3: return launch_read_f<T, B200_CACHE_FP8E4M3>(a, tokens, stream);
    case B200_CACHE_INT4: return launch_read_f<T, B200_CACHE_INT4>(a, tokens, stream);
    default: return launch_read_f<T, B200_CACHE_FP4_E2M1>(a, tokens, stream);
  }
}

static bool bad_index_dtype(int dt) { return dt != B200_DT_I32 && dt != B200_DT_I64; }
static bool real_dtype(int dt) { return dt == B200_DT_F16 || dt == B200_DT_BF16 || dt == B200_DT_F32; }

}  // namespace cache

int32_t check_cache(const b200_cache_desc *c) {
  if (c == nullptr) return b200_set_error(B200_ERR_INVALID, "null cache descriptor");
  if (c->format < B200_CACHE_INT8 || c->format > B200_CACHE_FP4_E2M1)
    return b200_set_error(B200_ERR_INVALID, "unknown cache format %d", c->format);
  if (c->scale_dtype != B200_DT_BF16 && c->scale_dtype != B200_DT_E8M0)
    return b200_set_error(B200_ERR_INVALID, "cache scales must be bfloat16 or E8M0 (got dtype %d)", c->scale_dtype);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return b200_set_error(B200_ERR_INVALID, "cache head_dim must be 64, 128 or 256 (got %d)", c->head_dim);
  if (c->block_size != 32 && c->block_size != c->head_dim)
    return b200_set_error(B200_ERR_INVALID, "cache block_size must be 32 or head_dim (got %d)", c->block_size);
  if (c->page_size < 16 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)) != 0)
    return b200_set_error(B200_ERR_INVALID, "cache page_size must be a power of two from 16 (got %d)", c->page_size);
  if (c->pages < 0 || c->kv_heads < 1 || c->kv_heads > 65535)
    return b200_set_error(B200_ERR_INVALID, "cache needs pages >= 0 and 1..65535 kv_heads");
  if (c->pages > INT32_MAX) return b200_set_error(B200_ERR_INVALID, "cache has more pages than int32 tables can name");
  if (c->pages > 0) {
    if (c->k == nullptr || c->v == nullptr || c->k_scales == nullptr || c->v_scales == nullptr)
      return b200_set_error(B200_ERR_INVALID, "null cache storage");
    for (int i = 0; i < 3; ++i)
      if (c->strides[i] < 0 || c->scale_strides[i] < 0)
        return b200_set_error(B200_ERR_INVALID, "cache strides must not be negative");
    constexpr int64_t most = 1ll << 30;
    if (c->strides[0] > most || c->scale_strides[0] > most || c->strides[2] > most / c->page_size ||
        c->scale_strides[2] > most / c->page_size)
      return b200_set_error(B200_ERR_UNSUPPORTED, "cache pages of more than 2^30 bytes, or as far apart");
    for (int i = 0; i < 3; ++i)
      if (c->strides[i] % 16) return b200_set_error(B200_ERR_INVALID, "cache strides must be multiples of 16 bytes");
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || (uintptr_t)c->k_scales % 16 || (uintptr_t)c->v_scales % 16)
      return b200_set_error(B200_ERR_INVALID, "cache storage must start on 16-byte boundaries");
  }
  return B200_OK;
}

int32_t launch_rotary(const void *x, int32_t dtype, int64_t batch, int64_t tokens, int32_t heads, int32_t head_dim,
                      const int64_t *xs, void *y, const int64_t *ys, const b200_rotary_desc *r, const void *pos,
                      int32_t pos_dtype, int32_t transpose, cudaStream_t stream) {
  using namespace cache;
  RotaryArgs a = {};
  a.x = x, a.y = y;
  a.xsb = xs[0], a.xst = xs[1], a.xsh = xs[2], a.ysb = ys[0], a.yst = ys[1], a.ysh = ys[2];
  a.heads = heads, a.dim = head_dim, a.rot = r->rotary_dim;
  a.cos = r->cos, a.sin = r->sin, a.rows = r->rows, a.pos = pos;
  a.pos_wide = pos_dtype == B200_DT_I64, a.interleaved = r->interleaved, a.sign = transpose ? -1.f : 1.f;
  switch (dtype) {
    case B200_DT_F16: return launch_rotary_dt<__half>(a, batch, tokens, stream);
    case B200_DT_BF16: return launch_rotary_dt<__nv_bfloat16>(a, batch, tokens, stream);
    default: return launch_rotary_dt<float>(a, batch, tokens, stream);
  }
}

int32_t check_rotary(const b200_rotary_desc *r, int32_t head_dim, const void *pos, int32_t pos_dtype) {
  if (r == nullptr || r->cos == nullptr || r->sin == nullptr || pos == nullptr)
    return b200_set_error(B200_ERR_INVALID, "rotary: null table or positions");
  if (r->rows < 0 || r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > head_dim)
    return b200_set_error(B200_ERR_INVALID, "rotary: rotary_dim must be even and at most head_dim (got %d of %d)",
                          r->rotary_dim, head_dim);
  if (cache::bad_index_dtype(pos_dtype)) return b200_set_error(B200_ERR_INVALID, "rotary: positions must be int32 or int64");
  return B200_OK;
}

int32_t launch_cache_write(const b200_cache_desc *c, const void *k, const void *v, int32_t dtype, int64_t tokens,
                           const int64_t *ks, const int64_t *vs, const void *slots, int32_t slots_dtype,
                           const b200_rotary_desc *r, const void *pos, int32_t pos_dtype, const void *q,
                           int32_t q_heads, const int64_t *qs, void *q_out, cudaStream_t stream) {
  using namespace cache;
  if (tokens > INT32_MAX) return b200_set_error(B200_ERR_UNSUPPORTED, "cache_write: too many tokens for one launch");
  WriteArgs a = {};
  a.c = *c, a.k = k, a.v = v, a.q = q, a.q_out = q_out, a.tokens = tokens, a.q_heads = q != nullptr ? q_heads : 0;
  a.kst = ks[0], a.ksh = ks[1], a.vst = vs[0], a.vsh = vs[1];
  if (q != nullptr) a.qst = qs[0], a.qsh = qs[1];
  a.slots = slots, a.slots_wide = slots_dtype == B200_DT_I64;
  while ((1 << a.page_shift) < c->page_size) ++a.page_shift;
  if (r != nullptr) {
    a.cos = r->cos, a.sin = r->sin, a.rows = r->rows, a.rot = r->rotary_dim, a.interleaved = r->interleaved;
    a.pos = pos, a.pos_wide = pos_dtype == B200_DT_I64;
    a.tvec = (a.rot / 2) % 8 == 0 && (uintptr_t)a.cos % 16 == 0 && (uintptr_t)a.sin % 16 == 0;
  }
  auto fits = [](const void *p, int64_t st, int64_t sh) { return (uintptr_t)p % 16 == 0 && st % 8 == 0 && sh % 8 == 0; };
  a.qvec = fits(q, a.qst, a.qsh), a.kvec = fits(k, a.kst, a.ksh), a.vvec = fits(v, a.vst, a.vsh);
  switch (dtype) {
    case B200_DT_F16: return launch_write_f<__half>(a, stream);
    case B200_DT_BF16: return launch_write_f<__nv_bfloat16>(a, stream);
    default: return launch_write_f<float>(a, stream);
  }
}

int32_t launch_cache_read(const b200_cache_desc *c, const void *slots, int32_t slots_dtype, int64_t tokens, void *k_out,
                          void *v_out, int32_t dtype, cudaStream_t stream) {
  using namespace cache;
  ReadArgs a = {*c, slots, slots_dtype == B200_DT_I64, 0, 0, k_out, v_out};
  while ((1 << a.page_shift) < c->page_size) ++a.page_shift;
  switch (dtype) {
    case B200_DT_F16: return launch_read_t<__half>(a, tokens, stream);
    case B200_DT_BF16: return launch_read_t<__nv_bfloat16>(a, tokens, stream);
    default: return launch_read_t<float>(a, tokens, stream);
  }
}

}  // namespace b200

// ---- C entries ---------------------------------------------------------------------------------
using namespace b200;

extern "C" {

int32_t b200_rotary(const void *x, int32_t dtype, int64_t batch, int64_t tokens, int32_t heads, int32_t head_dim,
                    int64_t x_stride_b, int64_t x_stride_t, int64_t x_stride_h, void *y, int64_t y_stride_b,
                    int64_t y_stride_t, int64_t y_stride_h, const b200_rotary_desc *table, const void *positions,
                    int32_t positions_dtype, int32_t transpose, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (batch < 0 || tokens < 0 || heads < 0 || head_dim < 1)
    return b200_set_error(B200_ERR_INVALID, "rotary: bad sizes");
  if (!cache::real_dtype(dtype)) return b200_set_error(B200_ERR_INVALID, "rotary: unsupported dtype %d", dtype);
  if (batch == 0 || tokens == 0 || heads == 0) return B200_OK;
  if (int32_t rc = check_rotary(table, head_dim, positions, positions_dtype)) return rc;
  if (x == nullptr || y == nullptr) return b200_set_error(B200_ERR_INVALID, "rotary: null x or y");
  const int64_t xs[3] = {x_stride_b, x_stride_t, x_stride_h}, ys[3] = {y_stride_b, y_stride_t, y_stride_h};
  return launch_rotary(x, dtype, batch, tokens, heads, head_dim, xs, y, ys, table, positions,
                       positions_dtype, transpose, (cudaStream_t)stream);
}

int32_t b200_cache_write(const b200_cache_desc *c, const void *k, int64_t k_stride_t, int64_t k_stride_h, const void *v,
                         int64_t v_stride_t, int64_t v_stride_h, int32_t dtype, int64_t tokens, const void *slots,
                         int32_t slots_dtype, const b200_rotary_desc *table, const void *positions,
                         int32_t positions_dtype, const void *q, int32_t q_heads, int64_t q_stride_t, int64_t q_stride_h,
                         void *q_out, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (int32_t rc = check_cache(c)) return rc;
  if (tokens < 0 || (q != nullptr && (q_heads < 1 || q_heads > 65535)))
    return b200_set_error(B200_ERR_INVALID, "cache_write: bad sizes");
  if (!cache::real_dtype(dtype)) return b200_set_error(B200_ERR_INVALID, "cache_write: unsupported dtype %d", dtype);
  if (cache::bad_index_dtype(slots_dtype)) return b200_set_error(B200_ERR_INVALID, "cache_write: slots must be int32 or int64");
  if (tokens == 0) return B200_OK;
  if (table != nullptr)
    if (int32_t rc = check_rotary(table, c->head_dim, positions, positions_dtype)) return rc;
  if (k == nullptr || v == nullptr || slots == nullptr || (q != nullptr && q_out == nullptr))
    return b200_set_error(B200_ERR_INVALID, "cache_write: null pointer");
  if ((uintptr_t)q_out % 16) return b200_set_error(B200_ERR_INVALID, "cache_write: q_out must start on a 16-byte boundary");
  const int64_t ks[2] = {k_stride_t, k_stride_h}, vs[2] = {v_stride_t, v_stride_h}, qs[2] = {q_stride_t, q_stride_h};
  return launch_cache_write(c, k, v, dtype, tokens, ks, vs, slots, slots_dtype, table, positions, positions_dtype, q,
                            q_heads, qs, q_out, (cudaStream_t)stream);
}

int32_t b200_cache_read(const b200_cache_desc *c, const void *slots, int32_t slots_dtype, int64_t tokens, void *k_out,
                        void *v_out, int32_t dtype, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (int32_t rc = check_cache(c)) return rc;
  if (tokens < 0) return b200_set_error(B200_ERR_INVALID, "cache_read: negative tokens");
  if (!cache::real_dtype(dtype)) return b200_set_error(B200_ERR_INVALID, "cache_read: unsupported dtype %d", dtype);
  if (cache::bad_index_dtype(slots_dtype)) return b200_set_error(B200_ERR_INVALID, "cache_read: slots must be int32 or int64");
  if (tokens == 0) return B200_OK;
  if (slots == nullptr || k_out == nullptr || v_out == nullptr) return b200_set_error(B200_ERR_INVALID, "cache_read: null pointer");
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
    return b200_set_error(B200_ERR_INVALID, "cache_read: outputs must start on 16-byte boundaries");
  return launch_cache_read(c, slots, slots_dtype, tokens, k_out, v_out, dtype, (cudaStream_t)stream);
}

}  // extern "C"
