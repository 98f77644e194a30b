// cache_ops.cu -- rotary positions, and the packed key/value cache's writing and reading back.
//
// All three move each value once and compute little: their floor is HBM bandwidth for prompts and
// the launch for single tokens. The reference has no attention; these feed cache_attn.cu.
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

// ---- rotary positions ----------------------------------------------------------------------------
// Pair (a, b) of a head becomes (a cos - b sin, b cos + a sin), the transposed map (the gradient)
// takes -sin. Products and sums are rounded one by one (no contraction): the same bits as the
// formula in fp32. A unit is VEC values of each side of VEC pairs (half layout), VEC values of
// VEC / 2 pairs (interleaved), or VEC values behind the rotated part, which are copied. A thread
// keeps its angles for HPT heads, so that the tables are read HPT times less often.
struct RotaryArgs {
  const void *x;
  void *y;
  int64_t xsb, xst, xsh, ysb, yst, ysh;
  int64_t batch, tokens;
  int heads, dim, rot;
  const float *cos, *sin;
  int64_t rows;
  const void *pos;
  int pos_wide, interleaved;
  float sign;
  int hgroups, units;
};

template <typename T, int VEC, int HPT>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  pdl_enter();
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int u = (int)(idx % a.units);
  const int64_t hi = idx / a.units;
  const int hg = (int)(hi % a.hgroups);
  const int64_t tok = hi / a.hgroups;
  if (tok >= a.batch * a.tokens) return;
  const int64_t b = tok / a.tokens, t = tok - b * a.tokens;
  const int half = a.rot / 2, ur = a.interleaved ? a.rot / VEC : half / VEC;
  const T *x = (const T *)a.x + b * a.xsb + t * a.xst;
  T *y = (T *)a.y + b * a.ysb + t * a.yst;
  constexpr bool V = VEC * sizeof(T) >= 16;
  const int h0 = hg * HPT;
  if (u >= ur) {  // behind the rotated part
    const int d = a.rot + (u - ur) * VEC;
#pragma unroll
    for (int i = 0; i < HPT; ++i)
      if (h0 + i < a.heads) {
        float f[VEC];
        load_n<T, VEC>(x + (int64_t)(h0 + i) * a.xsh + d, V, f);
        store_n<T, VEC>(y + (int64_t)(h0 + i) * a.ysh + d, V, f);
      }
    return;
  }
  const int64_t p = load_index(a.pos, tok, a.pos_wide);
  const bool ok = p >= 0 && p < a.rows;
  if (!ok) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
  const float nan = __uint_as_float(0x7FC00000u);
  if (!a.interleaved) {
    const int d = u * VEC;
    float c[VEC], s[VEC];
    if (ok) {
      load_n<float, VEC>(a.cos + p * half + d, V, c);
      load_n<float, VEC>(a.sin + p * half + d, V, s);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = ok ? c[i] : nan, s[i] = ok ? s[i] * a.sign : nan;
    float f[HPT][VEC], g[HPT][VEC];
#pragma unroll
    for (int i = 0; i < HPT; ++i)
      if (h0 + i < a.heads) {
        load_n<T, VEC>(x + (int64_t)(h0 + i) * a.xsh + d, V, f[i]);
        load_n<T, VEC>(x + (int64_t)(h0 + i) * a.xsh + half + d, V, g[i]);
      }
#pragma unroll
    for (int i = 0; i < HPT; ++i)
      if (h0 + i < a.heads) {
        float m[VEC], n[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          m[j] = __fsub_rn(__fmul_rn(f[i][j], c[j]), __fmul_rn(g[i][j], s[j]));
          n[j] = __fadd_rn(__fmul_rn(g[i][j], c[j]), __fmul_rn(f[i][j], s[j]));
        }
        store_n<T, VEC>(y + (int64_t)(h0 + i) * a.ysh + d, V, m);
        store_n<T, VEC>(y + (int64_t)(h0 + i) * a.ysh + half + d, V, n);
      }
  } else if constexpr (VEC >= 2) {
    const int d = u * VEC;
    constexpr bool VT = V && VEC * 2 >= 16;
    float c[VEC / 2], s[VEC / 2];
    if (ok) {
      load_n<float, VEC / 2>(a.cos + p * half + d / 2, VT, c);
      load_n<float, VEC / 2>(a.sin + p * half + d / 2, VT, s);
    }
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) c[i] = ok ? c[i] : nan, s[i] = ok ? s[i] * a.sign : nan;
    float f[HPT][VEC];
#pragma unroll
    for (int i = 0; i < HPT; ++i)
      if (h0 + i < a.heads) load_n<T, VEC>(x + (int64_t)(h0 + i) * a.xsh + d, V, f[i]);
#pragma unroll
    for (int i = 0; i < HPT; ++i)
      if (h0 + i < a.heads) {
        float m[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          m[j] = __fsub_rn(__fmul_rn(f[i][j], c[j / 2]), __fmul_rn(f[i][j + 1], s[j / 2]));
          m[j + 1] = __fadd_rn(__fmul_rn(f[i][j + 1], c[j / 2]), __fmul_rn(f[i][j], s[j / 2]));
        }
        store_n<T, VEC>(y + (int64_t)(h0 + i) * a.ysh + d, V, m);
      }
  }
}

template <typename T, int VEC, int HPT>
static int32_t launch_rotary_t(RotaryArgs a, cudaStream_t stream) {
  a.hgroups = (a.heads + HPT - 1) / HPT;
  a.units = (a.interleaved ? a.rot / VEC : a.rot / 2 / VEC) + (a.dim - a.rot) / VEC;
  const int64_t n = a.batch * a.tokens * a.hgroups * a.units, blocks = (n + 255) / 256;
  if (blocks > 0x7FFFFFFF) return b200_set_error(B200_ERR_UNSUPPORTED, "rotary: too many values for one launch");
  B200_CUDA_TRY(launch_pdl(rotary_kernel<T, VEC, HPT>, dim3((unsigned)blocks), dim3(256), stream, a));
  return B200_OK;
}

template <typename T>
static int32_t launch_rotary_dt(const RotaryArgs &a, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  auto fits = [](const void *p, int64_t sb, int64_t st, int64_t sh) {
    return (uintptr_t)p % 16 == 0 && sb % VEC == 0 && st % VEC == 0 && sh % VEC == 0;
  };
  const int side = a.interleaved ? a.rot : a.rot / 2;
  const bool vec = fits(a.x, a.xsb, a.xst, a.xsh) && fits(a.y, a.ysb, a.yst, a.ysh) && side % VEC == 0 &&
                   (a.dim - a.rot) % VEC == 0 && (uintptr_t)a.cos % 16 == 0 && (uintptr_t)a.sin % 16 == 0 &&
                   (a.rot / 2) % 4 == 0;
  if (!vec) return a.interleaved && (a.dim - a.rot) % 2 == 0 ? launch_rotary_t<T, 2, 1>(a, stream)
                   : a.interleaved ? b200_set_error(B200_ERR_UNSUPPORTED, "rotary: an odd head needs the half layout")
                                   : launch_rotary_t<T, 1, 1>(a, stream);
  // four heads a thread once that leaves every SM its 2048 threads twice over
  const int64_t threads = a.batch * a.tokens * ((a.heads + 3) / 4) * (a.dim / VEC);
  return threads >= 148 * 2048 * 2 ? launch_rotary_t<T, VEC, 4>(a, stream) : launch_rotary_t<T, VEC, 1>(a, stream);
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
  int qvec, kvec, vvec, tvec;
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
  const int64_t page = place ? slot / a.c.page_size : 0, offset = place ? slot - page * a.c.page_size : 0;
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
        constexpr float lo = 0x1p-100f, hi = 0x1p100f;
        const float rr = __fmul_rn(__uint_as_float(top), (float)(1.0 / CFmt<F>::qmax));
        const int h = isk ? r - a.q_heads : r - a.q_heads - kvh;
        const int64_t at = scale_row(a.c, page, h, offset) + lane_d / a.c.block_size;
        const bool writes = lane_d % a.c.block_size == 0;
        float sc;
        if (a.c.scale_dtype == B200_DT_E8M0) {
          uint32_t e = (__float_as_uint(rr) + 0x7FFFFFu) >> 23;
          e = rr != rr ? 255u : min(227u, max(27u, e));
          sc = e == 255u ? rr : __uint_as_float(e << 23);
          if (writes) ((uint8_t *)(isk ? a.c.k_scales : a.c.v_scales))[at] = (uint8_t)e;
        } else {
          sc = __bfloat162float(__float2bfloat16_rn(rr));
          sc = sc < lo ? lo : sc > hi ? hi : sc;
          if (writes) ((__nv_bfloat16 *)(isk ? a.c.k_scales : a.c.v_scales))[at] = __float2bfloat16_rn(sc);
        }
        // under a NaN scale codes are zeros: in attention the NaN then reaches only rows that see the key
        uint8_t *codes = (uint8_t *)(isk ? a.c.k : a.c.v) + code_row(a.c, page, h, offset) + lane_d * CFmt<F>::bits / 8;
        if (sc != sc)
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = 0.f;
        encode8<F>(y, __frcp_rn(sc != sc ? 1.f : sc), codes);
      }
    }
  }
}

template <typename T, int F>
static int32_t launch_write_t(const WriteArgs &a, cudaStream_t stream) {
  const int rows = a.q_heads + 2 * a.c.kv_heads, rpc = WT / (a.c.head_dim / 8);
  const int need = (rows + rpc - 1) / rpc;
  // few tokens: a CTA for every RPC rows; many: one CTA a token, its angles loaded once
  const int split = a.tokens >= 148 * 8 ? 1 : need;
  const dim3 grid((unsigned)a.tokens, (unsigned)split);
  if (a.c.head_dim == 64) B200_CUDA_TRY(launch_pdl(cache_write_kernel<T, F, 64>, grid, dim3(WT), stream, a));
  else if (a.c.head_dim == 128) B200_CUDA_TRY(launch_pdl(cache_write_kernel<T, F, 128>, grid, dim3(WT), stream, a));
  else B200_CUDA_TRY(launch_pdl(cache_write_kernel<T, F, 256>, grid, dim3(WT), stream, a));
  return B200_OK;
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
// gives 8 values. A negative slot reads zeros.
struct ReadArgs {
  b200_cache_desc c;
  const void *slots;
  int slots_wide;
  int64_t tokens;
  void *k_out, *v_out;
};

template <int F>
__device__ __forceinline__ void decode8(const uint8_t *src, float (&f)[8]) {
  uint32_t p[4];
  if constexpr (CFmt<F>::bits == 8) {
    const uint2 w = *reinterpret_cast<const uint2 *>(src);
    decode4_8bit<F>(w.x, p[0], p[1]);
    decode4_8bit<F>(w.y, p[2], p[3]);
  } else {
    decode8_4<F>(*reinterpret_cast<const uint32_t *>(src), p);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&p[i]));
    if constexpr (F == B200_CACHE_INT4) f[i] = v.x, f[i + 4] = v.y;
    else f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}

template <typename T, int F>
__global__ void __launch_bounds__(256) cache_read_kernel(ReadArgs a) {
  pdl_enter();
  const int D = a.c.head_dim, lpr = D / 8;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int d = (int)(idx % lpr) * 8;
  const int64_t hi = idx / lpr;
  const int h = (int)(hi % a.c.kv_heads);
  const int64_t t = hi / a.c.kv_heads;
  if (t >= a.tokens) return;
  const int64_t slot = load_index(a.slots, t, a.slots_wide);
  const int64_t cells = a.c.pages * a.c.page_size;
  const bool in = slot >= 0 && slot < cells;
  if (slot >= cells) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
  float k[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
  if (in) {
    const int64_t page = slot / a.c.page_size;
    const int64_t offset = slot - page * a.c.page_size;
    const bool e8 = a.c.scale_dtype == B200_DT_E8M0;
    const int64_t at = scale_row(a.c, page, h, offset) + d / a.c.block_size;
    const int64_t cd = code_row(a.c, page, h, offset) + d * CFmt<F>::bits / 8;
    const float ks = scale_f32(a.c.k_scales, at, e8), vs = scale_f32(a.c.v_scales, at, e8);
    decode8<F>((const uint8_t *)a.c.k + cd, k);
    decode8<F>((const uint8_t *)a.c.v + cd, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] *= ks, v[i] *= vs;
  }
  store_n<T, 8>((T *)a.k_out + (t * a.c.kv_heads + h) * D + d, true, k);
  store_n<T, 8>((T *)a.v_out + (t * a.c.kv_heads + h) * D + d, true, v);
}

template <typename T>
static int32_t launch_read_t(const ReadArgs &a, cudaStream_t stream) {
  const int64_t n = a.tokens * a.c.kv_heads * (a.c.head_dim / 8), blocks = (n + 255) / 256;
  if (blocks > 0x7FFFFFFF) return b200_set_error(B200_ERR_UNSUPPORTED, "cache_read: too many values for one launch");
  const dim3 grid((unsigned)blocks);
  switch (a.c.format) {
    case B200_CACHE_INT8: B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, B200_CACHE_INT8>, grid, dim3(256), stream, a)); break;
    case B200_CACHE_FP8E4M3: B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, B200_CACHE_FP8E4M3>, grid, dim3(256), stream, a)); break;
    case B200_CACHE_INT4: B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, B200_CACHE_INT4>, grid, dim3(256), stream, a)); break;
    default: B200_CUDA_TRY(launch_pdl(cache_read_kernel<T, B200_CACHE_FP4_E2M1>, grid, dim3(256), stream, a)); break;
  }
  return B200_OK;
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
  a.batch = batch, a.tokens = tokens, a.heads = heads, a.dim = head_dim, a.rot = r->rotary_dim;
  a.cos = r->cos, a.sin = r->sin, a.rows = r->rows, a.pos = pos;
  a.pos_wide = pos_dtype == B200_DT_I64, a.interleaved = r->interleaved, a.sign = transpose ? -1.f : 1.f;
  switch (dtype) {
    case B200_DT_F16: return launch_rotary_dt<__half>(a, stream);
    case B200_DT_BF16: return launch_rotary_dt<__nv_bfloat16>(a, stream);
    default: return launch_rotary_dt<float>(a, stream);
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
  ReadArgs a = {*c, slots, slots_dtype == B200_DT_I64, tokens, k_out, v_out};
  switch (dtype) {
    case B200_DT_F16: return launch_read_t<__half>(a, stream);
    case B200_DT_BF16: return launch_read_t<__nv_bfloat16>(a, stream);
    default: return launch_read_t<float>(a, stream);
  }
}

}  // namespace b200

// ---- C entries ---------------------------------------------------------------------------------
using namespace b200;

extern "C" {

int32_t b200_rotary(const void *x, int32_t dtype, int64_t batch, int64_t tokens, int32_t heads, int32_t head_dim,
                    const int64_t *x_strides, void *y, const int64_t *y_strides, const b200_rotary_desc *table,
                    const void *positions, int32_t positions_dtype, int32_t transpose, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (batch < 0 || tokens < 0 || heads < 0 || head_dim < 1 || x_strides == nullptr || y_strides == nullptr)
    return b200_set_error(B200_ERR_INVALID, "rotary: bad sizes");
  if (!cache::real_dtype(dtype)) return b200_set_error(B200_ERR_INVALID, "rotary: unsupported dtype %d", dtype);
  if (batch == 0 || tokens == 0 || heads == 0) return B200_OK;
  if (int32_t rc = check_rotary(table, head_dim, positions, positions_dtype)) return rc;
  if (x == nullptr || y == nullptr) return b200_set_error(B200_ERR_INVALID, "rotary: null x or y");
  return launch_rotary(x, dtype, batch, tokens, heads, head_dim, x_strides, y, y_strides, table, positions,
                       positions_dtype, transpose, (cudaStream_t)stream);
}

int32_t b200_cache_write(const b200_cache_desc *c, const void *k, const void *v, int32_t dtype, int64_t tokens,
                         const int64_t *k_strides, const int64_t *v_strides, const void *slots, int32_t slots_dtype,
                         const b200_rotary_desc *table, const void *positions, int32_t positions_dtype, const void *q,
                         int32_t q_heads, const int64_t *q_strides, void *q_out, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (int32_t rc = check_cache(c)) return rc;
  if (tokens < 0 || k_strides == nullptr || v_strides == nullptr || (q != nullptr && (q_heads < 1 || q_heads > 65535 || q_strides == nullptr)))
    return b200_set_error(B200_ERR_INVALID, "cache_write: bad sizes");
  if (!cache::real_dtype(dtype)) return b200_set_error(B200_ERR_INVALID, "cache_write: unsupported dtype %d", dtype);
  if (cache::bad_index_dtype(slots_dtype)) return b200_set_error(B200_ERR_INVALID, "cache_write: slots must be int32 or int64");
  if (tokens == 0) return B200_OK;
  if (table != nullptr)
    if (int32_t rc = check_rotary(table, c->head_dim, positions, positions_dtype)) return rc;
  if (k == nullptr || v == nullptr || slots == nullptr || (q != nullptr && q_out == nullptr))
    return b200_set_error(B200_ERR_INVALID, "cache_write: null pointer");
  if ((uintptr_t)q_out % 16) return b200_set_error(B200_ERR_INVALID, "cache_write: q_out must start on a 16-byte boundary");
  return launch_cache_write(c, k, v, dtype, tokens, k_strides, v_strides, slots, slots_dtype, table, positions,
                            positions_dtype, q, q_heads, q_strides, q_out, (cudaStream_t)stream);
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
