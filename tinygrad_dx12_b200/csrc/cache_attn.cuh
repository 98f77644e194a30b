// cache_attn.cuh -- what the attention kernels over the packed cache share: their arguments, the scale
// arithmetic, and how a row's result is finished. The mathematics is at the top of cache_attn.cu.
#pragma once

#include "cache.cuh"
#include "kernels.h"

namespace b200 {
namespace cattn {

using namespace cache;

constexpr float LAZY = 4.f;          // u may pass the running maximum by this before it moves
constexpr float BIAS = 15.f - LAZY;  // p = 2^(u - m + BIAS) uses fp16 up to 2^15, so small weights keep their bits
// A key adds p / vs to the denominator: up to 2^15 * 2^100 where its values are zero (a block of zeros has
// the scale 2^-100, no reference is below that), down to 2^11 / 2^100 where the largest are all that counts.
// Sums are kept as 2^-SUM_EXP of themselves: 2^31 keys stay below 2^126, and 2^-109 is an ordinary number.
// p below 2^-126 is flushed to zero: beside values whose scale is 2^13 (fp16's largest) a key of zeros counts
// down to 2^-24 of their weight, and fully, at equal scores, up to scales of 2^37.
constexpr int SUM_EXP = 20;
constexpr float SUM_UNIT = 1.f / (1 << SUM_EXP);

struct Params {
  const void *q;
  int64_t qsr, qsb, qsh;  // strides of q: request, token, head
  const uint8_t *k, *v;
  const void *ks, *vs;
  // strides in bytes: page, head, token; a page's extent and a page stride are below 2^31
  uint32_t cp, ct, sp, st;
  int64_t ch, sh;
  int e8m0, scale_vec, q_vec, q_bf16;
  int exact_keys;  // a prefix's share of results that come with logarithms
  int64_t pages;
  int page_shift, kv_heads, group;
  const int32_t *tables;
  int64_t table_stride;
  int max_pages;
  const int32_t *lengths;  // per request, or null: `fixed` for all
  int64_t fixed;
  int batch, rows, queries;  // rows: query rows of a (request, key head)
  int per_request;           // queries of a request (rows / group of them may span requests)
  int causal;
  float scale;  // softmax scale * log2 e
  int row_tiles, q_heads;
  // results: final (out, lse) or partial (po, pm, pl)
  void *out;
  float *lse;
  float *po, *pm, *pl;
  const float *fo, *fm, *fl;  // partials of the shared prefix, joined at the end
  int64_t row0;               // rows before these in fo, fm, fl
  int early;  // the launch before is the join_kernel that completes these partials: nothing else is waited for
  // split segments
  float *ws_o, *ws_ml;
  uint32_t *tickets;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <int BYTES>
__device__ __forceinline__ void lds(const uint8_t *p, uint32_t *w) {
  if constexpr (BYTES == 16) {
    const uint4 x = *reinterpret_cast<const uint4 *>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (BYTES == 8) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}

// 2^-(E - H): what a block's scale is multiplied by; 2^(E - H) is the row's scale, 2^-100 at least.
template <int F>
struct RowRef {
  static constexpr int H = CFmt<F>::bits == 4 ? 12 : 6;
  // `top`: bfloat16 bits of the row's largest scale
  __device__ static __forceinline__ int exponent(uint32_t top) { return max((int)((top >> 7) & 0xFF) - H, 27); }
  __device__ static __forceinline__ float inverse(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }
  __device__ static __forceinline__ float value(int e) { return __uint_as_float((uint32_t)e << 23); }
};

// The NB scales of a row in as few words as they fill.
template <int NB>
__device__ __forceinline__ void load_scales(const uint8_t *p, bool e8m0, bool vec, uint32_t (&raw)[(NB + 1) / 2]) {
  if constexpr (NB == 1) {
    raw[0] = e8m0 ? *p : *(const uint16_t *)p;
  } else if (vec && !e8m0) {
    lds<NB * 2>(p, raw);
  } else if (vec) {
    if constexpr (NB == 2) raw[0] = *(const uint16_t *)p;
    else lds<NB>(p, raw);
  } else {
#pragma unroll
    for (int i = 0; i < (NB + 1) / 2; ++i) raw[i] = 0;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (e8m0) raw[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
      else raw[i / 2] |= (uint32_t)((const uint16_t *)p)[i] << (16 * (i % 2));
    }
  }
}
// Them as fp32: E8M0's NaN byte reads infinity, which the product with zero turns into NaN (its
// byte 0, 2^-127, reads zero).
template <int NB>
__device__ __forceinline__ void widen(const uint32_t (&raw)[(NB + 1) / 2], bool e8m0, float (&f)[NB]) {
  if (e8m0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const float x = __uint_as_float(((raw[i / 4] >> (8 * (i % 4))) & 0xFFu) << 23);
      f[i] = fmaf(x, 0.f, x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NB; ++i) f[i] = __uint_as_float(i % 2 ? raw[i / 2] & 0xFFFF0000u : raw[i / 2] << 16);
  }
}

// Query row r of (entry, key head h): its offset in q, and its place among all rows of out.
struct RowAt {
  int64_t q, out;
};
__device__ __forceinline__ RowAt row_at(const Params &p, int b, int h, int r) {
  const int tok = p.rows == p.group ? 0 : r / p.group, head = h * p.group + (r - tok * p.group);
  const int rq = p.per_request == 1 ? tok : tok / p.per_request, qi = tok - rq * p.per_request;
  const int64_t req = b + rq;
  return {req * p.qsr + qi * p.qsb + head * p.qsh, (req * p.per_request + qi) * p.q_heads + head};
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T out_of(float v);
template <> __device__ __forceinline__ __half out_of<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 out_of<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// (o, m, l) with another share of the same row: numerators at `po`, maximum, denominator.
template <int D>
__device__ __forceinline__ void join(float4 &o, float &m, float &l, const float *po, float pm, float pl) {
  const float M = fmaxf(m, pm);
  const float a = m == -INFINITY ? 0.f : ex2(m - M), b = pm == -INFINITY ? 0.f : ex2(pm - M);
  const float4 f = *reinterpret_cast<const float4 *>(po);
  o.x = o.x * a + f.x * b, o.y = o.y * a + f.y * b, o.z = o.z * a + f.z * b, o.w = o.w * a + f.w * b;
  l = l * a + pl * b;
  m = M;
}

// What a numerator is multiplied by, one after the other: 2^-SUM_EXP / l in two parts that are ordinary numbers
// (and so are the products) whatever the sum. No key seen: zeros.
__device__ __forceinline__ float2 inverse_sum(float l) {
  const bool small = l < 1.f;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  return make_float2(small ? inv * SUM_UNIT : inv, small ? 1.f : SUM_UNIT);
}
// The natural logarithm of the softmax's sum.
__device__ __forceinline__ float log_sum(float m, float l) {
  return l == 0.f ? -INFINITY : (m - BIAS + (log2f(l) + SUM_EXP)) * 0.69314718055994531f;
}

// A row's result from its numerator (four values), maximum and denominator.
template <typename T, int D>
__device__ __forceinline__ void finish(const Params &p, int64_t row, int d, float4 o, float m, float l) {
  if (p.po != nullptr) {
    *reinterpret_cast<float4 *>(p.po + row * D + d) = o;
    if (d == 0) p.pm[row] = m, p.pl[row] = l;
    return;
  }
  if (p.fo != nullptr) {
    join<D>(o, m, l, p.fo + (p.row0 + row) * D + d, p.fm[p.row0 + row], p.fl[p.row0 + row]);
  }
  const float2 f = inverse_sum(l);
  T *dst = (T *)p.out + row * D + d;
  alignas(8) T r[4] = {out_of<T>(o.x * f.x * f.y), out_of<T>(o.y * f.x * f.y), out_of<T>(o.z * f.x * f.y),
                       out_of<T>(o.w * f.x * f.y)};
  *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(r);
  if (p.lse != nullptr && d == 0) p.lse[row] = log_sum(m, l);
}


// The many-row kernel (cache_attn_mma.cu): rows of p in tiles of 128 or 256 on the tcgen05 cores.
bool mma_supported(const Params &p, int dim);
int32_t launch_mma(Params &p, int q_dtype, int fmt, int dim, bool blk, cudaStream_t stream);

}  // namespace cattn
}  // namespace b200
