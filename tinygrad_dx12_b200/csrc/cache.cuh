// cache.cuh -- the packed key/value cache: formats, scales and the arithmetic shared by its kernels.
//
// A cache holds keys and values as codes of one format with a scale per block of `block` values
// along the head's axis (32 of them, or the whole head):
//   codes   [pages, kv_heads, page_size, head_dim * bits / 8]   lowest bits first, as packed weights
//   scales  [pages, kv_heads, page_size, head_dim / block]      bfloat16 or E8M0 bytes
// with strides of their own for pages, heads and tokens.
// Quantisation of a block: r = max|x| * (1 / QMAX), s = r rounded to bfloat16 (E8M0: the smallest
// power of two not below r, so nothing is clipped), held within [2^-100, 2^100] so that s, 1 / s and
// log2 s are ordinary fp32 numbers; the code is x * (1 / s) to the nearest, ties to even. Each of
// these is one IEEE operation in fp32, so codes are reproducible to the bit. A NaN in a block makes
// its scale NaN: what is read back, or attended to, is NaN whatever the format.
#pragma once

#include "common.cuh"
#include "decode.cuh"

namespace b200 {
namespace cache {

constexpr uint32_t DEVERR_BAD_INDEX = 2u;  // a slot, page or position outside its table

template <int F> struct CFmt;
template <> struct CFmt<B200_CACHE_INT8> { static constexpr int bits = 8; static constexpr double qmax = 127.0; };
template <> struct CFmt<B200_CACHE_FP8E4M3> { static constexpr int bits = 8; static constexpr double qmax = 448.0; };
template <> struct CFmt<B200_CACHE_INT4> { static constexpr int bits = 4; static constexpr double qmax = 7.0; };
template <> struct CFmt<B200_CACHE_FP4_E2M1> { static constexpr int bits = 4; static constexpr double qmax = 6.0; };

// Scale `i` of an array as the bits of a bfloat16 (an E8M0 byte b is bfloat16 2^(b-127) exactly).
__device__ __forceinline__ uint32_t scale_bits(const void *p, int64_t i, bool e8m0) {
  if (e8m0) {
    const uint32_t b = ((const uint8_t *)p)[i];
    return b == 0 ? 0x40u : b == 255 ? 0x7FC0u : b << 7;
  }
  return ((const uint16_t *)p)[i];
}
__device__ __forceinline__ float scale_f32(const void *p, int64_t i, bool e8m0) {
  return __uint_as_float(scale_bits(p, i, e8m0) << 16);
}

// Where (page, head, offset)'s row of codes (bytes) and of scales (elements) begins.
__device__ __forceinline__ int64_t code_row(const b200_cache_desc &c, int64_t page, int64_t h, int64_t offset) {
  return page * c.strides[0] + h * c.strides[1] + offset * c.strides[2];
}
__device__ __forceinline__ int64_t scale_row(const b200_cache_desc &c, int64_t page, int64_t h, int64_t offset) {
  return page * c.scale_strides[0] + h * c.scale_strides[1] + offset * c.scale_strides[2];
}

// ---- exact fp16 values of 8-bit codes ----------------------------------------------------------
// Bytes (b0, b1) and (b2, b3) of w -> two fp16 pairs. INT8: with the sign bit flipped a byte under
// 0x64 is fp16 1024 + (c + 128). E4M3 values are exact in fp16.
template <int F>
__device__ __forceinline__ void decode4_8bit(uint32_t w, uint32_t &p0, uint32_t &p1) {
  if constexpr (F == B200_CACHE_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t h0 = __byte_perm(u, 0x64646464u, 0x4140), h1 = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 c = __float2half2_rn(1152.f);
    const __half2 r0 = __hsub2(*reinterpret_cast<const __half2 *>(&h0), c);
    const __half2 r1 = __hsub2(*reinterpret_cast<const __half2 *>(&h1), c);
    p0 = *reinterpret_cast<const uint32_t *>(&r0);
    p1 = *reinterpret_cast<const uint32_t *>(&r1);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(p0), "=r"(p1)
        : "r"(w));
  }
}
// 8 nibbles -> 4 fp16 pairs: INT4 pairs (i, i + 4), FP4 pairs (2i, 2i + 1). INT4: with the sign bit
// flipped a nibble under 0x64 is fp16 1024 + (c + 8), four bits higher 1024 + 16 (c + 8): mask and flip
// are one operation.
template <int F>
__device__ __forceinline__ void decode8_4(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (F == B200_CACHE_INT4) {
    const uint32_t hi = w >> 8;
    const uint32_t h[4] = {(w & 0x000F000Fu) ^ 0x64086408u, (w & 0x00F000F0u) ^ 0x64806480u,
                           (hi & 0x000F000Fu) ^ 0x64086408u, (hi & 0x00F000F0u) ^ 0x64806480u};
    const __half2 one = __float2half2_rn(1032.f), sixteenth = __float2half2_rn(0.0625f), off = __float2half2_rn(-72.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 x = *reinterpret_cast<const __half2 *>(&h[i]);
      const __half2 r = i % 2 ? __hfma2(x, sixteenth, off) : __hsub2(x, one);
      p[i] = *reinterpret_cast<const uint32_t *>(&r);
    }
  } else {
    gemv::decode8_4bit<B200_FMT_FP4_E2M1>(w, p);
  }
}

}  // namespace cache
}  // namespace b200
