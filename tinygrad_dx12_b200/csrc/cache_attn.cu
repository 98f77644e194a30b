// cache_attn.cu -- attention of few query rows over the packed key/value cache.
//
//   s[r, t] = scale * q[r] . K[t],  K[t] = ks[t] * kc[t]        (codes times their row's scale)
//   out[r]  = sum_t w[r, t] V[t] / sum_t w[r, t],  w = exp(s), V[t] = vs[t] * vc[t]
//
// One pass over the keys. With everything in base 2, u = s + log2 vs[t] and a running maximum m of
// u, a key adds p * vc[t] (p = 2^(u - m + 11)) to the numerator and p / vs[t] to the denominator:
// codes enter the matrix instructions as they are stored, exact in fp16, and no scale is multiplied
// into them. p <= 2^15 is rounded to fp16 for the second product (11 bits down to 2^-25 of the
// largest weight); sums, statistics and the denominator are fp32. q is scaled by a power of two per row, so that bf16 values fit fp16.
// Blocks of 32 values with scales of their own: the codes are multiplied by scale / 2^E, with 2^E
// just above the row's largest scale (shifted up by fp16's headroom, so that blocks down to 2^-26,
// 8-bit 2^-20, of the largest keep their bits), and ks, vs above become 2^E.
//
// m16n8k16 takes keys as its 16 rows and query rows (heads that share a key head, and the tokens of
// a short block) as its 8 columns: s^T = K q^T, out^T = V^T p^T. Which value of the head sits at
// which k of an instruction is free as long as both operands agree, so a lane reads 16 consecutive
// bytes of a key row and q is laid out to match; a lane reads four values' worth of tokens of V^T
// at its 16 (8, 32) values of the head, and pairs of tokens are joined by byte permutes before
// the codes become fp16. p is turned with movmatrix. Keys therefore go from memory to registers
// to the tensor core: no shared memory, no barrier on the way. A warp works alone on units of 16
// or 32 keys, issues the loads of its next keys as soon as the registers are free, and 16 warps of
// an SM hide the latency.
//
// The units of all (request, key head, row tile) are laid end to end and cut into equal runs, one
// per CTA, from the lengths on the device: ragged batches balance, and the launch (a CUDA graph)
// does not depend on the lengths. A CTA's warps take its units in turn and join in shared memory;
// a segment cut over several CTAs is joined by the CTA that finishes last, always in the same order.
#include <map>
#include <mutex>

#include "cache.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace b200 {

int32_t cache_attn_device_error(unsigned int *v, bool clear) {
  B200_CUDA_TRY(tu_device_error(v, clear));
  return B200_OK;
}

namespace cattn {

using namespace cache;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int MAX_ENTRIES = 4096;  // (request, row tile) pairs of one launch
constexpr float LAZY = 4.f;         // u may pass the running maximum by this before it moves
constexpr float BIAS = 15.f - LAZY;  // p = 2^(u - m + BIAS) uses fp16 up to 2^15, so small weights keep their bits

struct Params {
  const void *q;
  int64_t qsr, qsb, qsh;  // strides of q: request, token, head
  const uint8_t *k, *v;
  const void *ks, *vs;
  int64_t cp, ch, ct, sp, sh, st;  // strides of codes (bytes) and scales: page, head, token
  int e8m0;
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
  // split segments
  float *ws_o, *ws_ml;
  uint32_t *tickets;
};

template <int F, int D, int NT>
struct Cfg {
  static constexpr int bits = CFmt<F>::bits;
  static constexpr int RB = D * bits / 8;                       // bytes of a row
  static constexpr int KCB = RB / 4 < 16 ? RB / 4 : 16;         // bytes of a lane's key chunk
  static constexpr int KCH = RB / 4 / KCB, KCW = KCB / 4;       // chunks, words of one
  static constexpr int KEC = KCB * 8 / bits;                    // values of one
  static constexpr int VCB = RB / 8 < 16 ? RB / 8 : 16;
  static constexpr int VCH = RB / 8 / VCB, VCW = VCB / 4;
  static constexpr int VEC = VCB * 8 / bits;
  static constexpr int KS = D / 16;                             // k steps of q K^T
  static constexpr int MT = D / 16;                             // tiles of V^T
  static constexpr int M2 = RB >= 128 ? 1 : 2;                  // blocks of 16 keys in a unit
  static constexpr int ROWS = 8 * NT;
  static constexpr int Q_BYTES = NT * KS * 32 * 8;
  static constexpr int ORS = D + 4;                             // row pitch of a warp's numerators (floats)
  static constexpr int JOIN_BYTES = WARPS * ROWS * ORS * 4;
  static constexpr int SMEM = Q_BYTES + JOIN_BYTES + WARPS * ROWS * 8 + ROWS * 16;
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
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t *w) {
  if constexpr (BYTES == 16) {
    const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (BYTES == 8) {
    const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
  }
}

// 2^-(E - H): what a block's scale is multiplied by; 2^(E - H) is the row's scale.
template <int F>
struct RowRef {
  static constexpr int H = CFmt<F>::bits == 4 ? 12 : 6;
  // `top`: bfloat16 bits of the row's largest scale
  __device__ static __forceinline__ int exponent(uint32_t top) { return max((int)((top >> 7) & 0xFF), H + 1) - H; }
  __device__ static __forceinline__ float inverse(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }
  __device__ static __forceinline__ float value(int e) { return __uint_as_float((uint32_t)e << 23); }
};

// A scale's bits, nothing for NaN: the NaN of a row travels in its denominator, which only rows that
// see the key take.
__device__ __forceinline__ uint32_t number(uint32_t bits) { return bits > 0x7F80u ? 0u : bits; }

// Where 16 keys' codes and scales begin.
struct At {
  int64_t code, scale;
};

// The codes and scales of 16 keys as a lane holds them.
template <int F, int D, int NT, bool BLK>
struct Keys {
  using C = Cfg<F, D, NT>;
  static constexpr int NB = D / 32;
  uint32_t k[2][C::KCH * C::KCW];
  uint32_t v[4][C::VCH * C::VCW];
  uint32_t ks[2][BLK ? C::KCH : 1];  // bfloat16 bits
  uint32_t vs[2];                    // of the two keys of this lane's scores (blocks: the largest)
  uint32_t kt[2];                    // blocks: the largest of the two keys'
  uint32_t vb[BLK ? 4 : 1][BLK ? C::VCH : 1];
};

template <int F, int D, int NT, bool BLK>
__device__ __forceinline__ void load_k(Keys<F, D, NT, BLK> &x, const Params &p, At at, int valid, int g, int t) {
  using C = Cfg<F, D, NT>;
  constexpr int NB = D / 32;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = 4 * (g >> 1) + (g & 1) + 2 * i;
    const bool in = tok < valid;
    const int64_t r = at.scale + tok * p.st;
    if (in) {
#pragma unroll
      for (int c = 0; c < C::KCH; ++c)
        load_words<C::KCB>(p.k + at.code + tok * p.ct + (t + 4 * c) * C::KCB, &x.k[i][c * C::KCW]);
    } else {
#pragma unroll
      for (int c = 0; c < C::KCH * C::KCW; ++c) x.k[i][c] = 0;
    }
    if constexpr (!BLK) {
      x.ks[i][0] = in ? scale_bits(p.ks, r, p.e8m0) : 0x3F80u;
      x.vs[i] = in ? scale_bits(p.vs, r, p.e8m0) : 0x3F80u;
    } else {
      uint32_t kt = 0, vt = 0;  // the largest over this lane's share of the blocks, then over the quad
#pragma unroll
      for (int c = 0; c < C::KCH; ++c)
        x.ks[i][c] = in ? scale_bits(p.ks, r + (t + 4 * c) * C::KEC / 32, p.e8m0) : 0u;
#pragma unroll
      for (int b = 0; b < (NB + 3) / 4; ++b) {
        const int nb = min(t + 4 * b, NB - 1);
        if (in) {
          kt = max(kt, scale_bits(p.ks, r + nb, p.e8m0));
          vt = max(vt, scale_bits(p.vs, r + nb, p.e8m0));
        }
      }
      x.kt[i] = kt, x.vs[i] = vt;
    }
  }
}
template <int F, int D, int NT, bool BLK>
__device__ __forceinline__ void load_v(Keys<F, D, NT, BLK> &x, const Params &p, At at, int valid, int g, int t) {
  using C = Cfg<F, D, NT>;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = 4 * t + i;
    if (tok < valid) {
#pragma unroll
      for (int c = 0; c < C::VCH; ++c) {
        load_words<C::VCB>(p.v + at.code + tok * p.ct + (g + 8 * c) * C::VCB, &x.v[i][c * C::VCW]);
        if constexpr (BLK)
          x.vb[i][c] = scale_bits(p.vs, at.scale + tok * p.st + (g + 8 * c) * C::VEC / 32, p.e8m0);
      }
    } else {  // nothing of a key that is not there: its codes may be anything
#pragma unroll
      for (int c = 0; c < C::VCH * C::VCW; ++c) x.v[i][c] = 0;
      if constexpr (BLK)
#pragma unroll
        for (int c = 0; c < C::VCH; ++c) x.vb[i][c] = 0;
    }
  }
}

// Query row r of (entry, key head h): its offset in q, and its place among all rows of out.
struct RowAt {
  int64_t q, out;
};
__device__ __forceinline__ RowAt row_at(const Params &p, int b, int h, int r) {
  const int tok = r / p.group, head = h * p.group + (r - tok * p.group);
  const int rq = tok / p.per_request, qi = tok - rq * p.per_request;
  const int64_t req = b + rq;
  return {req * p.qsr + qi * p.qsb + head * p.qsh, (req * p.per_request + qi) * p.q_heads + head};
}

// Half index in shared memory of value d of query row n: the order in which a lane's codes of a
// key row come out of their decoding.
template <int F, int D, int NT>
__device__ __forceinline__ int q_index(int n, int d) {
  using C = Cfg<F, D, NT>;
  const int chunk = d / C::KEC, t = chunk & 3, c = chunk >> 2, w = d % C::KEC;
  int step, reg, half;
  if constexpr (F == B200_CACHE_INT4) {  // words of 8: pairs (i, i + 4)
    const int pi = w & 3;
    step = (w >> 3) * 2 + (pi >> 1), reg = pi & 1, half = (w >> 2) & 1;
  } else {
    step = w >> 2, reg = (w >> 1) & 1, half = w & 1;
  }
  return ((((n >> 3) * C::KS + c * (C::KEC / 4) + step) * 32 + (n & 7) * 4 + t) * 2 + reg) * 2 + half;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T out_of(float v);
template <> __device__ __forceinline__ __half out_of<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 out_of<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A row's result from its numerator (four values), maximum and denominator.
template <typename T, int D>
__device__ __forceinline__ void finish(const Params &p, int64_t row, int d, float4 o, float m, float l) {
  if (p.po != nullptr) {
    *reinterpret_cast<float4 *>(p.po + row * D + d) = o;
    if (d == 0) p.pm[row] = m, p.pl[row] = l;
    return;
  }
  if (p.fo != nullptr) {
    const float pm = p.fm[row], M = fmaxf(m, pm);
    const float a = m == -INFINITY ? 0.f : ex2(m - M), b = pm == -INFINITY ? 0.f : ex2(pm - M);
    const float4 f = *reinterpret_cast<const float4 *>(p.fo + row * D + d);
    o.x = o.x * a + f.x * b, o.y = o.y * a + f.y * b, o.z = o.z * a + f.z * b, o.w = o.w * a + f.w * b;
    l = l * a + p.fl[row] * b;
    m = M;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key seen: zeros
  T *dst = (T *)p.out + row * D + d;
  alignas(8) T r[4] = {out_of<T>(o.x * inv), out_of<T>(o.y * inv), out_of<T>(o.z * inv), out_of<T>(o.w * inv)};
  *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(r);
  if (p.lse != nullptr && d == 0) p.lse[row] = l == 0.f ? -INFINITY : (m - BIAS + log2f(l)) * 0.69314718055994531f;
}

template <typename T, int F, int D, int NT, bool BLK>
__global__ void __launch_bounds__(THREADS, D == 256 || NT == 2 ? 1 : 2) attn_kernel(const Params p) {
  using C = Cfg<F, D, NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t *qf = (uint32_t *)smem;
  float *join_o = (float *)(smem + C::Q_BYTES);
  float *join_m = (float *)(smem + C::Q_BYTES + C::JOIN_BYTES), *join_l = join_m + WARPS * C::ROWS;
  float *qs_s = join_l + WARPS * C::ROWS;  // [ROWS] multiplier of a row's scores
  int *lim_s = (int *)(qs_s + C::ROWS);    // [ROWS] keys that a row sees
  __shared__ uint32_t prefix[MAX_ENTRIES + 1];
  __shared__ uint32_t scan[WARPS];
  __shared__ uint32_t last;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int entries = p.batch * p.row_tiles;
  constexpr int UNIT = 16 * C::M2;
  const int64_t cap = (int64_t)p.max_pages << p.page_shift;

  auto length_of = [&](int b) -> int64_t {
    const int64_t n = p.lengths != nullptr ? p.lengths[b] : p.fixed;
    return n < 0 ? 0 : n > cap ? cap : n;
  };
  // keys that the last row of an entry's tile sees
  auto keys_of = [&](int e) -> int64_t {
    const int b = e / p.row_tiles, rt = e - b * p.row_tiles;
    const int64_t n = length_of(b);
    if (!p.causal) return n;
    const int r1 = min(p.rows, (rt + 1) * C::ROWS) - 1;
    const int64_t lim = n - p.queries + r1 / p.group + 1;
    return lim < 0 ? 0 : lim;
  };

  // units of the entries, summed up
  {
    const int per = (entries + THREADS - 1) / THREADS, e0 = tid * per;
    uint32_t sum = 0;
    for (int i = 0; i < per; ++i)
      if (e0 + i < entries) sum += (uint32_t)((keys_of(e0 + i) + UNIT - 1) / UNIT);
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    uint32_t base = 0;
    for (int w = 0; w < warp; ++w) base += scan[w];
    uint32_t run = base + inc - sum;
    for (int i = 0; i < per; ++i)
      if (e0 + i < entries) {
        prefix[e0 + i] = run;
        run += (uint32_t)((keys_of(e0 + i) + UNIT - 1) / UNIT);
        if (e0 + i == entries - 1) prefix[entries] = run;
      }
    __syncthreads();
  }
  const int heads = p.kv_heads;
  const int64_t total = (int64_t)prefix[entries] * heads;

  // rows without a key: zeros (or what the prefix gave)
  for (int e = blockIdx.x; e < entries; e += gridDim.x) {
    if (prefix[e + 1] != prefix[e]) continue;
    const int b = e / p.row_tiles, rt = e - b * p.row_tiles;
    const int n = min(C::ROWS, p.rows - rt * C::ROWS);
    for (int i = tid; i < heads * n * (D / 4); i += THREADS) {
      const int d = (i % (D / 4)) * 4, rr = i / (D / 4);
      const RowAt at = row_at(p, b, rr / n, rt * C::ROWS + rr % n);
      finish<T, D>(p, at.out, d, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
  }

  // this CTA's run of units; without a workspace, whole segments in turn
  const bool split = p.ws_o != nullptr;
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < 2 * WARPS) per = 2 * WARPS;
  int64_t u = split ? (int64_t)blockIdx.x * per : 0;
  const int64_t u_end = split ? min(total, u + per) : total;
  int64_t skip = split ? 0 : blockIdx.x;  // segments to pass over
  int e = 0;
  while (u < u_end) {
    {  // the entry of unit u
      int lo = 0, hi = entries;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)prefix[mid] * heads <= u) lo = mid;
        else hi = mid;
      }
      e = lo;
    }
    const int units = (int)(prefix[e + 1] - prefix[e]);
    const int64_t first = (int64_t)prefix[e] * heads;
    const int h = (int)((u - first) / units);
    const int64_t seg0 = first + (int64_t)h * units, seg1 = seg0 + units;
    if (skip > 0) {
      --skip;
      u = seg1;
      continue;
    }
    if (!split) skip = gridDim.x - 1;
    const int b = e / p.row_tiles, rt = e - b * p.row_tiles, r0 = rt * C::ROWS;
    const int from = (int)(u - seg0), to = (int)(min(u_end, seg1) - seg0);
    const int n_rows = min(C::ROWS, p.rows - r0);
    const int64_t len = length_of(b), keys = keys_of(e);

    // q: fp16, each row scaled by a power of two, in the order of the keys' fragments
    __syncthreads();
    for (int n = warp; n < C::ROWS; n += WARPS) {
      constexpr int E = D / 32;
      float x[E], top = 0.f;
      bool bad = false;
      const bool in = n < n_rows;
      const T *src = in ? (const T *)p.q + row_at(p, b, h, r0 + n).q : nullptr;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[i] = in ? to_f32<T>(src[i * 32 + lane]) : 0.f;
        top = fmaxf(top, fabsf(x[i]));
        bad |= x[i] != x[i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      const int ex = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float((uint32_t)(254 - ex) << 23);
#pragma unroll
      for (int i = 0; i < E; ++i) ((__half *)qf)[q_index<F, D, NT>(n, i * 32 + lane)] = __float2half_rn(x[i] * down);
      if (lane == 0) {
        qs_s[n] = p.scale * __uint_as_float((uint32_t)ex << 23);
        const int64_t lim = !p.causal ? len : len - p.queries + (r0 + n) / p.group + 1;
        lim_s[n] = in ? (int)max((int64_t)0, lim) : 0;
      }
    }
    __syncthreads();

    float qs[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) qs[n][c] = qs_s[n * 8 + 2 * t + c], lim[n][c] = lim_s[n * 8 + 2 * t + c];

    float o[NT][C::MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < C::MT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][i][c] = 0.f;
    }

    const int32_t *table = p.tables + (int64_t)b * p.table_stride;
    const int page_blocks = p.page_shift - 4;  // blocks of 16 keys of a page, as a shift
    // where block blk (16 keys) is in the cache, and how many of its keys there are
    auto locate = [&](int blk, At &at, int &valid) {
      const int64_t left = keys - (int64_t)blk * 16;
      valid = left > 16 ? 16 : left < 0 ? 0 : (int)left;
      at = {0, 0};
      if (valid > 0) {
        const int32_t page = __ldg(table + (blk >> page_blocks));
        if (page < 0 || page >= p.pages) {
          if (lane == 0) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
          valid = 0;
        } else {
          const int64_t offset = (int64_t)(blk & ((1 << page_blocks) - 1)) << 4;
          at = {page * p.cp + h * p.ch + offset * p.ct, page * p.sp + h * p.sh + offset * p.st};
        }
      }
    };

    Keys<F, D, NT, BLK> x[C::M2];
    At row[C::M2];
    int valid[C::M2], unit = from + warp;
    if (unit < to) {
#pragma unroll
      for (int j = 0; j < C::M2; ++j) {
        locate(unit * C::M2 + j, row[j], valid[j]);
        load_k<F, D, NT, BLK>(x[j], p, row[j], valid[j], g, t);
      }
#pragma unroll
      for (int j = 0; j < C::M2; ++j) load_v<F, D, NT, BLK>(x[j], p, row[j], valid[j], g, t);
    }
    for (; unit < to; unit += WARPS) {
      float s[C::M2][NT][4], iv[C::M2][2], lv[C::M2][2];
      int ve[C::M2][2], seen[C::M2];
#pragma unroll
      for (int j = 0; j < C::M2; ++j) {
        seen[j] = valid[j];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[j][n][c] = 0.f;
        float krow[2];
        uint32_t kr[2][BLK ? C::KCH : 1];
        if constexpr (BLK) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t pk = x[j].kt[i] | (x[j].vs[i] << 16);
#pragma unroll
            for (int q = 1; q < 4; q <<= 1) {
              const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, pk, q);
              asm("max.u16x2 %0, %0, %1;" : "+r"(pk) : "r"(other));
            }
            const uint32_t kt = pk & 0xFFFFu, vt = pk >> 16;
            const int ke = RowRef<F>::exponent(kt);
            ve[j][i] = RowRef<F>::exponent(vt);
            // a NaN scale makes the whole row NaN
            krow[i] = kt > 0x7F80u ? __uint_as_float(0x7FC00000u) : RowRef<F>::value(ke);
            iv[j][i] = vt > 0x7F80u ? __uint_as_float(0x7FC00000u) : RowRef<F>::inverse(ve[j][i]);
            lv[j][i] = (float)(ve[j][i] - 127);
#pragma unroll
            for (int c = 0; c < C::KCH; ++c) {
              const float r = __uint_as_float(x[j].ks[i][c] << 16) * RowRef<F>::inverse(ke);
              kr[i][c] = pack_f16(r, r);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            krow[i] = __uint_as_float(x[j].ks[i][0] << 16);
            float vsc = __uint_as_float(x[j].vs[i] << 16);
            vsc = vsc < 0x1p-120f ? 0x1p-120f : vsc;  // a scale of zero: weight without a value
            iv[j][i] = 1.f / vsc;
            lv[j][i] = lg2(vsc);
          }
        }
        // s^T = K q^T
#pragma unroll
        for (int c = 0; c < C::KCH; ++c)
#pragma unroll
          for (int w = 0; w < C::KCW; ++w) {
            constexpr int STEPS = C::bits == 8 ? 1 : 2;
            uint32_t a[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t word = x[j].k[i][c * C::KCW + w];
              if constexpr (C::bits == 8) decode4_8bit<F>(word, a[i][0], a[i][1]);
              else decode8_4<F>(word, a[i]);
              if constexpr (BLK)
#pragma unroll
                for (int y = 0; y < 2 * STEPS; ++y) a[i][y] = hmul2(a[i][y], kr[i][c]);
            }
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
              const uint32_t frag[4] = {a[0][2 * st], a[1][2 * st], a[0][2 * st + 1], a[1][2 * st + 1]};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint2 bq = *reinterpret_cast<const uint2 *>(
                    &qf[((n * C::KS + c * (C::KEC / 4) + w * STEPS + st) * 32 + lane) * 2]);
                gemv::mma16816(s[j][n], frag, bq.x, bq.y);
              }
            }
          }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[j][n][c] *= krow[c >> 1];
      }
      // the next keys: their registers are free
      const int next = unit + WARPS;
      At nrow[C::M2];
      int nvalid[C::M2];
      if (next < to) {
#pragma unroll
        for (int j = 0; j < C::M2; ++j) {
          locate(next * C::M2 + j, nrow[j], nvalid[j]);
          load_k<F, D, NT, BLK>(x[j], p, nrow[j], nvalid[j], g, t);
        }
      }
      // u = s + log2 vs; keys that a row does not see: -inf
      bool up = false;
#pragma unroll
      for (int j = 0; j < C::M2; ++j) {
        const int tok = 4 * (g >> 1) + (g & 1), base = (unit * C::M2 + j) * 16 + tok;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = c >> 1, col = c & 1;
            const bool in = tok + 2 * i < seen[j] && base + 2 * i < lim[n][col];
            s[j][n][c] = in ? fmaf(s[j][n][c], qs[n][col], lv[j][i]) : -INFINITY;
            up |= s[j][n][c] > m[n][col] + LAZY;
          }
      }
      if (__any_sync(0xFFFFFFFFu, up)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int col = 0; col < 2; ++col) {
            float top = m[n][col];
#pragma unroll
            for (int j = 0; j < C::M2; ++j) top = fmaxf(top, fmaxf(s[j][n][col], s[j][n][col + 2]));
#pragma unroll
            for (int q = 4; q < 32; q <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, q));
            const float f = m[n][col] == -INFINITY ? 0.f : ex2(m[n][col] - top);
            m[n][col] = top;
            l[n][col] *= f;
#pragma unroll
            for (int i = 0; i < C::MT; ++i) o[n][i][col] *= f, o[n][i][col + 2] *= f;
          }
      }
#pragma unroll
      for (int j = 0; j < C::M2; ++j) {
        uint32_t bp[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float pr[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float mm = m[n][c & 1] == -INFINITY ? 0.f : m[n][c & 1] - BIAS;
            pr[c] = ex2(s[j][n][c] - mm);
            if (pr[c] != 0.f) l[n][c & 1] = fmaf(pr[c], iv[j][c >> 1], l[n][c & 1]);  // an unseen key's scale may be NaN
          }
          bp[n][0] = movmatrix_trans(pack_f16(pr[0], pr[1]));
          bp[n][1] = movmatrix_trans(pack_f16(pr[2], pr[3]));
        }
        uint32_t vr[2][BLK ? C::VCH : 1];  // scales of this lane's block of values, tokens in pairs
        if constexpr (BLK) {
          // keys 4t .. 4t + 3 are rows 2t, 2t + 1 of the scores: key 4t + i sits in lane 8t + 4 (i & 1)
          float inv[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ex = __shfl_sync(0xFFFFFFFFu, ve[j][i >> 1], 8 * t + 4 * (i & 1) + t);
            inv[i] = RowRef<F>::inverse(ex);
          }
#pragma unroll
          for (int c = 0; c < C::VCH; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              vr[i][c] = pack_f16(__uint_as_float(number(x[j].vb[2 * i][c]) << 16) * inv[2 * i],
                                  __uint_as_float(number(x[j].vb[2 * i + 1][c]) << 16) * inv[2 * i + 1]);
        }
        // out^T += V^T p^T
#pragma unroll
        for (int c = 0; c < C::VCH; ++c)
#pragma unroll
          for (int w = 0; w < C::VCW; ++w) {
            constexpr int DW = 32 / C::bits;  // values of a word
            uint32_t f[2][DW];                // [tokens (0, 1) or (2, 3)][value]
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w0 = x[j].v[2 * i][c * C::VCW + w], w1 = x[j].v[2 * i + 1][c * C::VCW + w];
              if constexpr (C::bits == 8) {
                decode4_8bit<F>(__byte_perm(w0, w1, 0x5140), f[i][0], f[i][1]);
                decode4_8bit<F>(__byte_perm(w0, w1, 0x7362), f[i][2], f[i][3]);
              } else if constexpr (F == B200_CACHE_INT4) {
                uint32_t lo[4], hi[4];
                decode8_4<F>(__byte_perm(w0, w1, 0x5410), lo);
                decode8_4<F>(__byte_perm(w0, w1, 0x7632), hi);
#pragma unroll
                for (int q = 0; q < 4; ++q) f[i][q] = lo[q], f[i][q + 4] = hi[q];
              } else {
                uint32_t ev[4], od[4];
                decode8_4<F>((w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), ev);
                decode8_4<F>(((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), od);
#pragma unroll
                for (int q = 0; q < 4; ++q) f[i][2 * q] = ev[q], f[i][2 * q + 1] = od[q];
              }
              if constexpr (BLK)
#pragma unroll
                for (int q = 0; q < DW; ++q) f[i][q] = hmul2(f[i][q], vr[i][c]);
            }
#pragma unroll
            for (int q = 0; q < DW / 2; ++q) {
              const uint32_t frag[4] = {f[0][2 * q], f[0][2 * q + 1], f[1][2 * q], f[1][2 * q + 1]};
              const int mt = (c * C::VCW + w) * (DW / 2) + q;
#pragma unroll
              for (int n = 0; n < NT; ++n) gemv::mma16816(o[n][mt], frag, bp[n][0], bp[n][1]);
            }
          }
      }
      if (next < to) {
#pragma unroll
        for (int j = 0; j < C::M2; ++j) {
          row[j] = nrow[j], valid[j] = nvalid[j];
          load_v<F, D, NT, BLK>(x[j], p, row[j], valid[j], g, t);
        }
      }
    }

    // join the warps: numerators [row][value] of each in shared memory
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int col = 0; col < 2; ++col) {
#pragma unroll
        for (int q = 4; q < 32; q <<= 1) l[n][col] += __shfl_xor_sync(0xFFFFFFFFu, l[n][col], q);
        const int r = n * 8 + 2 * t + col;
        if (g == 0) join_m[warp * C::ROWS + r] = m[n][col], join_l[warp * C::ROWS + r] = l[n][col];
        float *dst = join_o + (warp * C::ROWS + r) * C::ORS;
#pragma unroll
        for (int i = 0; i < C::MT; ++i) {
          constexpr int PER = C::VEC / 2;  // tiles of a chunk
          const int d = (g + 8 * (i / PER)) * C::VEC + 2 * (i % PER);
          *reinterpret_cast<float2 *>(dst + d) = make_float2(o[n][i][col], o[n][i][col + 2]);
        }
      }
    __syncthreads();
    const bool whole = from == 0 && to == units;
    const int64_t c0 = seg0 / per, c1 = (seg1 - 1) / per;  // CTAs of the segment
    const int slot = (int)(2 * blockIdx.x + (from == 0 ? 1 : 0));
    for (int i = tid; i < C::ROWS * (D / 4); i += THREADS) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, join_m[w * C::ROWS + r]);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float mw = join_m[w * C::ROWS + r], f = mw == -INFINITY ? 0.f : ex2(mw - M);
        const float4 y = *reinterpret_cast<const float4 *>(join_o + (w * C::ROWS + r) * C::ORS + d);
        a.x += y.x * f, a.y += y.y * f, a.z += y.z * f, a.w += y.w * f;
        L += join_l[w * C::ROWS + r] * f;
      }
      // NaN has no order: a warp whose scores are NaN keeps m = -inf but a NaN denominator
#pragma unroll
      for (int w = 0; w < WARPS; ++w)
        if (join_l[w * C::ROWS + r] != join_l[w * C::ROWS + r]) L = a.x = a.y = a.z = a.w = __uint_as_float(0x7FC00000u);
      if (whole) {
        if (r < n_rows) finish<T, D>(p, row_at(p, b, h, r0 + r).out, d, a, M, L);
      } else {
        *reinterpret_cast<float4 *>(p.ws_o + ((int64_t)slot * C::ROWS + r) * D + d) = a;
        if (d == 0) *reinterpret_cast<float2 *>(p.ws_ml + ((int64_t)slot * C::ROWS + r) * 2) = make_float2(M, L);
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) last = atomicAdd(&p.tickets[c0], 1u) == (uint32_t)(c1 - c0);
      __syncthreads();
      if (last) {
        __threadfence();
        for (int i = tid; i < n_rows * (D / 4); i += THREADS) {
          const int r = i / (D / 4), d = (i % (D / 4)) * 4;
          float M = -INFINITY, L = 0.f;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          bool nan = false;
          for (int64_t c = c0; c <= c1; ++c) {
            const int64_t sl = (2 * c + (c == c0 ? 1 : 0)) * C::ROWS + r;
            M = fmaxf(M, __ldcg((const float2 *)(p.ws_ml + sl * 2)).x);
          }
#pragma unroll 4
          for (int64_t c = c0; c <= c1; ++c) {
            const int64_t sl = (2 * c + (c == c0 ? 1 : 0)) * C::ROWS + r;
            const float2 ml = __ldcg((const float2 *)(p.ws_ml + sl * 2));
            const float4 y = __ldcg((const float4 *)(p.ws_o + sl * D + d));
            const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
            a.x += y.x * f, a.y += y.y * f, a.z += y.z * f, a.w += y.w * f;
            L += ml.y * f;
            nan |= ml.y != ml.y;
          }
          if (nan) L = a.x = a.y = a.z = a.w = __uint_as_float(0x7FC00000u);
          finish<T, D>(p, row_at(p, b, h, r0 + r).out, d, a, M, L);
        }
        if (tid == 0) p.tickets[c0] = 0u;  // ready for the next call on this workspace
      }
    }
    u = seg0 + to;
  }
}

// ---- per-(device, stream) workspace of split segments ---------------------------------------------
struct Workspace {
  float *o = nullptr, *ml = nullptr;
  uint32_t *tickets = nullptr;
  int grid = 0;
};
constexpr int MAX_ROWS_D = 16 * 128;  // ROWS * D of every variant is at most this

static std::mutex g_ws_mutex;
static std::map<std::pair<int, cudaStream_t>, Workspace> g_ws;

static int32_t workspace_for(cudaStream_t stream, Workspace &out) {
  int dev = 0, sms = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  B200_CUDA_TRY(device_sms(&sms));
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  auto it = g_ws.find({dev, stream});
  if (it != g_ws.end()) {
    out = it->second;
    return B200_OK;
  }
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  B200_CUDA_TRY(cudaStreamIsCapturing(stream, &cs));
  Workspace w;
  w.grid = 2 * sms;
  if (cs != cudaStreamCaptureStatusNone) {  // nothing can be allocated while capturing: whole segments
    out = w;
    return B200_OK;
  }
  const size_t slots = 2 * (size_t)w.grid;
  const size_t o_bytes = slots * MAX_ROWS_D * 4, ml_bytes = slots * 16 * 2 * 4, t_bytes = (size_t)w.grid * 4;
  uint8_t *base = nullptr;
  B200_CUDA_TRY(cudaMalloc((void **)&base, o_bytes + ml_bytes + t_bytes));
  w.o = (float *)base, w.ml = (float *)(base + o_bytes), w.tickets = (uint32_t *)(base + o_bytes + ml_bytes);
  // on the caller's stream, the only one that uses this workspace
  cudaError_t err = cudaMemsetAsync(w.tickets, 0, t_bytes, stream);
  if (err != cudaSuccess) {
    cudaFree(base);
    return b200_set_error(B200_ERR_CUDA, "cache_attention workspace: %s", cudaGetErrorString(err));
  }
  g_ws[{dev, stream}] = w;
  out = w;
  return B200_OK;
}

template <typename T, int F, int D, int NT, bool BLK>
static int32_t launch_t(Params p, cudaStream_t stream) {
  using C = Cfg<F, D, NT>;
  p.row_tiles = (p.rows + C::ROWS - 1) / C::ROWS;
  if (p.row_tiles > MAX_ENTRIES)
    return b200_set_error(B200_ERR_UNSUPPORTED, "cache_attention: too many query rows (%d of a key head)", p.rows);
  const int at_once = MAX_ENTRIES / p.row_tiles;
  if (p.batch > at_once) {  // a launch for each run of requests that the scan has room for
    const int all = p.batch;
    const Params base = p;
    for (int b = 0; b < all; b += at_once) {
      p = base;
      p.batch = all - b < at_once ? all - b : at_once;
      const int64_t rows = (int64_t)b * p.per_request * p.q_heads;
      p.q = (const T *)p.q + b * p.qsr;
      p.tables += b * p.table_stride, p.lengths += b;
      p.out = (T *)p.out + rows * D;
      if (p.lse != nullptr) p.lse += rows;
      if (p.fo != nullptr) p.fo += rows * D, p.fm += rows, p.fl += rows;
      if (int32_t rc = launch_t<T, F, D, NT, BLK>(p, stream)) return rc;
    }
    return B200_OK;
  }
  const int64_t entries = (int64_t)p.batch * p.row_tiles;
  Workspace w;
  if (int32_t rc = workspace_for(stream, w)) return rc;
  p.ws_o = w.o, p.ws_ml = w.ml, p.tickets = w.tickets;
  B200_CUDA_TRY((ensure_dynamic_smem<attn_kernel<T, F, D, NT, BLK>>(C::SMEM)));
  // no more CTAs than there can be runs of 2 * WARPS units
  const int64_t unit = 16 * C::M2;
  const int64_t cap = p.lengths != nullptr ? ((int64_t)p.max_pages << p.page_shift) : p.fixed;
  const int64_t most = entries * p.kv_heads * ((cap + unit - 1) / unit);
  int64_t grid = (most + 2 * WARPS - 1) / (2 * WARPS);
  const int64_t full = (D == 256 || NT == 2) ? w.grid / 2 : w.grid;
  if (grid > full) grid = full;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn_kernel<T, F, D, NT, BLK>, p));
  return B200_OK;
}

template <typename T, int F>
static int32_t launch_d(const Params &p, int dim, bool blk, cudaStream_t stream) {
  const bool two = p.rows > 8;  // 16 query rows share a pass over the keys
  if (dim == 64) {
    if (two) return blk ? launch_t<T, F, 64, 2, true>(p, stream) : launch_t<T, F, 64, 2, false>(p, stream);
    return blk ? launch_t<T, F, 64, 1, true>(p, stream) : launch_t<T, F, 64, 1, false>(p, stream);
  }
  if (dim == 128) {
    if (two) return blk ? launch_t<T, F, 128, 2, true>(p, stream) : launch_t<T, F, 128, 2, false>(p, stream);
    return blk ? launch_t<T, F, 128, 1, true>(p, stream) : launch_t<T, F, 128, 1, false>(p, stream);
  }
  return blk ? launch_t<T, F, 256, 1, true>(p, stream) : launch_t<T, F, 256, 1, false>(p, stream);
}
template <typename T>
static int32_t launch_f(const Params &p, int fmt, int dim, bool blk, cudaStream_t stream) {
  switch (fmt) {
    case B200_CACHE_INT8: return launch_d<T, B200_CACHE_INT8>(p, dim, blk, stream);
    case B200_CACHE_FP8E4M3: return launch_d<T, B200_CACHE_FP8E4M3>(p, dim, blk, stream);
    case B200_CACHE_INT4: return launch_d<T, B200_CACHE_INT4>(p, dim, blk, stream);
    default: return launch_d<T, B200_CACHE_FP4_E2M1>(p, dim, blk, stream);
  }
}

static int32_t attention(const b200_cache_desc *c, const b200_attention_args *a, cudaStream_t stream) {
  Params p = {};
  const int dim = c->head_dim;
  p.q = a->q;
  p.qsr = a->q_strides[0], p.qsb = a->q_strides[1], p.qsh = a->q_strides[2];
  p.k = (const uint8_t *)c->k, p.v = (const uint8_t *)c->v, p.ks = c->k_scales, p.vs = c->v_scales;
  p.cp = c->strides[0], p.ch = c->strides[1], p.ct = c->strides[2];
  p.sp = c->scale_strides[0], p.sh = c->scale_strides[1], p.st = c->scale_strides[2];
  p.e8m0 = c->scale_dtype == B200_DT_E8M0;
  p.pages = c->pages, p.kv_heads = c->kv_heads, p.group = a->heads / c->kv_heads, p.q_heads = a->heads;
  while ((1 << p.page_shift) < c->page_size) ++p.page_shift;
  p.scale = a->scale * 1.44269504088896341f;
  p.per_request = a->queries;
  const bool blk = c->block_size != dim;
  const int64_t all_rows = (int64_t)a->batch * a->queries * a->heads;
  auto run = [&](const Params &q) {
    return a->q_dtype == B200_DT_F16 ? launch_f<__half>(q, c->format, dim, blk, stream)
                                     : launch_f<__nv_bfloat16>(q, c->format, dim, blk, stream);
  };
  if (a->prefix_length > 0) {
    Params f = p;  // every row of the batch against the prefix: one request of batch * queries tokens
    f.tables = a->prefix, f.table_stride = 0, f.max_pages = (int)a->prefix_pages;
    f.fixed = a->prefix_length, f.batch = 1, f.queries = (int)(a->batch * a->queries), f.rows = f.queries * p.group;
    f.po = (float *)a->scratch, f.pm = f.po + all_rows * dim, f.pl = f.pm + all_rows;
    if (int32_t rc = run(f)) return rc;
    p.fo = f.po, p.fm = f.pm, p.fl = f.pl;
  }
  p.tables = a->tables, p.table_stride = a->table_stride, p.max_pages = (int)a->max_pages, p.lengths = a->lengths;
  p.batch = (int)a->batch, p.queries = (int)a->queries, p.rows = p.queries * p.group, p.causal = 1;
  p.out = a->out, p.lse = a->lse;
  return run(p);
}

}  // namespace cattn
}  // namespace b200

// ---- C entries ---------------------------------------------------------------------------------
using namespace b200;

extern "C" {

int64_t b200_cache_attention_scratch(int64_t batch, int64_t queries, int32_t heads, int32_t head_dim, int64_t prefix_length) {
  if (batch < 0 || queries < 0 || heads < 0 || head_dim < 0 || prefix_length <= 0) return 0;
  return batch * queries * heads * ((int64_t)head_dim + 2) * 4;
}

int32_t b200_cache_attention(const b200_cache_desc *c, const b200_attention_args *a, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (int32_t rc = check_cache(c)) return rc;
  if (a == nullptr) return b200_set_error(B200_ERR_INVALID, "cache_attention: null arguments");
  if (a->q_dtype != B200_DT_F16 && a->q_dtype != B200_DT_BF16)
    return b200_set_error(B200_ERR_INVALID, "cache_attention: q must be float16 or bfloat16 (got dtype %d)", a->q_dtype);
  if (a->batch < 0 || a->queries < 0 || a->heads < 1 || a->heads % c->kv_heads != 0)
    return b200_set_error(B200_ERR_INVALID, "cache_attention: %d heads over %d key heads", a->heads, c->kv_heads);
  if (a->max_pages < 0 || a->table_stride < 0 || a->prefix_pages < 0 || a->prefix_length < 0 ||
      a->prefix_length > a->prefix_pages * c->page_size)
    return b200_set_error(B200_ERR_INVALID, "cache_attention: bad table sizes");
  if (a->batch == 0 || a->queries == 0) return B200_OK;
  if (a->batch * a->queries * a->heads > INT32_MAX || a->max_pages * c->page_size > INT32_MAX - 64 ||
      a->prefix_pages * c->page_size > INT32_MAX - 64)
    return b200_set_error(B200_ERR_UNSUPPORTED, "cache_attention: more rows or keys than 32-bit counts hold");
  if (a->q == nullptr || a->out == nullptr || a->lengths == nullptr || (a->tables == nullptr && a->max_pages > 0) ||
      (a->prefix_length > 0 && (a->prefix == nullptr || a->scratch == nullptr)))
    return b200_set_error(B200_ERR_INVALID, "cache_attention: null pointer");
  if ((uintptr_t)a->out % 16 || (uintptr_t)a->scratch % 16)
    return b200_set_error(B200_ERR_INVALID, "cache_attention: out and scratch must start on 16-byte boundaries");
  try {
    return cattn::attention(c, a, (cudaStream_t)stream);
  } catch (...) {
    return b200_set_error(B200_ERR_CUDA, "cache_attention: out of host memory");
  }
}

}  // extern "C"
