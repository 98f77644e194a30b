// cache_attn_mma.cu -- attention of many query rows over the packed key/value cache, on the tcgen05 cores.
//
// The mathematics is cache_attn.cu's (base 2, u = s + log2 vs, codes as fp16 operands); here a tile of
// 128 query rows meets tiles of 128 keys: s = Q K^T (M = 128, N = 128, K = D) and O += p V (M = 128,
// N = D, K = 128) as tcgen05.mma with accumulators in tensor memory. Rows are those that see the same
// keys: all requests' heads of a key head over a shared prefix, or the tokens of a prompt's chunk times
// the heads of a group. One CTA an SM, 16 warps:
//   warps 0..7    two softmax warpgroups, a thread a row: scores from tensor memory, p back into it in
//                 the scores' place as the second product's left operand; O stays in tensor memory and
//                 is only touched when a row's maximum has grown by more than 2^4;
//   warps 8..11   codes -> fp16 into swizzled tiles in shared memory: keys row by row; values eight keys
//                 at a time, turned on the way so that keys are contiguous (pairs of keys are joined by
//                 byte permutes before they are decoded). Codes of the next tile are in registers;
//   warps 12, 13  one lane each issues a slot's MMAs (14, 15 are there for the registers' split).
// Two row tiles share every decoded key tile (256 rows); with up to 128 rows both warpgroups take the
// same rows and every other key tile each, and add up at the end. While one slot is in its softmax the
// other's products run. What bounds it: a tile pair is 2048 cycles of MMA, as many of the special
// function unit (one exponential a score) and about 9000 issue slots of four schedulers. It takes some
// 5300 cycles: a softmax (2400) and the round trip of its products (2650) follow one another in each
// slot, and the two slots fill each other's gaps only in part.
// Measured (bf16, 8 key heads of 128, device time): 1024 tokens of 32 heads against 8192 fp8 keys 215 us
// = 600 TFLOP/s (the few-row kernel 1087); 128 requests of 64 heads behind 16384 int4 keys, with their
// own 1 to 1024, 193 us (595).
//
// Tiles of all (row tile, key head) segments are laid end to end and cut into equal runs, one per CTA.
// A segment within a run is finished there; the others leave their share (numerators, maximum,
// denominator) in the CTA's two workspace slots, and join_kernel adds those up.
#include "cache_attn.cuh"
#include "sm100.cuh"

namespace b200 {

int32_t cache_attn_mma_device_error(unsigned int *v, bool clear) {
  B200_CUDA_TRY(tu_device_error(v, clear));
  return B200_OK;
}

namespace cattn {
namespace mma {

constexpr int KT = 128;                      // keys of a tile
constexpr int WG = 128, THREADS = 4 * WG;
// 128 x (2 x 168 + 120 + 56) = 512 x 128, the registers that the block is launched with
constexpr int SOFT_REGS = 168, DECODE_REGS = 120, ISSUE_REGS = 56;
constexpr int MAX_ENTRIES = 1024;
constexpr uint64_t WAIT_NS = 2000000000ull;

template <int F, int D, bool BLK>
struct Cfg {
  static constexpr int bits = CFmt<F>::bits;
  static constexpr int RB = D * bits / 8;
  static constexpr int U = 8, UD = D / U, UB = UD * bits / 8, UW = UB / 4;  // units of a row, values, bytes, words of one
  static constexpr int NB = D / 32, KNB = BLK ? NB : 1;
  static constexpr int QB = 128 * D * 2, KB = KT * D * 2, VB = KT * D * 2;
  static constexpr int RING = 4;                                            // tiles of scales
  static constexpr int SC = RING * KT * 12, RATIO = 2 * KNB * KT * 2;
  // scale exponents of a tile may differ by this for its codes to take them with all their bits in fp16
  static constexpr int SPAN = bits == 4 ? 24 : 11;
  static constexpr bool FOLD = BLK || bits == 4;                            // key codes always take their scales
  static constexpr int SMEM = 1024 + 2 * QB + 2 * KB + 2 * VB + SC + 2 * RATIO + 256;
};

// Pairs of fp32 in a register pair: one instruction for two.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ void unpair(uint64_t x, uint32_t &a, uint32_t &b) { asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(x)); }
__device__ __forceinline__ void unpair(uint64_t x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

__device__ __forceinline__ float2 wide2(const Params &p, uint32_t w) {
  if (p.q_bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <int D>
__device__ __forceinline__ void finish_any(const Params &p, int64_t row, int d, float4 o, float m, float l) {
  if (p.q_bf16) finish<__nv_bfloat16, D>(p, row, d, o, m, l);
  else finish<__half, D>(p, row, d, o, m, l);
}

__device__ __forceinline__ int length_of(const Params &p, int b) {
  const int64_t cap = (int64_t)p.max_pages << p.page_shift;
  const int64_t n = p.lengths != nullptr ? p.lengths[b] : p.fixed;
  return (int)(n < 0 ? 0 : n > cap ? cap : n);
}
__device__ __forceinline__ int keys_of(const Params &p, int e, int tile_rows) {
  const int b = p.row_tiles == 1 ? e : e / p.row_tiles, n = length_of(p, b);
  if (!p.causal) return n;
  const int r1 = min(p.rows, (e - b * p.row_tiles + 1) * tile_rows) - 1;
  return max(0, n - p.queries + r1 / p.group + 1);
}
// Tiles of a key head before each entry (request, row tile), by the first warp.
__device__ __forceinline__ void scan_entries(const Params &p, int tile_rows, uint32_t *prefix) {
  const int entries = p.batch * p.row_tiles, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    uint32_t carry = 0;
    for (int e0 = 0; e0 < entries; e0 += 32) {
      const int e = e0 + lane;
      const uint32_t n = e < entries ? ((uint32_t)keys_of(p, e, tile_rows) + KT - 1) / KT : 0;
      uint32_t inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      if (e < entries) prefix[e] = carry + inc - n;
      carry += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    if (lane == 0) prefix[entries] = carry;
  }
}

// A run of tiles, segment part by segment part.
struct Part {
  uint32_t u, u_end;         // where the run stands, and its end
  uint32_t seg0, tiles;      // the segment's first tile, and how many it has
  uint32_t from, to;         // this part of it
  int e, h, b, keys;
};

struct Bars {
  uint64_t qfull[2], sfull[2], pfull[2][2], pvdone[2], kfull[2], kfree[2], vfull[2], vfree[2], scfull[4];
  uint64_t done[3];  // one row tile: the first warpgroup's products; the second's share; that share's reading
  uint64_t drain[2]; // an issuer that gave up: its products in flight
};

// All N threads of barrier ID meet; whether every one of them is `ok`.
template <int ID, int N>
__device__ __forceinline__ bool meet(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok), "n"(ID), "n"(N)
      : "memory");
  return all != 0;
}

template <int REGS> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

// tcgen05.mma and its commit by one lane of a converged warp.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

// Value d (a multiple of four) of row `place` (slot * rows + row) of the shares of cut segments: four values of
// all rows side by side, as a thread a row writes them.
template <int D>
__device__ __forceinline__ int64_t cut_at(int64_t place, int rows, int d) {
  const int64_t slot = place / rows;
  return (slot * (D / 4) + d / 4) * rows * 4 + (place - slot * rows) * 4;
}

// Byte of 16-byte chunk g (8 values) of row r in a K-major tile of `rows` rows, 64 values a swizzled row.
__device__ __forceinline__ uint32_t tile_at(int rows, int r, int g) {
  return (uint32_t)((g >> 3) * rows * 128 + r * 128 + (((g & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// The type of q and out is a matter of a few instructions a row: a run-time one.
template <int F, int D, int RT, bool BLK>
__global__ void __launch_bounds__(THREADS, 1) attn_mma_kernel(const Params p) {
  using C = Cfg<F, D, BLK>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *qt = smem, *kt = qt + 2 * C::QB, *vt = kt + 2 * C::KB;
  float *sc = (float *)(vt + 2 * C::VB);             // [RING][key scale | log2 value scale | its inverse][KT]
  __half *kratio = (__half *)((uint8_t *)sc + C::SC), *vratio = kratio + C::RATIO / 2;  // [2][NB][KT]
  __shared__ Bars bars;
  __shared__ uint32_t prefix[MAX_ENTRIES + 1];
  __shared__ float2 share_ml[RT == 1 ? 128 : 1];
  __shared__ float4 tile_s[C::RING];   // (key scale, log2 of the value scale, its inverse, keys differ) of a tile
  __shared__ uint32_t span_s[2][4][5]; // of a warp's keys: largest and smallest exponents, any to be looked at one by one
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;
  volatile uint32_t *abort_flag = &abort_word;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int TR = 128 * RT;  // rows of a segment
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.qfull[i], WG), mbar_init(&bars.sfull[i], 1), mbar_init(&bars.pfull[i][0], WG), mbar_init(&bars.pfull[i][1], WG), mbar_init(&bars.pvdone[i], 1);
      mbar_init(&bars.kfull[i], WG), mbar_init(&bars.kfree[i], RT), mbar_init(&bars.vfull[i], WG), mbar_init(&bars.vfree[i], RT);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bars.scfull[i], WG);
    for (int i = 0; i < 3; ++i) mbar_init(&bars.done[i], WG);
    for (int i = 0; i < 2; ++i) mbar_init(&bars.drain[i], 1);
    abort_word = 0;
    fence_mbar_init();
  }
  scan_entries(p, TR, prefix);
  if (warp == 12) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int entries = p.batch * p.row_tiles, heads = p.kv_heads;
  const uint32_t total = prefix[entries] * (uint32_t)heads;
  const uint32_t per = max(1u, (total + gridDim.x - 1) / gridDim.x);

  // rows without a key: zeros (or what the prefix gave)
  for (int e = blockIdx.x; e < entries; e += gridDim.x) {
    if (prefix[e + 1] != prefix[e]) continue;
    const int b = p.row_tiles == 1 ? e : e / p.row_tiles, rt = e - b * p.row_tiles;
    const int n = min(TR, p.rows - rt * TR);
    for (int i = tid; i < heads * n * (D / 4); i += THREADS) {
      const int d = (i % (D / 4)) * 4, rr = i / (D / 4);
      const RowAt at = row_at(p, b, rr / n, rt * TR + rr % n);
      finish_any<D>(p, at.out, d, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
  }

  auto enter = [&](Part &w) {  // the segment of w.e, w.h, from w.u on
    w.tiles = prefix[w.e + 1] - prefix[w.e];
    w.seg0 = prefix[w.e] * heads + w.h * w.tiles;
    w.b = p.row_tiles == 1 ? w.e : w.e / p.row_tiles;
    w.keys = keys_of(p, w.e, TR);
    w.from = w.u - w.seg0;
    w.to = min(w.u_end - w.seg0, w.tiles);
  };
  auto next = [&](Part &w) {  // on to the next part; false at the end of the run
    w.u = w.seg0 + w.tiles;
    if (w.u >= w.u_end) return false;
    if (++w.h == heads) {
      w.h = 0;
      do ++w.e;
      while (prefix[w.e + 1] == prefix[w.e]);
    }
    enter(w);
    return true;
  };
  auto begin = [&](Part &w) {
    w.u = min(total, blockIdx.x * per);
    w.u_end = min(total, w.u + per);
    if (w.u >= w.u_end) return false;
    int lo = 0, hi = entries;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] * heads <= w.u) lo = mid;
      else hi = mid;
    }
    w.e = lo;
    w.h = (int)((w.u - prefix[lo] * heads) / (prefix[lo + 1] - prefix[lo]));
    enter(w);
    return true;
  };
  // Key codes take their scales before the products. With 8-bit codes and bfloat16 scales that rounds their
  // 15 bits to fp16's 11, 2^-12 at random: far below a bfloat16 result's half unit of 2^-8, but not below what
  // fp16 results and logarithms keep, whose scores take their key's scale instead.
  const bool fold = C::FOLD || p.e8m0 || (p.q_bf16 && p.lse == nullptr && p.exact_keys == 0);
  const int page_blocks = p.page_shift - 4;
  const uint32_t in_page = (1u << page_blocks) - 1;

  if (warp < 8) {
    // ================ softmax: thread = row of slot `slot` ================
    reg_inc<SOFT_REGS>();
    const int slot = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + (uint32_t)slot * 128, to = tmem + lanes + 256 + slot * D;
    uint32_t n0 = 0, ops = 0, parts = 0;  // tiles of the CTA so far; this slot's operations and parts
    Part w;
    bool alive = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {  // the warp's answer: what follows is for whole warps
      return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, WAIT_NS)) != 0;
    };
    for (bool more = begin(w); more && alive; more = next(w), ++parts) {
      const int rt = w.e - w.b * p.row_tiles, row = rt * TR + (RT == 2 ? slot * 128 : 0) + r;
      const bool in = row < p.rows;
      const int len = length_of(p, w.b);
      const int lim = !in ? 0 : p.causal ? len - p.queries + row / p.group + 1 : len;
      const RowAt at = in ? row_at(p, w.b, w.h, row) : RowAt{0, 0};
      const uint32_t first = RT == 2 ? w.from : w.from + ((n0 ^ slot) & 1);  // this slot's tiles: first, first + RT's step
      constexpr uint32_t STEP = RT == 2 ? 1 : 2;
      float m = -INFINITY, l = 0.f, qs = 0.f;
      const uint32_t ops0 = ops;
      if (first < w.to) {
        // q: fp16, scaled by a power of two, in the order that the keys' codes come out decoded
        // (a warp does its own 32 rows, whole rows at a time)
        constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes of a row, rows at once
        const int g = lane % LPR;
        uint32_t raw[LPR][4];
#pragma unroll
        for (int x = 0; x < LPR; ++x) {
          const int rr = x * RPI + lane / LPR;
          const int64_t q0 = __shfl_sync(0xFFFFFFFFu, at.q, rr);
          const bool there = __shfl_sync(0xFFFFFFFFu, (int)in, rr) != 0;
          const uint16_t *src = (const uint16_t *)p.q + q0 + 8 * g;
          if (!there) raw[x][0] = raw[x][1] = raw[x][2] = raw[x][3] = 0;
          else if (p.q_vec) lds<16>((const uint8_t *)src, raw[x]);
          else
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[x][i] = (uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16);
        }
        const uint32_t qa = smem_u32(qt + slot * C::QB);
#pragma unroll
        for (int x = 0; x < LPR; ++x) {
          float f[8], top = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = wide2(p, raw[x][i]);
            f[2 * i] = v.x, f[2 * i + 1] = v.y;
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
#pragma unroll
          for (int y = 1; y < LPR; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, y));
          const int ex = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
          const float down = copysignf(__uint_as_float((uint32_t)(254 - ex) << 23), p.scale);
          // not negative: the largest score is the largest product's
          const float up = __shfl_sync(0xFFFFFFFFu, fabsf(p.scale) * __uint_as_float((uint32_t)ex << 23), (lane % RPI) * LPR);
          if (lane / RPI == x) qs = up;
          uint32_t y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[i] = F == B200_CACHE_INT4 ? pack_f16(f[i] * down, f[i + 4] * down) : pack_f16(f[2 * i] * down, f[2 * i + 1] * down);
          sts128(qa + tile_at(128, (warp & 3) * 32 + x * RPI + lane / LPR, g), y[0], y[1], y[2], y[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&bars.qfull[slot]);
      }
      for (uint32_t j = first; j < w.to; j += STEP, ++ops) {
        const uint32_t n = n0 + (j - w.from);
        alive = wait(&bars.scfull[n & 3], (n >> 2) & 1) && wait(&bars.sfull[slot], ops & 1);
        if (!alive) break;
        tc_fence_after();
        const ulonglong2 *k4 = (const ulonglong2 *)(sc + (n & 3) * 3 * KT), *l4 = k4 + KT / 4, *i4 = l4 + KT / 4;
        const float4 tile = tile_s[n & 3];
        const bool edge = p.causal && __any_sync(0xFFFFFFFFu, (int)(j * KT + KT) > lim);  // keys that a row does not see
        // keys one by one: a tile that ends early, whose scales are far apart, or that some rows see in part
        const bool each = edge || tile.w != 0.f;
        const float qt_s = qs * tile.x;
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, most;
        uint32_t xa[32], xb[32];
        // `f` on the four chunks of 32 scores, the next chunk on its way meanwhile
        auto chunks = [&](auto f) {
          tmem_ld_32x32b_x32(ts, xa);
#pragma unroll 1
          for (int c = 0; c < 4; c += 2) {
            tmem_ld_wait();
            tmem_ld_32x32b_x32(ts + 32 * c + 32, xb);
            f(xa, c);
            tmem_ld_wait();
            if (c == 0) tmem_ld_32x32b_x32(ts + 64, xa);
            f(xb, c + 1);
          }
        };
        auto largest = [&](const uint32_t (&x)[32]) {
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            top[(i >> 1) & 3] = max3(top[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        };
        if (each) {  // u of every key in its score's place
          const uint64_t qs2 = pair(qs, qs);
          chunks([&](uint32_t(&x)[32], int c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const ulonglong2 k = k4[8 * c + i], a = l4[8 * c + i];
              unpair(fma2(mul2(pair(x[4 * i], x[4 * i + 1]), k.x), qs2, a.x), x[4 * i], x[4 * i + 1]);
              unpair(fma2(mul2(pair(x[4 * i + 2], x[4 * i + 3]), k.y), qs2, a.y), x[4 * i + 2], x[4 * i + 3]);
            }
            if (edge)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if ((int)(j * KT) + 32 * c + i >= lim) x[i] = 0xFF800000u;
            largest(x);
            tmem_st_32x32b_x32(ts + 32 * c, x);
          });
          tmem_st_wait();
          most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        } else if (fold) {  // one scale for all: it goes into the exponential's argument
          chunks([&](uint32_t(&x)[32], int) { largest(x); });
          most = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), qt_s, tile.y);
        } else {  // products take their key's scale
          chunks([&](uint32_t(&x)[32], int c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const ulonglong2 k = k4[8 * c + i];
              unpair(mul2(pair(x[4 * i], x[4 * i + 1]), k.x), x[4 * i], x[4 * i + 1]);
              unpair(mul2(pair(x[4 * i + 2], x[4 * i + 3]), k.y), x[4 * i + 2], x[4 * i + 3]);
            }
            largest(x);
            tmem_st_32x32b_x32(ts + 32 * c, x);
          });
          tmem_st_wait();
          most = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), qt_s, tile.y);
        }
        const bool up = most > m + LAZY;
        if (__any_sync(0xFFFFFFFFu, up)) {
          const float f = !up || m == -INFINITY ? 1.f : ex2(m - most);
          if (up) m = most, l *= f;
          if (ops != ops0) {  // what O holds
            alive = wait(&bars.pvdone[slot], (ops - 1) & 1);
            if (!alive) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(to + 16 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st_32x32b_x16(to + 16 * c, o);
            }
          }
        }
        const float mm = m == -INFINITY ? 0.f : m - BIAS;
        // the second product may begin with the first 64 keys
        auto half_done = [&]() {
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&bars.pfull[slot][0]);
        };
        // p of chunk c goes over the scores of chunk c / 2, which have been read
        uint64_t sum[2] = {0, 0};
        if (each) {
          const uint64_t mm2 = pair(-mm, -mm);
          chunks([&](uint32_t(&x)[32], int c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const ulonglong2 v = i4[8 * c + i];
              float e[4];
              unpair(add2(pair(x[4 * i], x[4 * i + 1]), mm2), e[0], e[1]);
              unpair(add2(pair(x[4 * i + 2], x[4 * i + 3]), mm2), e[2], e[3]);
#pragma unroll
              for (int y = 0; y < 4; ++y) e[y] = ex2(e[y]);
              sum[0] = fma2(pair(e[0], e[1]), v.x, sum[0]);
              sum[1] = fma2(pair(e[2], e[3]), v.y, sum[1]);
              pk[2 * i] = pack_f16(e[0], e[1]), pk[2 * i + 1] = pack_f16(e[2], e[3]);
            }
            tmem_st_32x32b_x16(ts + 16 * c, pk);
            if (c == 1) half_done();
          });
        } else {
          const uint64_t qs2 = pair(qt_s, qt_s), a2 = pair(tile.y - mm, tile.y - mm);
          chunks([&](uint32_t(&x)[32], int c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float e[4];
              unpair(fma2(pair(x[4 * i], x[4 * i + 1]), qs2, a2), e[0], e[1]);
              unpair(fma2(pair(x[4 * i + 2], x[4 * i + 3]), qs2, a2), e[2], e[3]);
#pragma unroll
              for (int y = 0; y < 4; ++y) e[y] = ex2(e[y]);
              sum[0] = add2(pair(e[0], e[1]), sum[0]);
              sum[1] = add2(pair(e[2], e[3]), sum[1]);
              pk[2 * i] = pack_f16(e[0], e[1]), pk[2 * i + 1] = pack_f16(e[2], e[3]);
            }
            tmem_st_32x32b_x16(ts + 16 * c, pk);
            if (c == 1) half_done();
          });
        }
        float s0, s1, s2, s3;
        unpair(sum[0], s0, s1);
        unpair(sum[1], s2, s3);
        l = fmaf((s0 + s1) + (s2 + s3), each ? 1.f : tile.z, l);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bars.pfull[slot][1]);
      }
      if (!alive) break;
      n0 += w.to - w.from;
      const bool any = ops != ops0;
      alive = !any || wait(&bars.pvdone[slot], (ops - 1) & 1);
      if (!alive) break;
      tc_fence_after();
      const bool whole = w.from == 0 && w.to == w.tiles;
      const int64_t place = (int64_t)(2 * blockIdx.x + (w.from == 0 ? 1 : 0)) * TR + (RT == 2 ? slot * 128 : 0) + r;
      if constexpr (RT == 2) {
        const bool plain = whole && p.po == nullptr && p.fo == nullptr;
        const float2 inv = inverse_sum(l);
        const uint32_t rowbuf = smem_u32(qt + slot * C::QB);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32b_x32(to + 32 * c, o);
          tmem_ld_wait();
          if (plain) {  // through this row's place in the query tile, so that whole rows are stored
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t y[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float f0 = __uint_as_float(o[i + 2 * x]) * inv.x * inv.y, f1 = __uint_as_float(o[i + 2 * x + 1]) * inv.x * inv.y;
                const __nv_bfloat162 h = __floats2bfloat162_rn(f0, f1);
                y[x] = p.q_bf16 ? *reinterpret_cast<const uint32_t *>(&h) : pack_f16(f0, f1);
              }
              sts128(rowbuf + r * (D * 2) + (((4 * c + i / 8) ^ (r & (D / 8 - 1))) << 4), y[0], y[1], y[2], y[3]);
            }
          } else if (in) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 x = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
              if (l != l) x = make_float4(l, l, l, l);
              if (whole) finish_any<D>(p, at.out, 32 * c + i, x, m, l);
              else *reinterpret_cast<float4 *>(p.ws_o + cut_at<D>(place, TR, 32 * c + i)) = x;
            }
          }
        }
        if (plain) {
          constexpr int LPR = D / 8, RPI = 32 / LPR;
          __syncwarp();
#pragma unroll 4
          for (int x = 0; x < LPR; ++x) {
            const int rr = x * RPI + lane / LPR, row_ = (warp & 3) * 32 + rr, g = lane % LPR;
            const int64_t to_row = __shfl_sync(0xFFFFFFFFu, at.out, rr);
            const bool there = __shfl_sync(0xFFFFFFFFu, (int)in, rr) != 0;
            const uint4 y = *reinterpret_cast<const uint4 *>(qt + slot * C::QB + row_ * (D * 2) + ((g ^ (row_ & (D / 8 - 1))) << 4));
            if (there) *reinterpret_cast<uint4 *>((uint16_t *)p.out + to_row * D + 8 * g) = y;
          }
          __syncwarp();
        }
        if (in && plain && p.lse != nullptr) p.lse[at.out] = log_sum(m, l);
        if (in && !whole) *reinterpret_cast<float2 *>(p.ws_ml + place * 2) = make_float2(m, l);
      } else {
        // the second warpgroup's share goes through its own and the first's query tile
        float *other = (float *)qt;  // [128][D], 16 bytes a lane in rows of their own order
        static_assert(C::QB * 2 >= 128 * D * 4, "query tiles hold the share");
        if (slot == 0) mbar_arrive(&bars.done[0]);
        if (slot == 1) {
          alive = wait(&bars.done[0], parts & 1);
          if (!alive) break;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(to + 16 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4 *>(other + (4 * c + i / 4) * 512 + r * 4) =
                  any ? make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]))
                      : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          share_ml[r] = make_float2(m, l);
          mbar_arrive(&bars.done[1]);
        } else {
          alive = wait(&bars.done[1], parts & 1);
          if (!alive) break;
          const float2 ml = share_ml[r];
          const float M = fmaxf(m, ml.x), fa = m == -INFINITY ? 0.f : ex2(m - M), fb = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
          const float L = l * fa + ml.y * fb;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(to + 16 * c, o);
            tmem_ld_wait();
            if (in)
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float4 y = *reinterpret_cast<const float4 *>(other + (4 * c + i / 4) * 512 + r * 4);
                const float z = any ? fa : 0.f;
                float4 x = make_float4(y.x * fb, y.y * fb, y.z * fb, y.w * fb);
                if (any) {
                  x.x += __uint_as_float(o[i]) * z, x.y += __uint_as_float(o[i + 1]) * z;
                  x.z += __uint_as_float(o[i + 2]) * z, x.w += __uint_as_float(o[i + 3]) * z;
                }
                if (L != L) x = make_float4(L, L, L, L);
                if (whole) finish_any<D>(p, at.out, 16 * c + i, x, M, L);
                else *reinterpret_cast<float4 *>(p.ws_o + cut_at<D>(place, TR, 16 * c + i)) = x;
              }
          }
          if (in && !whole) *reinterpret_cast<float2 *>(p.ws_ml + place * 2) = make_float2(M, L);
          mbar_arrive(&bars.done[2]);
        }
        alive = wait(&bars.done[2], parts & 1);  // the query tiles are free again
        if (!alive) break;
      }
      tc_fence_before();
    }
  } else if (warp < 12) {
    // ================ codes to fp16 ================
    reg_dec<DECODE_REGS>();
    const int w4 = warp & 3, i128 = tid & 127;
    // keys: unit kc of rows r0 + 4i; values: unit vc of keys 8 kg .. 8 kg + 7
    const int kc = lane & 7, r0 = 32 * w4 + (lane >> 3), vc = (lane >> 3) + 4 * (w4 & 1), kg = (lane & 7) + 8 * (w4 >> 1);
    uint32_t rawk[8][C::UW], rawv[8][C::UW];
    uint32_t rs[(C::KNB + 1) / 2], rv[(C::KNB + 1) / 2];  // the scales of this thread's key (i128)
    bool s_in = false;
    uint32_t page[3] = {0, 0, 0};  // of the keys' two blocks of 16 and the values' one, of the tile that is read next

    Part w;
    bool more = begin(w);
    uint32_t j = more ? w.from : 0;  // that tile
    auto read_pages = [&]() {
      if (!more) return;
      const int32_t *table = p.tables + w.b * p.table_stride;
      const int blk = (int)j * (KT / 16), blocks = (w.keys + 15) >> 4;
      const int at[3] = {blk + 2 * w4, blk + 2 * w4 + 1, blk + (kg >> 1)};
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        page[i] = 0xFFFFFFFFu;
        if (at[i] < blocks) page[i] = (uint32_t)__ldg(table + (at[i] >> page_blocks));
      }
    };
    auto read = [&](uint32_t (&raw)[8][C::UW], const uint8_t *codes, bool values) {
      const int blk = (int)j * (KT / 16), left = w.keys - (int)j * KT;
      const uint8_t *base = codes + w.h * p.ch + (values ? vc : kc) * C::UB;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int bk = values ? blk + (kg >> 1) : blk + 2 * w4 + half;
        const uint32_t pg = values ? page[2] : page[half];
        const bool ok = pg < (uint64_t)p.pages;
        const uint8_t *at = base + (uint64_t)(ok ? pg : 0) * p.cp + (bk & in_page) * 16 * p.ct;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = 4 * half + i, key = values ? 8 * kg + x : r0 + 4 * x;  // within the tile
          if (ok && key < left) {
            lds<C::UB>(at + (key & 15) * p.ct, raw[x]);
          } else {
#pragma unroll
            for (int y = 0; y < C::UW; ++y) raw[x][y] = 0;
          }
        }
      }
    };
    auto read_keys = [&]() {
      read(rawk, p.k, false);
      const int sb = (int)j * (KT / 16) + (i128 >> 4);
      const uint32_t pg = lane < 16 ? page[0] : page[1];
      const bool there = i128 < w.keys - (int)(j * KT);
      s_in = there && pg < (uint64_t)p.pages;
      if (there && !s_in) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
      if (s_in) {
        const uint8_t *at = (const uint8_t *)p.ks + w.h * p.sh + (uint64_t)pg * p.sp + ((sb & in_page) * 16 + (i128 & 15)) * p.st;
        load_scales<C::KNB>(at, p.e8m0, p.scale_vec, rs);
        load_scales<C::KNB>(at + ((uint64_t)p.vs - (uint64_t)p.ks), p.e8m0, p.scale_vec, rv);
      }
    };
    auto read_values = [&]() {  // then on to the next tile, whose pages are asked for
      read(rawv, p.v, true);
      if (++j == w.to) {
        more = next(w);
        j = w.from;
      }
      read_pages();
    };
    read_pages();
    bool here = more;
    if (here) {
      read_keys();
      read_values();
    }
    // A thread whose wait ran out leaves with all others, at meet(), or they would wait for it there.
    bool alive = true;
    for (uint32_t n = 0; here; ++n) {
      const uint32_t buf = n & 1, phase = ((n >> 1) - 1) & 1;
      const bool again = more;  // a tile follows this one
      alive = alive && (n < 2 || mbar_wait(&bars.kfree[buf], phase, abort_flag, WAIT_NS));
      // Scales. Where the tile's exponents lie close together, key and value codes take theirs relative to the
      // tile's (exactly, but for rounding products of 8-bit codes and bfloat16 scales to fp16) and the rows
      // need one of each; where not, or where a key is missing or NaN, relative to their own key's, and every
      // key leaves what the rows need of it.
      float kf[C::KNB], vf[C::KNB];
      widen<C::KNB>(rs, p.e8m0, kf);
      widen<C::KNB>(rv, p.e8m0, vf);
      uint32_t km = 0, vm = 0, kl = 0x7F800000u, vl = 0x7F800000u;  // magnitudes order as integers, NaN above all
#pragma unroll
      for (int i = 0; i < C::KNB; ++i) {
        const uint32_t a = __float_as_uint(kf[i]) & 0x7FFFFFFFu, b = __float_as_uint(vf[i]) & 0x7FFFFFFFu;
        km = max(km, a), vm = max(vm, b);
        if (a > 0x0E000000u) kl = min(kl, a);  // blocks of zeros have scales of 2^-100 and no say
        if (b > 0x0E000000u) vl = min(vl, b);
      }
      const bool kn = km >= 0x7F800000u, vn = vm >= 0x7F800000u;
      {
        uint32_t *sp = span_s[buf][w4];
        const uint32_t x0 = __reduce_max_sync(0xFFFFFFFFu, s_in ? km >> 23 : 0), x1 = __reduce_min_sync(0xFFFFFFFFu, s_in ? kl >> 23 : 255);
        const uint32_t x2 = __reduce_max_sync(0xFFFFFFFFu, s_in ? vm >> 23 : 0), x3 = __reduce_min_sync(0xFFFFFFFFu, s_in ? vl >> 23 : 255);
        const bool any = __any_sync(0xFFFFFFFFu, !s_in || kn || vn);
        if (lane == 0) sp[0] = x0, sp[1] = x1, sp[2] = x2, sp[3] = x3, sp[4] = any;
      }
      if (!meet<1, WG>(alive)) break;
      {
        uint32_t kx = 0, ki = 255, vx = 0, vi = 255;
        bool each = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t *sp = span_s[buf][i];
          kx = max(kx, sp[0]), ki = min(ki, sp[1]), vx = max(vx, sp[2]), vi = min(vi, sp[3]), each |= sp[4] != 0;
        }
        each = each || (fold && (int)(kx - ki) > C::SPAN) || (int)(vx - vi) > C::SPAN;
        const int ke = RowRef<F>::exponent((each ? km >> 23 : kx) << 7), ve = RowRef<F>::exponent((each ? vm >> 23 : vx) << 7);
        float *k_s = sc + (n & 3) * 3 * KT + i128;
        const float ks = fold ? RowRef<F>::value(ke) : kf[0], nan = __uint_as_float(0x7FC00000u);
        // a NaN scale: in the score, which rows that do not see the key drop
        k_s[0] = s_in && !kn ? ks : 0.f;
        k_s[KT] = !s_in ? -INFINITY : kn || vn ? nan : (float)(ve - 127);
        k_s[2 * KT] = s_in && !vn ? RowRef<F>::inverse(ve) * SUM_UNIT : 0.f;
        if (i128 == 0)
          tile_s[n & 3] = make_float4(fold ? ks : 1.f, (float)(ve - 127), RowRef<F>::inverse(ve) * SUM_UNIT, each ? 1.f : 0.f);
        const float kr = RowRef<F>::inverse(ke), vr = RowRef<F>::inverse(ve);
#pragma unroll
        for (int i = 0; i < C::KNB; ++i) {
          kratio[(buf * C::KNB + i) * KT + i128] = __float2half_rn(s_in && !kn ? kf[i] * kr : 0.f);
          vratio[(buf * C::KNB + i) * KT + i128] = __float2half_rn(s_in && !vn ? vf[i] * vr : 0.f);
        }
        mbar_arrive(&bars.scfull[n & 3]);
        meet<2, WG>(true);  // the ratios are there for all
      }
      const uint32_t ka = smem_u32(kt + buf * C::KB);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int row = r0 + 4 * x;
        uint32_t f[C::UD / 2];
        if constexpr (C::bits == 8) {
#pragma unroll
          for (int y = 0; y < C::UW; ++y) decode4_8bit<F>(rawk[x][y], f[2 * y], f[2 * y + 1]);
        } else {
#pragma unroll
          for (int y = 0; y < C::UW; ++y) decode8_4<F>(rawk[x][y], reinterpret_cast<uint32_t(&)[4]>(f[4 * y]));
        }
        if (fold) {
          const __half2 r2 = __half2half2(kratio[(buf * C::KNB + (BLK ? kc * C::UD / 32 : 0)) * KT + row]);
#pragma unroll
          for (int y = 0; y < C::UD / 2; ++y) f[y] = hmul2(f[y], *reinterpret_cast<const uint32_t *>(&r2));
        }
        if constexpr (C::UD == 16) {  // the upper units write their second half first: no bank twice
          const bool sw = kc >= 4;
          const uint32_t a0 = ka + tile_at(KT, row, 2 * kc), a1 = ka + tile_at(KT, row, 2 * kc + 1);
          sts128(sw ? a1 : a0, sw ? f[4] : f[0], sw ? f[5] : f[1], sw ? f[6] : f[2], sw ? f[7] : f[3]);
          sts128(sw ? a0 : a1, sw ? f[0] : f[4], sw ? f[1] : f[5], sw ? f[2] : f[6], sw ? f[3] : f[7]);
        } else {
          sts128(ka + tile_at(KT, row, kc), f[0], f[1], f[2], f[3]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&bars.kfull[buf]);
      if (again) read_keys();

      alive = n < 2 || mbar_wait(&bars.vfree[buf], phase, abort_flag, WAIT_NS);
      const uint32_t va = smem_u32(vt + buf * C::VB);
      uint32_t r4[4];
      lds<16>((const uint8_t *)&vratio[(buf * C::KNB + (BLK ? vc * C::UD / 32 : 0)) * KT + 8 * kg], r4);
      constexpr int DW = 32 / C::bits;
#pragma unroll
      for (int y = 0; y < C::UW; ++y) {
        uint32_t f[DW][4];  // [value][pair of keys]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w0 = rawv[2 * i][y], w1 = rawv[2 * i + 1][y];
          if constexpr (C::bits == 8) {
            decode4_8bit<F>(__byte_perm(w0, w1, 0x5140), f[0][i], f[1][i]);
            decode4_8bit<F>(__byte_perm(w0, w1, 0x7362), f[2][i], f[3][i]);
          } else if constexpr (F == B200_CACHE_INT4) {
            uint32_t lo[4], hi[4];
            decode8_4<F>(__byte_perm(w0, w1, 0x5410), lo);
            decode8_4<F>(__byte_perm(w0, w1, 0x7632), hi);
#pragma unroll
            for (int x = 0; x < 4; ++x) f[x][i] = lo[x], f[x + 4][i] = hi[x];
          } else {
            uint32_t ev[4], od[4];
            decode8_4<F>((w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), ev);
            decode8_4<F>(((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), od);
#pragma unroll
            for (int x = 0; x < 4; ++x) f[2 * x][i] = ev[x], f[2 * x + 1][i] = od[x];
          }
#pragma unroll
          for (int x = 0; x < DW; ++x) f[x][i] = hmul2(f[x][i], r4[i]);
        }
#pragma unroll
        for (int x = 0; x < DW; ++x) {
          const int d = vc * C::UD + y * DW + x;
          sts128(va + tile_at(D, d, kg), f[x][0], f[x][1], f[x][2], f[x][3]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&bars.vfull[buf]);
      here = again;
      if (here) read_values();
    }
  } else {
    reg_dec<ISSUE_REGS>();
    if (warp < 14) {
      // ================ MMA issuers: a warp a slot, so that neither waits for the other's softmax; the warp
      // stays together, so that descriptors live in uniform registers ================
      const uint32_t s = __shfl_sync(0xFFFFFFFFu, (uint32_t)warp - 12u, 0);
      constexpr uint32_t id_s = idesc_f16(0, 128, KT), id_o = idesc_f16(0, 128, D), STEP = RT == 2 ? 1 : 2;
      uint32_t qp = 0, pp = 0;  // parities of the queries' and weights' barriers
      auto wait = [&](uint64_t *bar, uint32_t phase) {
        return __all_sync(0xFFFFFFFFu, mbar_wait(bar, phase, abort_flag, WAIT_NS)) != 0;
      };
      const uint64_t qa = sw128_kmajor_desc(qt) + s * (C::QB / 16), k0 = sw128_kmajor_desc(kt), v0 = sw128_kmajor_desc(vt);
      const uint32_t ts = tmem + s * 128, to = tmem + 256 + s * D;
      auto scores = [&](uint32_t n) {
        if (!wait(&bars.kfull[n & 1], (n >> 1) & 1)) return false;
        tc_fence_after();
        const uint64_t kb = k0 + (n & 1) * (C::KB / 16);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {  // 128 x 128 bytes a 64 values, 32 bytes a step
          const uint64_t at = (x >> 2) * (128 * 128 / 16) + 2 * (x & 3);
          mma_ss(ts, qa + at, kb + at, id_s, x != 0);
        }
        commit(&bars.sfull[s]);
        commit(&bars.kfree[n & 1]);
        return true;
      };
      auto values = [&](uint32_t n, bool first) {
        if (!wait(&bars.vfull[n & 1], (n >> 1) & 1)) return false;
        const uint64_t vb = v0 + (n & 1) * (C::VB / 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 64 keys at a time
          if (!wait(&bars.pfull[s][h], pp)) return false;
          tc_fence_after();
#pragma unroll
          for (int x = 4 * h; x < 4 * h + 4; ++x)
            mma_ts(to, ts + 8 * x, vb + (x >> 2) * (D * 128 / 16) + 2 * (x & 3), id_o, !first || x != 0);
        }
        pp ^= 1;
        commit(&bars.pvdone[s]);
        commit(&bars.vfree[n & 1]);
        return true;
      };
      Part w;
      uint32_t n0 = 0;
      bool ok = true;
      for (bool more = begin(w); more && ok; more = next(w)) {
        const uint32_t end = n0 + __shfl_sync(0xFFFFFFFFu, w.to - w.from, 0), first = RT == 2 ? n0 : n0 + ((n0 ^ s) & 1);
        if (first < end) {
          ok = wait(&bars.qfull[s], qp) && scores(first);
          qp ^= 1;
          for (uint32_t n = first; n < end && ok; n += STEP) ok = values(n, n == first) && (n + STEP >= end || scores(n + STEP));
        }
        n0 = end;
      }
      if (!ok) {  // tensor memory is freed behind the products in flight (else every one has been waited for)
        commit(&bars.drain[s]);
        mbar_drain(&bars.drain[s], 0, 200000000ull);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// Joins the segments that were cut: a CTA takes 32 rows of one and as many of their values, a thread four.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const Params p, int tile_rows, uint32_t ctas) {
  __shared__ uint32_t prefix[MAX_ENTRIES + 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // only now: what starts from here on finds all launches before this one complete (Params::early)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  scan_entries(p, tile_rows, prefix);
  __syncthreads();
  const int entries = p.batch * p.row_tiles, chunks = tile_rows / 32 * (D / 32);
  const uint32_t total = prefix[entries] * (uint32_t)p.kv_heads, per = max(1u, (total + ctas - 1) / ctas);
  for (int x = blockIdx.x; x < entries * p.kv_heads * chunks; x += gridDim.x) {
    const int chunk = x % chunks, s = x / chunks, e = s / p.kv_heads, h = s - e * p.kv_heads;
    const uint32_t tiles = prefix[e + 1] - prefix[e], seg0 = prefix[e] * p.kv_heads + h * tiles;
    if (tiles == 0) continue;
    const uint32_t c0 = seg0 / per, c1 = (seg0 + tiles - 1) / per;
    if (c0 == c1) continue;
    const int b = e / p.row_tiles, rt = e - b * p.row_tiles;
    const int rr = chunk / (D / 32) * 32 + (threadIdx.x & 31), d = chunk % (D / 32) * 32 + (threadIdx.x >> 5) * 4;
    const int row = rt * tile_rows + rr;
    if (row >= p.rows) continue;
    auto place = [&](uint32_t c) { return (int64_t)(2 * c + (c == c0 ? 1 : 0)) * tile_rows + rr; };
    float M = -INFINITY, L = 0.f;
#pragma unroll 8
    for (uint32_t c = c0; c <= c1; ++c) M = fmaxf(M, ((const float2 *)p.ws_ml)[place(c)].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (uint32_t c = c0; c <= c1; ++c) {
      const float2 ml = ((const float2 *)p.ws_ml)[place(c)];
      const float4 y = *(const float4 *)(p.ws_o + cut_at<D>(place(c), tile_rows, d));
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
      L += ml.y * f;
    }
    if (L != L) o = make_float4(L, L, L, L);
    finish_any<D>(p, row_at(p, b, h, row).out, d, o, M, L);
  }
}

template <typename K>
static int32_t launch_pdl(K kernel, int grid, int block, size_t smem, cudaStream_t stream, const Params &p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return B200_OK;
}

template <int F, int D, int RT, bool BLK>
static int32_t launch_t(Params &p, cudaStream_t stream) {
  using C = Cfg<F, D, BLK>;
  constexpr int TR = 128 * RT;
  int sms = 0;
  B200_CUDA_TRY(device_sms(&sms));
  p.row_tiles = (p.rows + TR - 1) / TR;
  if (p.row_tiles > MAX_ENTRIES)
    return b200_set_error(B200_ERR_UNSUPPORTED, "cache_attention: too many query rows (%d of a key head)", p.rows);
  const int64_t cap = p.lengths != nullptr ? ((int64_t)p.max_pages << p.page_shift) : p.fixed;
  const int64_t tiles = (cap + KT - 1) / KT * p.kv_heads * p.row_tiles;  // of a request
  if (tiles > (1 << 30)) return b200_set_error(B200_ERR_UNSUPPORTED, "cache_attention: too many keys for one launch");
  int at_once = MAX_ENTRIES / p.row_tiles;
  if (tiles > 0 && tiles * at_once > (1 << 30)) at_once = (int)((1 << 30) / tiles);
  const size_t rows = (size_t)sms * 2 * 256;  // two shares a CTA
  uint8_t *ws = nullptr;
  if (int32_t rc = workspace_of(WS_ATTENTION_MMA, rows * (128 + 2) * 4, 0, stream, &ws)) return rc;
  p.ws_o = (float *)ws, p.ws_ml = (float *)(ws + rows * 128 * 4);
  B200_CUDA_TRY((ensure_dynamic_smem<attn_mma_kernel<F, D, RT, BLK>>(C::SMEM)));
  const Params base = p;
  for (int b = 0; b < base.batch; b += at_once) {  // a launch for each run of requests that the scan has room for
    p = base;
    p.batch = base.batch - b < at_once ? base.batch - b : at_once;
    if (b > 0) {
      const int64_t rows = (int64_t)b * p.per_request * p.q_heads;
      p.q = (const uint16_t *)p.q + b * p.qsr;
      p.tables += b * p.table_stride, p.lengths += b;
      p.out = (uint16_t *)p.out + rows * D;
      if (p.lse != nullptr) p.lse += rows;
      p.row0 += rows;
    }
    int64_t grid = tiles * p.batch;
    if (grid > sms) grid = sms;
    if (grid < 1) grid = 1;
    if (int32_t rc = launch_pdl(attn_mma_kernel<F, D, RT, BLK>, (int)grid, THREADS, C::SMEM, stream, p)) return rc;
    const int64_t chunks = (int64_t)p.batch * p.row_tiles * p.kv_heads * (TR / 32) * (D / 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(chunks < 8 * sms ? chunks : 8 * sms));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, join_kernel<D>, (const Params)p, TR, (uint32_t)grid));
  }
  return B200_OK;
}

template <int F>
static int32_t launch_d(Params &p, int dim, bool blk, cudaStream_t stream) {
  // Up to 128 rows: both softmax warpgroups on the same rows (64 rows, 8192 keys: 42.3 us, with one of
  // them idle 46.4).
  const bool two = p.rows > 128;
  if (dim == 64) {
    if (two) return blk ? launch_t<F, 64, 2, true>(p, stream) : launch_t<F, 64, 2, false>(p, stream);
    return blk ? launch_t<F, 64, 1, true>(p, stream) : launch_t<F, 64, 1, false>(p, stream);
  }
  if (two) return blk ? launch_t<F, 128, 2, true>(p, stream) : launch_t<F, 128, 2, false>(p, stream);
  return blk ? launch_t<F, 128, 1, true>(p, stream) : launch_t<F, 128, 1, false>(p, stream);
}
static int32_t launch_f(Params &p, int fmt, int dim, bool blk, cudaStream_t stream) {
  switch (fmt) {
    case B200_CACHE_INT8: return launch_d<B200_CACHE_INT8>(p, dim, blk, stream);
    case B200_CACHE_FP8E4M3: return launch_d<B200_CACHE_FP8E4M3>(p, dim, blk, stream);
    case B200_CACHE_INT4: return launch_d<B200_CACHE_INT4>(p, dim, blk, stream);
    default: return launch_d<B200_CACHE_FP4_E2M1>(p, dim, blk, stream);
  }
}

}  // namespace mma

// The few-row kernel reads and decodes the keys again for every 16 rows, this one for every 256, with a
// dearer start. Device us there and here: 8192 fp8 keys, 64 rows 34.9 and 43.1, 128 rows 50.0 and 41.6;
// 32768 keys, 64 rows 84 and 99, 128 rows 146 and 92; 16 requests of FP4 blocks, 48 rows 155 and 200, 64
// rows 202 and 202, 80 rows 248 and 204; an int4 prefix of 16384, 64 rows 72 and 80, 96 rows 88 and 83.
// The rule does not look at the number of keys, and over few of them the few-row kernel would be faster: 512
// fp8 keys, 96 rows 13.7 and 22.0, 128 rows 13.8 and 21.9, 192 rows 22.0 and 21.5, 256 rows 12.3 and 22.9; 64
// requests behind a prefix of 1024 keys 56.7 and 65.6.
bool mma_supported(const Params &p, int dim) { return dim <= 128 && p.rows > 64; }

int32_t launch_mma(Params &p, int q_dtype, int fmt, int dim, bool blk, cudaStream_t stream) {
  p.q_bf16 = q_dtype == B200_DT_BF16;
  return mma::launch_f(p, fmt, dim, blk, stream);
}

}  // namespace cattn
}  // namespace b200
