// cache_attn.cu -- attention of few query rows over the packed key/value cache.
//
//   s[r, t] = scale * q[r] . K[t],  K[t] = ks[t] * kc[t]        (codes times their row's scale)
//   out[r]  = sum_t w[r, t] V[t] / sum_t w[r, t],  w = exp(s), V[t] = vs[t] * vc[t]
//
// One pass over the keys. With everything in base 2, u = s + log2 vs[t] and a running maximum m of
// u, a key adds p * vc[t] (p = 2^(u - m + 11)) to the numerator and p / vs[t] to the denominator:
// codes enter the matrix instructions as they are stored, exact in fp16, and no scale is multiplied
// into them. vs is at least 2^-100 here, which stands for values of zero too, and the denominator is kept
// as 2^-20 of itself, so that it bears any number of such keys. p <= 2^15 is rounded to fp16 for the
// second product (11 bits down to 2^-25 of the largest weight); sums, statistics and the denominator are
// fp32. q is scaled by a power of two per row, so that bf16 values fit fp16.
// Blocks of 32 values with scales of their own: the codes are multiplied by scale / 2^E, with 2^E
// just above the row's largest scale (shifted up by fp16's headroom, so that blocks down to 2^-26,
// 8-bit 2^-20, of the largest keep their bits), and ks, vs above become 2^E.
//
// m16n8k16 takes keys as its 16 rows and query rows (heads that share a key head, and the tokens of
// a short block) as its 8 columns: s^T = K q^T, out^T = V^T p^T. Which value of the head sits at
// which k of an instruction is free as long as both operands agree: lane t of four holds values
// 8t .. 8t + 7 of each 32, so that a k step stays within one scale block, whose sum is multiplied by
// its scale in fp32. For V^T a lane reads its D / 8 neighbouring values of four keys; pairs of keys
// are joined by byte permutes before the codes become fp16. p is turned with movmatrix.
//
// Every warp works alone: it copies units of 16 to 64 keys (4 KB of codes, 8 KB for 256 values of 8 bits)
// into a ring of two of its own with cp.async, 16 bytes a lane, one unit ahead, chunks xor-ed by their row so
// that both operands' reads spread over the banks; a lane asks for the scales of a key two units ahead and
// leaves what the scores need of them beside the ring, and page numbers are asked for three units ahead.
// While a unit is computed the SM's 16 warps have 64 KB of codes on their way (8 warps 32 KB where 16 query
// rows share a pass), and no barrier stands between a segment's units.
//
// The units of all (request, key head, row tile) segments are laid end to end in rounds (a unit for
// each warp) and cut into equal runs, one per CTA, from the lengths on the device: ragged batches
// balance, and the launch (a CUDA graph) does not depend on the lengths. A CTA's warps join in
// shared memory; a segment cut over several CTAs is joined by the CTA that finishes last, always in
// the same order. Cuts pay down to single rounds: segments kept whole up to four rounds took 22.7 us
// instead of 12.2 for 4 requests of 4096 int4 keys, and 7.0 instead of 7.4 at 300 int8 keys.
//
// Measured (bf16, 8 key heads of 128, device time): 64 requests of 2048 to 8192 keys, 64 heads, FP4 in
// blocks: 127 us = 2.8 TB/s. Bound by instruction issue there: about 500 warp instructions for each 16
// keys of a key head, at 0.62 an SM quarter and cycle. 32 requests of 8192 keys, a scale a row: int8 116 us
// = 4.7 TB/s, fp8 104 us = 5.3 TB/s. One request of 257 int8 keys: 8.4 us, a chain of launch, lengths, page
// numbers, codes, two products, the warps' and the CTAs' joins.
#include "cache_attn.cuh"
#include "sm100.cuh"

namespace b200 {

int32_t cache_attn_device_error(unsigned int *v, bool clear) {
  B200_CUDA_TRY(tu_device_error(v, clear));
  return B200_OK;
}

namespace cattn {

constexpr int WARPS = 8, THREADS = WARPS * 32, STAGES = 2;
constexpr int MAX_ENTRIES = 4096;    // (request, row tile) pairs of one launch

template <int F, int D, int NT, bool BLK>
struct Cfg {
  static constexpr int bits = CFmt<F>::bits;
  static constexpr int RB = D * bits / 8;                              // bytes of a row
  static constexpr int T = RB == 32 ? 64 : RB == 64 ? 32 : 16;         // keys of a unit
  static constexpr int CPR = RB / 16;                                  // 16-byte chunks of a row
  static constexpr int RPI = 32 / CPR;                                 // rows that 32 lanes copy at once
  static constexpr int NB = D / 32;                                    // blocks of 32 values
  static constexpr int KNB = BLK ? NB : 1;                             // scales of a row
  static constexpr int VCB = RB / 8 < 16 ? RB / 8 : 16;                // bytes of a lane's value chunk
  static constexpr int VCH = RB / 8 / VCB, VCW = VCB / 4;              // chunks, words of one
  static constexpr int VEC = VCB * 8 / bits;                           // values of one
  static constexpr int MT = D / 16;                                    // tiles of V^T
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGE = 2 * T * RB;                             // codes of a unit
  // what the scores need of a unit's scales: (log2 of the value scale, its inverse) per key, key
  // scales, and in blocks the ratios of the value scales to their row's
  static constexpr int LVI = T * 8, KSB = T * KNB * 4, VRB = BLK ? T * NB * 2 : 0;
  static constexpr int SLOT = LVI + KSB + VRB;
  static constexpr int CTAS = D == 256 || NT == 2 ? 1 : 2;             // per SM
  static constexpr int RINGS = WARPS * STAGES * (STAGE + SLOT), STATS = 2 * WARPS * ROWS * 4;
  static constexpr int join_bytes(int passes) { return WARPS * ROWS * (D / passes + 4) * 4; }
  static constexpr bool fits(int passes) { return CTAS * (RINGS + join_bytes(passes) + STATS + 4096) <= 227 * 1024; }
  static constexpr int PASSES = fits(1) ? 1 : 2;                       // the warps join all of a row's values at once, or halves
  static_assert(fits(PASSES), "shared memory");
  static constexpr int PART = D / PASSES, ORS = PART + 4;              // values and row pitch of a pass
  static constexpr int SMEM = RINGS + join_bytes(PASSES) + STATS;

  // key of a unit's 16 that row r of an instruction's first 8 rows holds (row r + 8: the same + 8),
  // chosen with chunk() so that a read of 32 lanes meets no bank twice
  __device__ static __forceinline__ int key_of(int r) {
    if constexpr (bits == 4) return r;
    else if constexpr (RB == 64) return (r & 1) | ((r & 2) << 1) | ((r & 4) >> 1);
    else return 2 * (r & 3) + (r >> 2);
  }
  __device__ static __forceinline__ int row_of(int k) {  // the inverse
    if constexpr (bits == 4) return k;
    else if constexpr (RB == 64) return (k & 1) | ((k & 4) >> 1) | ((k & 2) << 1);
    else return (k >> 1) | ((k & 1) << 2);
  }
  // byte of chunk c of row `row` in a tile
  __device__ static __forceinline__ int chunk(int row, int c) {
    const int x = RB == 32 ? c ^ ((row >> 2) & 1) : RB == 64 ? c ^ ((row >> 1) & 3) : c ^ (row & 7);
    return row * RB + x * 16;
  }
};

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool in) {  // zeros where not `in`
  const int n = in ? 16 : 0;
  asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// A run of units of one segment, as a warp walks it.
struct Walk {
  uint32_t u, seg1;   // the round it stands at, and where its segment ends (both in the run's numbering)
  int e, h;           // entry and key head
  int b, keys;        // request, keys that the segment reads
  uint32_t seg0;
};

template <typename T, int F, int D, int NT, bool BLK>
__global__ void __launch_bounds__(THREADS, Cfg<F, D, NT, BLK>::CTAS) attn_kernel(const Params p) {
  using C = Cfg<F, D, NT, BLK>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t scan[WARPS];
  __shared__ uint32_t last;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  auto await = []() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  if (!p.early) await();  // else before the prefix's partials are read

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t *ring = smem + warp * STAGES * C::STAGE;
  uint8_t *slots = smem + WARPS * STAGES * C::STAGE + warp * STAGES * C::SLOT;
  float *join_o = (float *)(smem + WARPS * STAGES * (C::STAGE + C::SLOT));
  float *join_m = join_o + WARPS * C::ROWS * C::ORS, *join_l = join_m + WARPS * C::ROWS;
  uint32_t *prefix = (uint32_t *)(join_l + WARPS * C::ROWS);  // rounds of a key head before each entry
  const int entries = p.batch * p.row_tiles, heads = p.kv_heads;
  constexpr uint32_t ROUND = C::T * WARPS;
  const int64_t cap = (int64_t)p.max_pages << p.page_shift;

  auto length_of = [&](int b) -> int {
    const int64_t n = p.lengths != nullptr ? p.lengths[b] : p.fixed;
    return (int)(n < 0 ? 0 : n > cap ? cap : n);
  };
  // keys that the last row of an entry's tile sees
  auto keys_of = [&](int e) -> int {
    const int b = p.row_tiles == 1 ? e : e / p.row_tiles;
    const int n = length_of(b);
    if (!p.causal || p.queries == 1) return n;
    const int r1 = min(p.rows, (e - b * p.row_tiles + 1) * C::ROWS) - 1;
    return max(0, n - p.queries + r1 / p.group + 1);
  };
  auto rounds_of = [&](int keys) -> uint32_t { return ((uint32_t)keys + ROUND - 1) / ROUND; };

  uint32_t per;  // rounds of a CTA; the entries' are summed up
  {
    const int each = (entries + THREADS - 1) / THREADS, e0 = tid * each;
    uint32_t sum = 0;
    for (int i = 0; i < each; ++i)
      if (e0 + i < entries) {
        const uint32_t r = rounds_of(keys_of(e0 + i));
        prefix[e0 + i] = r;
        sum += r;
      }
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    uint32_t base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) base += scan[w];
      total += scan[w];
    }
    per = (uint32_t)(((uint64_t)total * heads + gridDim.x - 1) / gridDim.x);
    if (per == 0) per = 1;
    uint32_t run = base + inc - sum;
    for (int i = 0; i < each; ++i)
      if (e0 + i < entries) {
        const uint32_t r = prefix[e0 + i];
        prefix[e0 + i] = run;
        run += r;
        if (e0 + i == entries - 1) prefix[entries] = run;
      }
    __syncthreads();
  }
  const uint32_t total = prefix[entries] * (uint32_t)heads;

  // rows without a key: zeros (or what the prefix gave)
  for (int e = blockIdx.x; e < entries; e += gridDim.x) {
    if (prefix[e + 1] != prefix[e]) continue;
    if (p.early) await();
    const int b = e / p.row_tiles, rt = e - b * p.row_tiles;
    const int n = min(C::ROWS, p.rows - rt * C::ROWS);
    for (int i = tid; i < heads * n * (D / 4); i += THREADS) {
      const int d = (i % (D / 4)) * 4, rr = i / (D / 4);
      const RowAt at = row_at(p, b, rr / n, rt * C::ROWS + rr % n);
      finish<T, D>(p, at.out, d, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
    }
  }

  // this CTA's run of rounds
  const uint32_t u0 = min(total, blockIdx.x * per), u_end = min(total, u0 + per);

  auto enter = [&](Walk &w) {  // reads the segment that w.e, w.h name
    const uint32_t n = prefix[w.e + 1] - prefix[w.e];
    w.seg0 = prefix[w.e] * heads + w.h * n;
    w.seg1 = w.seg0 + n;
    w.b = p.row_tiles == 1 ? w.e : w.e / p.row_tiles;
    w.keys = keys_of(w.e);
  };
  auto next_segment = [&](Walk &w) {  // w.u stands at its end
    w.u = w.seg1;
    if (w.u >= u_end) return;
    if (++w.h == heads) {
      w.h = 0;
      do ++w.e;
      while (prefix[w.e + 1] == prefix[w.e]);
    }
    enter(w);
  };
  Walk c;
  c.u = u0, c.e = 0, c.h = 0;
  if (u0 < u_end) {
    int lo = 0, hi = entries;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] * heads <= u0) lo = mid;
      else hi = mid;
    }
    c.e = lo;
    c.h = (int)((u0 - prefix[lo] * heads) / (prefix[lo + 1] - prefix[lo]));
    enter(c);
  }

  // ---- what is on its way: pages of one unit, scales of the one before, codes of the one before that
  constexpr int BPU = C::T / 16;                 // blocks of 16 keys in a unit
  constexpr int KPL = (C::T + 31) / 32;          // keys of a lane
  constexpr int SW = (C::KNB + 1) / 2;
  Walk a = c;                                    // the unit whose pages are being read
  uint32_t page[BPU];
  const uint8_t *code[BPU];                      // key codes of the unit whose scales are being read
  int left = 0;                                  // its keys, none if there is no such unit
  uint32_t bad = 0;                              // its blocks on pages outside the cache
  uint32_t rk[KPL][SW], rv[KPL][SW];
  const int page_blocks = p.page_shift - 4;
  const uint32_t in_page = (1u << page_blocks) - 1;
  const int lr = lane / C::CPR, lc = lane % C::CPR;
  const uint32_t lane_code = lr * p.ct + lc * 16, lane_scale = (lane & 15) * p.st;
  const uint64_t v_of_k = (uint64_t)p.v - (uint64_t)p.k, vs_of_ks = (uint64_t)p.vs - (uint64_t)p.ks;

  auto read_pages = [&]() {
    if (a.u >= u_end) return;
    const int first = ((int)(a.u - a.seg0) * WARPS + warp) * BPU;
    const int32_t *table = p.tables + a.b * p.table_stride;
#pragma unroll
    for (int j = 0; j < BPU; ++j)
      page[j] = (first + j) * 16 < a.keys ? (uint32_t)__ldg(table + ((first + j) >> page_blocks)) : 0u;
  };
  auto read_scales = [&]() {  // of a's unit, whose pages are here; then a moves on and its next pages are asked for
    left = 0, bad = 0;
    if (a.u >= u_end) return;
    const int first = (int)(a.u - a.seg0) * WARPS + warp;
    left = a.keys - first * C::T;
    const uint8_t *kh = p.k + a.h * p.ch, *sh = (const uint8_t *)p.ks + a.h * p.sh;
#pragma unroll
    for (int j = 0; j < BPU; ++j) {
      if (page[j] >= (uint64_t)p.pages) {
        if (16 * j < left) {
          bad |= 1u << j;
          if (lane == 0) atomicOr(&g_device_error, DEVERR_BAD_INDEX);
        }
        page[j] = 0;
      }
      code[j] = kh + (uint64_t)page[j] * p.cp + ((first * BPU + j) & in_page) * 16 * p.ct;
    }
#pragma unroll
    for (int k = 0; k < KPL; ++k) {
      const int key = lane + 32 * k, j = key >> 4;
      uint32_t pg = page[0];
#pragma unroll
      for (int i = 1; i < BPU; ++i)
        if (j == i) pg = page[i];
      if (key < C::T && key < left && !((bad >> j) & 1)) {
        const uint8_t *at = sh + (uint64_t)pg * p.sp + ((first * BPU + j) & in_page) * 16 * p.st + lane_scale;
        load_scales<C::KNB>(at, p.e8m0, p.scale_vec, rk[k]);
        load_scales<C::KNB>(at + vs_of_ks, p.e8m0, p.scale_vec, rv[k]);
      }
    }
    if (++a.u == a.seg1) next_segment(a);
    read_pages();
  };
  // the codes of the unit whose scales were read last into stage s
  auto issue_codes = [&](int s) {
    if (left > 0) {
      const uint32_t kd = smem_u32(ring + s * C::STAGE), vd = kd + C::T * C::RB;
      if (left >= C::T && bad == 0) {
#pragma unroll
        for (int i = 0; i < C::T / C::RPI; ++i) {
          const uint8_t *src = code[(i * C::RPI) >> 4] + (lane_code + ((i * C::RPI) & 15) * p.ct);
          const int to = C::chunk(lr + i * C::RPI, lc);
          cp_async16(kd + to, src, true);
          cp_async16(vd + to, src + v_of_k, true);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < C::T / C::RPI; ++i) {
          const int row = lr + i * C::RPI, j = (i * C::RPI) >> 4;
          const bool in = row < left && !((bad >> j) & 1);
          const uint8_t *at = code[0];
#pragma unroll
          for (int x = 1; x < BPU; ++x)
            if (j == x) at = code[x];
          const uint8_t *src = at + (lane_code + ((i * C::RPI) & 15) * p.ct);
          const int to = C::chunk(row, lc);
          cp_async16(kd + to, src, in);
          cp_async16(vd + to, src + v_of_k, in);
        }
      }
    }
    cp_async_commit();
  };
  // what the scores need of its scales beside them
  auto store_scales = [&](int s) {
    if (left > 0) {
      float2 *lvi = (float2 *)(slots + s * C::SLOT);
      float *ks = (float *)(slots + s * C::SLOT + C::LVI);
      __half *vr = (__half *)(slots + s * C::SLOT + C::LVI + C::KSB);
#pragma unroll
      for (int k = 0; k < KPL; ++k) {
        const int key = lane + 32 * k;
        if (C::T < 32 && key >= C::T) continue;
        const bool in = key < left && !((bad >> (key >> 4)) & 1);
        float kf[C::KNB], vf[C::KNB];
        widen<C::KNB>(rk[k], p.e8m0, kf);
        widen<C::KNB>(rv[k], p.e8m0, vf);
        if constexpr (!BLK) {
          // values of zero, or a cell that was never written (scale 0): weight without a value
          const float vsc = vf[0] < 0x1p-100f ? 0x1p-100f : vf[0];
          lvi[key] = in ? make_float2(lg2(vsc), vsc == vsc ? __frcp_rn(vsc) * SUM_UNIT : 0.f) : make_float2(-INFINITY, 0.f);
          ks[key] = in ? kf[0] : 0.f;
        } else {
          uint32_t top = 0;  // magnitudes order as integers, NaN above all
#pragma unroll
          for (int i = 0; i < C::NB; ++i) top = max(top, __float_as_uint(vf[i]) & 0x7FFFFFFFu);
          const int e = RowRef<F>::exponent(top >> 16);
          float inv = RowRef<F>::inverse(e);
          // the row's NaN travels in its scores, which rows that do not see it drop
          lvi[key] = !in ? make_float2(-INFINITY, 0.f)
                     : top > 0x7F800000u ? make_float2(__uint_as_float(top), 0.f) : make_float2((float)(e - 127), inv * SUM_UNIT);
          const bool use = in && top <= 0x7F800000u;
          __half *vk = vr + (key & ~7) + C::row_of(key & 7);  // ratios in the order of the instruction's rows
#pragma unroll
          for (int i = 0; i < C::NB; ++i) vk[i * C::T] = __float2half_rn(use ? vf[i] * inv : 0.f);
#pragma unroll
          for (int i = 0; i < C::NB; i += 2)
            *(float2 *)(ks + key * C::NB + i) = in ? make_float2(kf[i], kf[i + 1]) : make_float2(0.f, 0.f);
        }
      }
    }
  };

  uint32_t raw_q[NT][C::NB][4];
  auto read_q = [&](const Walk &w) {
    const int r0 = (w.e - w.b * p.row_tiles) * C::ROWS;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 8 + g;
      const bool in = r < p.rows;
      const T *src = in ? (const T *)p.q + row_at(p, w.b, w.h, r).q + 8 * t : nullptr;
#pragma unroll
      for (int b = 0; b < C::NB; ++b) {
        if (in && p.q_vec) lds<16>((const uint8_t *)(src + 32 * b), raw_q[n][b]);
        else if (in)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            raw_q[n][b][i] = (uint32_t)*(const uint16_t *)(src + 32 * b + 2 * i) | ((uint32_t)*(const uint16_t *)(src + 32 * b + 2 * i + 1) << 16);
        else raw_q[n][b][0] = raw_q[n][b][1] = raw_q[n][b][2] = raw_q[n][b][3] = 0;
      }
    }
  };
  read_pages();
  if (c.u < u_end) read_q(c);
  // Of the unit that is computed, stage `stage` holds codes and scales; the next one's codes are asked for
  // first thing, and its scales, which were asked for a unit earlier, are stored last.
  int stage = 0;
  read_scales();
  issue_codes(0);
  store_scales(0);
  read_scales();

  while (c.u < u_end) {
    const uint32_t real = rounds_of(c.keys), from = c.u - c.seg0, to = min(u_end, c.seg1) - c.seg0;
    const int rt = c.e - c.b * p.row_tiles, r0 = rt * C::ROWS, n_rows = min(C::ROWS, p.rows - r0);
    const int len = length_of(c.b);

    // q as the second operand: fp16, each row scaled by a power of two, lane (g, t) of tile n holding
    // values 8t .. 8t + 7 of every block of 32 of row 8n + g, paired as the codes come out decoded
    uint32_t q[NT][C::NB][4];
    float qs[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = 0.f;
#pragma unroll
      for (int b = 0; b < C::NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T *v = reinterpret_cast<const T *>(&raw_q[n][b][i]);
          top = fmaxf(top, fmaxf(fabsf(to_f32(v[0])), fabsf(to_f32(v[1]))));
        }
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int ex = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float((uint32_t)(254 - ex) << 23);
#pragma unroll
      for (int b = 0; b < C::NB; ++b) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T *v = reinterpret_cast<const T *>(&raw_q[n][b][i]);
          x[2 * i] = to_f32(v[0]) * down, x[2 * i + 1] = to_f32(v[1]) * down;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[n][b][i] = F == B200_CACHE_INT4 ? pack_f16(x[i], x[i + 4]) : pack_f16(x[2 * i], x[2 * i + 1]);
      }
      const float mine = p.scale * __uint_as_float((uint32_t)ex << 23);
#pragma unroll
      for (int col = 0; col < 2; ++col) {
        qs[n][col] = __shfl_sync(0xFFFFFFFFu, mine, (2 * t + col) * 4);
        const int rc = n * 8 + 2 * t + col;
        lim[n][col] = rc >= n_rows ? 0 : p.causal && p.queries > 1 ? len - p.queries + (r0 + rc) / p.group + 1 : len;
      }
    }

    float o[NT][C::MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < C::MT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][i][x] = 0.f;
    }

    for (uint32_t round = from; round < to; ++round) {
      const int first = ((int)round * WARPS + warp) * C::T;  // the unit's first key
      issue_codes(stage ^ 1);
      cp_async_wait<1>();
      __syncwarp();
      const uint8_t *kt = ring + stage * C::STAGE, *vt = kt + C::T * C::RB;
      const float2 *lvi_s = (const float2 *)(slots + stage * C::SLOT);
      const float *ks_s = (const float *)(slots + stage * C::SLOT + C::LVI);
      const uint8_t *vr_s = slots + stage * C::SLOT + C::LVI + C::KSB;
#pragma unroll 1
      for (int sb = 0; sb < C::T && first + sb < c.keys; sb += 16) {
        const int k0 = sb + C::key_of(g), k1 = k0 + 8;  // this lane's two keys
        // s^T = K q^T
        float s[NT][4], s2[NT][4], sk0[C::KNB], sk1[C::KNB];
        lds<C::KNB * 4 < 16 ? C::KNB * 4 : 16>((const uint8_t *)(ks_s + k0 * C::KNB), (uint32_t *)sk0);
        lds<C::KNB * 4 < 16 ? C::KNB * 4 : 16>((const uint8_t *)(ks_s + k1 * C::KNB), (uint32_t *)sk1);
        if constexpr (C::KNB == 8) {
          lds<16>((const uint8_t *)(ks_s + k0 * C::KNB + 4), (uint32_t *)sk0 + 4);
          lds<16>((const uint8_t *)(ks_s + k1 * C::KNB + 4), (uint32_t *)sk1 + 4);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] = 0.f, s2[n][x] = 0.f;
#pragma unroll
        for (int b = 0; b < C::NB; ++b) {
          uint32_t f[2][4];  // [key][pairs of two k steps]
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = i ? k1 : k0;
            if constexpr (C::bits == 8) {
              uint32_t w[2];
              lds<8>(kt + C::chunk(row, 2 * b + (t >> 1)) + 8 * (t & 1), w);
              decode4_8bit<F>(w[0], f[i][0], f[i][1]);
              decode4_8bit<F>(w[1], f[i][2], f[i][3]);
            } else {
              uint32_t w[1];
              lds<4>(kt + C::chunk(row, b) + 4 * t, w);
              decode8_4<F>(w[0], f[i]);
            }
          }
          const uint32_t f0[4] = {f[0][0], f[1][0], f[0][1], f[1][1]}, f1[4] = {f[0][2], f[1][2], f[0][3], f[1][3]};
          if constexpr (BLK) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float y[4] = {0.f, 0.f, 0.f, 0.f};
              gemv::mma16816(y, f0, q[n][b][0], q[n][b][1]);
              gemv::mma16816(y, f1, q[n][b][2], q[n][b][3]);
              s[n][0] = fmaf(y[0], sk0[b], s[n][0]), s[n][1] = fmaf(y[1], sk0[b], s[n][1]);
              s[n][2] = fmaf(y[2], sk1[b], s[n][2]), s[n][3] = fmaf(y[3], sk1[b], s[n][3]);
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              gemv::mma16816(s[n], f0, q[n][b][0], q[n][b][1]);
              gemv::mma16816(s2[n], f1, q[n][b][2], q[n][b][3]);
            }
          }
        }
        const float2 lvi0 = lvi_s[k0], lvi1 = lvi_s[k1];
        // u = s + log2 vs: -inf for keys that are not there
        bool up = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float y = BLK ? s[n][x] : (s[n][x] + s2[n][x]) * (x < 2 ? sk0[0] : sk1[0]);
            s[n][x] = fmaf(y, qs[n][x & 1], x < 2 ? lvi0.x : lvi1.x);
          }
          if (p.causal && p.queries > 1) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (first + (x < 2 ? k0 : k1) >= lim[n][x & 1]) s[n][x] = -INFINITY;
          }
          up |= fmaxf(s[n][0], s[n][2]) > m[n][0] + LAZY || fmaxf(s[n][1], s[n][3]) > m[n][1] + LAZY;
        }
        if (__any_sync(0xFFFFFFFFu, up)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int col = 0; col < 2; ++col) {
              float top = fmaxf(m[n][col], fmaxf(s[n][col], s[n][col + 2]));
#pragma unroll
              for (int y = 4; y < 32; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, y));
              const float f = m[n][col] == -INFINITY ? 0.f : ex2(m[n][col] - top);
              m[n][col] = top;
              l[n][col] *= f;
#pragma unroll
              for (int i = 0; i < C::MT; ++i) o[n][i][col] *= f, o[n][i][col + 2] *= f;
            }
        }
        uint32_t bp[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float pr[4];
          const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0] - BIAS, m1 = m[n][1] == -INFINITY ? 0.f : m[n][1] - BIAS;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            pr[x] = ex2(s[n][x] - (x & 1 ? m1 : m0));
            l[n][x & 1] = fmaf(pr[x], x < 2 ? lvi0.y : lvi1.y, l[n][x & 1]);
          }
          bp[n][0] = movmatrix_trans(pack_f16(pr[0], pr[1]));
          bp[n][1] = movmatrix_trans(pack_f16(pr[2], pr[3]));
        }
        // out^T += V^T p^T: rows 2t, 2t + 1 (and + 8) of the scores are this lane's four keys
        const int kv[2] = {sb + C::key_of(2 * t), sb + C::key_of(2 * t + 1)};
#pragma unroll
        for (int ch = 0; ch < C::VCH; ++ch) {
          uint32_t w[4][C::VCW];  // keys kv[0], kv[1], kv[0] + 8, kv[1] + 8
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = kv[i & 1] + 8 * (i >> 1);
            const int at = (g + 8 * ch) * C::VCB;
            lds<C::VCB>(vt + C::chunk(row, at >> 4) + (at & 15), w[i]);
          }
          uint32_t vr[2] = {0, 0};
          if constexpr (BLK) {
            const uint8_t *at = vr_s + (((g + 8 * ch) * C::VEC / 32) * C::T + sb + 2 * t) * 2;
            vr[0] = *(const uint32_t *)at, vr[1] = *(const uint32_t *)(at + 16);
          }
#pragma unroll
          for (int y = 0; y < C::VCW; ++y) {
            constexpr int DW = 32 / C::bits;  // values of a word
            uint32_t f[2][DW];                // [keys of a pair][value]
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w0 = w[2 * i][y], w1 = w[2 * i + 1][y];
              if constexpr (C::bits == 8) {
                decode4_8bit<F>(__byte_perm(w0, w1, 0x5140), f[i][0], f[i][1]);
                decode4_8bit<F>(__byte_perm(w0, w1, 0x7362), f[i][2], f[i][3]);
              } else if constexpr (F == B200_CACHE_INT4) {
                uint32_t lo[4], hi[4];
                decode8_4<F>(__byte_perm(w0, w1, 0x5410), lo);
                decode8_4<F>(__byte_perm(w0, w1, 0x7632), hi);
#pragma unroll
                for (int x = 0; x < 4; ++x) f[i][x] = lo[x], f[i][x + 4] = hi[x];
              } else {
                uint32_t ev[4], od[4];
                decode8_4<F>((w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), ev);
                decode8_4<F>(((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), od);
#pragma unroll
                for (int x = 0; x < 4; ++x) f[i][2 * x] = ev[x], f[i][2 * x + 1] = od[x];
              }
              if constexpr (BLK)
#pragma unroll
                for (int x = 0; x < DW; ++x) f[i][x] = hmul2(f[i][x], vr[i]);
            }
#pragma unroll
            for (int x = 0; x < DW / 2; ++x) {
              const uint32_t frag[4] = {f[0][2 * x], f[0][2 * x + 1], f[1][2 * x], f[1][2 * x + 1]};
              const int mt = (ch * C::VCW + y) * (DW / 2) + x;
#pragma unroll
              for (int n = 0; n < NT; ++n) gemv::mma16816(o[n][mt], frag, bp[n][0], bp[n][1]);
            }
          }
        }
      }
      stage ^= 1;
      store_scales(stage);
      __syncwarp();  // this unit's stage may be filled again
      read_scales();
    }

    // join the warps
    if (p.early) await();
    Walk following = c;
    const bool whole = from == 0 && to == real;
    const uint32_t c0 = c.seg0 / per, c1 = (c.seg0 + real - 1) / per;  // CTAs of the segment
    const int slot = (int)(2 * blockIdx.x + (from == 0 ? 1 : 0));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int col = 0; col < 2; ++col) {
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) l[n][col] += __shfl_xor_sync(0xFFFFFFFFu, l[n][col], y);
        const int r = n * 8 + 2 * t + col;
        if (g == 0) join_m[warp * C::ROWS + r] = m[n][col], join_l[warp * C::ROWS + r] = l[n][col];
      }
#pragma unroll
    for (int pass = 0; pass < C::PASSES; ++pass) {
      // a lane's tiles pass * MT / PASSES .. side by side: 2 * MT / PASSES values
      constexpr int OWN = 2 * C::MT / C::PASSES;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int col = 0; col < 2; ++col) {
          float *dst = join_o + (warp * C::ROWS + n * 8 + 2 * t + col) * C::ORS + g * OWN;
#pragma unroll
          for (int i = 0; i < OWN / 2; ++i)
            *reinterpret_cast<float2 *>(dst + 2 * i) =
                make_float2(o[n][pass * (OWN / 2) + i][col], o[n][pass * (OWN / 2) + i][col + 2]);
        }
      if (pass == C::PASSES - 1) {  // the next segment's queries are on their way while the warps meet
        following.u = c.seg0 + to;
        if (following.u == following.seg1) next_segment(following);
        if (following.u < u_end) read_q(following);
      }
      __syncthreads();
      for (int i = tid; i < C::ROWS * (C::PART / 4); i += THREADS) {
        const int r = i / (C::PART / 4), at = (i % (C::PART / 4)) * 4;
        const int gg = at / OWN, place = pass * OWN + at % OWN;  // value `place` of lane gg's
        const int d = (gg + 8 * (place / C::VEC)) * C::VEC + place % C::VEC;
        float M = -INFINITY, L = 0.f, mw[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mw[w] = join_m[w * C::ROWS + r], M = fmaxf(M, mw[w]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float f = mw[w] == -INFINITY ? 0.f : ex2(mw[w] - M);
          const float4 y = *reinterpret_cast<const float4 *>(join_o + (w * C::ROWS + r) * C::ORS + at);
          x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
          L += join_l[w * C::ROWS + r] * f;  // NaN stays NaN, also where it left m at -inf
        }
        if (L != L) x.x = x.y = x.z = x.w = L;
        if (whole) {
          if (r < n_rows) finish<T, D>(p, row_at(p, c.b, c.h, r0 + r).out, d, x, M, L);
        } else {
          *reinterpret_cast<float4 *>(p.ws_o + ((int64_t)slot * C::ROWS + r) * D + d) = x;
          if (d == 0) *reinterpret_cast<float2 *>(p.ws_ml + ((int64_t)slot * C::ROWS + r) * 2) = make_float2(M, L);
        }
      }
      if (pass + 1 < C::PASSES) __syncthreads();
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) last = atomicAdd(&p.tickets[c0], 1u) == c1 - c0;
      __syncthreads();
      if (last) {
        __threadfence();
        for (int i = tid; i < n_rows * (D / 4); i += THREADS) {
          const int r = i / (D / 4), d = (i % (D / 4)) * 4;
          float M = -INFINITY, L = 0.f;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (uint32_t k = c0; k <= c1; ++k) {
            const int64_t sl = (int64_t)(2 * k + (k == c0 ? 1 : 0)) * C::ROWS + r;
            M = fmaxf(M, __ldcg((const float2 *)(p.ws_ml + sl * 2)).x);
          }
#pragma unroll 4
          for (uint32_t k = c0; k <= c1; ++k) {
            const int64_t sl = (int64_t)(2 * k + (k == c0 ? 1 : 0)) * C::ROWS + r;
            const float2 ml = __ldcg((const float2 *)(p.ws_ml + sl * 2));
            const float4 y = __ldcg((const float4 *)(p.ws_o + sl * D + d));
            const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
            x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
            L += ml.y * f;
          }
          if (L != L) x.x = x.y = x.z = x.w = L;
          finish<T, D>(p, row_at(p, c.b, c.h, r0 + r).out, d, x, M, L);
        }
        if (tid == 0) p.tickets[c0] = 0u;  // ready for the next call on this workspace
      }
    }
    __syncthreads();  // the join's memory is free
    c = following;
  }
  cp_async_wait<0>();
  if (p.early) await();  // the launch behind this one takes this one's end for that of all before it
}

// ---- workspace of split segments -------------------------------------------------------------------
constexpr int MAX_ROWS_D = 16 * 128;  // ROWS * D of every variant is at most this

// Two slots for each of the `grid` CTAs that a launch has at most, and their tickets.
static int32_t workspace_for(cudaStream_t stream, int grid, Params &p) {
  const size_t slots = 2 * (size_t)grid, o_bytes = slots * MAX_ROWS_D * 4, bytes = o_bytes + slots * 16 * 2 * 4;
  uint8_t *base = nullptr;
  if (int32_t rc = workspace_of(WS_ATTENTION, bytes, (size_t)grid * 4, stream, &base)) return rc;
  p.ws_o = (float *)base, p.ws_ml = (float *)(base + o_bytes), p.tickets = (uint32_t *)(base + bytes);
  return B200_OK;
}

template <typename T, int F, int D, int NT, bool BLK>
static int32_t launch_t(Params p, cudaStream_t stream) {
  using C = Cfg<F, D, NT, BLK>;
  p.row_tiles = (p.rows + C::ROWS - 1) / C::ROWS;
  if (p.row_tiles > MAX_ENTRIES)
    return b200_set_error(B200_ERR_UNSUPPORTED, "cache_attention: too many query rows (%d of a key head)", p.rows);
  const int64_t round = C::T * WARPS;
  const int64_t cap = p.lengths != nullptr ? ((int64_t)p.max_pages << p.page_shift) : p.fixed;
  const int64_t rounds = ((cap + round - 1) / round) * p.kv_heads * p.row_tiles;  // of a request
  if (rounds > (1 << 29)) return b200_set_error(B200_ERR_UNSUPPORTED, "cache_attention: too many keys for one launch");
  int at_once = MAX_ENTRIES / p.row_tiles;
  if (rounds * at_once > (1 << 29)) at_once = (int)((1 << 29) / rounds);
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
      p.row0 += rows;
      if (b > 0) p.early = 0;  // these share the workspace with the launch before
      if (int32_t rc = launch_t<T, F, D, NT, BLK>(p, stream)) return rc;
    }
    return B200_OK;
  }
  const int64_t entries = (int64_t)p.batch * p.row_tiles;
  int sms = 0;
  B200_CUDA_TRY(device_sms(&sms));
  if (int32_t rc = workspace_for(stream, 2 * sms, p)) return rc;
  B200_CUDA_TRY((ensure_dynamic_smem<attn_kernel<T, F, D, NT, BLK>>(C::SMEM + (MAX_ENTRIES + 1) * 4)));
  // no more CTAs than there can be rounds
  int64_t grid = entries * p.kv_heads * ((cap + round - 1) / round);
  const int64_t full = (int64_t)sms * C::CTAS;
  if (grid > full) grid = full;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM + (entries + 1) * 4;
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
  // Nine rows and more share a pass over the keys 16 at a time: two query tokens of 32 requests take 104
  // us instead of 141; where one request leaves SMs idle (4 tokens, 8192 keys), 19.8 us instead of 17.8.
  const bool two = p.rows > 8;
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
  const int64_t esz = c->scale_dtype == B200_DT_E8M0 ? 1 : 2;
  p.cp = (uint32_t)c->strides[0], p.ch = c->strides[1], p.ct = (uint32_t)c->strides[2];
  p.sp = (uint32_t)(c->scale_strides[0] * esz), p.sh = c->scale_strides[1] * esz, p.st = (uint32_t)(c->scale_strides[2] * esz);
  p.q_vec = (uintptr_t)p.q % 16 == 0 && p.qsr % 8 == 0 && p.qsb % 8 == 0 && p.qsh % 8 == 0;
  p.e8m0 = c->scale_dtype == B200_DT_E8M0;
  const int per_row = dim / c->block_size;  // a row's scales as one vector where they are aligned so
  p.scale_vec = p.sp % (per_row * esz) == 0 && p.sh % (per_row * esz) == 0 && p.st % (per_row * esz) == 0;
  p.pages = c->pages, p.kv_heads = c->kv_heads, p.group = a->heads / c->kv_heads, p.q_heads = a->heads;
  while ((1 << p.page_shift) < c->page_size) ++p.page_shift;
  p.scale = a->scale * 1.44269504088896341f;
  p.per_request = a->queries;
  const bool blk = c->block_size != dim;
  const int64_t all_rows = (int64_t)a->batch * a->queries * a->heads;
  auto run = [&](Params &q) {
    if (mma_supported(q, dim)) return launch_mma(q, a->q_dtype, c->format, dim, blk, stream);
    return a->q_dtype == B200_DT_F16 ? launch_f<__half>(q, c->format, dim, blk, stream)
                                     : launch_f<__nv_bfloat16>(q, c->format, dim, blk, stream);
  };
  bool joined = false;
  if (a->prefix_length > 0) {
    Params f = p;  // every row of the batch against the prefix: one request of batch * queries tokens
    f.tables = a->prefix, f.table_stride = 0, f.max_pages = (int)a->prefix_pages;
    f.fixed = a->prefix_length, f.batch = 1, f.queries = (int)(a->batch * a->queries), f.rows = f.queries * p.group;
    f.exact_keys = a->lse != nullptr;
    f.po = (float *)a->scratch, f.pm = f.po + all_rows * dim, f.pl = f.pm + all_rows;
    if (int32_t rc = run(f)) return rc;
    p.fo = f.po, p.fm = f.pm, p.fl = f.pl;
    joined = mma_supported(f, dim);
  }
  p.tables = a->tables, p.table_stride = a->table_stride, p.max_pages = (int)a->max_pages, p.lengths = a->lengths;
  p.batch = (int)a->batch, p.queries = (int)a->queries, p.rows = p.queries * p.group, p.causal = 1;
  p.out = a->out, p.lse = a->lse;
  // The few-row kernel works on its first keys while the many-row kernel's cut segments of the prefix are joined.
  p.early = joined && !mma_supported(p, dim);
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
  if (a->batch * a->queries * a->heads > INT32_MAX || a->max_pages > (INT32_MAX - 4096) / c->page_size ||
      a->prefix_pages > (INT32_MAX - 4096) / c->page_size)
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
