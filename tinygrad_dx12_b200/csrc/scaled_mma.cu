// scaled_mma.cu -- products of block-scaled 8-bit activations with packed FP4 / FP6 weights on the
// 5th-generation tensor cores, dense or through experts.
//
//   v[t, n] = sum_k x[t, k] 2^(xs[t, k/32]) w[n, k] 2^(ws[n, k/32]),  then bias, activation, gate, residual
//
// tcgen05.mma kind::mxf8f6f4 reads both sides as they are stored: E4M3 codes of x, FP4 / FP6 codes of w
// (TMA lays each 16 of them into a 16-byte slot), and a power of two for every 32 of either. No code is
// decoded on the CUDA cores, for one token or for thousands; products are exact and sums fp32.
//
// A tile is R x 128 weight rows (the MMA's M; R = 2 when gated: 128 gate rows and the 128 up rows that go
// with them, in two accumulators, so both are in one thread's hands) times up to NT tokens (its N, a
// multiple of 16, so an expert with few tokens costs few columns). K advances 128 codes a stage.
//   warps 0-7    epilogue, two groups of four that take turns at 16 tokens: tcgen05.ld (lane = weight
//                row, column = token), bias, activation, gate, residual; a warp's 32 rows are 32 neighbouring
//                columns of y, a block of the 8-bit output, whose largest value is one warp-wide maximum
//   warps 8-11   both sides' scale bytes, up to 12 stages ahead: a warp takes an atom (128 rows, four bytes a
//                stage) and loads 16 bytes of each row, four stages, which leave its registers as four atoms in the
//                layout that tcgen05.cp takes
//   warp 13      tcgen05.cp of a stage's scales into one of four sets of tensor-memory columns; commit
//                announces them to warp 12
//   warps 14-15  one thread each: TMA of the codes, the weights' and x's. Through experts x's rows lie in the
//                plan's order (gathered before, or written so by the product before), so a tile of tokens is a box
//   warp 12      four MMAs a stage and accumulator; commit frees the stage and its set. (One warp for
//                scales and MMAs took 0.5 us a stage: copies, waits and MMAs cost an issuing thread 25 to 45 ns each)
// Two accumulators of a tile's width, so that the epilogue of one tile runs under the products of the
// next: 2 x 224 columns, and four rotating sets of scale columns beside them.
//
// Work split: G CTAs take the tiles in turn, in the order of experts, weight rows and tokens, so that those
// of one time share their weights in L2 (64 experts' would not fit; in equal runs of neighbouring tiles 4001 tokens
// through them took 1730 us, not 1270). Neighbours read the same rows of x and of the
// weights, but not at the same time: each CTA begins at a K of its own and goes round (all at the same K, 4096 tokens
// x 1024 x 16384 took 324 us, not 112). The tiles of the last, partial wave are cut into units, (tile, K stage),
// laid end to end and shared out equally. The tiles of experts are counted on the device from the plan's offsets: a recorded
// launch fits every routing. A tile that a run's border cuts is finished by the last of its CTAs to arrive
// (acquire-release ticket), which adds the fp32 parts in the order of the CTAs: the same bits every time.
// No CTA waits for another. Every wait is bounded (sm100.cuh).
//
// Measured: 57344 x 8192 FP4, one token 52 us = 4.8 TB/s, bound by the stages' instructions (0.5 us for 16 KB an SM:
// issue, scales, barriers) and the ring's depth; 4096 x 14336 x 4096 238 us = 2021 TFLOP/s, bound by shared memory (MMA
// operands, codes in 16-byte slots, x); 64 tokens through 8 of 128 experts 114 + 73 us = 76 and 58 % of HBM.
#include <string.h>

#include "common.cuh"
#include "kernels.h"
#include "scaled_epilogue.cuh"
#include "sm100.cuh"

namespace b200 {

int32_t scaled_mma_device_error(unsigned int *v, bool clear) {
  B200_CUDA_TRY(tu_device_error(v, clear));
  return B200_OK;
}
int32_t scaled_mma_reset_tickets() { return workspace_zero(WS_SCALED); }

namespace scaled {

constexpr int TM = 128, KS = 128;            // weight rows of an MMA, codes of a stage
constexpr int EPI_WARPS = 8, SCALE_WARP0 = 8, SCALE_WARPS = 4, MMA_WARP = 12, SF_WARP = 13, W_WARP0 = 14, W_WARPS = 2;
constexpr int THREADS = 16 * 32;
constexpr int SLOTS = 12;                    // stages whose scales wait for tensor memory
constexpr int ACC_COLS = 224;                // columns of a set of accumulators that take turns: R * NT at most
constexpr int SF_SETS = 4;
constexpr int MAX_STAGES = 12;
constexpr int MAX_EXPERTS = 1024;
constexpr size_t TICKETS = 4096;             // one a CTA
constexpr int CH = 16;                       // tokens of an epilogue step: more unrolled code does not stay in the instruction cache
constexpr int SMEM_LIMIT = 227 * 1024;

struct Params {
  const uint8_t *xs, *ws;
  const int32_t *offsets, *order;
  int64_t rows, n;        // rows of y, weight rows of one matrix
  int64_t wrows;          // of all matrices
  int64_t second;         // the tile's other weight rows: up rows of a gate's, or the next 128
  int64_t nblk;           // scale bytes of a row
  int64_t cols;
  int experts, fan;
  int xs_rows;            // x's scales: B200_ROWS_* (its codes lie in the plan's order)
  int y_pairs;            // y's rows are pairs; else they lie in the plan's order (or there is no plan)
  int single_row;         // x is one token's row
  int vector;             // scale rows are whole 16 bytes
  int scale_warps;
  int nst;                // K stages
  int wtiles, tile_rows;  // tiles of weight rows of one matrix, columns of y in each
  int nt;                 // tokens of a tile, at most
  int grid, stages;
  int once;               // an expert's rows are one tile, most often
  int join, join_part;    // what joining a cut tile costs, in stages, and 16 times that for each part
  int sets;               // of scale columns in turn: no more than stages, whose barriers guard them
  uint32_t stage_bytes, b_off;        // weight codes, then x's
  uint32_t scale_bytes, sfb_off;      // of a slot: weight scales, then x's
  uint32_t tx;
  int bufs;               // accumulators that take turns: 2, or 1 of twice the width
  uint32_t acc_width, sf_col, sf_width, tmem_cols;
  uint32_t idesc;
  float *part;            // [grid][2][R][nt][128]
  unsigned int *tickets;  // [grid]: of the tile that the CTA's run ends in
};

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(EPI_WARPS * 32) : "memory"); }

// Whether the phase is over, without waiting.
__device__ __forceinline__ bool mbar_over(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Shared-memory descriptor of a scale atom: 32 rows of 16 bytes, no swizzle.
__device__ __forceinline__ uint64_t sf_desc(const void *atom) {
  const uint64_t addr = smem_u32(atom);
  return ((addr & 0x3FFFFull) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
// The tensor core's work is issued by one lane of a converged warp: descriptors stay in uniform registers.
// An atom into 4 columns of every lane quarter:
__device__ __forceinline__ void sf_copy(uint32_t taddr, uint64_t desc) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
      "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc) : "memory");
}
// The four products of a stage (K = 32 each: 32 bytes further along the rows, scale byte k): D (+)= A B^T.
__device__ __forceinline__ void mma_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t sfa,
                                          uint32_t sfb) {
  constexpr uint32_t ID = (1u << 4) | (1u << 29), SF = 1u << 30;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %2, %6, %10, [%14], [%18], p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %3, %7, %11, [%15], [%19], p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %4, %8, %12, [%16], [%20], p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %5, %9, %13, [%17], [%21], p;\n\t}" ::"r"(d),
      "r"(acc), "l"(a), "l"(a + 2), "l"(a + 4), "l"(a + 6), "l"(b), "l"(b + 2), "l"(b + 4), "l"(b + 6), "r"(idesc),
      "r"(idesc + ID), "r"(idesc + 2 * ID), "r"(idesc + 3 * ID), "r"(sfa), "r"(sfa + SF), "r"(sfa + 2 * SF), "r"(sfa + 3 * SF),
      "r"(sfb), "r"(sfb + SF), "r"(sfb + 2 * SF), "r"(sfb + 3 * SF)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

// What a tile is: expert, first weight row within its matrix, place of its first row, rows; width: rows rounded
// up to the MMA's N.
struct Tile {
  int e, w0, first, rows, width;
};

// Token tiles of `count` rows: as few as hold them, equally full.
__device__ __forceinline__ uint32_t tiles_of(const Params &p, int count) { return ((uint32_t)count + p.nt - 1) / (uint32_t)p.nt; }

// One copy of it for all warps, in 32 bits: every role asks for every tile, and code of its own that runs once a
// tile would come from L2 each time (inlined it took the scales' warps 4 us a tile).
__device__ __noinline__ uint4 find_tile(uint32_t tile, const int32_t *before, const int32_t *start, uint32_t experts, uint32_t rows,
                                        uint32_t wtiles, uint32_t nt) {
  uint32_t e = 0, first = 0, count = rows, at = tile;
  if (experts > 0) {
    const int32_t t = (int32_t)(tile / wtiles);
    uint32_t lo = 0, hi = experts;  // before[lo] <= t < before[hi]; empty experts have no tiles
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (before[mid] <= t) lo = mid;
      else hi = mid;
    }
    e = lo;
    at = tile - (uint32_t)before[e] * wtiles;
    first = (uint32_t)start[e];
    count = (uint32_t)start[e + 1] - first;
  }
  const uint32_t tt = (count + nt - 1) / nt, per = ((count + tt - 1) / tt + 15) / 16 * 16;
  const uint32_t w = at / tt, t = at - w * tt;
  return make_uint4(e, w, first + t * per, count - t * per < per ? count - t * per : per);
}
__device__ __forceinline__ Tile tile_at(const Params &p, const int32_t *before, const int32_t *start, int64_t tile) {
  const uint4 f = find_tile((uint32_t)tile, before, start, (uint32_t)p.experts, (uint32_t)p.rows, (uint32_t)p.wtiles, (uint32_t)p.nt);
  return Tile{(int)f.x, (int)f.y * p.tile_rows, (int)f.z, (int)f.w, ((int)f.w + 15) / 16 * 16};
}

// The row of x's scales of place `at`.
__device__ __forceinline__ int64_t scale_row(const Params &p, int64_t at) {
  if (p.xs_rows == B200_ROWS_PLAN) return at;
  const int32_t pair = p.order[at];
  return p.xs_rows == B200_ROWS_PAIRS ? pair : pair / p.fan;
}

// The CTA's work: `whole` tiles blockIdx, blockIdx + grid, ..., then units u0 .. u1 of the tiles behind `tiles`,
// the `units` of which are shared out among `ctas`.
struct Run {
  int64_t tiles, units, u0, u1;
  int whole, ctas, turn;
  __device__ __forceinline__ int64_t start(int64_t c) const { return c * units / ctas; }
};
struct Seg {
  int64_t tile;
  int s0, len;  // K stages s0, s0 + 1, ... (a whole tile's go on at 0 behind the last)
};
// The k-th part of the CTA's work; `u` goes through the shared units.
__device__ __forceinline__ bool next_seg(const Params &p, const Run &run, int &k, int64_t &u, Seg &g) {
  if (k < run.whole) {
    g.tile = blockIdx.x + (int64_t)k * p.grid;
    g.s0 = run.turn, g.len = p.nst;
    ++k;
    return true;
  }
  if (u >= run.u1) return false;
  const int64_t t = u / p.nst;
  g.tile = run.tiles + t;
  g.s0 = (int)(u - t * p.nst);
  g.len = (int)(p.nst - g.s0 < run.u1 - u ? p.nst - g.s0 : run.u1 - u);
  u += g.len;
  return true;
}

template <typename T>
__device__ __forceinline__ T to_out(float v) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
  else return v;
}
struct E4M3 {};

// One weight row's products with CH tokens, column `c` of y: finished and stored. `up`, with a gate: the products
// that the activated ones multiply. `at` is the row of y of token j in lane j (pairs: of any order).
template <bool GATED, typename OUT>
__device__ __forceinline__ void finish(const Epilogue &ep, float (&v)[CH], float bias, const float (&up)[CH], float up_bias, int c,
                                       int at, int count, bool pairs) {
  const int lane = threadIdx.x & 31;
  const bool live = c < ep.cols;
#pragma unroll
  for (int j = 0; j < CH; ++j) v[j] += bias;
  switch (ep.activation) {  // outside the loop: a column's functions run side by side
    case B200_ACT_RELU:
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = activate<B200_ACT_RELU>(v[j]);
      break;
    case B200_ACT_SILU:
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = activate<B200_ACT_SILU>(v[j]);
      break;
    case B200_ACT_GELU:
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = activate<B200_ACT_GELU>(v[j]);
      break;
    case B200_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = activate<B200_ACT_GELU_TANH>(v[j]);
      break;
  }
  if constexpr (GATED) {
#pragma unroll
    for (int j = 0; j < CH; ++j) v[j] = __fmul_rn(v[j], up[j] + up_bias);
  }
  const int cols = (int)ep.cols, lim = live ? count : 0;
  if (ep.residual != nullptr) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int row = __shfl_sync(0xffffffffu, at, j);
      if (j < lim) v[j] += load_as_f32(ep.residual, row * ep.rstride + c, ep.rdt);
    }
  }
  if constexpr (std::is_same<OUT, E4M3>::value) {  // y's columns are whole blocks: a warp's are all live or none
    uint32_t top = 0;  // of token j in lane j, which finds the scale for all
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const uint32_t t = __reduce_max_sync(0xffffffffu, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      if (lane == j) top = t;
    }
    const uint32_t byte = rows8::scale_byte(top);
    const float inv = rows8::inverse(byte);
    if (lane < lim) ep.ys[(int64_t)at * (cols >> 5) + (c >> 5)] = (uint8_t)byte;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int row = __shfl_sync(0xffffffffu, at, j);
      const float s = __shfl_sync(0xffffffffu, inv, j);
      if (j < lim) ((uint8_t *)ep.y)[(int64_t)row * cols + c] = (uint8_t)rows8::codes2(v[j], 0.f, s, s == 0.f);
    }
  } else if (!pairs) {  // rows side by side
    OUT *y = (OUT *)ep.y + (int64_t)__shfl_sync(0xffffffffu, at, 0) * cols + c;
#pragma unroll
    for (int j = 0; j < CH; ++j, y += cols)
      if (j < lim) *y = to_out<OUT>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int row = __shfl_sync(0xffffffffu, at, j);
      if (j < lim) ((OUT *)ep.y)[(int64_t)row * cols + c] = to_out<OUT>(v[j]);
    }
  }
}

template <int R, bool GATED, typename OUT>
__global__ void __launch_bounds__(THREADS, 1)
    scaled_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx, const __grid_constant__ Params p, const __grid_constant__ Epilogue ep) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int S = p.stages;
  uint8_t *scales = ring + (size_t)S * p.stage_bytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(scales + (size_t)SLOTS * p.scale_bytes);
  uint64_t *empty = full + S;
  uint64_t *fulls = empty + S, *frees = fulls + SLOTS;  // scales landed, scales in tensor memory
  uint64_t *sfready = frees + SLOTS;
  uint64_t *accfull = sfready + SF_SETS;
  uint64_t *accempty = accfull + 2;
  uint64_t *drain = accempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 2);
  volatile uint32_t *abort_flag = tmem_slot + 1;
  volatile uint32_t *last_flag = tmem_slot + 2;
  int32_t *start = reinterpret_cast<int32_t *>(tmem_slot + 4);  // [experts + 1] the plan's offsets
  int32_t *before = start + p.experts + 1;                      // [experts + 1] token tiles of earlier experts

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < SLOTS; ++b) {
      mbar_init(&fulls[b], p.scale_warps);
      mbar_init(&frees[b], 1);
    }
    for (int b = 0; b < SF_SETS; ++b) mbar_init(&sfready[b], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accfull[b], 1);
      mbar_init(&accempty[b], EPI_WARPS);
    }
    mbar_init(drain, 1);
    mbar_init(drain + 1, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmw);
  }
  // The next kernel's CTAs may start as this one's leave. Nothing is read or written before the kernel in front has ended,
  // the weights neither: it may be the one that writes them, and may let its followers start before it has. (Asked for at
  // once, one token x 10240 x 8192 behind its norm took 20.7 us, not 24.1.) No wait's bound runs until then.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = threadIdx.x; e <= p.experts && p.experts > 0; e += THREADS) start[e] = p.offsets[e];
  if (warp == MMA_WARP) tmem_alloc(tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  if (warp == 0 && p.experts > 0) {  // token tiles of the experts before each
    int carry = 0;
    for (int first = 0; first < p.experts; first += 32) {
      const int e = first + lane;
      const int own = e < p.experts ? (int)tiles_of(p, start[e + 1] - start[e]) : 0;
      int v = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (e < p.experts) before[e] = carry + v - own;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) before[p.experts] = carry;
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Run run;
  {
    const int64_t all = (p.experts > 0 ? (int64_t)before[p.experts] : (int64_t)tiles_of(p, (int)p.rows)) * p.wtiles;
    const int waves = (int)(all / p.grid), rest = (int)(all % p.grid);
    run.turn = (int)((int64_t)blockIdx.x * p.nst / p.grid);
    run.tiles = (int64_t)waves * p.grid;
    // The tiles of the last, partial wave go whole to as many CTAs, or are cut up among more of them, whichever
    // ends sooner by what joining the parts costs
    int least = p.nst;
    run.ctas = 0;
    for (int i = 0; i < 10 && rest > 0; ++i) {
      const int pieces = i == 0 ? 0 : i < 4 ? i + 1 : i < 7 ? 2 * i - 2 : 8 * i - 40;  // all CTAs; 2, 3, 4, 6, 8, 10, 16, 24, 32 a tile
      const int ctas = i == 0 ? p.grid : rest * pieces;
      if (ctas > p.grid || ctas <= rest) continue;
      const int parts = i == 0 ? p.grid / rest + 2 : pieces;
      const int cost = (rest * p.nst + ctas - 1) / ctas + p.join + parts * p.join_part / 16;
      if (cost < least) least = cost, run.ctas = ctas;
    }
    run.whole = waves + (run.ctas == 0 && (int)blockIdx.x < rest ? 1 : 0);
    run.units = run.ctas > 0 ? (int64_t)rest * p.nst : 0;
    // Weights that only one tile of tokens reads gain nothing from tiles in turn: equal runs of all of them, whose first
    // and last tiles are cut (33 tokens gated, 224 tiles: 66 us; a tile each, then parts of 76: 72), if that ends sooner
    // than a wave of the rest
    const int64_t equal = (all * p.nst + p.grid - 1) / p.grid + p.join + 3 * p.join_part / 16;
    if (p.once && waves > 0 && rest > 0 && equal < (int64_t)(waves + 1) * p.nst) {
      run.whole = 0;
      run.tiles = 0;
      run.units = all * p.nst;
      run.ctas = p.grid;
    }
    if (run.ctas == 0) run.ctas = 1;
    run.u0 = (int)blockIdx.x < run.ctas ? run.start(blockIdx.x) : 0;
    run.u1 = (int)blockIdx.x < run.ctas ? run.start(blockIdx.x + 1) : 0;
  }
  const int64_t n = (int64_t)run.whole * p.nst + run.u1 - run.u0;  // stages

  if (warp >= W_WARP0) {
    // ---------------- TMA of weight codes: warp w takes the stages i = w (mod W_WARPS) ----------------
    if (lane == 0) {
      const int turn = warp - W_WARP0, turns = S < W_WARPS ? S : W_WARPS;
      int64_t i = turn, u = run.u0, row = 0, first = 0;
      int s = turn, k = 0, slot = turn;  // s: stages into the segment, behind its end until the next is taken
      Seg g = {0, 0, 0};
      uint32_t round = 0;
      for (; i < n && turn < turns; i += turns) {
        while (s >= g.len) {
          s -= g.len;
          if (!next_seg(p, run, k, u, g)) break;
          const Tile t = tile_at(p, before, start, g.tile);
          row = (int64_t)t.e * p.n + t.w0;
          first = p.single_row ? 0 : t.first;
        }
        if (round > 0 && !mbar_wait(&empty[slot], (round - 1u) & 1u, abort_flag)) break;
        uint8_t *st = ring + (size_t)slot * p.stage_bytes;
        mbar_arrive_expect_tx(&full[slot], p.tx);
        const int x = (g.s0 + s < p.nst ? g.s0 + s : g.s0 + s - p.nst) * KS;
        tma_load_2d(st, &tmw, x, (int32_t)row, &full[slot]);
        if constexpr (R == 2) tma_load_2d(st + TM * KS, &tmw, x, (int32_t)(row + p.second), &full[slot]);
        tma_load_2d(st + p.b_off, &tmx, x, (int32_t)first, &full[slot]);
        s += turns;
        if ((slot += turns) >= S) slot -= S, ++round;
      }
      if (*abort_flag) {  // this thread's copies in flight land before the CTA exits
        for (int64_t q = turn; q < (i < n ? i : n); q += turns)
          if (q + S >= i) mbar_drain(&full[q % S], (uint32_t)((q / S) & 1), 200000000ull);
      }
    }
  } else if (warp >= SCALE_WARP0 && warp < SCALE_WARP0 + p.scale_warps) {
    // ---------------- scale bytes: one atom a warp, R of the weights, then one or two of x ----------------
    const int atom = warp - SCALE_WARP0;
    const bool mine = atom < R;  // weights
    uint8_t *dst = scales + atom * 512 + lane * 16;
    int slot = 0, k = 0;
    uint32_t round = 0;
    int64_t u = run.u0;
    Seg g;
    bool ok = true;
    while (ok && next_seg(p, run, k, u, g)) {
      const Tile t = tile_at(p, before, start, g.tile);
      // rows lane, lane + 32, ... of the atom, `has` of them: side by side, or where the plan says
      const int64_t row = mine ? (int64_t)t.e * p.n + atom * p.second + t.w0 + lane : t.first + (atom - R) * 128 + lane;
      const int64_t rest = mine ? p.wrows - row : (int64_t)t.rows - (atom - R) * 128 - lane;
      const int has = rest >= 97 ? 4 : rest <= 0 ? 0 : (int)((rest + 31) >> 5);
      const uint8_t *src[4];
      src[0] = (mine ? p.ws : p.xs) + row * p.nblk;
#pragma unroll
      for (int q = 1; q < 4; ++q) src[q] = src[q - 1] + 32 * p.nblk;
      if (!mine && p.xs_rows != B200_ROWS_PLAN) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < has) src[q] = p.xs + scale_row(p, row + 32 * q) * p.nblk;
      }
      // four stages' bytes of each row, from a multiple of four on
      auto load = [&](int s, uint32_t (&v)[4][4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (q < has) {
            const uint8_t *from = src[q] + 4 * s;
            if (p.vector) {
              w = *reinterpret_cast<const uint4 *>(from);
            } else {
              const uint32_t *word = reinterpret_cast<const uint32_t *>(from);
              w.x = word[0];
              if (s + 1 < p.nst) w.y = word[1];
              if (s + 2 < p.nst) w.z = word[2];
              if (s + 3 < p.nst) w.w = word[3];
            }
          }
          v[q][0] = w.x, v[q][1] = w.y, v[q][2] = w.z, v[q][3] = w.w;
        }
      };
      // stages begin .. end - 1, and behind the last those before the first
      int begin = g.s0, end = g.s0 + g.len < p.nst ? g.s0 + g.len : p.nst, left = g.len;
      uint32_t now[4][4], next[4][4];
      load(begin & ~3, next);
      for (int s = begin & ~3; left > 0 && ok; s += 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) now[q][j] = next[q][j];
        const int first = begin, behind = end, at = s;
        left -= (at + 4 < behind ? at + 4 : behind) - (at > first ? at : first);
        if (s + 4 >= end) s = -4, begin = 0, end = left;  // from the first stage on
        if (left > 0) load(s + 4, next);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (at + j < first || at + j >= behind || !ok) continue;
          if (round > 0) ok = __all_sync(0xffffffffu, mbar_wait(&frees[slot], (round - 1u) & 1u, abort_flag));
          if (!ok) continue;
          *reinterpret_cast<uint4 *>(dst + slot * p.scale_bytes) = make_uint4(now[0][j], now[1][j], now[2][j], now[3][j]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&fulls[slot]);
          if (++slot == SLOTS) slot = 0, ++round;
        }
      }
    }
  } else if (warp == MMA_WARP) {
    // ---------------- MMA issuer: the whole warp, one lane of it elected ----------------
    const uint64_t ad = sw128_kmajor_desc(ring), bd = sw128_kmajor_desc(ring + p.b_off);  // the slots' follow: address / 16
    int slot = 0, set = 0, seg = -1;
    uint64_t off = 0;
    uint32_t phase = 0, sphase = 0;  // of the scale set, of the stage
    bool ok = true, over = false;
    int k = 0;
    int64_t u = run.u0;
    Seg g;
    while (ok && next_seg(p, run, k, u, g)) {
      const Tile t = tile_at(p, before, start, g.tile);
      const int len = g.len;
      ++seg;
      const int buf = p.bufs == 2 ? seg & 1 : 0;
      const uint32_t turn = (uint32_t)(p.bufs == 2 ? seg >> 1 : seg);  // uses of the accumulator before
      if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(&accempty[buf], (turn - 1u) & 1u, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)buf * R * p.acc_width;
      const uint32_t idesc = p.idesc | ((uint32_t)(t.width >> 3) << 17);
      for (int j = 0; j < len; ++j) {
        if (!over) {
          ok = mbar_wait(&sfready[set], phase, abort_flag) && mbar_wait(&full[slot], sphase, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t sf = tmem + p.sf_col + p.sf_width * (uint32_t)set;
        if (++set == p.sets) set = 0, phase ^= 1u;
        const int now = slot;
        if (++slot == S) slot = 0, sphase ^= 1u;
        // the next stage is asked for before this one's MMAs are issued
        over = __all_sync(0xffffffffu, mbar_over(&sfready[set], phase) & mbar_over(&full[slot], sphase));
#pragma unroll
        for (int q = 0; q < R; ++q)
          mma_stage(acc + (uint32_t)q * p.acc_width, ad + off + (uint64_t)(q * (TM * KS >> 4)), bd + off, idesc, (uint32_t)j, sf + 4u * q,
                    sf + 4u * R);
        commit(&empty[now]);
        off = slot == 0 ? 0 : off + (p.stage_bytes >> 4);
      }
      if (ok) commit(&accfull[buf]);
    }
    // every MMA issued has completed before the CTA frees its tensor memory
    commit(&drain[0]);
    if (lane == 0) mbar_drain(&drain[0], 0, 200000000ull);
    __syncwarp();
  } else if (warp == SF_WARP) {
    // ---------------- scales into tensor memory ----------------
    const uint64_t da = sf_desc(scales), db = sf_desc(scales + p.sfb_off);
    uint64_t off = 0;
    int slot = 0, set = 0, back = 0;  // back: the ring slot of the stage p.sets before, whose MMAs read the set
    uint32_t phase = 0, bphase = 0;
    bool ok = true;
    for (int64_t i = 0; i < n; ++i) {
      const bool reuse = i >= p.sets;
      bool over = mbar_over(&fulls[slot], phase);
      if (reuse) over = over & mbar_over(&empty[back], bphase);
      if (!__all_sync(0xffffffffu, over)) {
        ok = mbar_wait(&fulls[slot], phase, abort_flag) && (!reuse || mbar_wait(&empty[back], bphase, abort_flag));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      fence_proxy_async_smem();  // threads wrote by the generic proxy, the tensor core reads by the other
      tc_fence_after();
      const uint32_t sf = tmem + p.sf_col + p.sf_width * (uint32_t)set;
#pragma unroll
      for (int q = 0; q < R; ++q) sf_copy(sf + 4u * q, da + off + 32u * q);
      sf_copy(sf + 4u * R, db + off);
      if (p.nt > 128) sf_copy(sf + 4u * R + 4u, db + off + 32u);
      commit(&sfready[set]);
      commit(&frees[slot]);
      off += p.scale_bytes >> 4;
      if (++slot == SLOTS) slot = 0, off = 0, phase ^= 1u;
      if (++set == p.sets) set = 0;
      if (reuse && ++back == S) back = 0, bphase ^= 1u;
    }
    // its copies have completed before the tensor memory is freed: the last MMAs followed them, but after a
    // wait that ran out they may not have
    commit(&drain[1]);
    if (lane == 0) mbar_drain(&drain[1], 0, 200000000ull);
    __syncwarp();
  } else if (warp < EPI_WARPS) {
    // ---------------- epilogue: weight row = tensor-memory lane, token = column ----------------
    constexpr int TOGETHER = GATED ? 2 : 1, PARTS = R / TOGETHER;
    const int quarter = warp & 3, group = warp >> 2;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    bool ok = true;  // this warp's waits; after one that ran out it still meets the others
    int seg = 0, k = 0;
    int64_t u = run.u0;
    Seg g;
    for (; next_seg(p, run, k, u, g); ++seg) {
      const bool whole = g.len == p.nst;
      const Tile t = tile_at(p, before, start, g.tile);
      const int c = (int)t.w0 + quarter * 32 + lane;  // column of y; ungated, the second accumulator's is c + 128
      float bias[R];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const int64_t row = q * p.second + c;
        bias[q] = ep.bias != nullptr && row < p.n ? load_as_f32(ep.bias, (int64_t)t.e * p.n + row, ep.bdt) : 0.f;
      }
      auto row_of = [&](int j0, int count) -> int {  // of y, of token j0 + lane
        const int at = t.first + j0 + (lane < count ? lane : 0);
        return p.y_pairs ? p.order[at] : at;
      };
      const int buf = p.bufs == 2 ? seg & 1 : 0;
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&accfull[buf], (uint32_t)((p.bufs == 2 ? seg >> 1 : seg) & 1), abort_flag));
      tc_fence_after();
      const uint32_t acc = tmem + lane_base + (uint32_t)buf * R * p.acc_width;
      // partial sums: of the first of the CTA's shared tiles in place 0, of the last in place 1
      const size_t place = (size_t)R * p.nt * TM;
      // four tokens of a row side by side
      float4 *mine = reinterpret_cast<float4 *>(p.part + ((size_t)blockIdx.x * 2 + (u - g.len == run.u0 ? 0 : 1)) * place) + quarter * 32 + lane;
      // steps of CH tokens, of one accumulator or of a gate's two; the groups take turns at them
      const int steps = PARTS * ((t.rows + CH - 1) / CH);
      if (group >= steps && lane == 0) mbar_arrive(&accempty[buf]);
#pragma unroll 1
      for (int step = group; step < steps; step += 2) {
        const int part = step % PARTS, j0 = step / PARTS * CH, count = t.rows - j0 < CH ? t.rows - j0 : CH;
        float v[TOGETHER][CH];
#pragma unroll
        for (int q = 0; q < TOGETHER; ++q) tmem_ld_32x32b_x16(acc + (uint32_t)(part + q) * p.acc_width + (uint32_t)(p.single_row ? 0 : j0), reinterpret_cast<uint32_t (&)[CH]>(v[q]));
        tmem_ld_wait();
        if (p.single_row) {  // a token that names an expert twice: its row is the first column's
#pragma unroll
          for (int q = 0; q < TOGETHER; ++q)
#pragma unroll
            for (int j = 1; j < CH; ++j) v[q][j] = v[q][0];
        }
        if (step + 2 >= steps) {  // the group's last columns are read: the accumulator may be used again
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&accempty[buf]);
        }
        if (!ok) continue;
        if (whole) {
          finish<GATED, OUT>(ep, v[0], part == 0 ? bias[0] : bias[R - 1], v[TOGETHER - 1], bias[R - 1], c + part * TM, row_of(j0, count), count, p.y_pairs);
        } else {
#pragma unroll
          for (int q = 0; q < TOGETHER; ++q)
#pragma unroll
            for (int j = 0; j < CH / 4; ++j)
              __stcg(mine + ((part + q) * p.nt + j0 + 4 * j) / 4 * TM, make_float4(v[q][4 * j], v[q][4 * j + 1], v[q][4 * j + 2], v[q][4 * j + 3]));
        }
      }
      if (!whole) {
        // the CTAs whose runs hold the tile's first and last unit; the tile's ticket is the first one's
        const int64_t tile = g.tile - run.tiles, a = tile * p.nst, b = a + p.nst - 1;
        int cf = (int)(a * run.ctas / run.units), cl = (int)(b * run.ctas / run.units);
        while (cf > 0 && run.start(cf) > a) --cf;
        while (cf + 1 < run.ctas && run.start(cf + 1) <= a) ++cf;
        while (cl > 0 && run.start(cl) > b) --cl;
        while (cl + 1 < run.ctas && run.start(cl + 1) <= b) ++cl;
        epi_sync();  // orders all parts' stores before the fence, which publishes them
        if (threadIdx.x == 0) {
          __threadfence();
          unsigned int old = ~0u;  // not counted: nobody finishes the tile
          if (ok && !*abort_flag) asm volatile("atom.add.acq_rel.gpu.u32 %0, [%1], 1;" : "=r"(old) : "l"(&p.tickets[cf]) : "memory");
          *last_flag = old == (unsigned int)(cl - cf) ? 1u : 0u;
        }
        epi_sync();
        if (*last_flag) {
#pragma unroll 1
          for (int step = group; step < steps; step += 2) {
            const int part = step % PARTS, j0 = step / PARTS * CH, count = t.rows - j0 < CH ? t.rows - j0 : CH;
            float v[TOGETHER][CH];
#pragma unroll
            for (int q = 0; q < TOGETHER; ++q)
#pragma unroll
              for (int j = 0; j < CH; ++j) v[q][j] = 0.f;
            for (int cc = cf; cc <= cl; cc += 2) {  // two parts' loads in flight together, added in turn
              float4 w[2][TOGETHER][CH / 4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int64_t first = run.start(cc + h < cl ? cc + h : cl) / p.nst;
                const float4 *src = reinterpret_cast<const float4 *>(p.part + ((size_t)(cc + h < cl ? cc + h : cl) * 2 + (first == tile ? 0 : 1)) * place) +
                                    quarter * 32 + lane;
#pragma unroll
                for (int q = 0; q < TOGETHER; ++q)
#pragma unroll
                  for (int j = 0; j < CH / 4; ++j) w[h][q][j] = __ldcg(src + ((part + q) * p.nt + j0 + 4 * j) / 4 * TM);
              }
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (cc + h > cl) break;
#pragma unroll
                for (int q = 0; q < TOGETHER; ++q)
#pragma unroll
                  for (int j = 0; j < CH / 4; ++j) {
                    v[q][4 * j] += w[h][q][j].x, v[q][4 * j + 1] += w[h][q][j].y;
                    v[q][4 * j + 2] += w[h][q][j].z, v[q][4 * j + 3] += w[h][q][j].w;
                  }
              }
            }
            finish<GATED, OUT>(ep, v[0], part == 0 ? bias[0] : bias[R - 1], v[TOGETHER - 1], bias[R - 1], c + part * TM, row_of(j0, count), count, p.y_pairs);
          }
          if (threadIdx.x == 0) p.tickets[cf] = 0u;  // ready for the next call
        }
        epi_sync();
      }
    }
    // rows of pairs that no expert has are zeros
    if (p.y_pairs) {
      const int64_t size = std::is_same<OUT, E4M3>::value ? 1 : sizeof(OUT), bytes = ep.cols * size;
      for (int64_t r = start[p.experts] + blockIdx.x; r < p.rows; r += gridDim.x) {
        const int64_t row = p.order[r];
        uint8_t *y = (uint8_t *)ep.y + row * bytes;
        for (int64_t o = threadIdx.x; o < bytes / size; o += EPI_WARPS * 32) {
          if (size == 4) ((uint32_t *)y)[o] = 0u;
          else if (size == 2) ((uint16_t *)y)[o] = 0u;
          else y[o] = 0u;
        }
        if constexpr (std::is_same<OUT, E4M3>::value)
          for (int64_t o = threadIdx.x; o < ep.cols >> 5; o += EPI_WARPS * 32) ep.ys[row * (ep.cols >> 5) + o] = 27u;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, p.tmem_cols);
}

// x's codes in the plan's order, 16 bytes a thread: a tile of an expert's tokens is one box then. It costs a
// write and a read of rows x cols bytes (32008 x 4096: 30 us beside 1000 us of products); copying the rows
// with cp.async within the product kept its load/store unit busy for longer than a stage takes.
__global__ void __launch_bounds__(256) gather_kernel(const uint8_t *x, uint8_t *out, const int32_t *offsets, const int32_t *order,
                                                     int experts, int fan, int pairs, int64_t cols) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_row = (int)(cols >> 4);
  const int64_t all = (int64_t)offsets[experts] * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t at = i / per_row;
    const int32_t pair = order[at];
    const int64_t row = pairs ? pair : pair / fan;
    reinterpret_cast<uint4 *>(out)[i] = reinterpret_cast<const uint4 *>(x)[row * per_row + (i - at * per_row)];
  }
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Rows that meet one matrix: all, or an expert's share.
static int64_t rows_of_one(const b200_scaled_args *a) {
  return a->experts > 0 ? (a->rows + a->experts - 1) / a->experts : a->rows;
}
// Gated, 113 to 224 tokens: accumulators of twice the width that do not take turns, so that the weights
// are read once (200 tokens x 57344 x 8192 112 us, with two tiles of tokens 122).
static bool single(const b200_scaled_args *a) {
  return a->experts == 0 && a->rows > ACC_COLS / 2 && a->rows <= ACC_COLS;
}

template <int R, bool GATED, typename OUT>
static int32_t launch_t(const b200_packed_desc *w, const b200_scaled_args *a, int bufs, cudaStream_t stream) {
  int sms = 0;
  B200_CUDA_TRY(device_sms(&sms));
  const int bits = fmt_bits(w->format);
  Params p;
  memset(&p, 0, sizeof(p));
  p.xs = (const uint8_t *)a->x_scales, p.ws = (const uint8_t *)w->scales;
  p.offsets = a->offsets, p.order = a->order;
  p.rows = a->rows;
  p.n = a->experts > 0 ? w->rows / a->experts : w->rows;
  p.wrows = w->rows;
  p.cols = w->cols;
  p.nblk = w->cols / 32;
  p.nst = (int)(w->cols / KS);
  p.experts = (int)a->experts, p.fan = a->experts > 0 ? a->fan : 1;
  p.xs_rows = a->experts > 0 ? a->x_rows : B200_ROWS_PLAN;
  p.y_pairs = a->experts > 0 && a->y_rows != B200_ROWS_PLAN;
  p.vector = p.nst % 4 == 0 && (uintptr_t)a->x_scales % 16 == 0 && (uintptr_t)w->scales % 16 == 0;
  const Epilogue ep = epilogue_of(w, a);
  p.second = GATED ? ep.cols : TM;
  p.tile_rows = R == 2 && !GATED ? 2 * TM : TM;
  p.wtiles = (int)((ep.cols + p.tile_rows - 1) / p.tile_rows);
  p.bufs = bufs;
  // tokens of a tile: equally full tiles; an expert's are as many as three times its share, in reason (fewer
  // leave room for more stages, and who has more takes several tiles)
  const int64_t limit = bufs == 2 ? ACC_COLS / R : ACC_COLS;
  int64_t most = a->rows;
  if (a->experts > 0) {
    const int64_t tokens = (a->rows + a->fan - 1) / a->fan, share = 3 * rows_of_one(a);
    most = share < 32 ? 32 : share;
    most = most < tokens ? most : tokens;
  }
  const int64_t tt = (most + limit - 1) / limit;
  p.nt = a->experts > 0 && tt > 1 ? (int)limit : (int)(((most + tt - 1) / tt + 15) / 16 * 16);
  p.b_off = (uint32_t)(R * TM * KS);
  p.stage_bytes = p.b_off + (uint32_t)((p.nt * KS + 1023) / 1024 * 1024);
  p.sfb_off = R * 512;
  p.scale_bytes = p.sfb_off + (p.nt > 128 ? 1024 : 512);
  p.scale_warps = R + (p.nt > 128 ? 2 : 1);
  static_assert(R + 2 <= SCALE_WARPS, "a warp for each atom");
  const size_t tail = 8 * (2 * MAX_STAGES + 2 * SLOTS + SF_SETS + 6) + 16 + 8 * ((size_t)p.experts + 1) + 16;
  int stages = (int)((SMEM_LIMIT - 1024 - tail - SLOTS * p.scale_bytes) / p.stage_bytes);
  p.stages = stages < MAX_STAGES ? stages : MAX_STAGES;
  p.sets = p.stages < SF_SETS ? p.stages : SF_SETS;
  p.tx = (uint32_t)(R * TM * KS * bits / 8);  // codes as they lie in global memory
  p.acc_width = (uint32_t)p.nt;
  p.sf_col = (uint32_t)bufs * R * p.acc_width;
  p.sf_width = 4 * R + (p.nt > 128 ? 8 : 4);
  p.tmem_cols = 32;
  while (p.tmem_cols < p.sf_col + p.sf_width * SF_SETS) p.tmem_cols *= 2;
  const uint32_t fmt = w->format == B200_FMT_FP4_E2M1 ? 5u : w->format == B200_FMT_FP6_E2M3 ? 3u : 4u;
  p.idesc = (fmt << 7) | (0u << 10) | (1u << 23) | ((uint32_t)(TM >> 4) << 24);  // B: E4M3; E8M0 scales
  p.grid = sms;
  // 200 tokens x 4096 x 4096, each tile cut in five: 38 us, 30 of them for the joining; a stage takes 0.45
  p.once = rows_of_one(a) <= p.nt;
  p.join = 6;
  p.join_part = p.nt * R * 14 / 16;
  const size_t part = (size_t)sms * 2 * 2 * ACC_COLS * TM * sizeof(float);
  uint8_t *base = nullptr;
  if (int32_t rc = workspace_of(WS_SCALED, part, TICKETS * sizeof(unsigned int), stream, &base)) return rc;
  p.part = reinterpret_cast<float *>(base);
  p.tickets = reinterpret_cast<unsigned int *>(base + part);

  CUtensorMap tmw;
  const uint64_t row_bytes = (uint64_t)w->cols * bits / 8;
  if (int32_t rc = make_tma_2d(&tmw, bits == 4 ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_16U6_ALIGN16B,
                               w->data, (uint64_t)w->cols, (uint64_t)w->rows, row_bytes, KS, TM, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  const uint8_t *xcodes = (const uint8_t *)a->x;
  int64_t xrows = a->rows;
  if (scaled_gathers(a)) {
    const int64_t ctas = (a->rows * (w->cols / 16) + 255) / 256;
    B200_CUDA_TRY(launch_dependent(gather_kernel, dim3((unsigned)(ctas < 8 * sms ? ctas : 8 * sms)), dim3(256), 0, stream, xcodes,
                                   (uint8_t *)a->scratch, a->offsets, a->order, (int)a->experts, (int)a->fan,
                                   (int)(a->x_rows == B200_ROWS_PAIRS), w->cols));
    xcodes = (const uint8_t *)a->scratch;
  } else if (a->experts > 0 && a->x_rows != B200_ROWS_PLAN) {
    p.single_row = 1;
    xrows = 1;
  }
  p.tx += (uint32_t)(p.nt * KS);
  CUtensorMap tmx;
  if (int32_t rc = make_tma_2d(&tmx, CU_TENSOR_MAP_DATA_TYPE_UINT8, xcodes, (uint64_t)w->cols, (uint64_t)xrows, (uint64_t)w->cols, KS,
                               (uint32_t)p.nt, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + SLOTS * p.scale_bytes + tail;
  B200_CUDA_TRY((ensure_dynamic_smem<scaled_kernel<R, GATED, OUT>>(SMEM_LIMIT)));
  B200_CUDA_TRY(launch_dependent(scaled_kernel<R, GATED, OUT>, dim3((unsigned)p.grid), dim3(THREADS), smem, stream, tmw, tmx, p, ep));
  return B200_OK;
}

template <int R, bool GATED>
static int32_t dispatch(const b200_packed_desc *w, const b200_scaled_args *a, int bufs, cudaStream_t stream) {
  switch (a->y_dtype) {
    case B200_DT_F16: return launch_t<R, GATED, __half>(w, a, bufs, stream);
    case B200_DT_BF16: return launch_t<R, GATED, __nv_bfloat16>(w, a, bufs, stream);
    case B200_DT_F32: return launch_t<R, GATED, float>(w, a, bufs, stream);
    default: return launch_t<R, GATED, E4M3>(w, a, bufs, stream);
  }
}

}  // namespace scaled

// Rows of x that are no tile as they lie: tokens' or pairs' rows, unless they are one.
bool scaled_gathers(const b200_scaled_args *a) {
  return a->experts > 0 && a->x_rows != B200_ROWS_PLAN && !(a->x_rows == B200_ROWS_TOKENS && a->rows <= a->fan) && a->rows > 1;
}

// What the checks of the entry have left: whole stages, and the alignment that TMA and the loads of scales ask for.
bool scaled_mma_takes(const b200_packed_desc *w, const b200_scaled_args *a) {
  if (w->cols % scaled::KS != 0 || w->cols > (1 << 24) || w->rows > (1ll << 31) - 256) return false;
  if ((uintptr_t)w->data % 32 != 0 || (uintptr_t)w->scales % 4 != 0) return false;
  if ((uintptr_t)a->x % 16 != 0 || (uintptr_t)a->x_scales % 4 != 0) return false;
  // tiles are counted in 31 bits: rows of y / 16 and some for the experts' last ones, times 128 rows of weights
  const int64_t n = a->experts > 0 ? w->rows / a->experts : w->rows;
  if ((a->rows / 16 + a->experts + 1) * (n / scaled::TM + 1) >= 1ll << 31) return false;
  return a->experts <= scaled::MAX_EXPERTS;
}

int32_t launch_scaled_mma(const b200_packed_desc *w, const b200_scaled_args *a, cudaStream_t stream) {
  // Two accumulators of 112 tokens halve a decode step's stages (one token x 57344 x 8192, us, with two / one: 48 / 60) and
  // load less for many tokens (2560 x 8192 x 8192 157 / 175, 4096 x 1024 x 16384 67 / 90); between, one of 224 goes over the weights
  // half as often (128 tokens x 57344 x 8192 97 / 82, 800 x 4096 x 14336 60 / 55, 1600 x 8192 x 8192 117 / 106, 2048 x 14336 x 4096
  // 132 / 127). Experts' tiles are seldom full, whatever their width: two at every share (224 tokens each x 4096 x 2048 64 / 77,
  // 500 118 / 137, 1100 259 / 264; of 2048 x 4096 128 tokens each 43 / 40, 500 97 / 102, 2500 401 / 462).
  if (a->gated) return scaled::dispatch<2, true>(w, a, scaled::single(a) ? 1 : 2, stream);
  if (a->experts > 0 || a->rows <= scaled::ACC_COLS / 2 || a->rows > 2304) return scaled::dispatch<2, false>(w, a, 2, stream);
  return scaled::dispatch<1, false>(w, a, 2, stream);
}

}  // namespace b200
