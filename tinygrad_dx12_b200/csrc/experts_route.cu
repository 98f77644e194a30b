// experts_route.cu -- which experts a row goes to, the order in which experts read their rows, and the
// sum of what they give back.
//
// Routing: a warp a row, expert e in lane e % 32. Choices become whole numbers that order like them (0:
// cannot be chosen), 32 bits where the logits decide and 64 where scores do, so a round of the k best is
// a warp-wide maximum, and a tie a warp-wide minimum of the index: no sort, and the same choice whatever
// else runs. Scores that decide are compared in 64 bits wherever 32 are not sure of the order: two experts
// whose scores differ by less than fp32 resolves are ordered as their definition has it.
// Plan: a stable counting sort of the pairs by expert. CTAs count their chunk's pairs, one warp an expert
// sums the counts over the chunks, and each CTA places its chunk: warps own consecutive pieces of it, so a
// pair's place is what lies before it in earlier chunks, earlier warps, earlier rounds and lower lanes.
// No atomics on places: the order is the same every time. Few pairs take one launch of one CTA.
// Bound by the launches up to some ten thousand pairs, then by the routing's instructions (32768 rows of 64 experts: issue 64 %).
#include <type_traits>

#include "kernels.h"
#include "common.cuh"

namespace b200 {
namespace route {

constexpr int MAX_EXPERTS = 1024, MAX_K = 32, MAX_GROUPS = 32;
constexpr int PLAN_WARPS = 32, PLAN_THREADS = 32 * PLAN_WARPS;

struct RouteParams {
  b200_route_args a;
};

// Whole numbers that order like the values; 0 stands for what cannot be chosen (and orders below all).
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order64(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float value32(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
// The same of a 16-bit logit that was widened: 16 bits, never 0. What stood for infinity stays above the type's
// largest value.
__device__ __forceinline__ uint32_t packed16(uint32_t k, int dtype) {
  if (dtype == B200_DT_BF16) return (k >> 16) + (k == order32(3.402823466e38f) ? 1u : 0u);
  const uint32_t h = (uint32_t)__half_as_ushort(__float2half_ru(value32(k)));
  return h ^ ((h >> 15) ? 0xFFFFu : 0x8000u);
}
__device__ __forceinline__ double value64(uint64_t k) {
  return __longlong_as_double((long long)(k ^ ((k >> 63) ? 1ull << 63 : ~0ull)));
}

// Launched behind a kernel that lets its followers start early: everything waits for it, and lets others start.
__device__ __forceinline__ void follow() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... KArgs, typename... Args>
static cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The lanes that hold the warp's largest key; empty if it is 0 everywhere. The low half is only compared where
// the high halves tie.
__device__ __forceinline__ uint32_t holders(uint32_t v) {
  const uint32_t top = __reduce_max_sync(0xffffffffu, v);
  return __ballot_sync(0xffffffffu, v == top && top != 0);
}
__device__ __forceinline__ uint32_t holders(uint64_t v) {
  const uint32_t hi = (uint32_t)(v >> 32), top = __reduce_max_sync(0xffffffffu, hi);
  uint32_t who = __ballot_sync(0xffffffffu, hi == top && v != 0);
  if (who & (who - 1)) {
    const uint32_t low = __reduce_max_sync(0xffffffffu, (who >> (threadIdx.x & 31) & 1u) ? (uint32_t)v : 0u);
    who &= __ballot_sync(0xffffffffu, (uint32_t)v == low);
  }
  return who;
}

// What a key is made of: a 16-bit logit and the index below it (one maximum a round finds both); a logit; a score
// in 32 bits; a score in 64 bits.
enum Mode { PACKED, LOGIT, QUICK, EXACT };

// One row, by a warp, N experts a lane. Scores that decide are compared in 32 bits first: where two neighbours in the
// order of what is chosen, or the last chosen and the next, lie closer than 32 bits are sure of, the answer is false
// and the row is done again in 64 (a row of 256 experts in 64 bits takes 4500 instructions, half of them exponentials).
// `smem` holds the warp's keys where there are groups: lane g goes through group g's.
template <int N, Mode MODE>
__device__ __forceinline__ bool route_row(const b200_route_args &a, int64_t row, void *smem) {
  constexpr bool WIDE = MODE == EXACT, SCORES = MODE == EXACT || MODE == QUICK;
  using Key = typename std::conditional<WIDE, uint64_t, uint32_t>::type;
  const int lane = threadIdx.x & 31;
  int32_t *indices = a.indices + row * a.k;
  float *weights = a.weights + row * a.k;
  if (a.live != nullptr && row >= *a.live) {
    if (lane < a.k) indices[lane] = -1, weights[lane] = 0.f;
    return true;
  }
  // logits; -inf for what cannot be chosen by them
  float x[N];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = lane + 32 * i;
    float v = -INFINITY;
    if (e < a.experts) {
      if (a.dtype == B200_DT_F32) v = ((const float *)a.logits)[row * a.stride + e];
      else if (a.dtype == B200_DT_F16) v = __half2float(((const __half *)a.logits)[row * a.stride + e]);
      else v = __bfloat162float(((const __nv_bfloat16 *)a.logits)[row * a.stride + e]);
      v = v != v ? -INFINITY : fminf(v, 3.402823466e38f);
    }
    x[i] = v;
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // the softmax's denominator, over all experts with a logit; weights over their sum do without
  float total = 0.f;
  if (!a.sigmoid && (!a.renormalize || MODE == QUICK)) {
#pragma unroll
    for (int i = 0; i < N; ++i) total += x[i] == -INFINITY ? 0.f : expf(x[i] - top);
    total = warp_sum(total);
  }
  Key key[N];
  float span = 0.f;  // the largest |bias|
  if constexpr (WIDE) {
    double all = 1.0;
    if (!a.sigmoid) {
      all = 0.0;
#pragma unroll
      for (int i = 0; i < N; ++i) all += x[i] == -INFINITY ? 0.0 : exp((double)x[i] - (double)top);
      all = warp_sum(all);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      key[i] = 0;
      if (x[i] == -INFINITY) continue;
      double c = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[i])) : exp((double)x[i] - (double)top) / all;
      if (a.bias != nullptr) {
        const float b = a.bias[lane + 32 * i];
        if (b != b || b == -INFINITY) continue;
        c += (double)fminf(b, 3.402823466e38f);
      }
      key[i] = order64(c == 0.0 ? 0.0 : c);  // one zero
    }
  } else if constexpr (MODE == QUICK) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      key[i] = 0;
      if (x[i] == -INFINITY) continue;
      float c = a.sigmoid ? __fdividef(1.f, 1.f + expf(-x[i])) : __fdividef(expf(x[i] - top), total);
      if (a.bias != nullptr) {
        const float b = a.bias[lane + 32 * i];
        if (b != b || b == -INFINITY) continue;
        c += fminf(b, 3.402823466e38f);
        span = fmaxf(span, fabsf(b));
      }
      key[i] = order32(c == 0.f ? 0.f : c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) span = fmaxf(span, __shfl_xor_sync(0xffffffffu, span, o));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      key[i] = x[i] == -INFINITY ? 0u : order32(x[i] == 0.f ? 0.f : x[i]);
      if (MODE == PACKED && key[i] != 0) key[i] = (packed16(key[i], a.dtype) << 16) | (0xFFFFu - (uint32_t)(lane + 32 * i));
    }
  }
  // What 32 bits are not sure of. A score c = e^(x - top) / total is off by E c: the subtraction's rounding is up to 2^-18
  // of an exponent (x - top beyond -64), the total's up to (N + 5) 2^-24 <= 2^-18.8 (lanes' terms, then the tree), exponentials
  // and division 5 ulp: 9e-6 in all; a sigmoid has only the last, 8e-7. A choice is c + bias, a group's sum two of them, so the
  // scores in it add up to at most |sum| + 2 span, and two sums that differ by more than 2 E (|higher| + 2 span) and what the
  // additions round (2^-24 of the same) are in order. Below 2^-126 a score is off by steps of 2^-149 whatever its size, and the fast
  // division gives zero: 2^-100 covers that. What is no number (infinite sums) is not sure either.
  const float unsure = a.sigmoid ? 4e-6f : 2e-5f;
  auto close = [&](float higher, float lower) { return !(higher - lower > fmaf(unsure, fabsf(higher) + 2.f * span, 7.9e-31f)); };
  if (a.groups > 1) {
    const int size = a.experts / a.groups;
    Key *keys = (Key *)smem;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < a.experts) keys[lane + 32 * i] = key[i];
    __syncwarp();
    // lane g: group g's best and next best, from a place of its own on, so that lanes read different banks
    Key mine = 0, next = 0;
    if (lane < a.groups) {
      const Key *group = keys + lane * size;
      int at = lane % size;
      for (int j = 0; j < size; ++j) {
        const Key v = group[at];
        at = at + 1 == size ? 0 : at + 1;
        next = max(next, min(mine, v));
        mine = max(mine, v);
      }
      if constexpr (SCORES) {
        if (a.group_best == 2 && next != 0) {
          if constexpr (WIDE) {
            const double sum = value64(mine) + value64(next);
            mine = order64(sum == 0.0 ? 0.0 : sum);
          } else {
            const float sum = value32(mine) + value32(next);
            mine = order32(sum == 0.f ? 0.f : sum);
          }
        }
      }
    }
    uint32_t kept = 0;
    float before = 0.f;
    for (int r = 0; r < a.top_groups + (MODE == QUICK ? 1 : 0); ++r) {
      const uint32_t who = holders(mine);
      if (who == 0) break;
      const int g = __ffs(who) - 1;  // the lowest on a tie
      if constexpr (MODE == QUICK) {  // which groups, not in what order
        const float score = value32(__shfl_sync(0xffffffffu, mine, g));
        if (r == a.top_groups) {
          if (close(before, score)) return false;
          break;
        }
        before = score;
      }
      kept |= 1u << g;
      if (lane == g) mine = 0;
    }
    if (lane < a.groups && !(kept >> lane & 1u)) {
      int at = lane % size;
      for (int j = 0; j < size; ++j) {
        keys[lane * size + at] = 0;
        at = at + 1 == size ? 0 : at + 1;
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < a.experts) key[i] = keys[lane + 32 * i];
    __syncwarp();
  }
  // the k best, round by round: lane j keeps the j-th
  int chosen = -1;
  float logit = -INFINITY, before = 0.f;
  for (int j = 0; j < a.k + (MODE == QUICK ? 1 : 0); ++j) {
    Key best = 0;
    float value = 0.f;
    uint32_t index = 0xFFFFFFFFu, at;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (key[i] > best) best = key[i], value = x[i], index = lane + 32 * i;  // the lower index on a tie
    if constexpr (MODE == PACKED) {
      const uint32_t first = __reduce_max_sync(0xffffffffu, best);
      if (first == 0) break;
      at = 0xFFFFu - (first & 0xFFFFu);
    } else {
      const uint32_t who = holders(best);
      if (who == 0) break;
      at = __shfl_sync(0xffffffffu, index, __ffs(who) - 1);
      if (who & (who - 1)) at = __reduce_min_sync(0xffffffffu, (who >> lane & 1u) ? index : 0xFFFFFFFFu);
      if constexpr (MODE == QUICK) {
        const float choice = value32(__shfl_sync(0xffffffffu, best, __ffs(who) - 1));
        if (j > 0 && close(before, choice)) return false;
        if (j == a.k) break;
        before = choice;
      }
    }
    value = __shfl_sync(0xffffffffu, value, at & 31);
    if (lane == j) chosen = (int)at, logit = value;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((int)at == lane + 32 * i) key[i] = 0;
  }
  float w = 0.f;
  if (a.renormalize) {
    // scores over their sum, both divided by the largest softmax numerator of the chosen (exp(min(0, the
    // largest logit)) for sigmoids): neither vanishes, however small the scores are
    float most = logit;
    if constexpr (SCORES) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    } else {
      most = __shfl_sync(0xffffffffu, most, 0);  // by logits the first chosen has the largest
    }
    if (chosen >= 0) {
      if (!a.sigmoid) w = expf(logit - most);
      else if (most >= 0.f) w = 1.f / (1.f + expf(-logit));
      else w = expf(logit - most) / (1.f + expf(logit));
    }
    const float sum = warp_sum(w);
    w = chosen >= 0 ? w / sum : 0.f;
  } else if (chosen >= 0) {
    w = a.sigmoid ? 1.f / (1.f + expf(-logit)) : expf(logit - top) / total;
  }
  if (lane < a.k) indices[lane] = chosen, weights[lane] = w * a.scale;
  return true;
}

// (the exact one's code apart: a kernel of much straight code waits for its instructions)
template <int N>
__device__ __noinline__ void route_row_exactly(const b200_route_args &a, int64_t row, void *smem) {
  route_row<N, EXACT>(a, row, smem);
}

template <int N, Mode MODE>
__global__ void __launch_bounds__(128) route_kernel(const __grid_constant__ RouteParams rp) {
  __shared__ __align__(8) uint8_t keys[4][N * 32 * 8];
  follow();
  const int warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 4 + warp;
  if (row < rp.a.rows && !route_row<N, MODE>(rp.a, row, keys[warp])) route_row_exactly<N>(rp.a, row, keys[warp]);
}

// ---- the plan -------------------------------------------------------------------------------------
struct PlanParams {
  const int32_t *indices;
  int64_t pairs;
  int first, experts;
  int32_t *offsets, *order;
  int32_t *counts;  // [experts + 1][chunks]: pairs of a chunk, then those of earlier chunks
  int32_t *totals;  // [experts + 1]
  int64_t chunk;    // pairs a chunk, a multiple of PLAN_THREADS
  int chunks;
};

__device__ __forceinline__ int bin_of(const PlanParams &p, int64_t i) {
  const uint32_t e = (uint32_t)p.indices[i] - (uint32_t)p.first;  // below `first`: wraps far beyond
  return p.indices[i] >= p.first && e < (uint32_t)p.experts ? (int)e : p.experts;
}

// Pairs [begin, end) of each warp of CTA `c`: consecutive pieces of whole rounds of 32.
__device__ __forceinline__ void piece(const PlanParams &p, int c, int warp, int64_t &begin, int64_t &end) {
  const int64_t per = p.chunk / PLAN_WARPS;
  begin = c * p.chunk + warp * per;
  end = begin + per < p.pairs ? begin + per : p.pairs;
}

// hist[warp][bin] = pairs of each bin in the warp's piece.
__device__ __forceinline__ void count_pieces(const PlanParams &p, int c, int32_t *hist) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bins = p.experts + 1;
  for (int i = threadIdx.x; i < PLAN_WARPS * bins; i += PLAN_THREADS) hist[i] = 0;
  __syncthreads();
  int64_t begin, end;
  piece(p, c, warp, begin, end);
#pragma unroll 4
  for (int64_t i = begin + lane; i < end; i += 32) atomicAdd(&hist[warp * bins + bin_of(p, i)], 1);
  __syncthreads();
}

// base[bin] = where the bin begins, from the totals in `base`: an exclusive sum in place (bins <= 1056).
__device__ __forceinline__ void exclusive(int32_t *base, int bins) {
  __shared__ int32_t part[PLAN_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int carry = 0;
  for (int first = 0; first < bins; first += PLAN_THREADS) {
    const int i = first + threadIdx.x;
    const int own = i < bins ? base[i] : 0;
    int v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) part[warp] = v;
    __syncthreads();
    int before = carry, all = 0;
    for (int w = 0; w < PLAN_WARPS; ++w) {
      if (w < warp) before += part[w];
      all += part[w];
    }
    if (i < bins) base[i] = before + v - own;
    carry += all;
    __syncthreads();
  }
}

// Places the warps' pieces: base[bin] is where the chunk's pairs of a bin begin, hist the pieces' counts.
__device__ __forceinline__ void place_pieces(const PlanParams &p, int c, int32_t *hist, const int32_t *base) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bins = p.experts + 1;
  for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) {
    int at = base[b];
    for (int w = 0; w < PLAN_WARPS; ++w) {
      const int n = hist[w * bins + b];
      hist[w * bins + b] = at;
      at += n;
    }
  }
  __syncthreads();
  int64_t begin, end;
  piece(p, c, warp, begin, end);
  int32_t *next = hist + warp * bins;
  int coming = begin + lane < end ? bin_of(p, begin + lane) : -1;
  for (int64_t i = begin; i < end; i += 32) {
    const int b = coming;
    const bool live = b >= 0;
    coming = i + 32 + lane < end ? bin_of(p, i + 32 + lane) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, b);
    const int at = live ? next[b] : 0;
    __syncwarp();
    if (live) {
      p.order[at + __popc(same & ((1u << lane) - 1))] = (int32_t)(i + lane);
      if ((same >> lane) == 1u) next[b] = at + __popc(same);  // the last of them
    }
    __syncwarp();
  }
}

__device__ __forceinline__ void plan_whole(const PlanParams &p, int32_t *smem) {
  const int bins = p.experts + 1;
  int32_t *base = smem, *hist = smem + bins;
  count_pieces(p, 0, hist);
  for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) {
    int n = 0;
    for (int w = 0; w < PLAN_WARPS; ++w) n += hist[w * bins + b];
    base[b] = n;
  }
  __syncthreads();
  exclusive(base, bins);
  for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) p.offsets[b] = base[b];
  place_pieces(p, 0, hist, base);
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_whole_kernel(const PlanParams p) {
  extern __shared__ int32_t smem[];
  follow();
  plan_whole(p, smem);
}

// A few rows and their plan in one launch of one CTA.
template <int N, Mode MODE>
__global__ void __launch_bounds__(PLAN_THREADS) route_whole_kernel(const __grid_constant__ RouteParams rp, const PlanParams p) {
  extern __shared__ int32_t smem[];
  follow();
  const int warp = threadIdx.x >> 5;
  uint8_t *keys = reinterpret_cast<uint8_t *>(smem) + warp * (N * 32 * 8);  // the plan's counts come after
  for (int64_t row = warp; row < rp.a.rows; row += PLAN_WARPS)
    if (!route_row<N, MODE>(rp.a, row, keys)) route_row_exactly<N>(rp.a, row, keys);
  __syncthreads();  // the indices are this CTA's own
  plan_whole(p, smem);
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_count_kernel(const PlanParams p) {
  extern __shared__ int32_t smem[];
  follow();
  const int bins = p.experts + 1;
  count_pieces(p, blockIdx.x, smem);
  for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) {
    int n = 0;
    for (int w = 0; w < PLAN_WARPS; ++w) n += smem[w * bins + b];
    p.counts[(int64_t)b * p.chunks + blockIdx.x] = n;
  }
}

// A warp a bin: counts over the chunks become those of earlier chunks.
__global__ void __launch_bounds__(128) plan_sum_kernel(const PlanParams p) {
  follow();
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b > p.experts) return;
  int32_t *row = p.counts + (int64_t)b * p.chunks;
  int carry = 0;
  for (int first = 0; first < p.chunks; first += 32) {
    const int c = first + lane;
    const int own = c < p.chunks ? row[c] : 0;
    int v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (c < p.chunks) row[c] = carry + v - own;
    carry += __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) p.totals[b] = carry;
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_place_kernel(const PlanParams p) {
  extern __shared__ int32_t smem[];
  follow();
  const int bins = p.experts + 1;
  int32_t *base = smem, *hist = smem + bins;
  for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) base[b] = p.totals[b];
  __syncthreads();
  exclusive(base, bins);
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) p.offsets[b] = base[b];
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += PLAN_THREADS) base[b] += p.counts[(int64_t)b * p.chunks + blockIdx.x];
  __syncthreads();
  count_pieces(p, blockIdx.x, hist);
  place_pieces(p, blockIdx.x, hist, base);
}

// Up to this many pairs one CTA does it all.
constexpr int64_t WHOLE = 4096;
constexpr int MAX_CHUNKS = 256;

static int64_t chunk_of(int64_t pairs) {
  if (pairs <= WHOLE) return (pairs + PLAN_THREADS - 1) / PLAN_THREADS * PLAN_THREADS;
  int64_t c = (pairs + MAX_CHUNKS - 1) / MAX_CHUNKS;
  c = c < 1024 ? 1024 : c;
  return (c + PLAN_THREADS - 1) / PLAN_THREADS * PLAN_THREADS;
}

static int32_t plan(const int32_t *indices, int64_t pairs, int first, int experts, int32_t *offsets, int32_t *order,
                    void *scratch, cudaStream_t stream) {
  PlanParams p{indices, pairs, first, experts, offsets, order, nullptr, nullptr, chunk_of(pairs), 1};
  const int bins = experts + 1;
  const size_t smem = (size_t)(PLAN_WARPS + 1) * bins * 4;  // at most 135 KB
  if (pairs <= WHOLE) {
    B200_CUDA_TRY((ensure_dynamic_smem<plan_whole_kernel>(140 * 1024)));
    B200_CUDA_TRY(launch(plan_whole_kernel, dim3(1), PLAN_THREADS, smem, stream, p));
  } else {
    p.chunks = (int)((pairs + p.chunk - 1) / p.chunk);
    p.counts = (int32_t *)scratch;
    p.totals = p.counts + (int64_t)bins * p.chunks;
    B200_CUDA_TRY((ensure_dynamic_smem<plan_count_kernel>(140 * 1024)));
    B200_CUDA_TRY((ensure_dynamic_smem<plan_place_kernel>(140 * 1024)));
    B200_CUDA_TRY(launch(plan_count_kernel, dim3((unsigned)p.chunks), PLAN_THREADS, smem, stream, p));
    B200_CUDA_TRY(launch(plan_sum_kernel, dim3((unsigned)(bins + 3) / 4), 128, 0, stream, p));
    B200_CUDA_TRY(launch(plan_place_kernel, dim3((unsigned)p.chunks), PLAN_THREADS, smem, stream, p));
  }
  return B200_OK;
}

// Up to this many rows (two a warp) routing and plan are one launch: 5.7 us for one row, in two launches 6.8.
constexpr int64_t FEW_ROWS = 2 * PLAN_WARPS;

template <int N, Mode MODE>
static int32_t launch_keyed(const RouteParams &rp, cudaStream_t stream) {
  if constexpr (N <= 8) {
    if (rp.a.rows <= FEW_ROWS) {  // at most 2048 pairs
      const int64_t pairs = rp.a.rows * rp.a.k;
      const PlanParams p{rp.a.indices, pairs, 0, rp.a.experts, rp.a.offsets, rp.a.order, nullptr, nullptr, chunk_of(pairs), 1};
      const size_t counts = (size_t)(PLAN_WARPS + 1) * (rp.a.experts + 1) * 4, keys = (size_t)PLAN_WARPS * N * 32 * 8;
      B200_CUDA_TRY((ensure_dynamic_smem<route_whole_kernel<N, MODE>>(140 * 1024)));
      B200_CUDA_TRY(launch(route_whole_kernel<N, MODE>, dim3(1), PLAN_THREADS, counts > keys ? counts : keys, stream, rp, p));
      return B200_OK;
    }
  }
  B200_CUDA_TRY(launch(route_kernel<N, MODE>, dim3((unsigned)((rp.a.rows + 3) / 4)), 128, 0, stream, rp));
  return plan(rp.a.indices, rp.a.rows * rp.a.k, 0, rp.a.experts, rp.a.offsets, rp.a.order, rp.a.scratch, stream);
}

template <int N>
static int32_t launch_route(const RouteParams &rp, bool wide, cudaStream_t stream) {
  if (wide) return launch_keyed<N, QUICK>(rp, stream);
  return rp.a.dtype == B200_DT_F32 ? launch_keyed<N, LOGIT>(rp, stream) : launch_keyed<N, PACKED>(rp, stream);
}

// ---- the weighted sum -------------------------------------------------------------------------------
struct CombineParams {
  const void *y;
  const float *weights;
  const int32_t *indices;
  const void *residual;
  void *out;
  int64_t cols, rstride;
  int first, experts, fan, ydt, rdt, odt;
};

// VEC neighbouring columns a thread; four pairs' rows are asked for together and added in their order (one after
// another a token's four took 4 us).
template <int VEC>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ CombineParams p) {
  follow();
  const int64_t t = blockIdx.y, c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
  if (c >= p.cols) return;
  float sum[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
  for (int j0 = 0; j0 < p.fan; j0 += 4) {
    float w[4], v[4][VEC];
    bool has[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t pair = t * p.fan + (j0 + j < p.fan ? j0 + j : p.fan - 1);
      const int32_t e = p.indices[pair];
      has[j] = j0 + j < p.fan && e >= p.first && e - p.first < p.experts;
      w[j] = p.weights[pair];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t pair = t * p.fan + j0 + j;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = 0.f;
      if (!has[j]) continue;
      if constexpr (VEC == 4) {
        if (p.ydt == B200_DT_F32) {
          const float4 u = *reinterpret_cast<const float4 *>((const float *)p.y + pair * p.cols + c);
          v[j][0] = u.x, v[j][1] = u.y, v[j][2] = u.z, v[j][3] = u.w;
          continue;
        }
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = load_as_f32(p.y, pair * p.cols + c + i, p.ydt);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (has[j]) sum[i] = fmaf(w[j], v[j][i], sum[i]);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (p.residual != nullptr) sum[i] += load_as_f32(p.residual, t * p.rstride + c + i, p.rdt);
#pragma unroll
  for (int i = 0; i < VEC; ++i) store_f32(p.out, t * p.cols + c + i, p.odt, sum[i]);
}

static bool real(int dt) { return dt == B200_DT_F16 || dt == B200_DT_BF16 || dt == B200_DT_F32; }

}  // namespace route
}  // namespace b200

using namespace b200;
using namespace b200::route;

extern "C" {

int64_t b200_expert_plan_scratch(int64_t pairs, int32_t experts) {
  if (pairs <= WHOLE || experts < 1 || experts > MAX_EXPERTS) return 0;
  const int64_t chunks = (pairs + chunk_of(pairs) - 1) / chunk_of(pairs);
  return (chunks + 1) * (experts + 1) * 4;
}

int32_t b200_expert_plan(const int32_t *indices, int64_t pairs, int32_t first, int32_t experts, int32_t *offsets,
                         int32_t *order, void *scratch, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (pairs < 0 || first < 0 || experts < 1 || experts > MAX_EXPERTS || pairs > 0x7FFFFFFF)
    return b200_set_error(B200_ERR_INVALID, "expert_plan: 1 to %d experts and fewer than 2^31 pairs", MAX_EXPERTS);
  if (offsets == nullptr || (pairs > 0 && (indices == nullptr || order == nullptr)) || (pairs > WHOLE && scratch == nullptr))
    return b200_set_error(B200_ERR_INVALID, "expert_plan: null pointer");
  return plan(indices, pairs, first, experts, offsets, order, scratch, (cudaStream_t)stream);
}

int32_t b200_route_experts(const b200_route_args *a, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (a == nullptr) return b200_set_error(B200_ERR_INVALID, "route_experts: null arguments");
  if (!real(a->dtype) || a->rows < 0 || a->experts < 1 || a->experts > MAX_EXPERTS || a->k < 1 || a->k > MAX_K || a->k > a->experts)
    return b200_set_error(B200_ERR_INVALID, "route_experts: k of at most %d out of 1 to %d experts, float16, bfloat16 or float32",
                          MAX_K, MAX_EXPERTS);
  if (a->groups < 1 || a->groups > MAX_GROUPS || a->experts % a->groups != 0 || a->top_groups < 1 || a->top_groups > a->groups ||
      (a->group_best != 1 && a->group_best != 2) || a->k > a->experts / a->groups * a->top_groups)
    return b200_set_error(B200_ERR_INVALID, "route_experts: groups do not divide the experts, or leave fewer than k");
  if (a->rows * a->k > 0x7FFFFFFF) return b200_set_error(B200_ERR_UNSUPPORTED, "route_experts: 2^31 pairs or more");
  if (a->offsets == nullptr || (a->rows > 0 && (a->logits == nullptr || a->indices == nullptr || a->weights == nullptr || a->order == nullptr)))
    return b200_set_error(B200_ERR_INVALID, "route_experts: null pointer");
  if (a->rows * a->k > WHOLE && a->scratch == nullptr) return b200_set_error(B200_ERR_INVALID, "route_experts: null scratch");
  cudaStream_t s = (cudaStream_t)stream;
  const RouteParams rp{*a};
  const bool wide = a->bias != nullptr || (a->groups > 1 && a->group_best == 2);
  if (a->rows == 0) return plan(a->indices, 0, 0, a->experts, a->offsets, a->order, a->scratch, s);
  if (a->experts <= 64) return launch_route<2>(rp, wide, s);
  if (a->experts <= 128) return launch_route<4>(rp, wide, s);
  if (a->experts <= 256) return launch_route<8>(rp, wide, s);
  if (a->experts <= 512) return launch_route<16>(rp, wide, s);
  return launch_route<32>(rp, wide, s);
}

int32_t b200_expert_combine(const b200_combine_args *a, void *stream) {
  if (int32_t rc = b200_injected()) return rc;
  if (a == nullptr || !real(a->y_dtype) || !real(a->out_dtype) || (a->residual != nullptr && !real(a->residual_dtype)) || a->fan < 1 ||
      a->tokens < 0 || a->cols < 0)
    return b200_set_error(B200_ERR_INVALID, "expert_combine: float16, bfloat16 or float32 rows");
  const int64_t tokens = a->tokens, cols = a->cols;
  if (tokens == 0 || cols == 0) return B200_OK;
  if (a->y == nullptr || a->weights == nullptr || a->indices == nullptr || a->out == nullptr)
    return b200_set_error(B200_ERR_INVALID, "expert_combine: null pointer");
  const int32_t fan = a->fan;
  cudaStream_t s = (cudaStream_t)stream;
  const CombineParams p{a->y, a->weights, a->indices, a->residual, a->out, cols, a->residual_stride, a->first, a->experts, fan, a->y_dtype,
                        a->residual_dtype, a->out_dtype};
  const bool vec = cols % 4 == 0 && (uintptr_t)a->y % 16 == 0;
  for (int64_t t0 = 0; t0 < tokens; t0 += 65535) {  // the grid's second axis
    const int64_t n = tokens - t0 < 65535 ? tokens - t0 : 65535;
    CombineParams q = p;
    q.y = (const uint8_t *)a->y + t0 * fan * cols * dt_size(a->y_dtype);
    q.weights += t0 * fan;
    q.indices += t0 * fan;
    if (a->residual != nullptr) q.residual = (const uint8_t *)a->residual + t0 * a->residual_stride * dt_size(a->residual_dtype);
    q.out = (uint8_t *)a->out + t0 * cols * dt_size(a->out_dtype);
    if (vec) B200_CUDA_TRY(launch(combine_kernel<4>, dim3((unsigned)((cols + 1023) / 1024), (unsigned)n), 256, 0, s, q));
    else B200_CUDA_TRY(launch(combine_kernel<1>, dim3((unsigned)((cols + 255) / 256), (unsigned)n), 256, 0, s, q));
  }
  return B200_OK;
}

int32_t b200_expert_mlp(const b200_packed_desc *up, const b200_scaled_args *first, const b200_packed_desc *down,
                        const b200_scaled_args *second, const b200_combine_args *combine, void *stream) {
  if (int32_t rc = b200_scaled_linear(up, first, stream)) return rc;
  if (int32_t rc = b200_scaled_linear(down, second, stream)) return rc;
  return b200_expert_combine(combine, stream);
}

}  // extern "C"
