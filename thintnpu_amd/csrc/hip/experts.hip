// Expert blocks: routing of tokens to experts, the move of their rows to the
// experts and the weighted sum of the rows that come back.
#include "rows.h"

#include <string.h>

#include <algorithm>

namespace thin {
namespace {

constexpr uint32_t kThreads = 256;
constexpr int64_t kMaxExperts = 1024;
constexpr int64_t kMaxChosen = 32;
constexpr int64_t kMaxGroups = 64;

// ---------------------------------------------------------------- routing
struct RoutePlan {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* experts;
  int64_t row, bias_step;            // strides of the logits' rows and of the bias
  int64_t wt, wk, et, ek;            // strides of weights and experts
  uint32_t tokens, count;            // tokens, experts
  int32_t k, groups, top, size;      // chosen, groups, kept groups, experts a group
  int32_t softmax, renormalize;
  FastDiv by_size;
  float scale;
};

constexpr float kLog2e = 1.4426950408889634f;

// Scores s of a row held by G lanes: softmax or sigmoid of x in V.
template <int G, int PER>
__device__ __forceinline__ void scores32(const float (&x)[PER], uint32_t first, uint32_t count, bool softmax,
                                         float (&s)[PER], float& total) {
  if (softmax) {
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (first + j < count) m = fmaxf(m, x[j]);
    m = dev::group_max<G>(m);
    total = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      s[j] = first + j < count ? __builtin_amdgcn_exp2f((x[j] - m) * kLog2e) : 0.f;
      total += s[j];
    }
    total = dev::group_sum<G>(total);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] /= total;
  } else {
    total = 1.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = dev::sigmoid_fast(x[j]);
  }
}
template <int G>
__device__ double group_sum64(double v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int G, int PER>
__device__ void scores64(const float (&x)[PER], uint32_t first, uint32_t count, bool softmax, double (&s)[PER]) {
  if (softmax) {
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (first + j < count) m = fmaxf(m, x[j]);
    m = dev::group_max<G>(m);
    double total = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      s[j] = first + j < count ? exp((double)x[j] - (double)m) : 0.0;
      total += s[j];
    }
    total = group_sum64<G>(total);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] /= total;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = 1.0 / (1.0 + exp(-(double)x[j]));
  }
}

// How near two 32-bit choice scores may be before their order is settled in
// 64 bits.  A score s <= 1 is off by less than 2^-22 (softmax: s |x - m| 2^-23
// <= 0.37 * 2^-23 from the exponent's argument, 2^-23 from exp2 and the sum
// each), the bias adds half a step of c: the two sides together stay below
// 2^-20 + 2^-22 |c|.  A group's score adds two of them.
__device__ __forceinline__ bool near_tie(float above, float below, float terms) {
  return above - below <= terms * (0x1p-20f + 0x1p-22f * fabsf(above));
}

// Drops the keys of groups that are not among the `top` best.  `near`: the
// last kept and the first dropped group are too near for 32 bits.
template <int G, int PER, bool BIAS, typename K>
__device__ __forceinline__ bool keep_groups(const RoutePlan& p, K (&key)[PER], uint32_t g, K* staged, K* group_key,
                                            uint8_t* kept, K* border) {
  const uint32_t first = g * PER;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (first + j < p.count) staged[first + j] = key[j];
  dev::wave_lds_fence();
  for (int q = (int)g; q < p.groups; q += G) {
    K best = 0, second = 0;
    int i = q % p.size;  // lanes start at different banks
    for (int n = 0; n < p.size; ++n) {
      const K v = staged[q * p.size + i];
      second = v > best ? best : v > second ? v : second;
      best = v > best ? v : best;
      i = i + 1 == p.size ? 0 : i + 1;
    }
    if (BIAS && p.size > 1) best = dev::score_key(dev::key_score(best) + dev::key_score(second));
    group_key[q] = best;
  }
  dev::wave_lds_fence();
  for (int q = (int)g; q < p.groups; q += G) {
    const K mine = group_key[q];
    int rank = 0;
    for (int o = 0; o < p.groups; ++o) {
      const K other = group_key[o];
      rank += other > mine || (other == mine && o < q);
    }
    kept[q] = rank < p.top;
    if (rank == p.top - 1) border[0] = mine;
    if (rank == p.top) border[1] = mine;
  }
  dev::wave_lds_fence();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t e = min(first + j, p.count - 1);
    if (!kept[p.by_size.div(e)]) key[j] = 0;
  }
  if constexpr (sizeof(K) == 4 && BIAS) {
    return near_tie(dev::key_score((uint32_t)border[0]), dev::key_score((uint32_t)border[1]), 2.f);
  } else {
    return false;
  }
}

// G lanes a token, lane g holding the logits of experts g * PER + j.  Without
// a bias the choice follows the logits, whose order is that of the scores.
// With one it follows s + bias in 32 bits, and where two of the k + 1 best (or
// the border of the groups) are nearer than that arithmetic can tell apart the
// token is chosen again in 64 bits; equal logits with equal biases are equal
// in either.
template <typename T, int G, int PER, bool BIAS, bool GROUPED>
__global__ __launch_bounds__(kThreads) void route_kernel(RoutePlan p) {
  constexpr int kTokens = kThreads / G;
  __shared__ int32_t chosen[kTokens][kMaxChosen + 1];
  __shared__ float choice[BIAS ? kTokens : 1][kMaxChosen + 1];
  __shared__ uint64_t group_key[GROUPED ? kTokens : 1][kMaxGroups];
  __shared__ uint64_t border[GROUPED ? kTokens : 1][2];
  __shared__ uint8_t kept[GROUPED ? kTokens : 1][kMaxGroups];
  extern __shared__ uint64_t staged_lds[];  // GROUPED: a key for each expert of each token

  const uint32_t g = threadIdx.x % G, slot = threadIdx.x / G;
  const uint32_t token = blockIdx.x * kTokens + slot;
  const bool live = token < p.tokens;  // every lane joins the group's exchanges
  const T* row = static_cast<const T*>(p.logits) + (int64_t)min(token, p.tokens - 1) * p.row;
  const uint32_t first = g * PER;
  float x[PER];
  if (first + PER <= p.count) {
    dev::load_pack<T, PER>(row + first, x);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = first + j < p.count ? (float)row[first + j] : 0.f;
  }

  uint32_t key[PER];
  float total = 1.f;
  if constexpr (BIAS) {
    float s[PER];
    scores32<G, PER>(x, first, p.count, p.softmax, s, total);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      key[j] = first + j < p.count ? dev::score_key(s[j] + p.bias[(first + j) * p.bias_step]) : 0u;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = first + j < p.count ? dev::score_key(x[j]) : 0u;
  }
  constexpr size_t kKey = BIAS ? 8 : 4;
  char* staged = reinterpret_cast<char*>(staged_lds) + slot * (size_t)p.count * kKey;
  bool close = false;
  if constexpr (GROUPED)
    close = keep_groups<G, PER, BIAS, uint32_t>(p, key, g, reinterpret_cast<uint32_t*>(staged),
                                                reinterpret_cast<uint32_t*>(group_key[slot]), kept[slot],
                                                reinterpret_cast<uint32_t*>(border[slot]));
  const int open = GROUPED ? p.top * p.size : (int)p.count;
  const int n = BIAS && p.k < open ? p.k + 1 : p.k;
  dev::take_best<G, PER>(key, n, g, [&](int i, uint32_t e, uint32_t k) {
    chosen[slot][i] = (int32_t)e;
    if constexpr (BIAS) choice[slot][i] = dev::key_score(k);
  });
  dev::wave_lds_fence();
  if constexpr (BIAS) {
    for (int i = (int)g; i < n - 1; i += G) {
      if (!near_tie(choice[slot][i], choice[slot][i + 1], 1.f)) continue;
      const int32_t a = chosen[slot][i], b = chosen[slot][i + 1];
      close = close || (float)row[a] != (float)row[b] || p.bias[a * p.bias_step] != p.bias[b * p.bias_step];
    }
    if (dev::group_ballot<G>(close)) {
      double s[PER];
      scores64<G, PER>(x, first, p.count, p.softmax, s);
      uint64_t key64[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j)
        key64[j] = first + j < p.count ? dev::score_key(s[j] + (double)p.bias[(first + j) * p.bias_step]) : 0u;
      if constexpr (GROUPED)
        keep_groups<G, PER, BIAS, uint64_t>(p, key64, g, reinterpret_cast<uint64_t*>(staged), group_key[slot],
                                            kept[slot], border[slot]);
      dev::take_best<G, PER>(key64, p.k, g, [&](int i, uint32_t e, uint64_t) { chosen[slot][i] = (int32_t)e; });
      dev::wave_lds_fence();
    }
  }

  // weights of the chosen, from their logits
  float top = -__builtin_inff();
  if (p.softmax) {
    if (p.renormalize) {  // the sum over all experts cancels: any common maximum serves
      for (int i = (int)g; i < p.k; i += G) top = fmaxf(top, (float)row[chosen[slot][i]]);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (first + j < p.count) top = fmaxf(top, x[j]);
    }
    top = dev::group_max<G>(top);
  }
  float sum = 0.f;
  if (p.renormalize) {
    for (int i = (int)g; i < p.k; i += G) {
      const float v = (float)row[chosen[slot][i]];
      sum += p.softmax ? expf(v - top) : 1.0f / (1.0f + expf(-v));
    }
    sum = dev::group_sum<G>(sum);
    if (BIAS && p.softmax && total != total) sum = total;  // a NaN anywhere is in every score of the row
  } else if (p.softmax) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (first + j < p.count) sum += expf(x[j] - top);
    sum = dev::group_sum<G>(sum);
  } else {
    sum = 1.f;
  }
  if (!live) return;
  for (int i = (int)g; i < p.k; i += G) {
    const int32_t e = chosen[slot][i];
    const float v = (float)row[e];
    const float s = p.softmax ? expf(v - top) : 1.0f / (1.0f + expf(-v));
    p.weights[(int64_t)token * p.wt + i * p.wk] = s / sum * p.scale;
    p.experts[(int64_t)token * p.et + i * p.ek] = e;
  }
}

template <typename T, int G, int PER>
thin_status launch_route(const RoutePlan& p, hipStream_t stream) {
  const uint32_t tokens = kThreads / G;
  const dim3 grid((p.tokens + tokens - 1) / tokens), block(kThreads);
  const bool grouped = p.top < p.groups;
  const uint32_t lds = grouped ? (uint32_t)(tokens * p.count * (p.bias ? 8 : 4)) : 0u;
  if (p.bias) {
    if (grouped) hipLaunchKernelGGL((route_kernel<T, G, PER, true, true>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((route_kernel<T, G, PER, true, false>), grid, block, 0, stream, p);
  } else {
    if (grouped) hipLaunchKernelGGL((route_kernel<T, G, PER, false, true>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((route_kernel<T, G, PER, false, false>), grid, block, 0, stream, p);
  }
  THIN_LAUNCH_CHECK("expert_route");
  return THIN_OK;
}

// ---------------------------------------------------------------- rows
// A row of `bytes` bytes goes in 16-byte vectors; the last one ends with the
// row and may repeat bytes of the one before.  Rows below 16 bytes go element
// by element.
struct RowsPlan {
  const char* x;
  char* rows;
  const int32_t* experts;
  int32_t* offsets;
  int32_t* slots;
  int32_t* counts;                   // workspace: [blocks][count] assignments of each expert
  int64_t xs, rs, et, ek, os;        // byte strides of x and rows, element strides of experts and offsets
  int64_t st, sk;                    // element strides of slots
  uint32_t tokens, assigned;         // assigned = tokens * k
  int32_t k, count;                  // experts a token, experts
  uint32_t bytes, elem;              // bytes of a row, of an element
  uint32_t lanes;                    // threads that copy one row (a power of two)
  uint32_t chunk;                    // assignments a wave of the counting kernels
  FastDiv by_k;
};

typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ int32_t expert_of(const RowsPlan& p, uint32_t a) {
  const uint32_t t = p.by_k.div(a);
  const int32_t e = p.experts[(int64_t)t * p.et + (int64_t)(a - t * p.k) * p.ek];
  return (uint32_t)e < (uint32_t)p.count ? e : -1;
}

// Vector v of token t's row, copied to the rows its slots name.
template <typename Slot>
__device__ __forceinline__ void copy_row(const RowsPlan& p, uint32_t t, uint32_t v, Slot slot) {
  const char* src = p.x + (int64_t)t * p.xs;
  if (p.bytes >= 16) {
    const uint32_t at = min(v * 16, p.bytes - 16);
    const u4u w = *reinterpret_cast<const u4u*>(src + at);
    for (int j = 0; j < p.k; ++j) {
      const int32_t s = slot(j);
      if (s >= 0) *reinterpret_cast<u4u*>(p.rows + (int64_t)s * p.rs + at) = w;
    }
  } else {
    for (int j = 0; j < p.k; ++j) {
      const int32_t s = slot(j);
      if (s < 0) continue;
      for (uint32_t b = 0; b < p.bytes; b += 2)
        *reinterpret_cast<uint16_t*>(p.rows + (int64_t)s * p.rs + b) = *reinterpret_cast<const uint16_t*>(src + b);
    }
  }
}

// Few assignments: block (t, y) counts for each of its token's assignments the
// ones before it in the order (expert, assignment) among all, and copies 256
// vectors of the row; block (tokens, 0) writes the offsets.  One launch.
constexpr uint32_t kCountedAssignments = 4096;
__global__ __launch_bounds__(kThreads) void dispatch_small_kernel(RowsPlan p) {
  constexpr int kWaves = kThreads / 64, kAtOnce = 8;
  __shared__ int32_t ids[kCountedAssignments];
  __shared__ int32_t part[kWaves][kMaxChosen];
  __shared__ int32_t scan[kMaxExperts];
  for (uint32_t a = threadIdx.x; a < p.assigned; a += kThreads) ids[a] = expert_of(p, a);
  if (blockIdx.x == p.tokens) {
    if (blockIdx.y) return;
    for (int e = threadIdx.x; e < p.count; e += kThreads) scan[e] = 0;
    __syncthreads();
    for (uint32_t a = threadIdx.x; a < p.assigned; a += kThreads)
      if (ids[a] >= 0) atomicAdd(&scan[ids[a]], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= p.count; e += kThreads) {
      int32_t before = 0;
      for (int o = 0; o < e; ++o) before += scan[o];
      p.offsets[e * p.os] = before;
    }
    return;
  }
  __syncthreads();
  const uint32_t t = blockIdx.x;
  for (int j0 = 0; j0 < p.k; j0 += kAtOnce) {
    int32_t mine[kAtOnce], before[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      mine[j] = j0 + j < p.k ? ids[t * p.k + j0 + j] : -1;
      before[j] = 0;
    }
    for (uint32_t a = threadIdx.x; a < p.assigned; a += kThreads) {
      const int32_t e = ids[a];
      if (e < 0) continue;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) before[j] += e < mine[j] || (e == mine[j] && a < t * p.k + j0 + j);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      int32_t s = before[j];
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      if ((threadIdx.x & 63u) == 0 && j0 + j < p.k) part[threadIdx.x >> 6][j0 + j] = s;
    }
  }
  __syncthreads();
  if (threadIdx.x < (uint32_t)p.k) {
    int32_t s = 0;
    for (int w = 0; w < kWaves; ++w) s += part[w][threadIdx.x];
    s = ids[t * p.k + threadIdx.x] < 0 ? -1 : s;
    part[0][threadIdx.x] = s;
    if (blockIdx.y == 0) p.slots[(int64_t)t * p.st + threadIdx.x * p.sk] = s;
  }
  __syncthreads();
  const uint32_t v = blockIdx.y * kThreads + threadIdx.x;
  if (v * 16 < p.bytes) copy_row(p, t, v, [&](int j) { return part[0][j]; });
}

// Many assignments, in three launches: counts of each block's assignments by
// expert, slots from them, the copy.  A block's four waves take runs of
// `chunk` assignments each, in order.
__global__ __launch_bounds__(kThreads) void dispatch_count_kernel(RowsPlan p) {
  __shared__ int32_t counts[kMaxExperts];
  for (int e = threadIdx.x; e < p.count; e += kThreads) counts[e] = 0;
  __syncthreads();
  const uint32_t begin = blockIdx.x * p.chunk * (kThreads / 64);
  const uint32_t end = min(begin + p.chunk * (kThreads / 64), p.assigned);
  for (uint32_t a = begin + threadIdx.x; a < end; a += kThreads) {
    const int32_t e = expert_of(p, a);
    if (e >= 0) atomicAdd(&counts[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.count; e += kThreads) p.counts[(int64_t)blockIdx.x * p.count + e] = counts[e];
}

__global__ __launch_bounds__(kThreads) void dispatch_slots_kernel(RowsPlan p) {
  constexpr uint32_t kWaves = kThreads / 64;
  __shared__ int32_t next[kWaves][kMaxExperts];  // next slot of each expert in each wave's run
  __shared__ int32_t sums[kThreads];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
  // each thread owns a run of experts: total of all blocks and of those before this one
  const int per = (p.count + (int)kThreads - 1) / (int)kThreads;
  const int e0 = (int)threadIdx.x * per;
  int32_t total[kMaxExperts / kThreads], before[kMaxExperts / kThreads];
  int32_t own = 0;
#pragma unroll
  for (int i = 0; i < (int)(kMaxExperts / kThreads); ++i) {
    total[i] = before[i] = 0;
    if (i < per && e0 + i < p.count) {
      for (uint32_t b = 0; b < gridDim.x; ++b) {
        const int32_t c = p.counts[(int64_t)b * p.count + e0 + i];
        total[i] += c;
        if (b < blockIdx.x) before[i] += c;
      }
      own += total[i];
    }
  }
  sums[threadIdx.x] = own;
  __syncthreads();
  for (uint32_t o = 1; o < kThreads; o <<= 1) {
    const int32_t add = threadIdx.x >= o ? sums[threadIdx.x - o] : 0;
    __syncthreads();
    sums[threadIdx.x] += add;
    __syncthreads();
  }
  int32_t start = sums[threadIdx.x] - own;
#pragma unroll
  for (int i = 0; i < (int)(kMaxExperts / kThreads); ++i) {
    if (i < per && e0 + i < p.count) {
      if (blockIdx.x == 0) p.offsets[(int64_t)(e0 + i) * p.os] = start;
      next[0][e0 + i] = start + before[i];
      for (uint32_t w = 1; w < kWaves; ++w) next[w][e0 + i] = 0;
      start += total[i];
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == kThreads - 1) p.offsets[(int64_t)p.count * p.os] = sums[kThreads - 1];
  __syncthreads();
  const uint32_t begin = (blockIdx.x * kWaves + wave) * p.chunk;
  const uint32_t end = min(begin + p.chunk, p.assigned);
  if (wave + 1 < kWaves)
    for (uint32_t a = begin + lane; a < end; a += 64) {
      const int32_t e = expert_of(p, a);
      if (e >= 0) atomicAdd(&next[wave + 1][e], 1);
    }
  __syncthreads();
  for (int e = threadIdx.x; e < p.count; e += kThreads)
    for (uint32_t w = 1; w < kWaves; ++w) next[w][e] += next[w - 1][e];
  __syncthreads();
  // 64 assignments at a time: the lanes of one expert take consecutive slots
  for (uint32_t a0 = begin; a0 < end; a0 += 64) {
    const uint32_t a = a0 + lane;
    const int32_t e = a < end ? expert_of(p, a) : -1;
    uint64_t same = __ballot(e >= 0);
    for (int bit = 0; (1 << bit) < p.count; ++bit) {
      const uint64_t set = __ballot((e >> bit) & 1);
      same &= (e >> bit) & 1 ? set : ~set;
    }
    if (e >= 0) {
      const int leader = __builtin_ctzll(same);
      int32_t base = 0;
      if ((int)lane == leader) base = atomicAdd(&next[wave][e], __builtin_popcountll(same));
      base = __shfl(base, leader, 64);
      const uint32_t t = p.by_k.div(a);
      p.slots[(int64_t)t * p.st + (int64_t)(a - t * p.k) * p.sk] =
          base + __builtin_popcountll(same & ((1ull << lane) - 1));
    } else if (a < end) {
      const uint32_t t = p.by_k.div(a);
      p.slots[(int64_t)t * p.st + (int64_t)(a - t * p.k) * p.sk] = -1;
    }
  }
}

__global__ __launch_bounds__(kThreads) void dispatch_copy_kernel(RowsPlan p) {
  const uint32_t t = blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes;
  const uint32_t v = blockIdx.y * p.lanes + threadIdx.x % p.lanes;
  if (t >= p.tokens || v * 16 >= p.bytes) return;
  copy_row(p, t, v, [&](int j) { return p.slots[(int64_t)t * p.st + j * p.sk]; });
}

// ---------------------------------------------------------------- sums
struct CombinePlan {
  const void* y;
  void* out;
  const float* weights;
  const int32_t* slots;
  int64_t ys, os, wt, wk, st, sk;
  uint32_t tokens, rows, width;  // width: elements of a row
  int32_t k;
  uint32_t lanes;
};

// out[t] = sum_j weights[t, j] * y[slots[t, j]], in the order of j, in fp32
// with one rounding; slots outside y contribute nothing.
template <typename T>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombinePlan p) {
  constexpr uint32_t V = 16 / sizeof(T);
  const uint32_t t = blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes;
  const uint32_t v = blockIdx.y * p.lanes + threadIdx.x % p.lanes;
  if (t >= p.tokens || v * V >= p.width) return;
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out) + (int64_t)t * p.os;
  const float* w = p.weights + (int64_t)t * p.wt;
  const int32_t* slot = p.slots + (int64_t)t * p.st;
  if (p.width >= V) {
    const uint32_t at = min(v * V, p.width - V);
    float sum[V] = {};
    for (int j = 0; j < p.k; ++j) {
      const uint32_t s = (uint32_t)slot[j * p.sk];
      if (s >= p.rows) continue;
      float r[V];
      dev::load_pack<T, V>(y + (int64_t)s * p.ys + at, r);
      const float f = w[j * p.wk];
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) sum[i] = __builtin_fmaf(f, r[i], sum[i]);
    }
    dev::store_pack<T, V>(out + at, sum);
  } else {
    for (uint32_t i = 0; i < p.width; ++i) {
      float sum = 0.f;
      for (int j = 0; j < p.k; ++j) {
        const uint32_t s = (uint32_t)slot[j * p.sk];
        if (s < p.rows) sum = __builtin_fmaf(w[j * p.wk], (float)y[(int64_t)s * p.ys + i], sum);
      }
      out[i] = (T)sum;
    }
  }
}

// Threads that share a row of `vectors` vectors.
uint32_t row_lanes(uint64_t vectors) {
  uint32_t lanes = 1;
  while (lanes < kThreads && lanes < vectors) lanes *= 2;
  return lanes;
}

// Blocks of the counting kernels and assignments a wave of them takes: at
// least 512 a wave, at most 256 blocks (each block reads the counts of all).
uint32_t count_blocks(int64_t assigned, uint32_t* chunk) {
  const int64_t wave = std::max<int64_t>(512, (assigned + 1023) / 1024);
  *chunk = (uint32_t)((wave + 63) / 64 * 64);
  return (uint32_t)((assigned + (int64_t)*chunk * 4 - 1) / ((int64_t)*chunk * 4));
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" thin_status thin_expert_route(const thin_desc* logits, const thin_desc* bias, int32_t softmax,
                                         int64_t groups, int64_t top_groups, int32_t renormalize, float scale,
                                         const thin_desc* weights, const thin_desc* experts, hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(logits) && (!bias || desc_valid(bias)) && desc_valid(weights) && desc_valid(experts),
               THIN_ERR_INVALID, "expert_route: invalid descriptor");
  THIN_REQUIRE(float_type(logits->dtype) && logits->rank == 2, THIN_ERR_INVALID,
               "expert_route takes float16, bfloat16 or float32 logits [tokens, experts]");
  const int64_t T = logits->sizes[0], E = logits->sizes[1];
  THIN_REQUIRE(E >= 1 && E <= kMaxExperts && T < (1ll << 31), THIN_ERR_UNSUPPORTED,
               "expert_route takes 1..%lld experts and below 2^31 tokens", (long long)kMaxExperts);
  THIN_REQUIRE(weights->rank == 2 && weights->dtype == THIN_F32 && weights->sizes[0] == T && experts->rank == 2 &&
                   experts->dtype == THIN_I32 && experts->sizes[0] == T && experts->sizes[1] == weights->sizes[1],
               THIN_ERR_INVALID, "expert_route writes float32 weights and int32 experts [tokens, k]");
  const int64_t k = weights->sizes[1];
  THIN_REQUIRE(groups >= 1 && groups <= kMaxGroups && E % groups == 0 && top_groups >= 1 && top_groups <= groups,
               THIN_ERR_INVALID, "expert_route: %lld groups (1..%lld, equal), of which %lld stay", (long long)groups,
               (long long)kMaxGroups, (long long)top_groups);
  THIN_REQUIRE(k >= 1 && k <= kMaxChosen && k <= E / groups * top_groups, THIN_ERR_INVALID,
               "expert_route chooses 1..%lld of the %lld experts that the kept groups hold, not %lld",
               (long long)kMaxChosen, (long long)(E / groups * top_groups), (long long)k);
  THIN_REQUIRE(!bias || (bias->dtype == THIN_F32 && bias->rank == 1 && bias->sizes[0] == E), THIN_ERR_INVALID,
               "expert_route: the bias is float32 [experts]");
  THIN_REQUIRE(E == 1 || logits->strides[1] == 1, THIN_ERR_UNSUPPORTED,
               "expert_route: the logits of a token must be adjacent");
  if (T == 0) return THIN_OK;
  THIN_REQUIRE(!overlap(weights, logits) && !overlap(experts, logits) && !overlap(weights, experts) &&
                   (!bias || (!overlap(weights, bias) && !overlap(experts, bias))), THIN_ERR_INVALID,
               "expert_route: an output overlaps another operand");
  RoutePlan p;
  memset(&p, 0, sizeof p);
  p.logits = logits->data;
  p.bias = bias ? static_cast<const float*>(bias->data) : nullptr;
  p.bias_step = bias ? bias->strides[0] : 0;
  p.weights = static_cast<float*>(weights->data);
  p.experts = static_cast<int32_t*>(experts->data);
  p.row = logits->strides[0];
  p.wt = weights->strides[0]; p.wk = weights->strides[1];
  p.et = experts->strides[0]; p.ek = experts->strides[1];
  p.tokens = (uint32_t)T;
  p.count = (uint32_t)E;
  p.k = (int32_t)k;
  p.groups = (int32_t)groups;
  p.top = (int32_t)top_groups;
  p.size = (int32_t)(E / groups);
  p.by_size = FastDiv::make((uint32_t)p.size);
  p.softmax = softmax ? 1 : 0;
  p.renormalize = renormalize ? 1 : 0;
  p.scale = scale;
  return with_float_type(logits->dtype, [&](auto zero) {
    using T_ = decltype(zero);
    if (E <= 16) return launch_route<T_, 4, 4>(p, stream);
    if (E <= 32) return launch_route<T_, 8, 4>(p, stream);
    if (E <= 64) return launch_route<T_, 16, 4>(p, stream);
    if (E <= 128) return launch_route<T_, 16, 8>(p, stream);
    if (E <= 256) return launch_route<T_, 16, 16>(p, stream);
    if (E <= 512) return launch_route<T_, 32, 16>(p, stream);
    return launch_route<T_, 64, 16>(p, stream);
  });
}

extern "C" size_t thin_expert_dispatch_workspace(int64_t tokens, int64_t top_k, int64_t num_experts) {
  if (tokens <= 0 || top_k <= 0 || num_experts <= 0 || tokens > (1ll << 31) / top_k) return 0;
  if (tokens * top_k <= kCountedAssignments) return 0;
  uint32_t chunk;
  return (size_t)count_blocks(tokens * top_k, &chunk) * (size_t)num_experts * sizeof(int32_t);
}

extern "C" thin_status thin_expert_dispatch(const thin_desc* x, const thin_desc* experts, int64_t num_experts,
                                            const thin_desc* rows, const thin_desc* offsets, const thin_desc* slots,
                                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(x) && desc_valid(experts) && desc_valid(rows) && desc_valid(offsets) && desc_valid(slots),
               THIN_ERR_INVALID, "expert_dispatch: invalid descriptor");
  THIN_REQUIRE(float_type(x->dtype) && x->rank == 2 && rows->dtype == x->dtype && rows->rank == 2, THIN_ERR_INVALID,
               "expert_dispatch takes float16, bfloat16 or float32 x [tokens, width] and rows of its type");
  const int64_t T = x->sizes[0], H = x->sizes[1];
  THIN_REQUIRE(experts->rank == 2 && experts->dtype == THIN_I32 && experts->sizes[0] == T, THIN_ERR_INVALID,
               "expert_dispatch takes int32 experts [tokens, k]");
  const int64_t k = experts->sizes[1];
  THIN_REQUIRE(num_experts >= 1 && num_experts <= kMaxExperts && k >= 1 && k <= kMaxChosen, THIN_ERR_UNSUPPORTED,
               "expert_dispatch takes 1..%lld experts and 1..%lld of them a token", (long long)kMaxExperts,
               (long long)kMaxChosen);
  THIN_REQUIRE(T * k < (1ll << 31) && H < (1ll << 28), THIN_ERR_UNSUPPORTED, "expert_dispatch: tensors too large");
  THIN_REQUIRE(rows->sizes[0] == T * k && rows->sizes[1] == H && slots->rank == 2 && slots->dtype == THIN_I32 &&
                   slots->sizes[0] == T && slots->sizes[1] == k && offsets->rank == 1 && offsets->dtype == THIN_I32 &&
                   offsets->sizes[0] == num_experts + 1,
               THIN_ERR_INVALID,
               "expert_dispatch writes rows [tokens * k, width], int32 offsets [experts + 1] and int32 slots [tokens, k]");
  THIN_REQUIRE(H <= 1 || (x->strides[1] == 1 && rows->strides[1] == 1), THIN_ERR_UNSUPPORTED,
               "expert_dispatch: the elements of a row must be adjacent");
  THIN_REQUIRE(!overlap(rows, x) && !overlap(rows, experts) && !overlap(slots, experts) && !overlap(offsets, experts) &&
                   !overlap(slots, x) && !overlap(offsets, x) && !overlap(slots, rows) && !overlap(offsets, rows) &&
                   !overlap(offsets, slots),
               THIN_ERR_INVALID, "expert_dispatch: an output overlaps another operand");
  const size_t need = thin_expert_dispatch_workspace(T, k, num_experts);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "expert_dispatch needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  const uint32_t elem = (uint32_t)dtype_size(x->dtype);
  RowsPlan p;
  memset(&p, 0, sizeof p);
  p.x = static_cast<const char*>(x->data);
  p.rows = static_cast<char*>(rows->data);
  p.experts = static_cast<const int32_t*>(experts->data);
  p.offsets = static_cast<int32_t*>(offsets->data);
  p.slots = static_cast<int32_t*>(slots->data);
  p.counts = static_cast<int32_t*>(workspace);
  p.xs = x->strides[0] * elem;
  p.rs = rows->strides[0] * elem;
  p.et = experts->strides[0]; p.ek = experts->strides[1];
  p.os = offsets->strides[0];
  p.st = slots->strides[0]; p.sk = slots->strides[1];
  p.tokens = (uint32_t)T;
  p.assigned = (uint32_t)(T * k);
  p.k = (int32_t)k;
  p.count = (int32_t)num_experts;
  p.bytes = (uint32_t)(H * elem);
  p.elem = elem;
  p.by_k = FastDiv::make((uint32_t)k);
  const uint64_t vectors = (p.bytes + 15) / 16;
  if (p.assigned <= kCountedAssignments) {
    const uint64_t columns = std::max<uint64_t>(1, (vectors + kThreads - 1) / kThreads);
    THIN_REQUIRE(columns < 65536, THIN_ERR_UNSUPPORTED, "expert_dispatch: rows too long");
    hipLaunchKernelGGL(dispatch_small_kernel, dim3(p.tokens + 1, (uint32_t)columns), dim3(kThreads), 0, stream, p);
    THIN_LAUNCH_CHECK("expert_dispatch");
    return THIN_OK;
  }
  const uint32_t blocks = count_blocks(p.assigned, &p.chunk);
  hipLaunchKernelGGL(dispatch_count_kernel, dim3(blocks), dim3(kThreads), 0, stream, p);
  THIN_LAUNCH_CHECK("expert_dispatch_count");
  hipLaunchKernelGGL(dispatch_slots_kernel, dim3(blocks), dim3(kThreads), 0, stream, p);
  THIN_LAUNCH_CHECK("expert_dispatch_slots");
  if (H == 0) return THIN_OK;
  p.lanes = row_lanes(vectors);
  const uint32_t per = kThreads / p.lanes;
  const uint64_t columns = (vectors + p.lanes - 1) / p.lanes;
  THIN_REQUIRE(columns < 65536, THIN_ERR_UNSUPPORTED, "expert_dispatch: rows too long");
  hipLaunchKernelGGL(dispatch_copy_kernel, dim3((p.tokens + per - 1) / per, (uint32_t)columns), dim3(kThreads), 0,
                     stream, p);
  THIN_LAUNCH_CHECK("expert_dispatch_copy");
  return THIN_OK;
}

extern "C" thin_status thin_expert_combine(const thin_desc* y, const thin_desc* weights, const thin_desc* slots,
                                           const thin_desc* out, hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(y) && desc_valid(weights) && desc_valid(slots) && desc_valid(out), THIN_ERR_INVALID,
               "expert_combine: invalid descriptor");
  THIN_REQUIRE(float_type(y->dtype) && y->rank == 2 && out->dtype == y->dtype && out->rank == 2 &&
                   out->sizes[1] == y->sizes[1],
               THIN_ERR_INVALID,
               "expert_combine takes float16, bfloat16 or float32 y [rows, width] and writes [tokens, width] of its type");
  const int64_t T = out->sizes[0], H = out->sizes[1], S = y->sizes[0];
  THIN_REQUIRE(weights->rank == 2 && weights->dtype == THIN_F32 && slots->rank == 2 && slots->dtype == THIN_I32 &&
                   weights->sizes[0] == T && slots->sizes[0] == T && weights->sizes[1] == slots->sizes[1],
               THIN_ERR_INVALID, "expert_combine takes float32 weights and int32 slots [tokens, k]");
  THIN_REQUIRE(T < (1ll << 31) && S < (1ll << 31) && H < (1ll << 28) && slots->sizes[1] < (1ll << 31),
               THIN_ERR_UNSUPPORTED, "expert_combine: tensors too large");
  THIN_REQUIRE(H <= 1 || (y->strides[1] == 1 && out->strides[1] == 1), THIN_ERR_UNSUPPORTED,
               "expert_combine: the elements of a row must be adjacent");
  if (T == 0 || H == 0) return THIN_OK;
  THIN_REQUIRE(!overlap(out, y) && !overlap(out, weights) && !overlap(out, slots), THIN_ERR_INVALID,
               "expert_combine: the output overlaps an input");
  CombinePlan p;
  memset(&p, 0, sizeof p);
  p.y = y->data;
  p.out = out->data;
  p.weights = static_cast<const float*>(weights->data);
  p.slots = static_cast<const int32_t*>(slots->data);
  p.ys = y->strides[0]; p.os = out->strides[0];
  p.wt = weights->strides[0]; p.wk = weights->strides[1];
  p.st = slots->strides[0]; p.sk = slots->strides[1];
  p.tokens = (uint32_t)T;
  p.rows = (uint32_t)S;
  p.width = (uint32_t)H;
  p.k = (int32_t)slots->sizes[1];
  const uint32_t V = 16 / (uint32_t)dtype_size(y->dtype);
  const uint64_t vectors = ((uint64_t)H + V - 1) / V;
  p.lanes = row_lanes(vectors);
  const uint32_t per = kThreads / p.lanes;
  const uint64_t columns = (vectors + p.lanes - 1) / p.lanes;
  THIN_REQUIRE(columns < 65536, THIN_ERR_UNSUPPORTED, "expert_combine: rows too long");
  const dim3 grid((p.tokens + per - 1) / per, (uint32_t)columns), block(kThreads);
  return with_float_type(y->dtype, [&](auto zero) {
    hipLaunchKernelGGL((combine_kernel<decltype(zero)>), grid, block, 0, stream, p);
    THIN_LAUNCH_CHECK("expert_combine");
    return THIN_OK;
  });
}
