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
// Tokens up to which each has a whole wavefront: with few of them the latency of
// one counts (256 bf16 logits, bias and groups: 16 tokens 5.2 us against 7.4 by 16
// lanes a token, 1024 9.2 against 11.1, 4096 14.8 against 15.0; fp16 without a
// bias: 1024 3.8 against 4.2, 2048 4.2 against 4.3, 4096 5.4 against 4.3).
constexpr int64_t kFewTokens = 1024;

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
  int32_t group_lanes;               // lanes of a group that is whole lanes, a power of two; else 0
  uint32_t staged;                   // 64-bit words of LDS that a wave stages keys in
  int32_t softmax, renormalize;
  FastDiv by_size;
  float scale;
};

constexpr float kLog2e = 1.4426950408889634f;

// Scores s of a row held by G lanes: softmax or sigmoid of x in V.
template <int G, int PER>
__device__ __forceinline__ void scores32(const float (&x)[PER], const dev::Part<PER, false>& part, bool softmax,
                                         float (&s)[PER], float& total) {
  if (softmax) {
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (part.own(j)) m = fmaxf(m, x[j]);
    m = dev::group_max<G>(m);
    total = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      s[j] = part.own(j) ? __builtin_amdgcn_exp2f((x[j] - m) * kLog2e) : 0.f;
      total += s[j];
    }
    total = dev::group_sum<G>(total);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] *= 1.0f / total;
  } else {
    total = 1.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = dev::sigmoid_fast(x[j]);
  }
}
// How near two 32-bit choice scores may be before their order is settled in
// 64 bits: further apart than the scores' two errors (the slack) and the half
// steps of c = s + bias on either side (2^-23 |c|, which counts twice here).
//
// Slack of two sigmoids: each is off by at most 2 * 2^-23 (0.23 from the
// exponent's argument, as s (1 - s) |x| <= 0.23, 0.25 from exp2, 0.5 from the
// sum, 1 from the reciprocal), so 2^-21; taken as 2^-20.
// Slack of two softmax scores s = e / total, in units of u = 2^-24 and of the
// row's highest score 1 / total.  With y = m - x, each e is off by (2.25 y + 2) u
// and its product by u, and s y <= 0.37 / total: 8 for two of them.  What the
// total is off by moves both alike, and their difference by no more than the
// highest score times it: 2 for the reciprocal, 2 + 2.25 * 4.5 for the terms
// (the mean of y, weighted by s, is at most 4.5 for 1024 experts), and 15 sums in
// a lane and 6 joins, each of which may lose half a step of the whole: 21.  That
// makes 44; taken as 48.
__device__ __forceinline__ float slack_of(bool softmax, float total) { return softmax ? 0x1.8p-19f / total : 0x1p-20f; }
__device__ __forceinline__ bool near_tie(float above, float below, float slack) {
  return above - below <= slack + 0x1p-22f * fabsf(above);
}
// The same for a group's score, the mean of its two highest c, a and b: two
// groups together are off by the slack, each by the half steps of its a and b
// (2^-24 of their mean size, however near the mean itself is to 0) and of its own
// (no more; the two count twice here).  A group stays clear of the border if it
// lies further than that from the middle of the last kept and the first dropped
// score.  Infinities and NaN are exact in either arithmetic, and near nothing.
__device__ __forceinline__ float group_reach(float size, float slack) { return 0.5f * slack + 0x1p-22f * size; }

// The best two keys of two sets.
template <typename K>
__device__ __forceinline__ void join_best(K& best, K& second, K b, K s) {
  second = max(min(best, b), max(second, s));
  best = max(best, b);
}
template <int O>
__device__ __forceinline__ void join_lane(uint32_t& best, uint32_t& second) {
  join_best(best, second, dev::lane_xor_bits<O>(best), dev::lane_xor_bits<O>(second));
}
// A group's score: with a bias the mean of its two highest, whose order is that
// of the sum and which no finite scores take past the range.
template <bool BIAS, typename K>
__device__ __forceinline__ K group_score(K best, K second, int size) {
  return BIAS && size > 1 ? dev::score_key(0.5f * dev::key_score(best) + 0.5f * dev::key_score(second)) : best;
}
// The mean size of what group_score() adds.
__device__ __forceinline__ float group_size(uint32_t best, uint32_t second, int size) {
  const float a = fabsf(dev::key_score(best));
  return size > 1 ? 0.5f * a + 0.5f * fabsf(dev::key_score(second)) : a;
}

// Drops the keys of groups that are not among the `top` best, in 32 bits;
// true in some lane if a group is too near the border for that.  Where a group
// is a power of two of whole lanes, its score comes from registers; any other
// size goes through LDS, where its size then takes the place of its first key.
struct GroupLds {
  uint32_t key[kMaxGroups];
  uint32_t border[2];
};
template <int G, int PER, bool BIAS>
__device__ __forceinline__ bool keep_groups(const RoutePlan& p, uint32_t (&key)[PER], const dev::Part<PER, false>& part,
                                            uint32_t g, float slack, uint32_t* staged, GroupLds& lds) {
  const uint32_t first = g * PER;
  const bool whole = p.group_lanes != 0;
  uint32_t own = 0;  // whole: the score of this lane's group
  float own_size = 0.f;
  bool near = false;
  if (whole) {
    uint32_t best = 0, second = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) join_best(best, second, key[j], 0u);
    if (p.group_lanes > 1) join_lane<1>(best, second);
    if (p.group_lanes > 2) join_lane<2>(best, second);
    if constexpr (G > 4) {
      if (p.group_lanes > 4) join_lane<4>(best, second);
    }
    if constexpr (G > 8) {
      if (p.group_lanes > 8) join_lane<8>(best, second);
    }
    if constexpr (G > 16) {
      if (p.group_lanes > 16) join_lane<16>(best, second);
    }
    if constexpr (G > 32) {
      if (p.group_lanes > 32) join_lane<32>(best, second);
    }
    own = group_score<BIAS>(best, second, p.size);
    if constexpr (BIAS) own_size = group_size(best, second, p.size);
    if (first < p.count) lds.key[p.by_size.div(first)] = own;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (part.own(j)) staged[part.from + j] = key[j];
    dev::wave_lds_fence();
    for (int q = (int)g; q < p.groups; q += G) {
      uint32_t best = 0, second = 0;
      int i = q % p.size;  // lanes start at different banks
      for (int n = 0; n < p.size; ++n) {
        join_best(best, second, staged[q * p.size + i], 0u);
        i = i + 1 == p.size ? 0 : i + 1;
      }
      lds.key[q] = group_score<BIAS>(best, second, p.size);
      if constexpr (BIAS) staged[q * p.size] = __builtin_bit_cast(uint32_t, group_size(best, second, p.size));
    }
  }
  dev::wave_lds_fence();
  const auto rank_of = [&](int q, uint32_t mine) {
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < p.groups; ++o) {
      const uint32_t other = lds.key[o];
      rank += other > mine || (other == mine && o < q);
    }
    if (rank == p.top - 1) lds.border[0] = mine;
    if (rank == p.top) lds.border[1] = mine;
    return rank;
  };
  const auto near_border = [&](bool kept, uint32_t key, float size) {
    const float middle = 0.5f * dev::key_score(lds.border[0]) + 0.5f * dev::key_score(lds.border[1]);
    const float score = dev::key_score(key), reach = group_reach(size, slack);
    return kept ? score - reach < middle : score + reach > middle;
  };
  if (whole) {
    const bool kept = first >= p.count || rank_of((int)p.by_size.div(first), own) < p.top;
    if (!kept) {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = 0;
    }
    dev::wave_lds_fence();
    if constexpr (BIAS) near = first < p.count && near_border(kept, own, own_size);
  } else {
    uint32_t kept[(kMaxGroups + G - 1) / G];
#pragma unroll
    for (int i = 0; i < (int)((kMaxGroups + G - 1) / G); ++i) {
      const int q = (int)g + i * G;
      kept[i] = q < p.groups && rank_of(q, lds.key[min(q, p.groups - 1)]) < p.top;
    }
    dev::wave_lds_fence();
#pragma unroll
    for (int i = 0; i < (int)((kMaxGroups + G - 1) / G); ++i) {
      const int q = (int)g + i * G;
      if (q >= p.groups) continue;
      if constexpr (BIAS)
        near = near || near_border(kept[i], lds.key[q], __builtin_bit_cast(float, staged[q * p.size]));
      lds.key[q] = kept[i];
    }
    dev::wave_lds_fence();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (!lds.key[p.by_size.div(min(part.from + j, p.count - 1))]) key[j] = 0;
  }
  dev::wave_lds_fence();
  return near;
}

// The choice of one token in 64 bits by a whole wavefront; rolled loops, as it
// is rare (a few tokens in a thousand of 256 experts).  Rows that all need it cost
// more: 16384 tokens of 256 experts whose groups tie 64 us, where others take 21,
// and peaked softmax rows with a bias of zeros 38, where flatter ones take 20.
struct WideLds {
  uint64_t group_key[kMaxGroups];
  uint32_t kept[kMaxGroups];
};
template <typename T>
__device__ __forceinline__ void choose64(const RoutePlan& p, const T* row, uint64_t* staged, WideLds& lds, int32_t* chosen) {
  const uint32_t lane = threadIdx.x & 63u;
  double top = 0.0, total = 1.0;
  if (p.softmax) {
    float m = -__builtin_inff();
    for (uint32_t e = lane; e < p.count; e += 64) m = fmaxf(m, (float)row[e]);
    top = (double)dev::group_max<64>(m);
    total = 0.0;
#pragma unroll 1
    for (uint32_t e = lane; e < p.count; e += 64) total += exp((double)(float)row[e] - top);
#pragma unroll 1
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
  }
#pragma unroll 1
  for (uint32_t e = lane; e < p.count; e += 64) {
    const double x = (double)(float)row[e], v = exp(p.softmax ? x - top : -x);
    staged[e] = dev::score_key((p.softmax ? v / total : 1.0 / (1.0 + v)) + (double)p.bias[e * p.bias_step]);
  }
  dev::wave_lds_fence();
  if (p.top < p.groups) {
    for (int q = (int)lane; q < p.groups; q += 64) {
      uint64_t best = 0, second = 0;
#pragma unroll 1
      for (int i = 0; i < p.size; ++i) join_best(best, second, staged[q * p.size + i], (uint64_t)0);
      lds.group_key[q] = group_score<true>(best, second, p.size);
    }
    dev::wave_lds_fence();
    for (int q = (int)lane; q < p.groups; q += 64) {
      int rank = 0;
#pragma unroll 1
      for (int o = 0; o < p.groups; ++o)
        rank += lds.group_key[o] > lds.group_key[q] || (lds.group_key[o] == lds.group_key[q] && o < q);
      lds.kept[q] = rank < p.top;
    }
    dev::wave_lds_fence();
    for (uint32_t e = lane; e < p.count; e += 64)
      if (!lds.kept[p.by_size.div(e)]) staged[e] = 0;
    dev::wave_lds_fence();
  }
#pragma unroll 1
  for (int i = 0; i < p.k; ++i) {
    uint64_t best = 0;
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll 1
    for (uint32_t e = lane; e < p.count; e += 64)
      if (staged[e] > best) {
        best = staged[e];
        at = e;
      }
    const uint64_t most = dev::group_max_key<64>(best);
    const uint32_t first = ~dev::group_max_key<64>(best == most ? ~at : 0u);  // the lowest of the equals
    if (lane == 0) {
      chosen[i] = (int32_t)first;
      staged[first] = 0;
    }
    dev::wave_lds_fence();
  }
}

// G lanes a token, lane g holding the logits of experts g * PER + j.  Without
// a bias the choice follows the logits, whose order is that of the scores.
// With one it follows s + bias in 32 bits, and where two of the k + 1 best (or
// the border of the groups) are nearer than that arithmetic can tell apart the
// token is chosen again in 64 bits; equal logits with equal biases are equal
// in either.
//
// The logits are read once, at the start; what bounds the kernel is the issue of
// instructions, not their bytes.  16384 tokens of 256 fp32 logits, 8 of them out
// of 4 of 8 groups: 21 us (0.85 TB/s; 1480 VALU instructions a wave of 4 tokens;
// of 25k cycles the loads take 3.5k, the scores 5.5k, the groups 3.4k, without the
// 80 instructions of their reach, and the selection 10.7k).  51200 tokens of 60
// fp16 logits, 4 of them: 7.8 us.  Hence the shape: as few lanes a token as hold
// its logits 4 to 16 each, so that a wave's reductions serve several tokens, and
// keys that are whole numbers, so that a maximum is one instruction and needs no
// second one for its place.
template <typename T, int G, int PER, bool BIAS, bool GROUPED>
__global__ __launch_bounds__(kThreads) void route_kernel(RoutePlan p) {
  constexpr int kTokens = kThreads / G;
  constexpr bool kPlaces = !BIAS && sizeof(T) == 2;  // a 16-bit logit and its place in one key
  __shared__ int32_t chosen[kTokens][kMaxChosen + 1];
  __shared__ float choice[BIAS ? kTokens : 1][kMaxChosen + 1];
  __shared__ GroupLds groups[GROUPED ? kTokens : 1];
  __shared__ WideLds wide[BIAS ? kThreads / 64 : 1];
  extern __shared__ uint64_t staged_lds[];

  const uint32_t g = threadIdx.x % G, slot = threadIdx.x / G;
  const uint32_t token = blockIdx.x * kTokens + slot;
  const bool live = token < p.tokens;  // every lane joins the group's exchanges
  // this wave's own, as waves do not wait for each other: 32-bit keys of all its tokens, then 64-bit ones of one
  uint64_t* staged = staged_lds + (threadIdx.x >> 6) * p.staged;
  const T* row = static_cast<const T*>(p.logits) + (int64_t)min(token, p.tokens - 1) * p.row;
  const dev::Part<PER, false> part(g, p.count);
  float x[PER];
  part.load(row, x);

  uint32_t key[PER];
  float total = 1.f;
  if constexpr (BIAS) {
    float b[PER];
    if (p.bias_step == 1) {
      part.load(p.bias, b);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) b[j] = p.bias[min(part.from + j, p.count - 1) * p.bias_step];
    }
    float s[PER];
    scores32<G, PER>(x, part, p.softmax, s, total);
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = part.own(j) ? dev::score_key(s[j] + b[j]) : 0u;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if constexpr (kPlaces) key[j] = part.own(j) ? dev::place_key<T>(x[j], part.from + j) : 0u;
      else key[j] = part.own(j) ? dev::score_key(x[j]) : 0u;
    }
  }
  const float slack = slack_of(p.softmax, total);
  bool close = false;
  if constexpr (GROUPED)
    close = keep_groups<G, PER, BIAS>(p, key, part, g, slack,
                                      reinterpret_cast<uint32_t*>(staged) + slot % (64 / G) * p.count, groups[slot]);
  const int open = GROUPED ? p.top * p.size : (int)p.count;
  const int n = BIAS && p.k < open ? p.k + 1 : p.k;
  if constexpr (kPlaces) {
    dev::take_places<G, PER>(key, n, g, [&](int i, uint32_t k) { chosen[slot][i] = (int32_t)dev::place_index(k); });
  } else {
    dev::take_best<G, PER>(key, n, g, [&](int i, uint32_t e, uint32_t k) {
      chosen[slot][i] = (int32_t)(e - part.skip);
      if constexpr (BIAS) choice[slot][i] = dev::key_score(k);
    });
  }
  dev::wave_lds_fence();
  if constexpr (BIAS) {
    for (int i = (int)g; i < n - 1; i += G) {
      if (!near_tie(choice[slot][i], choice[slot][i + 1], slack)) continue;
      const int32_t a = chosen[slot][i], b = chosen[slot][i + 1];
      close = close || (float)row[a] != (float)row[b] || p.bias[a * p.bias_step] != p.bias[b * p.bias_step];
    }
    uint64_t again = __ballot(close && live);
    if (again) {
      const uint32_t wave = threadIdx.x >> 6;
      while (again) {
        const uint32_t in_wave = (uint32_t)__builtin_ctzll(again) / G;  // token of the wave
        again &= ~((G == 64 ? ~0ull : (1ull << G) - 1) << (in_wave * G));
        const uint32_t s = wave * (64 / G) + in_wave;
        choose64(p, static_cast<const T*>(p.logits) + (int64_t)(blockIdx.x * kTokens + s) * p.row,
                 staged, wide[wave], chosen[s]);
      }
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
        if (part.own(j)) top = fmaxf(top, x[j]);
    }
    top = dev::group_max<G>(top);
  }
  bool low = false;
  const auto score = [&](float v) {
    if (low) return expf(v - top) / (1.0f + expf(v));
    return p.softmax ? expf(v - top) : 1.0f / (1.0f + expf(-v));
  };
  // (one weight a lane in most calls: kept for the second use)
  float mine = 0.f, sum = 0.f;
  if ((int)g < p.k) mine = score((float)row[chosen[slot][g]]);
  if (p.renormalize) {
    const auto add_scores = [&]() {
      float s = mine;
#pragma unroll 1
      for (int i = (int)g + G; i < p.k; i += G) s += score((float)row[chosen[slot][i]]);
      return dev::group_sum<G>(s);
    };
    sum = add_scores();
    // Logits below -86 leave less and less of 1 / (1 + e^-v) in 32 bits, which
    // matters where no sigmoid reaches 1/2: there the terms are
    // e^(v - top) / (1 + e^v), top being the highest chosen logit, whose
    // exponential cancels.
    if (!p.softmax && __any(sum < 0.5f)) {
      bool lost = false;
      for (int i = (int)g; i < p.k; i += G) {
        const float v = (float)row[chosen[slot][i]];
        lost = lost || v < -86.f;
        top = fmaxf(top, v);
      }
      low = sum < 0.5f && dev::group_ballot<G>(lost) != 0;  // the same for the lanes of a token
      if (__any(low)) {
        top = dev::group_max<G>(top);
        if ((int)g < p.k) mine = score((float)row[chosen[slot][g]]);
        sum = add_scores();
      }
    }
    if (BIAS && p.softmax && total != total) sum = total;  // a NaN anywhere is in every score of the row
  } else if (p.softmax) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (part.own(j)) sum += expf(x[j] - top);
    sum = dev::group_sum<G>(sum);
  } else {
    sum = 1.f;
  }
  if (!live) return;
#pragma unroll 1
  for (int i = (int)g; i < p.k; i += G) {
    const int32_t e = chosen[slot][i];
    if (i != (int)g) mine = score((float)row[e]);
    p.weights[(int64_t)token * p.wt + i * p.wk] = mine / sum * p.scale;
    p.experts[(int64_t)token * p.et + i * p.ek] = e;
  }
}

template <typename T, int G, int PER>
thin_status launch_route(RoutePlan p, hipStream_t stream) {
  const uint32_t tokens = kThreads / G;
  const dim3 grid((p.tokens + tokens - 1) / tokens), block(kThreads);
  THIN_REQUIRE(launchable(grid.x, kThreads), THIN_ERR_UNSUPPORTED, "expert_route: too many tokens");
  const bool grouped = p.top < p.groups;
  const uint32_t lanes = (uint32_t)p.size / PER;
  p.group_lanes = (uint32_t)p.size % PER == 0 && (lanes & (lanes - 1)) == 0 ? (int32_t)lanes : 0;
  p.staged = std::max<uint32_t>(p.bias ? p.count : 0u, grouped && !p.group_lanes ? (64 / G * p.count + 1) / 2 : 0u);
  const uint32_t lds = kThreads / 64 * p.staged * 8;
  if (p.bias) {
    if (grouped) hipLaunchKernelGGL((route_kernel<T, G, PER, true, true>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((route_kernel<T, G, PER, true, false>), grid, block, lds, stream, p);
  } else {
    if (grouped) hipLaunchKernelGGL((route_kernel<T, G, PER, false, true>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((route_kernel<T, G, PER, false, false>), grid, block, lds, stream, p);
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
  uint32_t bytes;                    // of a row
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

// Vector v of token t's row, copied to the rows its slots name.  NT: streaming
// stores, for rows that leave the caches anyway (604 MB: 104 us against 109
// without and 117 with the loads streaming too).
template <bool NT, typename Slot>
__device__ __forceinline__ void copy_row(const RowsPlan& p, uint32_t t, uint32_t v, Slot slot) {
  const char* src = p.x + (int64_t)t * p.xs;
  if (p.bytes >= 16) {
    const uint32_t at = min(v * 16, p.bytes - 16);
    const u4u w = *reinterpret_cast<const u4u*>(src + at);
    for (int j = 0; j < p.k; ++j) {
      const int32_t s = slot(j);
      if (s < 0) continue;
      u4u* to = reinterpret_cast<u4u*>(p.rows + (int64_t)s * p.rs + at);
      if constexpr (NT) __builtin_nontemporal_store(w, to);
      else *to = w;
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
// vectors of the row; block (tokens, 0) writes the offsets.  One launch, bound by
// latency: the ids' load, a pass over them in LDS and the row's own load and
// stores one after another (48 tokens of 4096 bf16, 8 experts each: 6.3 us for
// 3.5 MB, where counting, planning and copying in launches of their own would
// cost three times the launch alone).  Up to 4096 assignments: to 256 experts 128
// of them take 4.9 us against 9.6 in three launches, 2048 10.0 against 12.7, 4096
// 16.1 against 14.1.  To 1024 experts the offsets, a sum of its own for each, take
// 24 us of one block whatever the assignments, three launches 11 to 16.
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
  if (v * 16 < p.bytes) copy_row<false>(p, t, v, [&](int j) { return part[0][j]; });
}

// Many assignments, in three launches: counts of each block's assignments by
// expert, slots from them, the copy.  A block's 16 waves take runs of `chunk`
// assignments each, in order, so that no slot depends on the order of atomics.
// The first two are bound by latency, a load of ids and LDS atomics in turn;
// loads therefore go four or more at a time (131072 assignments to 256 experts:
// 4.8 and 8.4 us; with one wave's loads one after another the slots took 25 us).
constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// f(assignment, expert) of the assignments in [begin, end) of a thread that
// takes every step-th from begin + first on.
template <typename F>
__device__ __forceinline__ void each_assignment(const RowsPlan& p, uint32_t first, uint32_t end, uint32_t step, F f) {
  constexpr int U = 4;
#pragma unroll 1
  for (uint32_t a = first; a < end; a += U * step) {
    int32_t e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = expert_of(p, min(a + u * step, p.assigned - 1));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (a + u * step < end) f(a + u * step, e[u]);
  }
}

__global__ __launch_bounds__(kPlanThreads) void dispatch_count_kernel(RowsPlan p) {
  __shared__ int32_t counts[kMaxExperts];
  for (int e = threadIdx.x; e < p.count; e += kPlanThreads) counts[e] = 0;
  __syncthreads();
  const uint32_t begin = blockIdx.x * p.chunk * kPlanWaves, end = min(begin + p.chunk * kPlanWaves, p.assigned);
  each_assignment(p, begin + threadIdx.x, end, kPlanThreads, [&](uint32_t, int32_t e) {
    if (e >= 0) atomicAdd(&counts[e], 1);
  });
  __syncthreads();
  for (int e = threadIdx.x; e < p.count; e += kPlanThreads) p.counts[(int64_t)blockIdx.x * p.count + e] = counts[e];
}

__global__ __launch_bounds__(kPlanThreads) void dispatch_slots_kernel(RowsPlan p) {
  static_assert(kMaxExperts <= kPlanThreads, "a thread an expert");
  extern __shared__ int32_t next[];  // [waves][count]: next slot of each expert in each wave's run
  __shared__ int32_t sums[kPlanWaves];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
  const uint32_t begin = (blockIdx.x * kPlanWaves + wave) * p.chunk, end = min(begin + p.chunk, p.assigned);
  // counts of each wave's run, for the waves behind it
  for (int i = threadIdx.x; i < (int)kPlanWaves * p.count; i += kPlanThreads) next[i] = 0;
  __syncthreads();
  if (wave + 1 < kPlanWaves)
    each_assignment(p, begin + lane, end, 64, [&](uint32_t, int32_t e) {
      if (e >= 0) atomicAdd(&next[(wave + 1) * p.count + e], 1);
    });
  // a thread an expert: its assignments in all blocks, and in those before this one
  const int mine = (int)threadIdx.x;
  int32_t total = 0, before = 0;
  if (mine < p.count) {
    constexpr uint32_t U = 16;
    for (uint32_t b0 = 0; b0 < gridDim.x; b0 += U) {
      int32_t c[U];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) c[u] = p.counts[(int64_t)min(b0 + u, gridDim.x - 1) * p.count + mine];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        if (b0 + u < gridDim.x) total += c[u];
        if (b0 + u < blockIdx.x) before += c[u];
      }
    }
  }
  int32_t upto = total;  // sum of the experts' totals up to this one
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int32_t add = __shfl_up(upto, o, 64);
    if ((int)lane >= o) upto += add;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) upto += sums[w];
  if (mine < p.count) {
    if (blockIdx.x == 0) {
      p.offsets[(int64_t)mine * p.os] = upto - total;
      if (mine == p.count - 1) p.offsets[(int64_t)p.count * p.os] = upto;
    }
    int32_t at = upto - total + before;
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
      const int32_t in_wave = next[w * p.count + mine];  // of the wave before
      at += in_wave;
      next[w * p.count + mine] = at;
    }
  }
  __syncthreads();
  // 64 assignments at a time: the lanes of one expert take consecutive slots
  int32_t ahead = begin + lane < end ? expert_of(p, begin + lane) : -1;
  for (uint32_t a0 = begin; a0 < end; a0 += 64) {
    const uint32_t a = a0 + lane;
    const int32_t e = ahead;
    ahead = a + 64 < end ? expert_of(p, a + 64) : -1;
    uint64_t same = __ballot(e >= 0);
    for (int bit = 0; (1 << bit) < p.count; ++bit) {
      const uint64_t set = __ballot((e >> bit) & 1);
      same &= (e >> bit) & 1 ? set : ~set;
    }
    int32_t slot = -1;
    if (e >= 0) {
      const int leader = __builtin_ctzll(same);
      int32_t base = 0;
      if ((int)lane == leader) base = atomicAdd(&next[wave * p.count + e], __builtin_popcountll(same));
      slot = __shfl(base, leader, 64) + __builtin_popcountll(same & ((1ull << lane) - 1));
    }
    if (a < end) {
      const uint32_t t = p.by_k.div(a);
      p.slots[(int64_t)t * p.st + (int64_t)(a - t * p.k) * p.sk] = slot;
    }
  }
}

// The copy: HBM alone.  16384 rows of 4 KB to 8 places each: 104 us for 604 MB
// (5.8 TB/s); the stores by themselves, with no row read, also take 104 us.  A
// row is read once and written k times from registers.
template <bool NT>
__global__ __launch_bounds__(kThreads) void dispatch_copy_kernel(RowsPlan p) {
  const uint32_t t = blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes;
  const uint32_t v = blockIdx.y * p.lanes + threadIdx.x % p.lanes;
  if (t >= p.tokens || v * 16 >= p.bytes) return;
  copy_row<NT>(p, t, v, [&](int j) { return p.slots[(int64_t)t * p.st + j * p.sk]; });
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
// with one rounding; slots outside y contribute nothing.  A thread owns 16 bytes
// of out[t], so sums need neither LDS nor atomics.  Bound by HBM: 16384 tokens, 8
// rows of 4 KB each, 604 MB in 117 us (5.2 TB/s; rows of 4 KB at random places
// stay below a copy's 6.4).  Eight rows are loaded at a time (one after another
// 125 us; streaming loads changed nothing).
template <typename T, int N>
__device__ __forceinline__ void add_rows(const CombinePlan& p, uint32_t t, uint32_t at, float (&sum)[N]) {
  constexpr int U = 8;
  typedef typename dev::Pack<T, N>::type P;
  const T* y = static_cast<const T*>(p.y) + at;
  const float* w = p.weights + (int64_t)t * p.wt;
  const int32_t* slot = p.slots + (int64_t)t * p.st;
#pragma unroll 1
  for (int j = 0; j < p.k; j += U) {
    uint32_t s[U];
    float f[U];
    P r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(j + u, p.k - 1);
      s[u] = (uint32_t)slot[i * p.sk];
      f[u] = w[i * p.wk];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const P* from = reinterpret_cast<const P*>(y + (int64_t)min(s[u], p.rows - 1) * p.ys);
      r[u] = *from;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s[u] >= p.rows || j + u >= p.k) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] = __builtin_fmaf(f[u], (float)r[u][i], sum[i]);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombinePlan p) {
  constexpr uint32_t V = 16 / sizeof(T);
  const uint32_t t = p.lanes == kThreads ? blockIdx.x : blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes;
  const uint32_t v = blockIdx.y * p.lanes + threadIdx.x % p.lanes;
  if (t >= p.tokens || v * V >= p.width) return;
  T* out = static_cast<T*>(p.out) + (int64_t)t * p.os;
  if (p.width >= V) {
    const uint32_t at = min(v * V, p.width - V);
    float sum[V] = {};
    if (p.rows) add_rows<T, V>(p, t, at, sum);
    dev::store_pack<T, V>(out + at, sum);
  } else {
    for (uint32_t i = 0; i < p.width; ++i) {
      float sum[1] = {};
      if (p.rows) add_rows<T, 1>(p, t, i, sum);
      out[i] = (T)sum[0];
    }
  }
}

// Threads that share a row of `vectors` vectors.
uint32_t row_lanes(uint64_t vectors) {
  uint32_t lanes = 1;
  while (lanes < kThreads && lanes < vectors) lanes *= 2;
  return lanes;
}

// Blocks of the planning kernels and assignments a wave of them takes: at least
// 256 a wave, at most 256 blocks (each block reads the counts of all).
uint32_t plan_blocks(int64_t assigned, uint32_t* chunk) {
  const int64_t wave = std::max<int64_t>(256, (assigned + 256 * kPlanWaves - 1) / (256 * kPlanWaves));
  *chunk = (uint32_t)((wave + 63) / 64 * 64);
  return (uint32_t)((assigned + (int64_t)*chunk * kPlanWaves - 1) / ((int64_t)*chunk * kPlanWaves));
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
  THIN_REQUIRE(!repeats(weights) && !repeats(experts), THIN_ERR_INVALID, "expert_route: an output has a stride of 0");
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
    if (E < 4) return launch_route<T_, 64, 1>(p, stream);  // (a lane's part is no longer than the row)
    if (T <= kFewTokens) {
      if (E <= 64) return launch_route<T_, 64, 1>(p, stream);
      if (E <= 128) return launch_route<T_, 64, 2>(p, stream);
      if (E <= 256) return launch_route<T_, 64, 4>(p, stream);
      if (E <= 512) return launch_route<T_, 64, 8>(p, stream);
    }
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
  return (size_t)plan_blocks(tokens * top_k, &chunk) * (size_t)num_experts * sizeof(int32_t);
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
  THIN_REQUIRE(!repeats(rows) && !repeats(offsets) && !repeats(slots), THIN_ERR_INVALID,
               "expert_dispatch: an output has a stride of 0");
  const uint32_t elem = (uint32_t)dtype_size(x->dtype);
  const int64_t vectors = (H * elem + 15) / 16;
  const bool small = T * k <= kCountedAssignments;
  const int64_t lanes = small ? kThreads : row_lanes(vectors), per = kThreads / lanes;
  const dim3 grid((uint32_t)(small ? T + 1 : (T + per - 1) / per), (uint32_t)std::max<int64_t>(1, (vectors + lanes - 1) / lanes));
  THIN_REQUIRE(launchable(grid.x, kThreads) && grid.y < 65536, THIN_ERR_UNSUPPORTED, "expert_dispatch: tensors too large");
  const size_t need = thin_expert_dispatch_workspace(T, k, num_experts);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "expert_dispatch needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  THIN_REQUIRE(need == 0 || workspace_aligned(workspace), THIN_ERR_WORKSPACE,
               "expert_dispatch: the workspace must be 4-byte aligned");
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
  p.by_k = FastDiv::make((uint32_t)k);
  p.lanes = (uint32_t)lanes;
  if (small) {
    hipLaunchKernelGGL(dispatch_small_kernel, grid, dim3(kThreads), 0, stream, p);
    THIN_LAUNCH_CHECK("expert_dispatch");
    return THIN_OK;
  }
  const uint32_t blocks = plan_blocks(p.assigned, &p.chunk);
  hipLaunchKernelGGL(dispatch_count_kernel, dim3(blocks), dim3(kPlanThreads), 0, stream, p);
  THIN_LAUNCH_CHECK("expert_dispatch_count");
  hipLaunchKernelGGL(dispatch_slots_kernel, dim3(blocks), dim3(kPlanThreads),
                     kPlanWaves * (uint32_t)p.count * sizeof(int32_t), stream, p);
  THIN_LAUNCH_CHECK("expert_dispatch_slots");
  if (H == 0) return THIN_OK;
  if ((int64_t)p.assigned * p.bytes >= kStreamingBytes)
    hipLaunchKernelGGL((dispatch_copy_kernel<true>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((dispatch_copy_kernel<false>), grid, dim3(kThreads), 0, stream, p);
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
  THIN_REQUIRE(!repeats(out), THIN_ERR_INVALID, "expert_combine: the output has a stride of 0");
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
  const dim3 grid((p.tokens + per - 1) / per, (uint32_t)columns), block(kThreads);
  THIN_REQUIRE(columns < 65536 && launchable(grid.x, kThreads), THIN_ERR_UNSUPPORTED, "expert_combine: tensors too large");
  return with_float_type(y->dtype, [&](auto zero) {
    hipLaunchKernelGGL((combine_kernel<decltype(zero)>), grid, block, 0, stream, p);
    THIN_LAUNCH_CHECK("expert_combine");
    return THIN_OK;
  });
}
