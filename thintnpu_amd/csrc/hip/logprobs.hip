// Log probabilities of given tokens, with the entropy of each row and its most
// likely alternatives, from rows of logits.
//
// Everything is kept in powers of two: with L = log2(e) and m the maximum of the
// elements at hand, each contributes e = 2^y, y = (x - m) L, to s = sum e and
// u = sum e y.  Then
//   log p(x) = (x - m) - log2(s) ln 2,    entropy = (log2 s - u / s) ln 2,
// in which no term is larger than the result's own range.  y is one fma against
// M = fl(m L), whose rounding d = m L - M is taken back from the sums:
// s 2^-d and (u - d s) 2^-d.  That holds while d is small (plain_range()); larger
// maxima take x - m first.
#include "rows.h"

#include <string.h>

#include <algorithm>

namespace thin {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int64_t kMaxTop = 32;
constexpr int64_t kShortRow = 1024;   // longest row that one group of lanes holds
constexpr uint32_t kRun = 64;         // elements whose maximum is kept
constexpr uint32_t kTile = kRun * 64;  // elements of a wavefront
constexpr int64_t kMaxWidth = 8388608;
// Rows from which a wavefront finishes each instead of 16 (50001 wide, 5 and 20
// alternatives: 512 rows 8.4 and 14.2 against 7.2 and 8.0 us, 1000 rows 9.0 and
// 14.8 against 12.6 and 14.2).
constexpr int64_t kManyRows = 768;

struct LogprobsPlan {
  const void* logits;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  int64_t row, token_step, lp_step, h_step, tr, tk, ir, ik;  // element strides
  uint32_t rows, width, tiles;
  int32_t top;
  uint32_t* run_keys;   // workspace: [rows][tiles * 64] order of the runs' maxima
  uint32_t* tile_keys;  // [rows][tiles]
  float* tile_sums;     // [rows][tiles][2]: s and u against the tile's own maximum
  FastDiv by_tiles;
};

struct RowSums {
  float m, s, u;
};

// s and u of the elements against their maximum m.  The plain form needs a
// maximum in plain_range() and finite logits (-inf weighs nothing but would leave
// 0 * -inf in u) whose products with L are finite too; the careful one takes
// every value.
template <bool CAREFUL>
__device__ __forceinline__ void add_element(RowSums& r, float x, float top, float base) {
  const float y = CAREFUL ? (x - top) * kLog2e : __builtin_fmaf(x, kLog2e, -base);
  const float e = __builtin_amdgcn_exp2f(y);
  r.s += e;
  r.u = CAREFUL && e == 0.f ? r.u : __builtin_fmaf(e, y, r.u);
}
template <bool CAREFUL, typename L, int N>
__device__ __forceinline__ RowSums sums_of(const L (&v)[N], float m) {
  RowSums r{m, 0.f, 0.f};
  const float top = CAREFUL && m == -__builtin_inff() ? 0.f : m;
  const float base = top * kLog2e;
#pragma unroll
  for (int l = 0; l < N; ++l)
#pragma unroll
    for (int j = 0; j < L::V; ++j) add_element<CAREFUL>(r, v[l].at(j), top, base);
  return r;
}
// The plain form's sums against m itself.
__device__ __forceinline__ void take_back_rounding(RowSums& r) {
  const float d = __builtin_fmaf(r.m, kLog2e, -(r.m * kLog2e)), f = __builtin_amdgcn_exp2f(-d);
  r.u = __builtin_fmaf(-d, r.s, r.u) * f;
  r.s *= f;
}
// |d| <= 2^-4 (from about 2^30 on it passes the exponent's range, and sums and
// their factor of 0 and infinity would meet).
__device__ __forceinline__ bool plain_range(float m) { return fabsf(m) < 0x1p20f; }

__device__ __forceinline__ float rest_of(const RowSums& r) { return __builtin_log2f(r.s) * kLn2; }
// The given token's logit, loaded ahead of what store_row() waits for.
struct Given {
  float x;
  bool known;
};
template <typename T>
__device__ __forceinline__ Given given_of(const LogprobsPlan& p, uint32_t row, const T* x) {
  const int64_t token = p.tokens[(int64_t)row * p.token_step];
  const bool known = (uint64_t)token < (uint64_t)p.width;
  return {(float)x[known ? token : 0], known};
}
__device__ __forceinline__ void store_row(const LogprobsPlan& p, uint32_t row, const Given& given, const RowSums& r) {
  p.logprob[(int64_t)row * p.lp_step] = given.known ? (given.x - r.m) - rest_of(r) : __builtin_nanf("");
  p.entropy[(int64_t)row * p.h_step] = (__builtin_log2f(r.s) - r.u / r.s) * kLn2;
}
__device__ __forceinline__ void store_alternative(const LogprobsPlan& p, uint32_t row, int i, uint32_t id, float x,
                                                  float m, float rest) {
  p.top_logprobs[(int64_t)row * p.tr + i * p.tk] = (x - m) - rest;
  p.top_ids[(int64_t)row * p.ir + i * p.ik] = (int64_t)id;
}

// What stands in the place of elements that a row does not have: finite (an -inf
// would leave 0 * -inf), of weight 0 next to any maximum above kLowest, and the
// lowest value whose product with L is finite.  A lower element leaves a NaN in
// u, for which a tile is summed again without what stands in; so where it stays,
// it raises no run's maximum above that of the run's own elements.
template <typename T> constexpr float kAbsent = -0x1.62e42ep127f;
template <> constexpr float kAbsent<__bf16> = -0x1.62p127f;
template <> constexpr float kAbsent<_Float16> = -65504.f;
template <typename T> constexpr float kLowest = -0x1p20f;
template <> constexpr float kLowest<_Float16> = -65000.f;

// ---------------------------------------------------------------- short rows
// G lanes a row, lane g holding elements g * PER + j, so that a row is read once
// and everything after it is registers.  Bound by the issue of instructions, above
// all those of the alternatives, taken one after another: 200000 rows of 1000
// bf16, 400 MB, 97 us with none (4.1 TB/s), 216 with 5 and 396 with 20 (fp32 130,
// 251 and 664: its keys leave no room for the index, so that the one taken has to
// be found and removed); of 80, 32 MB, 14, 29 and 57.
template <typename T, int G, int PER>
__global__ __launch_bounds__(256) void short_rows_kernel(LogprobsPlan p) {
  const uint32_t g = threadIdx.x % G;
  const uint32_t row = blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row < p.rows;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)min(row, p.rows - 1) * p.row;
  const Given given = given_of(p, min(row, p.rows - 1), x);
  const dev::Part<PER, true> part(g, p.width);
  float v[PER];
  part.load(x, v);
  float m = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    v[j] = part.own(j) ? v[j] : kAbsent<float>;
    m = fmaxf(m, v[j]);
  }
  RowSums r{dev::group_max<G>(m), 0.f, 0.f};
  const bool plain = r.m > kLowest<float> && plain_range(r.m);
  const float base = r.m * kLog2e;
#pragma unroll
  for (int j = 0; j < PER; ++j) add_element<false>(r, v[j], r.m, base);
  r.s = dev::group_sum<G>(r.s);
  r.u = dev::group_sum<G>(r.u);
  take_back_rounding(r);
  if (!plain || r.u != r.u) {  // the same for the lanes of a row
    m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      v[j] = part.own(j) ? v[j] : -__builtin_inff();
      m = fmaxf(m, v[j]);
    }
    r = {dev::group_max<G>(m), 0.f, 0.f};
    const float top = r.m == -__builtin_inff() ? 0.f : r.m;
#pragma unroll
    for (int j = 0; j < PER; ++j) add_element<true>(r, v[j], top, 0.f);
    r.s = dev::group_sum<G>(r.s);
    r.u = dev::group_sum<G>(r.u);
  }
  if (live && g == 0) store_row(p, row, given, r);
  if (p.top == 0) return;
  const float rest = rest_of(r);
  uint32_t key[PER];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = part.own(j) ? dev::place_key<T>(v[j], part.from + j) : 0u;
    dev::take_places<G, PER>(key, p.top, g, [&](int i, uint32_t k) {
      if (live) store_alternative(p, row, i, dev::place_index(k), dev::place_score<T>(k), r.m, rest);
    });
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = part.own(j) ? dev::score_key(v[j]) : 0u;
    dev::take_best<G, PER>(key, p.top, g, [&](int i, uint32_t id, uint32_t k) {
      if (live) store_alternative(p, row, i, id - part.skip, dev::key_score(k), r.m, rest);
    });
  }
}

// ---------------------------------------------------------------- long rows
// NaN before everything.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  __asm__("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Sixteen bytes of a row as loaded.  (Maxima of pairs of halves, which leave the
// conversion to a mixed-precision fma, measured slower: 71.6 against 67.6 us for
// 4001 rows of 50001 halves.)
template <typename T>
struct Lane16 {
  static constexpr int V = 16 / sizeof(T);
  typename dev::Pack<T, V>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const typename dev::Pack<T, V>::type*>(p); }
  __device__ __forceinline__ void set(int j, T x) { raw[j] = x; }
  __device__ __forceinline__ void fill(T x) {
#pragma unroll
    for (int j = 0; j < V; ++j) raw[j] = x;
  }
  __device__ __forceinline__ float at(int j) const { return (float)raw[j]; }
  __device__ __forceinline__ float maximum() const {
    if constexpr (V == 8) {
      return max3(max3(max3(at(0), at(1), at(2)), at(3), at(4)), max3(at(5), at(6), at(7)), at(7));
    } else {
      return max3(max3(at(0), at(1), at(2)), at(3), at(3));
    }
  }
};

// Maxima over runs of N lanes of N values each lane: lane i of a run ends with
// the maximum of value i.  Each step halves the values: a lane keeps one of a
// pair, and hands the other to the lane across.
template <int O>
__device__ __forceinline__ float lane_xor_max(float keep, float send) {
  const float got = dev::lane_xor<O>(send);
  return max3(keep, got, got);
}
template <int N>
__device__ __forceinline__ float run_maximum(const float (&v)[N]) {
  if constexpr (N == 1) {
    return v[0];
  } else {
    constexpr int H = N / 2;
    const bool up = threadIdx.x & H;
    float half[H];
#pragma unroll
    for (int i = 0; i < H; ++i) half[i] = lane_xor_max<H>(up ? v[i + H] : v[i], up ? v[i] : v[i + H]);
    return run_maximum<H>(half);
  }
}

// A wavefront's tile of 4096 elements, in registers: the maximum first, then the
// sums against it, so that no running maximum rescales them.  Tiles begin at
// 16-byte aligned addresses whatever the row's own start, which leaves the odd
// elements to a row's first and last tile.  Sums and maximum (the same in every
// lane), and in lane l the maximum of run run_of(l).
template <typename T>
__device__ __forceinline__ uint32_t run_of() {
  constexpr uint32_t kLoads = kRun / Lane16<T>::V;
  const uint32_t lane = threadIdx.x & 63u;
  return lane % kLoads * (64 / kLoads) + lane / kLoads;
}
// The tile whose 16-byte aligned first position is at x; the row has positions
// [lo, hi) of it.
template <typename T>
__device__ __forceinline__ RowSums tile_sums(const T* x, int32_t lo, int32_t hi, float& run_top) {
  constexpr int V = Lane16<T>::V;   // elements of a load
  constexpr int kLoads = kRun / V;  // loads of a lane, and lanes that hold a run
  typedef typename dev::Pack<T, V>::type P;
  const int32_t lane = (int32_t)(threadIdx.x & 63u);
  const bool whole = lo <= 0 && hi >= (int32_t)kTile;  // the same for the whole wave
  Lane16<T> v[kLoads];
  if (whole) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      typedef T aligned __attribute__((ext_vector_type(V)));
      v[l].raw = __builtin_bit_cast(P, *reinterpret_cast<const aligned*>(x + (l * 64 + lane) * V));
    }
  } else {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int32_t at = (l * 64 + lane) * V;
      v[l].fill((T)kAbsent<T>);
      if (at >= lo && at + V <= hi) v[l].load(x + at);
    }
    // the vectors in which the row begins and ends, element by element
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      const int32_t edge = e ? hi : lo;
      if (edge <= 0 || edge >= (int32_t)kTile || edge % V == 0 || (e && lo > 0 && lo / V == hi / V)) continue;
      const int32_t vec = edge / V;
      if (lane != vec % 64) continue;
      Lane16<T> part;
#pragma unroll
      for (int j = 0; j < V; ++j) part.set(j, vec * V + j >= lo && vec * V + j < hi ? x[vec * V + j] : (T)kAbsent<T>);
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
        if (l == vec / 64) v[l] = part;
    }
  }
  float m;
  const auto maxima = [&]() {
    float part[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l) part[l] = v[l].maximum();
    run_top = run_maximum<kLoads>(part);
    m = lane_xor_max<32>(run_top, run_top);
    m = lane_xor_max<16>(m, m);
    m = lane_xor_max<8>(m, m);
    m = lane_xor_max<4>(m, m);
    m = lane_xor_max<2>(m, m);
    m = lane_xor_max<1>(m, m);
  };
  maxima();
  RowSums r{m, 0.f, __builtin_nanf("")};
  if (m > kLowest<T> && plain_range(m)) {
    r = sums_of<false>(v, m);
    r.s = dev::group_sum<64>(r.s);
    r.u = dev::group_sum<64>(r.u);
    take_back_rounding(r);
  }
  if (r.u != r.u) {
    if (!whole) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int32_t at = (l * 64 + lane) * V + j;
          if (at < lo || at >= hi) v[l].set(j, (T)-__builtin_inff());
        }
      maxima();
    }
    r = sums_of<true>(v, m);
    r.s = dev::group_sum<64>(r.s);
    r.u = dev::group_sum<64>(r.u);
  }
  return r;
}
// The order of the maximum of this lane's run, 0 if the row has none of it.
template <typename T>
__device__ __forceinline__ uint32_t run_key(float run_top, int32_t lo, int32_t hi) {
  const int32_t at = (int32_t)(run_of<T>() * kRun);
  return at + (int32_t)kRun > lo && at < hi ? dev::score_key(run_top) : 0u;
}

// A row in 16-byte aligned positions: x[at - skew] is at position `at`.
template <typename T>
struct Row {
  const T* x;
  int32_t skew;
  __device__ __forceinline__ Row(const LogprobsPlan& p, uint32_t row)
      : x(static_cast<const T*>(p.logits) + (int64_t)row * p.row),
        skew((int32_t)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T))) {}
  __device__ __forceinline__ RowSums tile(const LogprobsPlan& p, uint32_t t, uint32_t& key) const {
    const int32_t from = (int32_t)(t * kTile) - skew, lo = -from, hi = (int32_t)p.width - from;
    float run_top;
    const RowSums r = tile_sums(x + from, lo, hi, run_top);
    key = run_key<T>(run_top, lo, hi);
    return r;
  }
  // the order of the element at a position, 0 if the row has none there
  __device__ __forceinline__ uint32_t key(const LogprobsPlan& p, uint32_t at) const {
    const uint32_t i = at - (uint32_t)skew;
    const uint32_t key = dev::score_key((float)x[min(i, p.width - 1)]);
    return i < p.width ? key : 0u;
  }
};

// Adds a tile's sums to the row's, whose maximum r.m is known.
__device__ __forceinline__ void join(RowSums& r, float m, float s, float u) {
  if (s == 0.f) return;
  const float shift = (m - r.m) * kLog2e;
  const float f = __builtin_amdgcn_exp2f(shift);
  r.s = __builtin_fmaf(f, s, r.s);
  if (f != 0.f) r.u = __builtin_fmaf(f, __builtin_fmaf(shift, s, u), r.u);
}

// The K best of `items` x 64 keys by one wavefront, key(i) being item i of this
// lane and standing for index(i): entry r of best[], r < n, becomes the r-th
// best as key << 32 | ~index.  Where K lanes hold a key as high as some bound,
// the K best are among the keys not below it; those are listed and ranked by
// counting.  Where equal keys make the list too long, the best are taken one by
// one.  Keys in LDS and rolled loops: a row runs this twice, and
// fetching the instructions took longer than running them (unrolled over 32
// keys a lane in registers, 25 KB of code, three of these took 17 us).
constexpr int kListed = 256;
__device__ __forceinline__ uint32_t index_of(uint64_t entry) { return ~(uint32_t)entry; }
__device__ __forceinline__ uint32_t key_of(uint64_t entry) { return (uint32_t)(entry >> 32); }
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
struct Lists {
  uint64_t list[kListed];
  uint64_t best[kMaxTop];
};

template <typename Key, typename Index>
__device__ __forceinline__ int best_of(Key key, Index index, int items, int K, Lists& lds) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t top = 0;
#pragma unroll 4
  for (int i = 0; i < items; ++i) top = max(top, key(i));
  // the ceil(K / 4)-th best maximum of each 16 lanes (or less, where maxima are
  // equal): the lowest of the four
  uint32_t bound = dev::group_max_key<16>(top);
#pragma unroll 1
  for (int k = 4; k < K; k += 4) {
    if (top >= bound) top = 0;
    bound = dev::group_max_key<16>(top);
  }
  bound = min(bound, dev::lane_xor_bits<16>(bound));
  bound = max(1u, min(bound, dev::lane_xor_bits<32>(bound)));
  int listed = 0;
  const auto entry = [&](int i, uint32_t k) { return (uint64_t)k << 32 | (uint32_t)~index(i); };
#pragma unroll 1
  for (int i = 0; i < items; i += 4) {
    uint32_t k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = key(min(i + u, items - 1));
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool hit = k[u] >= bound && i + u < items;
      const uint64_t here = __ballot(hit);
      if (here == 0) continue;
      const int at = listed + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(here >> 32),
                                                             __builtin_amdgcn_mbcnt_lo((uint32_t)here, 0));
      if (hit && at < kListed) lds.list[at] = entry(i + u, k[u]);
      listed += __builtin_popcountll(here);
    }
  }
  dev::wave_lds_fence();
  const int n = min(K, listed);
  if (listed <= 64) {
    const uint64_t own = (int)lane < listed ? lds.list[lane] : 0;
    int before = 0;
    for (int o = 0; o < listed; ++o) before += lane_value(own, o) > own;
    if ((int)lane < listed && before < K) lds.best[before] = own;
  } else if (listed <= kListed) {
    for (int i = (int)lane; i < listed; i += 64) {
      const uint64_t own = lds.list[i];
      int before = 0;
#pragma unroll 4
      for (int o = 0; o < listed; ++o) before += lds.list[o] > own;
      if (before < K) lds.best[before] = own;
    }
  } else {
    uint64_t last = 0;
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      uint64_t next = 0;
#pragma unroll 1
      for (int i = 0; i < items; ++i) {
        const uint64_t own = entry(i, key(i));
        if ((k == 0 || own < last) && own > next) next = own;
      }
      last = dev::group_max_key<64>(next);
      if (lane == 0) lds.best[k] = last;
    }
  }
  dev::wave_lds_fence();
  return n;
}

// The row's K best elements by one wavefront, from `items` x 64 staged keys of
// its runs or of its tiles (any element outside has K better ones before it).
// The K best items of a level become the next level's, 64 adjacent keys of each.
template <typename T>
__device__ __forceinline__ void alternatives(const LogprobsPlan& p, uint32_t row, const Row<T>& x, uint32_t* staged,
                                             int items, bool runs, float m, float rest, Lists& lds) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t* run_keys = p.run_keys + (uint64_t)row * p.tiles * 64;
  uint32_t chosen = lane;  // in lane i: what item i stands for
  const auto item = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)chosen, i) * 64 + lane; };
  int n = items;
#pragma unroll 1
  for (int level = runs ? 1 : 0;; ++level) {  // tiles, runs, elements
    n = best_of([&](int i) { return staged[i * 64 + lane]; }, item, n, p.top, lds);
    chosen = (int)lane < n ? index_of(lds.best[lane]) : 0u;
    if (level == 2) break;
#pragma unroll 1
    for (int i = 0; i < n; i += 8) {  // eight loads in flight
      uint32_t key[8];
      if (level) {
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = x.key(p, item(min(i + u, n - 1)));
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = run_keys[item(min(i + u, n - 1))];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u < n) staged[(i + u) * 64 + lane] = key[u];
    }
    dev::wave_lds_fence();
  }
  if ((int)lane < n)
    store_alternative(p, row, (int)lane, chosen - (uint32_t)x.skew, dev::key_score(key_of(lds.best[lane])), m, rest);
}

// The sums of all tiles, in every lane.  The first 64 tiles' are loaded before
// anything else of a row's end, whose loads would otherwise wait for each other.
struct TileSums {
  const uint32_t* keys;
  const float* sums;
  uint32_t tiles, key;
  float s, u;
  __device__ __forceinline__ TileSums(const LogprobsPlan& p, uint32_t row)
      : keys(p.tile_keys + (uint64_t)row * p.tiles), sums(p.tile_sums + 2 * (uint64_t)row * p.tiles), tiles(p.tiles) {
    const uint32_t lane = threadIdx.x & 63u, t = min(lane, tiles - 1);
    key = keys[t];
    s = sums[2 * t];
    u = sums[2 * t + 1];
    if (lane >= tiles) s = 0.f;
  }
  __device__ __forceinline__ RowSums row() const {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t top = key;
    for (uint32_t t = lane + 64; t < tiles; t += 64) top = max(top, keys[t]);
    RowSums r{dev::key_score(dev::group_max_key<64>(top)), 0.f, 0.f};
    join(r, dev::key_score(key), s, u);
    for (uint32_t t = lane + 64; t < tiles; t += 64) join(r, dev::key_score(keys[t]), sums[2 * t], sums[2 * t + 1]);
    r.s = dev::group_sum<64>(r.s);
    r.u = dev::group_sum<64>(r.u);
    return r;
  }
};

// Rows of one tile, a wavefront each, in one launch: 40000 rows of 4000 bf16 53 us
// (6.1 TB/s), 93 with 5 alternatives and 148 with 20, by the issue of their
// selection; of 1100, which leave three quarters of the tile empty, 41, 86 and 131.
template <typename T>
__global__ __launch_bounds__(64) void tile_rows_kernel(LogprobsPlan p) {
  __shared__ Lists lds;
  __shared__ uint32_t staged[kMaxTop * 64];
  const uint32_t row = blockIdx.x;
  const Row<T> x(p, row);
  const Given given = given_of(p, row, x.x);
  uint32_t key;
  const RowSums r = x.tile(p, 0, key);
  if (threadIdx.x == 0) store_row(p, row, given, r);
  if (p.top == 0) return;
  staged[run_of<T>()] = key;
  dev::wave_lds_fence();
  alternatives(p, row, x, staged, 1, true, r.m, rest_of(r), lds);
}

// Longer rows, two launches: tiles anywhere on the device, however few the rows,
// then the joins.  The first is bound by HBM and, next to it, by issue (550 VALU
// instructions a tile, 64 of them exponentials): 4001 rows of 50001, 400 MB, 64 us
// in bf16 (6.3 TB/s) and 72 us in fp16 (5.5, a conversion an element more); 48
// rows of 128000 5.8 us.
template <typename T>
__global__ __launch_bounds__(256) void tiles_kernel(LogprobsPlan p) {
  const uint32_t wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t row = p.by_tiles.div(wave);
  if (row >= p.rows) return;
  uint32_t key;
  const RowSums r = Row<T>(p, row).tile(p, wave - row * p.tiles, key);
  if ((threadIdx.x & 63u) == 0) {
    p.tile_keys[wave] = dev::score_key(r.m);
    p.tile_sums[2 * (uint64_t)wave] = r.s;
    p.tile_sums[2 * (uint64_t)wave + 1] = r.u;
  }
  if (p.top) p.run_keys[(uint64_t)wave * 64 + run_of<T>()] = key;
}

// Many rows: a wavefront each, which the others on the device hide (as much LDS
// as the row needs, so that more of them fit).  Bound by the issue of the
// selection's instructions: 4001 rows of 13 tiles, 5 alternatives, 14 us (740
// VALU instructions a row for 10 MB of keys).
constexpr uint32_t kStaged = 33;  // items of 64: the tiles of the longest row, the runs of 33 tiles
uint32_t staged_items(uint32_t tiles, int64_t top) {
  return top ? std::max<uint32_t>(tiles <= kStaged ? tiles : (tiles + 63) / 64, (uint32_t)top) : 0u;
}
template <typename T>
__global__ __launch_bounds__(64) void finish_many_kernel(LogprobsPlan p) {
  __shared__ Lists lds;
  extern __shared__ uint32_t staged[];  // staged_items() x 64
  const uint32_t lane = threadIdx.x, row = blockIdx.x;
  const Row<T> x(p, row);
  const Given given = given_of(p, row, x.x);
  const TileSums sums(p, row);
  const bool runs = p.tiles <= kStaged;
  const int items = runs ? (int)p.tiles : (int)((p.tiles + 63) / 64);
  if (p.top) {
    const uint32_t* keys = runs ? p.run_keys + (uint64_t)row * p.tiles * 64 : sums.keys;
    const uint32_t count = runs ? p.tiles * 64 : p.tiles;
#pragma unroll 1
    for (int i = 0; i < items; i += 16) {  // 16 loads in flight
      uint32_t key[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) key[u] = keys[min((i + u) * 64 + lane, count - 1)];
#pragma unroll
      for (int u = 0; u < 16; ++u)
        if (i + u < items) staged[(i + u) * 64 + lane] = (i + u) * 64 + lane < count ? key[u] : 0u;
    }
  }
  const RowSums r = sums.row();
  if (lane == 0) store_row(p, row, given, r);
  dev::wave_lds_fence();
  if (p.top) alternatives(p, row, x, staged, items, runs, r.m, rest_of(r), lds);
}

// Few rows: 16 wavefronts each, for the latency, which is all there is: loads of
// the keys, two or three rounds of counting and ranking, and between them loads
// of what was chosen (48 rows of 32 tiles, 20 alternatives: 7.3 us).
// best_of() by a workgroup of 16 wavefronts, item i of a thread standing for
// index(i): the same bound from the maxima of the 64 lane columns, its counts
// and ranks shared out over the waves (in one wave each of their steps waits
// for the last: 11400 cycles for 20 of 2048 keys, a tenth of that here).
constexpr int kFinishThreads = 1024;
constexpr int kHeld = 8;  // keys of a thread
struct WideLists {
  uint64_t list[kListed];
  uint64_t best[kMaxTop];
  uint64_t wave_best[kFinishThreads / 64];
  uint32_t rank[kListed];
  uint32_t column[64];
  uint32_t higher[64];
  uint32_t count;
};
template <typename Index>
__device__ __forceinline__ int wide_best_of(const uint32_t (&key)[kHeld], Index index, int K, WideLists& lds) {
  constexpr uint32_t W = kFinishThreads / 64;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  if (threadIdx.x < 64) {
    lds.column[threadIdx.x] = 0;
    lds.higher[threadIdx.x] = 0;
  }
  if (threadIdx.x < (uint32_t)kListed) lds.rank[threadIdx.x] = 0;
  if (threadIdx.x == 0) lds.count = 0;
  __syncthreads();
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kHeld; ++i) top = max(top, key[i]);
  if (top) atomicMax(&lds.column[lane], top);
  __syncthreads();
  const uint32_t mine = lds.column[lane];
  uint32_t higher = 0;
#pragma unroll
  for (uint32_t o = 0; o < 64 / W; ++o) higher += lds.column[wave * (64 / W) + o] > mine;
  if (higher) atomicAdd(&lds.higher[lane], higher);
  __syncthreads();
  // the lowest maximum that fewer than K others pass
  const uint32_t bound = max(1u, ~dev::group_max_key<64>(lds.higher[lane] < (uint32_t)K ? ~mine : 0u));
  if (top >= bound) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (key[i] >= bound) {
        const uint32_t at = atomicAdd(&lds.count, 1u);
        if (at < (uint32_t)kListed) lds.list[at] = (uint64_t)key[i] << 32 | (uint32_t)~index(i);
      }
  }
  __syncthreads();
  const int listed = (int)lds.count, n = min(K, listed);
  if (listed <= kListed) {
    for (int e = (int)lane; e < listed; e += 64) {
      const uint64_t own = lds.list[e];
      uint32_t before = 0;
      for (int o = (int)wave; o < listed; o += W) before += lds.list[o] > own;
      if (before) atomicAdd(&lds.rank[e], before);
    }
    __syncthreads();
    if ((int)threadIdx.x < listed && lds.rank[threadIdx.x] < (uint32_t)K)
      lds.best[lds.rank[threadIdx.x]] = lds.list[threadIdx.x];
  } else {
    uint64_t last = 0;
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
      uint64_t next = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const uint64_t own = (uint64_t)key[i] << 32 | (uint32_t)~index(i);
        if (key[i] && (k == 0 || own < last) && own > next) next = own;
      }
      next = dev::group_max_key<64>(next);
      if (lane == 0) lds.wave_best[wave] = next;
      __syncthreads();
      last = 0;
#pragma unroll 1
      for (uint32_t w = 0; w < W; ++w) last = lds.wave_best[w] > last ? lds.wave_best[w] : last;
      __syncthreads();
      if (threadIdx.x == 0) lds.best[k] = last;
    }
  }
  __syncthreads();
  return n;
}

template <typename T>
__global__ __launch_bounds__(kFinishThreads) void finish_few_kernel(LogprobsPlan p) {
  constexpr uint32_t W = kFinishThreads / 64;
  __shared__ WideLists lds;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x;
  const Row<T> x(p, row);
  const Given given = given_of(p, row, x.x);
  const TileSums sums(p, row);
  const uint32_t* run_keys = p.run_keys + (uint64_t)row * p.tiles * 64;
  // the runs of all tiles at once, or first the tiles
  int level = p.tiles <= kHeld * W ? 1 : 0, n = 0;
  uint32_t key[kHeld];
  if (p.top) {
    const uint32_t* keys = level ? run_keys : sums.keys;
    const uint32_t count = level ? p.tiles * 64 : p.tiles;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const uint32_t at = i * kFinishThreads + threadIdx.x, k = keys[min(at, count - 1)];
      key[i] = at < count ? k : 0u;
    }
  }
  const RowSums r = sums.row();
  if (threadIdx.x == blockDim.x - 64) store_row(p, row, given, r);
  if (p.top == 0) return;
  uint32_t first[kMaxTop / W] = {};  // this wave's items of a level after the first: 64 indices each
#pragma unroll 1
  for (int step = 0;; ++step, ++level) {  // tiles, runs, elements
    n = wide_best_of(key, [&](int i) { return step ? (first[i & 1] + lane) : i * kFinishThreads + threadIdx.x; }, p.top, lds);
    if (level == 2) break;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int item = (int)wave + i * (int)W;
      key[i] = 0;
      if (i < (int)(kMaxTop / W) && item < n) {
        first[i & 1] = index_of(lds.best[item]) * 64;
        const uint32_t at = first[i & 1] + lane;
        key[i] = level == 0 ? run_keys[at] : x.key(p, at);
      }
    }
    __syncthreads();
  }
  if ((int)threadIdx.x < n) {
    const uint64_t found = lds.best[threadIdx.x];
    store_alternative(p, row, (int)threadIdx.x, index_of(found) - (uint32_t)x.skew, dev::key_score(key_of(found)), r.m,
                      rest_of(r));
  }
}

// Tiles of a row, wherever in 16 bytes it begins.
uint32_t tiles_of(int64_t width, int elem) { return (uint32_t)((width + 16 / elem - 1 + kTile - 1) / kTile); }

template <typename T, int G, int PER>
thin_status launch_short(const LogprobsPlan& p, hipStream_t stream) {
  const uint32_t rows = 256 / G;
  THIN_REQUIRE(launchable((p.rows + rows - 1) / rows, 256), THIN_ERR_UNSUPPORTED, "token_logprobs: tensor too large");
  hipLaunchKernelGGL((short_rows_kernel<T, G, PER>), dim3((p.rows + rows - 1) / rows), dim3(256), 0, stream, p);
  THIN_LAUNCH_CHECK("token_logprobs");
  return THIN_OK;
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" size_t thin_token_logprobs_workspace(int64_t rows, int64_t width, int64_t top) {
  // (as for 16-bit rows, which may begin further into their first 16 bytes)
  if (rows <= 0 || width <= kShortRow || width > kMaxWidth) return 0;
  const int64_t tiles = tiles_of(width, 2);
  return tiles == 1 ? 0 : (size_t)rows * tiles * (top > 0 ? 64 + 3 : 3) * 4;
}

extern "C" thin_status thin_token_logprobs(const thin_desc* logits, const thin_desc* tokens, const thin_desc* logprobs,
                                           const thin_desc* entropy, const thin_desc* top_logprobs,
                                           const thin_desc* top_ids, void* workspace, size_t workspace_bytes,
                                           hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(logits) && desc_valid(tokens) && desc_valid(logprobs) && desc_valid(entropy) &&
                   desc_valid(top_logprobs) && desc_valid(top_ids),
               THIN_ERR_INVALID, "token_logprobs: invalid descriptor");
  THIN_REQUIRE(float_type(logits->dtype) && logits->rank == 2, THIN_ERR_INVALID,
               "token_logprobs takes float16, bfloat16 or float32 logits [rows, width]");
  const int64_t R = logits->sizes[0], V = logits->sizes[1];
  THIN_REQUIRE(tokens->rank == 1 && tokens->dtype == THIN_I64 && tokens->sizes[0] == R && logprobs->rank == 1 &&
                   logprobs->dtype == THIN_F32 && logprobs->sizes[0] == R && entropy->rank == 1 &&
                   entropy->dtype == THIN_F32 && entropy->sizes[0] == R,
               THIN_ERR_INVALID, "token_logprobs takes int64 tokens [rows], float32 logprobs and entropy [rows]");
  THIN_REQUIRE(top_logprobs->rank == 2 && top_logprobs->dtype == THIN_F32 && top_logprobs->sizes[0] == R &&
                   top_ids->rank == 2 && top_ids->dtype == THIN_I64 && top_ids->sizes[0] == R &&
                   top_ids->sizes[1] == top_logprobs->sizes[1],
               THIN_ERR_INVALID, "token_logprobs writes float32 top_logprobs and int64 top_ids [rows, top]");
  const int64_t K = top_ids->sizes[1];
  THIN_REQUIRE(V >= 1 && K <= V && K <= kMaxTop, THIN_ERR_INVALID,
               "token_logprobs gives up to %lld alternatives of the row's %lld, not %lld", (long long)kMaxTop,
               (long long)V, (long long)K);
  THIN_REQUIRE(V <= kMaxWidth && R < (1ll << 31) && (V <= kShortRow || launchable(R * tiles_of(V, 2) + 3, 64)),
               THIN_ERR_UNSUPPORTED, "token_logprobs: tensor too large");
  THIN_REQUIRE(V == 1 || logits->strides[1] == 1, THIN_ERR_UNSUPPORTED,
               "token_logprobs: the logits of a row must be adjacent");
  if (R == 0) return THIN_OK;
  const thin_desc* outs[4] = {logprobs, entropy, top_logprobs, top_ids};
  for (int i = 0; i < 4; ++i) {
    THIN_REQUIRE(!repeats(outs[i]), THIN_ERR_INVALID, "token_logprobs: an output has a stride of 0");
    THIN_REQUIRE(!overlap(outs[i], logits) && !overlap(outs[i], tokens), THIN_ERR_INVALID,
                 "token_logprobs: an output overlaps an input");
    for (int j = 0; j < i; ++j)
      THIN_REQUIRE(!overlap(outs[i], outs[j]), THIN_ERR_INVALID, "token_logprobs: two outputs overlap");
  }
  const size_t need = thin_token_logprobs_workspace(R, V, K);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "token_logprobs needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  THIN_REQUIRE(need == 0 || workspace_aligned(workspace), THIN_ERR_WORKSPACE,
               "token_logprobs: the workspace must be 4-byte aligned");
  LogprobsPlan p;
  memset(&p, 0, sizeof p);
  p.logits = logits->data;
  p.tokens = static_cast<const int64_t*>(tokens->data);
  p.logprob = static_cast<float*>(logprobs->data);
  p.entropy = static_cast<float*>(entropy->data);
  p.top_logprobs = static_cast<float*>(top_logprobs->data);
  p.top_ids = static_cast<int64_t*>(top_ids->data);
  p.row = logits->strides[0];
  p.token_step = tokens->strides[0];
  p.lp_step = logprobs->strides[0];
  p.h_step = entropy->strides[0];
  p.tr = top_logprobs->strides[0]; p.tk = top_logprobs->strides[1];
  p.ir = top_ids->strides[0]; p.ik = top_ids->strides[1];
  p.rows = (uint32_t)R;
  p.width = (uint32_t)V;
  p.top = (int32_t)K;
  return with_float_type(logits->dtype, [&](auto zero) {
    using T = decltype(zero);
    if (V <= 16) return launch_short<T, 4, 4>(p, stream);
    if (V <= 32) return launch_short<T, 8, 4>(p, stream);
    if (V <= 64) return launch_short<T, 16, 4>(p, stream);
    if (V <= 128) return launch_short<T, 16, 8>(p, stream);
    if (V <= 256) return launch_short<T, 16, 16>(p, stream);
    if (V <= 512) return launch_short<T, 32, 16>(p, stream);
    if (V <= kShortRow) return launch_short<T, 64, 16>(p, stream);
    p.tiles = tiles_of(V, 2);
    if (p.tiles == 1) {
      hipLaunchKernelGGL((tile_rows_kernel<T>), dim3(p.rows), dim3(64), 0, stream, p);
      THIN_LAUNCH_CHECK("token_logprobs_rows");
      return THIN_OK;
    }
    p.by_tiles = FastDiv::make(p.tiles);
    const uint64_t waves = (uint64_t)p.rows * p.tiles;
    p.tile_sums = static_cast<float*>(workspace);
    p.tile_keys = reinterpret_cast<uint32_t*>(p.tile_sums + 2 * waves);
    p.run_keys = p.tile_keys + waves;
    hipLaunchKernelGGL((tiles_kernel<T>), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, stream, p);
    THIN_LAUNCH_CHECK("token_logprobs_tiles");
    if (R < kManyRows) hipLaunchKernelGGL((finish_few_kernel<T>), dim3(p.rows), dim3(p.top ? kFinishThreads : 64), 0, stream, p);
    else hipLaunchKernelGGL((finish_many_kernel<T>), dim3(p.rows), dim3(64), staged_items(p.tiles, K) * 256, stream, p);
    THIN_LAUNCH_CHECK("token_logprobs_finish");
    return THIN_OK;
  });
}
