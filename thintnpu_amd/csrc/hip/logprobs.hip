// Log probabilities of given tokens, with the entropy of each row and its most
// likely alternatives, from rows of logits.
//
// Everything is kept in powers of two: with L = log2(e) and m the maximum of the
// elements at hand, each contributes e = 2^y, y = (x - m) L, to s = sum e and
// u = sum e y.  Then
//   log p(x) = (x - m) - log2(s) ln 2,    entropy = (log2 s - u / s) ln 2,
// in which no term is larger than the result's own range.  y is one fma against
// M = fl(m L), whose rounding d = m L - M is taken back from the sums:
// s 2^-d and (u - d s) 2^-d.
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
constexpr int64_t kMaxTiles = 64 * kMaxTop;

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

// s and u of the elements against their maximum m.  The plain form needs
// finite logits (-inf weighs nothing but would leave 0 * -inf in u) whose
// products with L are finite too; the careful one takes every value.
template <bool CAREFUL, int N, int V>
__device__ __forceinline__ RowSums sums_of(const float (&v)[N][V], float m) {
  RowSums r{m, 0.f, 0.f};
  const float top = CAREFUL && m == -__builtin_inff() ? 0.f : m;
  const float base = top * kLog2e;
#pragma unroll
  for (int l = 0; l < N; ++l)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float y = CAREFUL ? (v[l][j] - top) * kLog2e : __builtin_fmaf(v[l][j], kLog2e, -base);
      const float e = __builtin_amdgcn_exp2f(y);
      r.s += e;
      r.u = CAREFUL ? (e == 0.f ? r.u : __builtin_fmaf(e, y, r.u)) : __builtin_fmaf(e, y, r.u);
    }
  return r;
}
// The plain form's sums against m itself.
__device__ __forceinline__ void take_back_rounding(RowSums& r) {
  const float d = __builtin_fmaf(r.m, kLog2e, -(r.m * kLog2e)), f = __builtin_amdgcn_exp2f(-d);
  r.u = __builtin_fmaf(-d, r.s, r.u) * f;
  r.s *= f;
}
__device__ __forceinline__ bool plain_range(float m) { return fabsf(m) < 1e38f; }

__device__ __forceinline__ float rest_of(const RowSums& r) { return __builtin_log2f(r.s) * kLn2; }
template <typename T>
__device__ __forceinline__ void store_row(const LogprobsPlan& p, uint32_t row, const T* x, const RowSums& r) {
  const float rest = rest_of(r);
  const int64_t token = p.tokens[(int64_t)row * p.token_step];
  const bool known = (uint64_t)token < (uint64_t)p.width;
  p.logprob[(int64_t)row * p.lp_step] = known ? ((float)x[token] - r.m) - rest : __builtin_nanf("");
  p.entropy[(int64_t)row * p.h_step] = (__builtin_log2f(r.s) - r.u / r.s) * kLn2;
}
__device__ __forceinline__ void store_alternative(const LogprobsPlan& p, uint32_t row, int i, uint32_t id, float x,
                                                  float m, float rest) {
  p.top_logprobs[(int64_t)row * p.tr + i * p.tk] = (x - m) - rest;
  p.top_ids[(int64_t)row * p.ir + i * p.ik] = (int64_t)id;
}

// ---------------------------------------------------------------- short rows
// G lanes a row, lane g holding elements g * PER + j.
template <typename T, int G, int PER>
__global__ __launch_bounds__(256) void short_rows_kernel(LogprobsPlan p) {
  const uint32_t g = threadIdx.x % G;
  const uint32_t row = blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row < p.rows;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)min(row, p.rows - 1) * p.row;
  const uint32_t first = g * PER;
  float v[1][PER];
  if (first + PER <= p.width) {
    dev::load_pack<T, PER>(x + first, v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) v[0][j] = first + j < p.width ? (float)x[first + j] : -__builtin_inff();
  }
  float m = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < PER; ++j) m = fmaxf(m, v[0][j]);
  RowSums r = sums_of<true>(v, dev::group_max<G>(m));
  r.s = dev::group_sum<G>(r.s);
  r.u = dev::group_sum<G>(r.u);
  if (live && g == 0) store_row(p, row, x, r);
  if (p.top == 0) return;
  const float rest = rest_of(r);
  uint32_t key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) key[j] = first + j < p.width ? dev::score_key(v[0][j]) : 0u;
  dev::take_best<G, PER>(key, p.top, g, [&](int i, uint32_t id, uint32_t k) {
    if (live) store_alternative(p, row, i, id, dev::key_score(k), r.m, rest);
  });
}

// ---------------------------------------------------------------- long rows
// A wavefront takes a tile of 4096 elements of a row: its sums, and the
// maximum of each run of 64, whose order is all that the second launch needs
// to find the alternatives.
template <typename T>
__global__ __launch_bounds__(256) void tiles_kernel(LogprobsPlan p) {
  constexpr uint32_t V = 16 / sizeof(T);     // elements of a load
  constexpr uint32_t kLoads = kRun / V;      // loads of a lane
  constexpr uint32_t kLanes = kRun / V;      // lanes that hold a run
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t row = p.by_tiles.div(wave);
  if (row >= p.rows) return;
  const uint32_t tile = wave - row * p.tiles;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.row;
  float v[kLoads][V];
#pragma unroll
  for (uint32_t l = 0; l < kLoads; ++l) {
    const uint32_t at = tile * kTile + l * 64 * V + lane * V;
    if (at + V <= p.width) {
      dev::load_pack<T, V>(x + at, v[l]);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < V; ++j) v[l][j] = at + j < p.width ? (float)x[at + j] : -__builtin_inff();
    }
  }
  float m = -__builtin_inff();
  uint32_t run_key = 0;
#pragma unroll
  for (uint32_t l = 0; l < kLoads; ++l) {
    float top = v[l][0];
#pragma unroll
    for (uint32_t j = 1; j < V; ++j) top = __builtin_elementwise_maximum(top, v[l][j]);
#pragma unroll
    for (uint32_t o = 1; o < kLanes; o <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o, 64));
    // the lanes of a run keep one load's maximum each
    const uint32_t at = tile * kTile + l * 64 * V + (lane & ~(kLanes - 1)) * V;
    if (lane % kLanes == l) run_key = at < p.width ? dev::score_key(top) : 0u;
    m = __builtin_elementwise_maximum(m, top);
  }
#pragma unroll
  for (uint32_t o = kLanes; o < 64; o <<= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o, 64));
  // wave-uniform: every lane holds m and the sums
  RowSums r{m, 0.f, __builtin_nanf("")};
  if ((tile + 1) * kTile <= p.width && plain_range(m)) {
    r = sums_of<false>(v, m);
    r.s = dev::group_sum<64>(r.s);
    r.u = dev::group_sum<64>(r.u);
    take_back_rounding(r);
  }
  if (r.u != r.u) {
    r = sums_of<true>(v, m);
    r.s = dev::group_sum<64>(r.s);
    r.u = dev::group_sum<64>(r.u);
  }
  const uint64_t at = (uint64_t)row * p.tiles + tile;
  if (lane == 0) {
    p.tile_keys[at] = dev::score_key(m);
    p.tile_sums[2 * at] = r.s;
    p.tile_sums[2 * at + 1] = r.u;
  }
  if (p.top) p.run_keys[at * 64 + lane % kLanes * (64 / kLanes) + lane / kLanes] = run_key;
}

// The K best of the keys of a wavefront, item i of lane l standing for index
// base[i] * 64 + l, base ascending.  At least K lanes hold a key as high as the
// K-th best of the lanes' maxima: what lies above it, and of its equals the
// first K in the order of the index, contains the K best.  `list` then holds
// them (at most (K - 1) items of each of the K - 1 lanes above, and K), and
// ranks by counting put them in order.  Returns how many there are.
struct Found {
  uint32_t key, index;
};
constexpr int kListed = (int)((kMaxTop - 1) * kMaxTop + kMaxTop);

__device__ int best_of(const uint32_t (&key)[kMaxTop], int items, const uint32_t* base, int K, Found* list,
                       uint32_t* lane_keys, Found* best) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < (int)kMaxTop; ++i)
    if (i < items) top = max(top, key[i]);
  lane_keys[lane] = top;
  dev::wave_lds_fence();
  int rank = 0;
  for (int o = 0; o < 64; ++o) {
    const uint32_t other = lane_keys[o];
    rank += other > top || (other == top && o < (int)lane);
  }
  const uint64_t last = __ballot(rank == K - 1);
  const uint32_t bound = max(1u, (uint32_t)__builtin_amdgcn_readlane((int)top, __builtin_ctzll(last)));
  int above = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < (int)kMaxTop; ++i) {
    if (i >= items) continue;
    const uint64_t over = __ballot(key[i] > bound), same = __ballot(key[i] == bound);
    const uint64_t below = (1ull << lane) - 1;
    if (key[i] > bound) list[kMaxTop + above + __builtin_popcountll(over & below)] = Found{key[i], base[i] * 64 + lane};
    const int place = equal + __builtin_popcountll(same & below);
    if (key[i] == bound && place < K) list[place] = Found{key[i], base[i] * 64 + lane};
    above += __builtin_popcountll(over);
    equal = min(K, equal + (int)__builtin_popcountll(same));
  }
  dev::wave_lds_fence();
  const int n = min(K, above + equal);
  for (int i = (int)lane; i < above + equal; i += 64) {
    const Found mine = i < equal ? list[i] : list[kMaxTop + i - equal];
    int before = 0;
    for (int o = 0; o < above + equal; ++o) {
      const Found other = o < equal ? list[o] : list[kMaxTop + o - equal];
      before += other.key > mine.key || (other.key == mine.key && other.index < mine.index);
    }
    if (before < K) best[before] = mine;
  }
  dev::wave_lds_fence();
  return n;
}

// Indices of `best` in ascending order.
__device__ void ascending(const Found* best, int n, uint32_t* index) {
  const int lane = (int)(threadIdx.x & 63u);
  if (lane < n) {
    const uint32_t mine = best[lane].index;
    int before = 0;
    for (int o = 0; o < n; ++o) before += best[o].index < mine;
    index[before] = mine;
  }
  dev::wave_lds_fence();
}

// A wavefront a row: joins the tiles' sums, then descends from the K tiles
// with the best maxima to their K best runs and the K best elements of those
// (any element outside has K better ones before it).
template <typename T>
__global__ __launch_bounds__(64) void finish_kernel(LogprobsPlan p) {
  __shared__ Found list[kListed];
  __shared__ Found best[kMaxTop];
  __shared__ uint32_t lane_keys[64];
  __shared__ uint32_t base[kMaxTop];
  const uint32_t lane = threadIdx.x, row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.row;
  const uint32_t* tile_keys = p.tile_keys + (uint64_t)row * p.tiles;
  const float* tile_sums = p.tile_sums + 2 * (uint64_t)row * p.tiles;
  uint32_t top = 0;
  for (uint32_t t = lane; t < p.tiles; t += 64) top = max(top, tile_keys[t]);
  top = dev::group_max_key<64>(top);
  RowSums r{dev::key_score(top), 0.f, 0.f};
  for (uint32_t t = lane; t < p.tiles; t += 64) {
    const float s = tile_sums[2 * t], u = tile_sums[2 * t + 1];
    if (s == 0.f) continue;
    const float shift = (dev::key_score(tile_keys[t]) - r.m) * kLog2e;
    const float f = __builtin_amdgcn_exp2f(shift);
    r.s = __builtin_fmaf(f, s, r.s);
    if (f != 0.f) r.u = __builtin_fmaf(f, __builtin_fmaf(shift, s, u), r.u);
  }
  r.s = dev::group_sum<64>(r.s);
  r.u = dev::group_sum<64>(r.u);
  if (lane == 0) store_row(p, row, x, r);
  if (p.top == 0) return;
  const float rest = rest_of(r);

  uint32_t key[kMaxTop];
  if (lane < (uint32_t)kMaxTop) base[lane] = lane;
  dev::wave_lds_fence();
  const int items = (int)((p.tiles + 63) / 64);
#pragma unroll
  for (int i = 0; i < (int)kMaxTop; ++i) key[i] = i < items && i * 64 + lane < p.tiles ? tile_keys[i * 64 + lane] : 0u;
  int n = best_of(key, items, base, p.top, list, lane_keys, best);
  ascending(best, n, base);
  const uint32_t* run_keys = p.run_keys + (uint64_t)row * p.tiles * 64;
#pragma unroll
  for (int i = 0; i < (int)kMaxTop; ++i) key[i] = i < n ? run_keys[base[i] * 64 + lane] : 0u;
  n = best_of(key, n, base, p.top, list, lane_keys, best);
  ascending(best, n, base);
#pragma unroll
  for (int i = 0; i < (int)kMaxTop; ++i)
    key[i] = i < n && base[i] * 64 + lane < p.width ? dev::score_key((float)x[base[i] * 64 + lane]) : 0u;
  n = best_of(key, n, base, p.top, list, lane_keys, best);
  if ((int)lane < n) store_alternative(p, row, (int)lane, best[lane].index, dev::key_score(best[lane].key), r.m, rest);
}

uint32_t tiles_of(int64_t width) { return (uint32_t)((width + kTile - 1) / kTile); }

template <typename T, int G, int PER>
thin_status launch_short(const LogprobsPlan& p, hipStream_t stream) {
  const uint32_t rows = 256 / G;
  hipLaunchKernelGGL((short_rows_kernel<T, G, PER>), dim3((p.rows + rows - 1) / rows), dim3(256), 0, stream, p);
  THIN_LAUNCH_CHECK("token_logprobs");
  return THIN_OK;
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" size_t thin_token_logprobs_workspace(int64_t rows, int64_t width, int64_t top) {
  if (rows <= 0 || width <= kShortRow || width > kMaxTiles * (int64_t)kTile) return 0;
  return (size_t)rows * tiles_of(width) * (top > 0 ? 64 + 3 : 3) * 4;
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
  THIN_REQUIRE(V <= kMaxTiles * (int64_t)kTile && R < (1ll << 31) && R * tiles_of(V) < (1ll << 31),
               THIN_ERR_UNSUPPORTED, "token_logprobs: tensor too large");
  THIN_REQUIRE(V == 1 || logits->strides[1] == 1, THIN_ERR_UNSUPPORTED,
               "token_logprobs: the logits of a row must be adjacent");
  if (R == 0) return THIN_OK;
  const thin_desc* outs[4] = {logprobs, entropy, top_logprobs, top_ids};
  for (int i = 0; i < 4; ++i) {
    THIN_REQUIRE(!overlap(outs[i], logits) && !overlap(outs[i], tokens), THIN_ERR_INVALID,
                 "token_logprobs: an output overlaps an input");
    for (int j = 0; j < i; ++j)
      THIN_REQUIRE(!overlap(outs[i], outs[j]), THIN_ERR_INVALID, "token_logprobs: two outputs overlap");
  }
  const size_t need = thin_token_logprobs_workspace(R, V, K);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "token_logprobs needs %zu bytes of workspace, got %zu", need, workspace_bytes);
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
    p.tiles = tiles_of(V);
    p.by_tiles = FastDiv::make(p.tiles);
    const uint64_t waves = (uint64_t)p.rows * p.tiles;
    p.tile_sums = static_cast<float*>(workspace);
    p.tile_keys = reinterpret_cast<uint32_t*>(p.tile_sums + 2 * waves);
    p.run_keys = p.tile_keys + waves;
    hipLaunchKernelGGL((tiles_kernel<T>), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, stream, p);
    THIN_LAUNCH_CHECK("token_logprobs_tiles");
    hipLaunchKernelGGL((finish_kernel<T>), dim3(p.rows), dim3(64), 0, stream, p);
    THIN_LAUNCH_CHECK("token_logprobs_finish");
    return THIN_OK;
  });
}
