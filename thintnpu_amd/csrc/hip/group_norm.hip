// Group norm with an optional SiLU over channels-last rows [N, ..., C] and the
// channel-blocked layout NC1HWC0 [N, C1, H, W, 16]:
//   mean, var over the rows and channels of a group, y = (x - mean) /
//   sqrt(var + eps) * weight + bias, then y * sigmoid(y).
//
// Statistics are fp32.  x has to be read before the first of y is known: either
// a workgroup holds all rows of its groups in registers (one launch, x read
// once), or the moments take a launch of their own and x is read again, from the
// Infinity Cache where it fits.
#include "rows.h"

#include <string.h>

#include <algorithm>
#include <numeric>
#include <type_traits>

namespace thin {
namespace {

constexpr uint32_t kThreads = 256;
// One launch with fewer than kFillingTiles workgroups only where each holds few
// vectors: in the blocked layout, whose tiles are runs of memory, 8192 (frames of
// 128 channels in 32 groups, recorded into a graph: [64,64] 8.4 us against 9.9 in
// two launches, [80,80] 9.9 against 10.0, [100,100] 13.2 against 11.0; a call of
// its own [80,80] 10.8 against 13.9), else 2048 (channels last: [40,40] 7.2 against
// 10.6, [64,64] 9.7 against 10.7, [80,80] 12.2 against 11.2, two of them 17.5
// against 11.6).
constexpr int64_t kFillingTiles = 128;
constexpr int64_t kFewVectors = 2048, kFewBlockedVectors = 8192;
constexpr int64_t kHeldVectors = 16384;  // 16-byte vectors that 1024 threads hold, 16 each
constexpr int64_t kBlocks = 1024;     // workgroups that fill the device

struct NormPlan {
  const void* x;
  void* out;
  const void* weight;
  const void* bias;
  float* partial;                    // workspace: [samples][groups][chunks][2]
  int64_t xn, xb, xh, xw;            // element strides: sample, block of 16 channels, row dims
  int64_t on, ob, oh, ow;
  int64_t ws, bs;                    // of weight and bias
  uint32_t samples, rows, inner;     // rows = outer * inner
  uint32_t channels, padded;         // padded: channels that memory holds (blocked layout)
  uint32_t groups, per_group;
  uint32_t tile_groups, tiles;       // groups a workgroup takes; workgroups across the channels
  uint32_t width;                    // channels of a vector
  uint32_t vectors, lanes, lines;    // vectors of a tile; threads across (lanes) and down (lines)
  uint32_t slots_per_group;
  uint32_t chunks, chunk_rows;
  uint32_t spans;                    // whole runs of 8 samples
  FastDiv by_inner, by_lanes, by_chunks, by_tiles, by_group, by_slots, by_span;
  int32_t blocked, silu, weight32, bias32;
  float eps;
};

// Address of row r, channel c (a vector does not cross a block of 16).
__device__ __forceinline__ int64_t offset_of(const NormPlan& p, int64_t b, int64_t h, int64_t w, uint32_t r,
                                             uint32_t c) {
  const uint32_t q = p.by_inner.div(r);
  const int64_t at = (int64_t)q * h + (int64_t)(r - q * p.inner) * w;
  return p.blocked ? at + (int64_t)(c >> 4) * b + (c & 15u) : at + c;
}

// A vector at c of a row; past the channels of a channels-last row are zeros
// (EDGE: the vector ends behind them.  Kept out of the other rows' loop, where
// the choice made every load wait).
template <typename T, bool EDGE>
__device__ __forceinline__ typename dev::Pack<T, 16 / sizeof(T)>::type load_vector(const NormPlan& p, const T* x, uint32_t c) {
  typedef typename dev::Pack<T, 16 / sizeof(T)>::type P;
  if constexpr (!EDGE) return *reinterpret_cast<const P*>(x);
  P v;
#pragma unroll
  for (int j = 0; j < (int)(16 / sizeof(T)); ++j) v[j] = c + j < p.channels ? x[j] : (T)0.f;
  return v;
}

// Where a workgroup works: its groups hold channels [c0, c1), which it walks in
// vectors from `from` on (a whole vector of the blocked layout).
struct Place {
  uint32_t sample, tile, chunk;
  uint32_t first, count;  // groups
  uint32_t from, c0, c1;
};
__device__ __forceinline__ Place place_of(const NormPlan& p, uint32_t block) {
  Place at;
  const uint32_t q = p.by_chunks.div(block);
  at.chunk = block - q * p.chunks;
  at.sample = p.by_tiles.div(q);
  at.tile = q - at.sample * p.tiles;
  at.first = at.tile * p.tile_groups;
  at.count = min(p.tile_groups, p.groups - at.first);
  at.c0 = at.first * p.per_group;
  at.c1 = at.c0 + at.count * p.per_group;
  at.from = p.blocked ? at.c0 & ~(p.width - 1) : at.c0;
  return at;
}

template <typename T>
__device__ __forceinline__ float param(const void* w, int32_t is32, int64_t at) {
  return is32 ? static_cast<const float*>(w)[at] : (float)static_cast<const T*>(w)[at];
}
template <typename T, bool SILU>
__device__ __forceinline__ float activate(float y) {
  if constexpr (!SILU) return y;
  else return sizeof(T) == 2 ? y * dev::sigmoid_fast(y) : y / (1.0f + expf(-y));
}

// (x - mean) * scale + shift as x * scale + (shift - mean * scale) where that
// loses nothing next to a 16-bit result: the products are below 32, so that
// their rounding stays under 2^-18.
template <typename T>
__device__ __forceinline__ bool folds(float mean, float scale) {
  return sizeof(T) == 2 && fabsf(mean * scale) < 32.f;
}

// One launch, where tiles and channels end at whole vectors: a workgroup holds
// all rows of its groups in registers, H vectors a thread, so that x is read once.
__device__ __forceinline__ void add_lines(float& v, uint32_t lanes) {  // over the lines of a wavefront
  if (lanes <= 32) v += dev::lane_xor<32>(v);
  if (lanes <= 16) v += dev::lane_xor<16>(v);
  if (lanes <= 8) v += dev::lane_xor<8>(v);
  if (lanes <= 4) v += dev::lane_xor<4>(v);
  if (lanes <= 2) v += dev::lane_xor<2>(v);
  if (lanes <= 1) v += dev::lane_xor<1>(v);
}
// Sums of a value a segment over the workgroup's lines and each group's
// segments, into group[].  part: [waves][lanes * SEG].
template <int SEG, int THREADS>
__device__ __forceinline__ void add_up(const NormPlan& p, const Place& at, float (&v)[SEG], float* part, float* group) {
  constexpr uint32_t W = THREADS / 64;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, width = p.lanes * SEG;
#pragma unroll
  for (int s = 0; s < SEG; ++s) {
    add_lines(v[s], p.lanes);
    if (lane < p.lanes) part[wave * width + lane * SEG + s] = v[s];
  }
  __syncthreads();
  const uint32_t entries = W * p.slots_per_group;
  for (uint32_t g0 = 0; g0 < at.count; g0 += THREADS / 16) {
    const uint32_t g = g0 + threadIdx.x / 16;
    float sum = 0.f;
    if (g < at.count)
      for (uint32_t k = threadIdx.x % 16; k < entries; k += 16) {
        const uint32_t w = p.by_slots.div(k);
        sum += part[w * width + g * p.slots_per_group + (k - w * p.slots_per_group)];
      }
    sum = dev::group_sum<16>(sum);
    if (g < at.count && threadIdx.x % 16 == 0) group[g] = sum;
  }
  __syncthreads();
}

// A thread's sums of x - k and its square over n elements of each segment, k
// being the first of them that it reads, so that a mean far from zero cancels
// before the squares are formed.
template <int SEG>
struct Sums {
  float k[SEG], s1[SEG], s2[SEG], n[SEG];
};
// Sums of the workgroup's `count` elements of each group: off[g] = sum of x -
// reference (the group's first element in the workgroup's first row), and
// dev2[g] = sum of squared deviations from the mean that gives.  Each thread's
// mean goes against the reference, then its squares with their distance from
// the mean of all.  Sums alone: joined pair by pair with a division each, this
// took longer than reading the rows (15.6 us for 33 MB).
// lds: part of add_up(), then off, dev2 and the references, one a group each.
struct Reference {
  float first, second;  // of groups threadIdx.x and threadIdx.x + THREADS (a tile has at most 512)
};
template <typename T, int THREADS>
__device__ __forceinline__ Reference reference_of(const NormPlan& p, const Place& at, const T* x, uint32_t r) {
  const auto element = [&](uint32_t g) {
    return g < at.count ? (float)x[offset_of(p, p.xb, p.xh, p.xw, r, at.c0 + g * p.per_group)] : 0.f;
  };
  return {element(threadIdx.x), element(threadIdx.x + THREADS)};
}
struct Joined {
  const float* off;
  const float* dev2;
  const float* reference;
};
template <int SEG, int W, int THREADS>
__device__ __forceinline__ Joined join_threads(const NormPlan& p, const Place& at, const uint32_t (&of)[SEG],
                                               const Reference& reference, float inverse, const Sums<SEG>& t,
                                               float* lds) {
  float* off = lds + THREADS / 64 * p.lanes * SEG;
  float* dev2 = off + p.tile_groups;
  float* against = dev2 + p.tile_groups;
  if (threadIdx.x < at.count) against[threadIdx.x] = reference.first;
  if (threadIdx.x + THREADS < at.count) against[threadIdx.x + THREADS] = reference.second;
  __syncthreads();
  float mean[SEG], m2[SEG], sum[SEG];
#pragma unroll
  for (int s = 0; s < SEG; ++s) {
    const float d = t.n[s] != 0.f ? t.s1[s] * (1.0f / t.n[s]) : 0.f, m = t.s2[s] - t.s1[s] * d;
    mean[s] = t.k[s] - against[of[s]] + d;
    m2[s] = m < 0.f ? 0.f : m;
    sum[s] = t.n[s] != 0.f ? mean[s] * t.n[s] : 0.f;
  }
  add_up<SEG, THREADS>(p, at, sum, lds, off);
#pragma unroll
  for (int s = 0; s < SEG; ++s) {
    const float d = mean[s] - off[of[s]] * inverse;
    sum[s] = t.n[s] != 0.f ? __builtin_fmaf(d * d, t.n[s], m2[s]) : 0.f;
  }
  add_up<SEG, THREADS>(p, at, sum, lds, dev2);
  return {off, dev2, against};
}
// 32 samples of [80,80,128] fp16 in 32 groups with SiLU, 105 MB: 26.5 us (4 TB/s;
// blocked 24.5).  One workgroup of 16 waves fills a CU's registers, so that its
// phases do not overlap: 9.6 us of loads (5.4 TB/s), 2 of joins, 8 of SiLU and
// stores, the rest of ramps.  A single blocked frame: 11.4 us by 16 workgroups, 9.9
// where launches follow each other, each bound by its own CU's loads.
template <typename T, int SEG, int THREADS, int H>
__global__ __launch_bounds__(THREADS) void norm_held_kernel(NormPlan p) {
  constexpr int V = 16 / sizeof(T), W = V / SEG;
  typedef typename dev::Pack<T, V>::type P;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  extern __shared__ float lds[];
  // neighbouring tiles on one XCD, whose L2 then holds the lines they share: each
  // of 8 samples on its own, of fewer samples an eighth each (3 of [40,40,256]
  // 10.5 us without, 7.0 with)
  uint32_t block = blockIdx.x;
  const uint32_t span = 8 * p.tiles, q = p.by_span.div(block);
  if (q < p.spans) {
    const uint32_t r = block - q * span;
    block = q * span + (r & 7u) * p.tiles + (r >> 3);
  } else if (p.tiles % 8 == 0) {
    const uint32_t t = block - p.by_tiles.div(block) * p.tiles;
    block += (t & 7u) * (p.tiles >> 3) + (t >> 3) - t;
  }
  const Place at = place_of(p, block);
  const uint32_t tx = threadIdx.x & (p.lanes - 1), ty = p.by_lanes.div(threadIdx.x);
  const uint32_t c = min(at.c0 + tx * V, at.c1 - V);
  const bool live = tx < p.vectors;
  const T* x = static_cast<const T*>(p.x) + (int64_t)at.sample * p.xn;
  T* out = static_cast<T*>(p.out) + (int64_t)at.sample * p.on;
  // what the ends need first, so that the rows can be added as they arrive
  float scale[V], shift[V];
  const Reference reference = reference_of<T, THREADS>(p, at, x, 0);
  uint32_t of[SEG];  // group of a segment
#pragma unroll
  for (int j = 0; j < V; ++j) {
    scale[j] = p.weight ? param<T>(p.weight, p.weight32, (c + j) * p.ws) : 1.f;
    shift[j] = p.bias ? param<T>(p.bias, p.bias32, (c + j) * p.bs) : 0.f;
  }
#pragma unroll
  for (int s = 0; s < SEG; ++s) of[s] = p.by_group.div(c + s * W) - at.first;
  // as integers, so that no pass keeps the fp32 values of another alive; rows
  // past the last load the last (a load under a condition makes the wait for
  // any of them a wait for all)
  u4 v[H];
  const auto at_hand = [&](int h, int j) { return (float)__builtin_bit_cast(P, v[h])[j]; };
#pragma unroll
  for (int h = 0; h < H; ++h)
    v[h] = __builtin_bit_cast(
        u4, *reinterpret_cast<const P*>(x + offset_of(p, p.xb, 0, p.xw, min(ty + h * p.lines, p.rows - 1), c)));
  Sums<SEG> t = {};
#pragma unroll
  for (int s = 0; s < SEG; ++s) t.k[s] = at_hand(0, s * W);
  uint32_t mine = 0;  // rows of this thread
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if (ty + h * p.lines < p.rows) {
      ++mine;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = at_hand(h, j) - t.k[j / W];
        t.s1[j / W] += d;
        t.s2[j / W] = __builtin_fmaf(d, d, t.s2[j / W]);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < SEG; ++s) t.n[s] = live ? (float)(mine * W) : 0.f;
  const float inverse = 1.0f / (float)(p.rows * p.per_group);
  const Joined joined = join_threads<SEG, W, THREADS>(p, at, of, reference, inverse, t, lds);
  float mean[SEG];
#pragma unroll
  for (int s = 0; s < SEG; ++s) {
    mean[s] = __builtin_fmaf(joined.off[of[s]], inverse, joined.reference[of[s]]);
    const float inv = 1.0f / __builtin_sqrtf(__builtin_fmaf(joined.dev2[of[s]], inverse, p.eps));
#pragma unroll
    for (int j = 0; j < W; ++j) scale[s * W + j] *= inv;
  }
  if (!live) return;
  bool fold = true;
#pragma unroll
  for (int j = 0; j < V; ++j) fold = fold && folds<T>(mean[j / W], scale[j]);
  if (fold) {
#pragma unroll
    for (int j = 0; j < V; ++j) shift[j] = __builtin_fmaf(-mean[j / W], scale[j], shift[j]);
  }
  const auto rows = [&](auto silu, auto folded) {
    T* to = out + offset_of(p, p.ob, 0, p.ow, ty, c);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      __asm__ volatile("" : "+v"(v[h]));
      if (ty + h * p.lines < p.rows) {
        P y;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = decltype(folded)::value ? at_hand(h, j) : at_hand(h, j) - mean[j / W];
          y[j] = (T)activate<T, decltype(silu)::value>(__builtin_fmaf(d, scale[j], shift[j]));
        }
        *reinterpret_cast<P*>(to) = y;
      }
      to += p.lines * p.ow;
    }
  };
  const auto with_silu = [&](auto folded) {
    if (p.silu) rows(std::true_type{}, folded);
    else rows(std::false_type{}, folded);
  };
  if constexpr (sizeof(T) == 2) {
    if (fold) return with_silu(std::true_type{});
  }
  with_silu(std::false_type{});
}

// Two launches: moments of a chunk of rows, then the rows with the moments of
// all chunks joined.  Both are bound by memory and by what comes before a
// workgroup's first load and after its last: 5 samples of [61,83,648] bf16 (half
// the channels of 1296), 33 MB, moments 13.7 us and rows 15.6 us; of 210 MB 46 us
// (4.6 TB/s).
template <typename T, int SEG>
__global__ __launch_bounds__(kThreads) void norm_moments_kernel(NormPlan p) {
  constexpr int V = 16 / sizeof(T), W = V / SEG, U = 4;  // rows at hand; as many are on their way
  typedef typename dev::Pack<T, V>::type P;
  extern __shared__ float lds[];
  const Place at = place_of(p, blockIdx.x);
  const uint32_t begin = at.chunk * p.chunk_rows, end = min(begin + p.chunk_rows, p.rows);
  const uint32_t ty = p.by_lanes.div(threadIdx.x), tx = threadIdx.x & (p.lanes - 1);
  const T* x = static_cast<const T*>(p.x) + (int64_t)at.sample * p.xn;
  const Reference reference = reference_of<T, kThreads>(p, at, x, begin);
  uint32_t of[SEG];  // group of a segment
#pragma unroll
  for (int s = 0; s < SEG; ++s) of[s] = p.by_group.div(min(max(at.from + tx * V + s * W, at.c0), at.c1 - 1)) - at.first;
  Sums<SEG> t = {};
  bool fresh = true;
  // (one turn, or several over the vectors of a single wide group)
  for (uint32_t c = at.from + tx * V; c < at.c1 && begin + ty < end; c += p.lanes * V) {
    const bool whole = c >= at.c0 && c + V <= at.c1;
    uint32_t seen = 0;
    const auto row_loop = [&](auto edge) {
      P ahead[U];
      const auto load = [&](uint32_t r) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          ahead[u] = load_vector<T, decltype(edge)::value>(
              p, x + offset_of(p, p.xb, p.xh, p.xw, min(r + u * p.lines, end - 1), c), c);
      };
      load(begin + ty);
      for (uint32_t r = begin + ty; r < end; r += U * p.lines) {
        P v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = ahead[u];
        if (r + U * p.lines < end) load(r + U * p.lines);
        if (fresh) {
#pragma unroll
          for (int s = 0; s < SEG; ++s) {
            t.k[s] = (float)v[0][s * W];
            // a vector that begins before the group: what stands there is another group's
            if constexpr (decltype(edge)::value) {
#pragma unroll
              for (int j = 1; j < W; ++j)
                if (c + s * W + j <= at.c0) t.k[s] = (float)v[0][s * W + j];
            }
          }
          fresh = false;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r + u * p.lines >= end) continue;
          ++seen;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float d = (float)v[u][j] - t.k[j / W];
            if constexpr (decltype(edge)::value) d = c + j >= at.c0 && c + j < at.c1 ? d : 0.f;
            t.s1[j / W] += d;
            t.s2[j / W] = __builtin_fmaf(d, d, t.s2[j / W]);
          }
        }
      }
    };
    if (whole) row_loop(std::false_type{});
    else row_loop(std::true_type{});
#pragma unroll
    for (int s = 0; s < SEG; ++s) {
      const uint32_t lo = max(c + s * W, at.c0), hi = min(c + s * W + W, at.c1);
      t.n[s] += lo < hi ? (float)(seen * (hi - lo)) : 0.f;
    }
  }
  const float inverse = 1.0f / (float)((end - begin) * p.per_group);
  const Joined joined = join_threads<SEG, W, kThreads>(p, at, of, reference, inverse, t, lds);
  for (uint32_t g = threadIdx.x; g < at.count; g += kThreads) {
    float* o = p.partial + (((uint64_t)at.sample * p.groups + at.first + g) * p.chunks + at.chunk) * 2;
    o[0] = __builtin_fmaf(joined.off[g], inverse, joined.reference[g]);
    o[1] = joined.dev2[g];
  }
}

// Mean and 1 / sqrt(var + eps) of the tile's groups from the chunks' moments:
// the mean from the chunks' means (against the first, so that a common offset
// cancels), then the squares' sum with each chunk's distance from it.
constexpr int kChunkLanes = 16, kHeldChunks = 8;  // lanes of a group, chunks of a lane
__device__ __forceinline__ void join_chunks(const NormPlan& p, const Place& at, float* group) {
  for (uint32_t g0 = 0; g0 < at.count; g0 += kThreads / kChunkLanes) {
    const uint32_t g = min(g0 + threadIdx.x / kChunkLanes, at.count - 1);
    const float* part = p.partial + ((uint64_t)at.sample * p.groups + at.first + g) * p.chunks * 2;
    float mean[kHeldChunks], m2[kHeldChunks], n[kHeldChunks];
#pragma unroll
    for (int i = 0; i < kHeldChunks; ++i) {
      const uint32_t k = threadIdx.x % kChunkLanes + i * kChunkLanes, held = min(k, p.chunks - 1);
      mean[i] = part[2 * held];
      m2[i] = part[2 * held + 1];
      n[i] = k < p.chunks ? (float)(min(p.chunk_rows, p.rows - k * p.chunk_rows) * p.per_group) : 0.f;
    }
    const float first = part[0], total = (float)(p.rows * p.per_group);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kHeldChunks; ++i)
      if (n[i] != 0.f) sum = __builtin_fmaf(mean[i] - first, n[i], sum);
    const float mu = first + dev::group_sum<kChunkLanes>(sum) / total;
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < kHeldChunks; ++i)
      if (n[i] != 0.f) squares += __builtin_fmaf((mean[i] - mu) * (mean[i] - mu), n[i], m2[i]);
    squares = dev::group_sum<kChunkLanes>(squares);
    if (g0 + threadIdx.x / kChunkLanes < at.count && threadIdx.x % kChunkLanes == 0) {
      group[2 * g] = mu;
      group[2 * g + 1] = 1.0f / __builtin_sqrtf(squares / total + p.eps);
    }
  }
  __syncthreads();
}

// NT: streaming stores, where a tile's rows are whole lines of a large output.
// They leave the caches to the next x (moments of 210 MB after such a pass 46
// us, after plain stores 64); in parts of lines they cost more than the whole
// (52 MB in 32-byte parts by the one launch: 71 against 27 us).
template <typename T, bool SILU, bool NT>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(NormPlan p) {
  constexpr int V = 16 / sizeof(T), U = 4;
  extern __shared__ float lds[];
  const Place at = place_of(p, blockIdx.x);
  const uint32_t begin = at.chunk * p.chunk_rows, end = min(begin + p.chunk_rows, p.rows);
  const uint32_t ty = p.by_lanes.div(threadIdx.x), tx = threadIdx.x & (p.lanes - 1);
  const T* x = static_cast<const T*>(p.x) + (int64_t)at.sample * p.xn;
  T* out = static_cast<T*>(p.out) + (int64_t)at.sample * p.on;
  // the last tile of a blocked tensor also writes the padding channels (zeros)
  const uint32_t last = at.c1 == p.channels ? p.padded : at.c1;
  uint32_t c = at.from + tx * V;
  const bool busy = c < last && begin + ty < end;
  typedef typename dev::Pack<T, V>::type P;
  // U rows from r on; the first ones are on their way while the moments are joined
  const auto load = [&](uint32_t r, P (&v)[U], auto edge) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = load_vector<T, decltype(edge)::value>(
          p, x + offset_of(p, p.xb, p.xh, p.xw, min(r + u * p.lines, end - 1), c), c);
  };
  // memory past the channels of a row is not this tensor's, in the blocked layout its padding
  const auto inside = [&]() { return p.blocked || c + V <= p.channels; };
  float scale[V], shift[V];
  const auto params = [&]() {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t ch = min(max(c + j, at.c0), at.c1 - 1);
      scale[j] = p.weight ? param<T>(p.weight, p.weight32, ch * p.ws) : 1.f;
      shift[j] = p.bias ? param<T>(p.bias, p.bias32, ch * p.bs) : 0.f;
    }
  };
  P v[U];
  if (busy) {
    params();
    if (inside()) load(begin + ty, v, std::false_type{});
  }
  join_chunks(p, at, lds);
  if (!busy) return;
  for (; c < last; c += p.lanes * V) {
    if (c != at.from + tx * V) {
      params();
      if (inside()) load(begin + ty, v, std::false_type{});
    }
    if (!inside()) load(begin + ty, v, std::true_type{});
    float mean[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t g = p.by_group.div(min(max(c + j, at.c0), at.c1 - 1)) - at.first;
      mean[j] = lds[2 * g];
      scale[j] *= lds[2 * g + 1];
    }
    bool fold = true;
#pragma unroll
    for (int j = 0; j < V; ++j) fold = fold && folds<T>(mean[j], scale[j]);
    const bool inner = c >= at.c0 && c + V <= at.c1;
    if (fold && inner) {
#pragma unroll
      for (int j = 0; j < V; ++j) shift[j] = __builtin_fmaf(-mean[j], scale[j], shift[j]);
    }
    const auto row_loop = [&](auto folded, auto edge) {
    for (uint32_t r = begin + ty; r < end;) {
      P y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] = v[u];
      const uint32_t now = r;
      r += U * p.lines;
      if (r < end) load(r, v, edge);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t row = now + u * p.lines;
        if (row >= end) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = decltype(folded)::value ? (float)y[u][j] : (float)y[u][j] - mean[j];
          y[u][j] = (T)activate<T, SILU>(__builtin_fmaf(d, scale[j], shift[j]));
        }
        T* to = out + offset_of(p, p.ob, p.oh, p.ow, row, c);
        if constexpr (!decltype(edge)::value) {
          if constexpr (NT) __builtin_nontemporal_store(y[u], reinterpret_cast<P*>(to));
          else *reinterpret_cast<P*>(to) = y[u];
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (c + j >= at.c0 && c + j < last) to[j] = c + j < p.channels ? y[u][j] : (T)0.f;
        }
      }
    }
    };
    if (!inner) row_loop(std::false_type{}, std::true_type{});
    else if (sizeof(T) == 2 && fold) row_loop(std::true_type{}, std::false_type{});
    else row_loop(std::false_type{}, std::false_type{});
  }
}

// How the work is cut, from sizes alone (the workspace's size follows it).
struct Cut {
  uint32_t tile_groups, tiles, vectors, lanes, lines, segments, slots_per_group, chunks, chunk_rows;
  uint32_t threads, held;  // one launch: threads of a workgroup and vectors of a thread; else 0
};
uint32_t power_of_two(uint32_t n) {
  uint32_t p = 1;
  while (p < n) p *= 2;
  return p;
}
// The parts that follow from tg groups a tile.
void cut_tile(Cut& c, int64_t tg, int64_t groups, int64_t per, int64_t V, bool blocked) {
  tg = std::min(tg, groups);
  c.tile_groups = (uint32_t)tg;
  c.tiles = (uint32_t)((groups + tg - 1) / tg);
  c.vectors = (uint32_t)((tg * per + V - 1) / V);
  // channels of a vector that one sum takes: all where they are of one group
  int64_t width = per % V == 0 ? V : V % per == 0 ? per : 1;
  c.slots_per_group = (uint32_t)(per / width);
  if (tg == 1) {
    if (blocked && c.tiles > 1 && per % V) ++c.vectors;  // it may start inside a vector
    width = V;
    c.slots_per_group = c.vectors;
  }
  c.segments = (uint32_t)(V / width);
}
Cut cut_of(int64_t samples, int64_t rows, bool flat, int64_t channels, int64_t groups, int elem, bool blocked) {
  Cut c;
  memset(&c, 0, sizeof c);
  const int64_t V = 16 / elem, per = channels / groups;
  // a tile holds whole groups, where few enough so many that it starts and ends
  // at a whole vector (a whole block of 16), else one
  const int64_t unit = V / std::gcd(per, V), most_channels = 64 * V;  // a wavefront across
  const bool aligned = unit * per <= most_channels;
  // one launch: the widest tile whose rows registers hold, narrower (down to 32
  // bytes) while there are too few of them for the device
  int64_t tg = aligned ? std::min(unit, groups) : 1;
  cut_tile(c, tg, groups, per, V, blocked);
  const auto fits = [&](const Cut& k) {
    const int64_t lanes = power_of_two(k.vectors);
    if (!flat || channels % (blocked ? 16 : V) || k.tile_groups * per % V) return false;
    return lanes <= 32 && lanes * k.segments <= 256 && lanes * rows <= kHeldVectors;
  };
  if (fits(c) && (samples * c.tiles >= kFillingTiles || (int64_t)c.vectors * rows <= (blocked ? kFewBlockedVectors : kFewVectors))) {
    while (aligned) {
      Cut wider = c;
      cut_tile(wider, tg * 2, groups, per, V, blocked);
      if (wider.tiles >= c.tiles || !fits(wider)) break;
      if (samples * wider.tiles < 256 && (c.vectors >= 2 || samples * wider.tiles < kFillingTiles)) break;
      c = wider;
      tg *= 2;
    }
    c.lanes = power_of_two(c.vectors);
    const int64_t vectors = c.lanes * rows;
    c.threads = vectors <= 1024 ? 256 : 1024;
    c.held = vectors <= 4096 ? 4 : vectors <= 8192 ? 8 : 16;
    c.lines = c.threads / c.lanes;
    c.chunks = 1;
    c.chunk_rows = (uint32_t)rows;
    return c;
  }
  // two launches: tiles of at least 256 bytes a row where whole vectors allow
  // (a whole block of 16 in the blocked layout, which is one run of memory)
  const int64_t least = blocked ? 16 : 256 / elem;
  cut_tile(c, aligned ? std::min((least + unit * per - 1) / (unit * per), most_channels / (unit * per)) * unit : 1,
           groups, per, V, blocked);
  c.lanes = std::min<uint32_t>(power_of_two(c.vectors), 64);
  c.lines = kThreads / c.lanes;
  if (c.tile_groups == 1) c.slots_per_group = c.lanes;
  // rows a thread: few while that gives the device enough workgroups, and the
  // second launch not more chunks than it joins
  int64_t each = 2;
  const auto chunks = [&](int64_t m) { return (rows + c.lines * m - 1) / (c.lines * m); };
  while (chunks(each) > kChunkLanes * kHeldChunks || (chunks(each) > 1 && samples * c.tiles * chunks(each) > kBlocks)) each *= 2;
  c.chunk_rows = (uint32_t)std::min<int64_t>(rows, c.lines * each);
  c.chunks = (uint32_t)chunks(each);
  return c;
}

// Samples, rows and the strides between them of x and out jointly.
struct Shape {
  int64_t samples, rows, outer, inner, channels;
  int64_t strides[2][4];  // of x, out: sample, block, outer, inner
  bool ok;
};
Shape shape_of(const thin_desc* x, const thin_desc* out, bool blocked) {
  Shape s;
  memset(&s, 0, sizeof s);
  const int first = blocked ? 2 : 1, last = x->rank - 1;
  thin_desc mid[2];
  const thin_desc* both[2] = {x, out};
  for (int k = 0; k < 2; ++k) {
    mid[k] = *both[k];
    mid[k].rank = last - first;
    for (int d = first; d < last; ++d) {
      mid[k].sizes[d - first] = both[k]->sizes[d];
      mid[k].strides[d - first] = both[k]->strides[d];
    }
    s.strides[k][0] = both[k]->strides[0];
    s.strides[k][1] = blocked ? both[k]->strides[1] : 0;
  }
  const thin_desc* ops[2] = {&mid[0], &mid[1]};
  const Coalesced c = coalesce(ops, 2);
  s.ok = c.nd <= 2;
  if (!s.ok) return s;
  s.samples = x->sizes[0];
  s.inner = c.size[c.nd - 1];
  s.outer = c.nd == 2 ? c.size[0] : 1;
  s.rows = s.inner * s.outer;
  for (int k = 0; k < 2; ++k) {
    s.strides[k][3] = c.stride[k][c.nd - 1];
    s.strides[k][2] = c.nd == 2 ? c.stride[k][0] : 0;
  }
  return s;
}

template <typename T, int SEG>
thin_status launch_norm(const NormPlan& p, const Cut& c, bool streaming, hipStream_t stream) {
  const uint32_t blocks = p.samples * p.tiles * p.chunks;
  if (c.held) {
    const size_t lds = sizeof(float) * (c.threads / 64 * p.lanes * SEG + 3 * p.tile_groups);
    if (c.threads == 256)
      hipLaunchKernelGGL((norm_held_kernel<T, SEG, 256, 4>), dim3(blocks), dim3(256), lds, stream, p);
    else if (c.held == 4)
      hipLaunchKernelGGL((norm_held_kernel<T, SEG, 1024, 4>), dim3(blocks), dim3(1024), lds, stream, p);
    else if (c.held == 8)
      hipLaunchKernelGGL((norm_held_kernel<T, SEG, 1024, 8>), dim3(blocks), dim3(1024), lds, stream, p);
    else
      hipLaunchKernelGGL((norm_held_kernel<T, SEG, 1024, 16>), dim3(blocks), dim3(1024), lds, stream, p);
    THIN_LAUNCH_CHECK("group_norm");
    return THIN_OK;
  }
  const size_t lds = sizeof(float) * (kThreads / 64 * p.lanes * SEG + 3 * p.tile_groups);
  hipLaunchKernelGGL((norm_moments_kernel<T, SEG>), dim3(blocks), dim3(kThreads), lds, stream, p);
  THIN_LAUNCH_CHECK("group_norm_moments");
  const size_t group = sizeof(float) * 2 * p.tile_groups;
  const dim3 grid(blocks), block(kThreads);
  if (p.silu && streaming) hipLaunchKernelGGL((norm_apply_kernel<T, true, true>), grid, block, group, stream, p);
  else if (p.silu) hipLaunchKernelGGL((norm_apply_kernel<T, true, false>), grid, block, group, stream, p);
  else if (streaming) hipLaunchKernelGGL((norm_apply_kernel<T, false, true>), grid, block, group, stream, p);
  else hipLaunchKernelGGL((norm_apply_kernel<T, false, false>), grid, block, group, stream, p);
  THIN_LAUNCH_CHECK("group_norm_apply");
  return THIN_OK;
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" size_t thin_group_norm_workspace(const thin_desc* x, const thin_desc* out, int32_t blocked, int64_t channels,
                                            int64_t groups) {
  if (!desc_valid(x) || !desc_valid(out) || !same_sizes(x, out) || !float_type(x->dtype) || x->rank < (blocked ? 5 : 2) || groups < 1 || channels < groups ||
      channels % groups || numel(x) == 0)
    return 0;
  int64_t rows = 1;
  for (int d = blocked ? 2 : 1; d < x->rank - 1; ++d) rows *= x->sizes[d];
  const bool flat = shape_of(x, out, blocked != 0).outer == 1;
  const Cut c = cut_of(x->sizes[0], rows, flat, channels, groups, dtype_size(x->dtype), blocked != 0);
  return !c.held ? (size_t)x->sizes[0] * groups * c.chunks * 2 * sizeof(float) : 0;
}

extern "C" thin_status thin_group_norm(const thin_desc* x, int32_t blocked, int64_t channels, int64_t groups,
                                       const thin_desc* weight, const thin_desc* bias, double eps, int32_t silu,
                                       const thin_desc* out, void* workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(x) && desc_valid(out) && (!weight || desc_valid(weight)) && (!bias || desc_valid(bias)),
               THIN_ERR_INVALID, "group_norm: invalid descriptor");
  THIN_REQUIRE(float_type(x->dtype) && out->dtype == x->dtype && same_sizes(x, out), THIN_ERR_INVALID,
               "group_norm takes float16, bfloat16 or float32 x and an output of its type and sizes");
  THIN_REQUIRE(blocked ? x->rank == 5 && x->sizes[4] == 16 : x->rank >= 2, THIN_ERR_INVALID,
               "group_norm takes channels-last [N, ..., C] or blocked [N, C1, H, W, 16]");
  THIN_REQUIRE(blocked ? channels >= 1 && (channels + 15) / 16 == x->sizes[1] : channels == x->sizes[x->rank - 1],
               THIN_ERR_INVALID, "group_norm: %lld channels do not fit x", (long long)channels);
  THIN_REQUIRE(groups >= 1 && channels >= 1 && channels % groups == 0, THIN_ERR_INVALID,
               "group_norm: %lld channels do not divide into %lld groups", (long long)channels, (long long)groups);
  THIN_REQUIRE(eps >= 0, THIN_ERR_INVALID, "group_norm: eps must not be negative");
  const thin_desc* params[2] = {weight, bias};
  for (int i = 0; i < 2; ++i)
    THIN_REQUIRE(!params[i] || (params[i]->rank == 1 && params[i]->sizes[0] == channels &&
                                (params[i]->dtype == x->dtype || params[i]->dtype == THIN_F32)),
                 THIN_ERR_INVALID, "group_norm: weight and bias hold one value a channel, of x's type or float32");
  if (numel(x) == 0) return THIN_OK;
  THIN_REQUIRE((x->sizes[x->rank - 1] == 1 || x->strides[x->rank - 1] == 1) &&
                   (out->sizes[out->rank - 1] == 1 || out->strides[out->rank - 1] == 1),
               THIN_ERR_UNSUPPORTED, "group_norm: the channels of a row must be adjacent");
  const Shape s = shape_of(x, out, blocked != 0);
  THIN_REQUIRE(s.ok, THIN_ERR_UNSUPPORTED, "group_norm: the rows of a sample need more than two strides");
  bool same = x->data == out->data;
  for (int d = 0; d < x->rank; ++d) same = same && (x->sizes[d] == 1 || x->strides[d] == out->strides[d]);
  THIN_REQUIRE(!repeats(out), THIN_ERR_INVALID, "group_norm: the output has a stride of 0");
  THIN_REQUIRE(same || !overlap(out, x), THIN_ERR_INVALID, "group_norm: the output overlaps x without being x");
  for (int i = 0; i < 2; ++i)
    THIN_REQUIRE(!params[i] || !overlap(out, params[i]), THIN_ERR_INVALID, "group_norm: the output overlaps a parameter");
  const int elem = dtype_size(x->dtype);
  THIN_REQUIRE(s.rows < (1ll << 31) && channels < (1ll << 31) && s.samples < (1ll << 31) &&
                   s.rows * (channels / groups) < (1ll << 31),
               THIN_ERR_UNSUPPORTED, "group_norm: tensor too large");
  const Cut c = cut_of(s.samples, s.rows, s.outer == 1, channels, groups, elem, blocked != 0);
  THIN_REQUIRE(launchable(s.samples * c.tiles * (int64_t)c.chunks, c.held ? c.threads : kThreads), THIN_ERR_UNSUPPORTED,
               "group_norm: tensor too large");
  const size_t need = !c.held ? (size_t)s.samples * groups * c.chunks * 2 * sizeof(float) : 0;
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "group_norm needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  THIN_REQUIRE(need == 0 || workspace_aligned(workspace), THIN_ERR_WORKSPACE,
               "group_norm: the workspace must be 4-byte aligned");
  NormPlan p;
  memset(&p, 0, sizeof p);
  p.x = x->data;
  p.out = out->data;
  p.weight = weight ? weight->data : nullptr;
  p.bias = bias ? bias->data : nullptr;
  p.ws = weight ? weight->strides[0] : 0;
  p.bs = bias ? bias->strides[0] : 0;
  p.weight32 = weight && weight->dtype == THIN_F32;
  p.bias32 = bias && bias->dtype == THIN_F32;
  p.partial = static_cast<float*>(workspace);
  p.xn = s.strides[0][0]; p.xb = s.strides[0][1]; p.xh = s.strides[0][2]; p.xw = s.strides[0][3];
  p.on = s.strides[1][0]; p.ob = s.strides[1][1]; p.oh = s.strides[1][2]; p.ow = s.strides[1][3];
  p.samples = (uint32_t)s.samples;
  p.rows = (uint32_t)s.rows;
  p.inner = (uint32_t)s.inner;
  p.channels = (uint32_t)channels;
  p.padded = blocked ? (uint32_t)(x->sizes[1] * 16) : (uint32_t)channels;
  p.groups = (uint32_t)groups;
  p.per_group = (uint32_t)(channels / groups);
  p.tile_groups = c.tile_groups;
  p.tiles = c.tiles;
  p.width = 16u / (uint32_t)elem;
  p.vectors = c.vectors;
  p.lanes = c.lanes;
  p.lines = c.lines;
  p.slots_per_group = c.slots_per_group;
  p.chunks = c.chunks;
  p.chunk_rows = c.chunk_rows;
  p.by_inner = FastDiv::make(p.inner);
  p.by_lanes = FastDiv::make(p.lanes);
  p.by_chunks = FastDiv::make(p.chunks);
  p.by_tiles = FastDiv::make(p.tiles);
  p.by_group = FastDiv::make(p.per_group);
  p.by_slots = FastDiv::make(p.slots_per_group);
  p.by_span = FastDiv::make(8 * p.tiles);
  p.spans = p.samples / 8;
  p.blocked = blocked ? 1 : 0;
  p.silu = silu ? 1 : 0;
  p.eps = (float)eps;
  const bool streaming = numel(x) * elem >= kStreamingBytes &&
                         (blocked ? p.ow == 16 : c.vectors % 8 == 0 && s.strides[1][3] * elem % 128 == 0);
  return with_float_type(x->dtype, [&](auto zero) {
    using T = decltype(zero);
    switch (c.segments) {
      case 1: return launch_norm<T, 1>(p, c, streaming, stream);
      case 2: return launch_norm<T, 2>(p, c, streaming, stream);
      case 4: return launch_norm<T, 4>(p, c, streaming, stream);
      default:
        if constexpr (sizeof(T) == 2) return launch_norm<T, 8>(p, c, streaming, stream);
        else return THIN_ERR_UNSUPPORTED;
    }
  });
}
