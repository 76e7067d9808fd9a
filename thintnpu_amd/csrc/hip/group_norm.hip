// Group norm with an optional SiLU over channels-last rows [N, ..., C] and the
// channel-blocked layout NC1HWC0 [N, C1, H, W, 16]:
//   mean, var over the rows and channels of a group, y = (x - mean) /
//   sqrt(var + eps) * weight + bias, then y * sigmoid(y).
//
// Statistics are fp32: a thread sums x - K and its square, K being the first
// element that it reads of the group, so that a mean far from zero cancels
// before the squares are formed; partial (count, mean, sum of squared
// deviations) are joined by Chan, Golub and LeVeque's pairwise rule.
#include "rows.h"

#include <string.h>

#include <algorithm>
#include <numeric>

namespace thin {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxSlots = 1536;  // group segments of a tile that LDS holds
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
  FastDiv by_inner, by_lanes, by_chunks, by_tiles, by_group;
  int32_t blocked, silu, weight32, bias32;
  float eps;
};

struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
  if (b.n == 0.f) return a;
  if (a.n == 0.f) return b;
  const float n = a.n + b.n, d = b.mean - a.mean, part = b.n / n;
  return {n, __builtin_fmaf(d, part, a.mean), a.m2 + b.m2 + d * d * a.n * part};
}
template <int G>
__device__ __forceinline__ Moments join_lanes(Moments m) {
#pragma unroll
  for (int o = 1; o < G; o <<= 1)
    m = join(m, Moments{__shfl_xor(m.n, o, 64), __shfl_xor(m.mean, o, 64), __shfl_xor(m.m2, o, 64)});
  return m;
}

// Address of row r, channel c (a vector does not cross a block of 16).
__device__ __forceinline__ int64_t offset_of(const NormPlan& p, int64_t b, int64_t h, int64_t w, uint32_t r,
                                             uint32_t c) {
  const uint32_t q = p.by_inner.div(r);
  const int64_t at = (int64_t)q * h + (int64_t)(r - q * p.inner) * w;
  return p.blocked ? at + (int64_t)(c >> 4) * b + (c & 15u) : at + c;
}

// V channels from c on; those past the last are zero.  Blocked memory holds
// whole blocks, so only channels-last rows end inside a vector.
template <typename T, int V>
__device__ __forceinline__ void load_channels(const NormPlan& p, const T* x, uint32_t c, float (&v)[V]) {
  if (p.blocked || c + V <= p.channels) {
    dev::load_pack<T, V>(x, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = c + j < p.channels ? (float)x[j] : 0.f;
  }
}

// Where a workgroup works: its groups hold channels [c0, c1), which it walks in
// vectors from `from` on (a whole vector of the blocked layout).
struct Place {
  uint32_t sample, tile, chunk;
  uint32_t first, count;  // groups
  uint32_t from, c0, c1;
};
__device__ __forceinline__ Place place_of(const NormPlan& p) {
  Place at;
  const uint32_t q = p.by_chunks.div(blockIdx.x);
  at.chunk = blockIdx.x - q * p.chunks;
  at.sample = p.by_tiles.div(q);
  at.tile = q - at.sample * p.tiles;
  at.first = at.tile * p.tile_groups;
  at.count = min(p.tile_groups, p.groups - at.first);
  at.c0 = at.first * p.per_group;
  at.c1 = at.c0 + at.count * p.per_group;
  at.from = p.blocked ? at.c0 & ~(p.width - 1) : at.c0;
  return at;
}

// Moments of the tile's groups over rows [begin, end), into group[].
template <typename T, int SEG>
__device__ void tile_moments(const NormPlan& p, const Place& at, uint32_t begin, uint32_t end, Moments* lines,
                             Moments* slots, Moments* group) {
  constexpr int V = 16 / sizeof(T), W = V / SEG;  // channels of a vector, of a segment
  constexpr int U = 4;                            // rows in flight
  const uint32_t ty = p.by_lanes.div(threadIdx.x), tx = threadIdx.x - ty * p.lanes;
  const T* x = static_cast<const T*>(p.x) + (int64_t)at.sample * p.xn;
  for (uint32_t v0 = 0; v0 < p.vectors; v0 += p.lanes) {
    const uint32_t vec = v0 + tx, c = at.from + vec * V;
    const bool live = ty < p.lines && vec < p.vectors && c < at.c1;
    Moments m[SEG];
#pragma unroll
    for (int s = 0; s < SEG; ++s) m[s] = {0.f, 0.f, 0.f};
    if (live && begin + ty < end) {
      float k[SEG], s1[SEG] = {}, s2[SEG] = {};
      uint32_t n = 0;
      for (uint32_t r = begin + ty; r < end; r += U * p.lines) {
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t row = min(r + u * p.lines, end - 1);
          load_channels<T, V>(p, x + offset_of(p, p.xb, p.xh, p.xw, row, c), c, v[u]);
        }
        if (n == 0) {
#pragma unroll
          for (int s = 0; s < SEG; ++s) k[s] = v[0][s * W];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r + u * p.lines >= end) continue;
          ++n;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float d = c + j >= at.c0 && c + j < at.c1 ? v[u][j] - k[j / W] : 0.f;
            s1[j / W] += d;
            s2[j / W] = __builtin_fmaf(d, d, s2[j / W]);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < SEG; ++s) {
        const uint32_t lo = max(c + s * W, at.c0), hi = min(c + s * W + W, at.c1);
        if (lo >= hi) continue;
        const float count = (float)(n * (hi - lo)), mean = s1[s] / count;
        const float m2 = s2[s] - s1[s] * mean;
        m[s] = {count, k[s] + mean, m2 < 0.f ? 0.f : m2};
      }
    }
    // down the lines of the workgroup, a tree
    for (uint32_t left = p.lines; left > 1;) {
      const uint32_t half = (left + 1) / 2;
      if (live && ty >= half && ty < left) {
#pragma unroll
        for (int s = 0; s < SEG; ++s) lines[((ty - half) * p.lanes + tx) * SEG + s] = m[s];
      }
      __syncthreads();
      if (live && ty + half < left) {
#pragma unroll
        for (int s = 0; s < SEG; ++s) m[s] = join(m[s], lines[(ty * p.lanes + tx) * SEG + s]);
      }
      __syncthreads();
      left = half;
    }
    if (ty == 0 && vec < p.vectors) {
#pragma unroll
      for (int s = 0; s < SEG; ++s) slots[vec * SEG + s] = m[s];
    }
  }
  __syncthreads();
  // across the segments of a group: 8 lanes each
  for (uint32_t g0 = 0; g0 < at.count; g0 += kThreads / 8) {
    const uint32_t g = g0 + threadIdx.x / 8;
    Moments m = {0.f, 0.f, 0.f};
    if (g < at.count)
      for (uint32_t s = threadIdx.x % 8; s < p.slots_per_group; s += 8) m = join(m, slots[g * p.slots_per_group + s]);
    m = join_lanes<8>(m);
    if (g < at.count && threadIdx.x % 8 == 0) group[g] = m;
  }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ float param(const void* w, int32_t is32, int64_t at) {
  return is32 ? static_cast<const float*>(w)[at] : (float)static_cast<const T*>(w)[at];
}

// y of rows [begin, end) from the group's moments (m2 already 1 / sqrt).
template <typename T>
__device__ void apply_rows(const NormPlan& p, const Place& at, uint32_t begin, uint32_t end, const Moments* group) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const uint32_t ty = p.by_lanes.div(threadIdx.x), tx = threadIdx.x - ty * p.lanes;
  if (ty >= p.lines) return;
  const T* x = static_cast<const T*>(p.x) + (int64_t)at.sample * p.xn;
  T* out = static_cast<T*>(p.out) + (int64_t)at.sample * p.on;
  // the last tile of a blocked tensor also writes the padding channels (zeros)
  const uint32_t last = at.c1 == p.channels ? p.padded : at.c1;
  for (uint32_t c = at.from + tx * V; c < last; c += p.lanes * V) {
    float mean[V], scale[V], shift[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t ch = min(max(c + j, at.c0), at.c1 - 1);
      const Moments g = group[p.by_group.div(ch) - at.first];
      mean[j] = g.mean;
      scale[j] = p.weight ? g.m2 * param<T>(p.weight, p.weight32, ch * p.ws) : g.m2;
      shift[j] = p.bias ? param<T>(p.bias, p.bias32, ch * p.bs) : 0.f;
    }
    for (uint32_t r = begin + ty; r < end; r += U * p.lines) {
      float v[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t row = min(r + u * p.lines, end - 1);
        load_channels<T, V>(p, x + offset_of(p, p.xb, p.xh, p.xw, row, c), c, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t row = r + u * p.lines;
        if (row >= end) continue;
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          y[j] = __builtin_fmaf(v[u][j] - mean[j], scale[j], shift[j]);
          if (p.silu) y[j] = sizeof(T) == 2 ? y[j] * dev::sigmoid_fast(y[j]) : y[j] / (1.0f + expf(-y[j]));
        }
        T* o = out + offset_of(p, p.ob, p.oh, p.ow, row, c);
        if (c >= at.c0 && c + V <= at.c1) {
          dev::store_pack<T, V>(o, y);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (c + j >= at.c0 && c + j < last) o[j] = c + j < p.channels ? (T)y[j] : (T)0.f;
        }
      }
    }
  }
}

__device__ __forceinline__ float inverse_deviation(const NormPlan& p, const Moments& m) {
  return 1.0f / __builtin_sqrtf(m.m2 / m.n + p.eps);
}

// One launch: a workgroup takes all rows of its groups, twice.
template <typename T, int SEG>
__global__ __launch_bounds__(kThreads) void norm_whole_kernel(NormPlan p) {
  extern __shared__ float lds[];
  Moments* lines = reinterpret_cast<Moments*>(lds);
  Moments* slots = lines + kThreads * SEG;
  Moments* group = slots + p.vectors * SEG;
  const Place at = place_of(p);
  tile_moments<T, SEG>(p, at, 0, p.rows, lines, slots, group);
  for (uint32_t g = threadIdx.x; g < at.count; g += kThreads) group[g].m2 = inverse_deviation(p, group[g]);
  __syncthreads();
  apply_rows<T>(p, at, 0, p.rows, group);
}

// Two launches: moments of a chunk of rows, then the rows with the moments of
// all chunks joined.
template <typename T, int SEG>
__global__ __launch_bounds__(kThreads) void norm_moments_kernel(NormPlan p) {
  extern __shared__ float lds[];
  Moments* lines = reinterpret_cast<Moments*>(lds);
  Moments* slots = lines + kThreads * SEG;
  Moments* group = slots + p.vectors * SEG;
  const Place at = place_of(p);
  const uint32_t begin = at.chunk * p.chunk_rows, end = min(begin + p.chunk_rows, p.rows);
  tile_moments<T, SEG>(p, at, begin, end, lines, slots, group);
  for (uint32_t g = threadIdx.x; g < at.count; g += kThreads) {
    float* o = p.partial + (((uint64_t)at.sample * p.groups + at.first + g) * p.chunks + at.chunk) * 2;
    o[0] = group[g].mean;
    o[1] = group[g].m2;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(NormPlan p) {
  extern __shared__ float lds[];
  Moments* group = reinterpret_cast<Moments*>(lds);
  const Place at = place_of(p);
  for (uint32_t g0 = 0; g0 < at.count; g0 += kThreads / 8) {
    const uint32_t g = g0 + threadIdx.x / 8;
    Moments m = {0.f, 0.f, 0.f};
    if (g < at.count) {
      const float* part = p.partial + ((uint64_t)at.sample * p.groups + at.first + g) * p.chunks * 2;
      for (uint32_t k = threadIdx.x % 8; k < p.chunks; k += 8) {
        const uint32_t rows = min(p.chunk_rows, p.rows - k * p.chunk_rows);
        m = join(m, Moments{(float)(rows * p.per_group), part[2 * k], part[2 * k + 1]});
      }
    }
    m = join_lanes<8>(m);
    if (g < at.count && threadIdx.x % 8 == 0) group[g] = {m.n, m.mean, inverse_deviation(p, m)};
  }
  __syncthreads();
  const uint32_t begin = at.chunk * p.chunk_rows;
  apply_rows<T>(p, at, begin, min(begin + p.chunk_rows, p.rows), group);
}

// How the work is cut, from sizes alone (the workspace's size follows it).
struct Cut {
  uint32_t tile_groups, tiles, vectors, lanes, lines, segments, slots_per_group, chunks, chunk_rows;
  bool ok;
};
Cut cut_of(int64_t samples, int64_t rows, int64_t channels, int64_t groups, int elem, bool blocked) {
  Cut c;
  memset(&c, 0, sizeof c);
  const int64_t V = 16 / elem, per = channels / groups;
  // a tile holds whole groups, where few enough so many that it starts and ends
  // at a whole vector (a whole block of 16), else one
  const int64_t whole = blocked ? 16 : V, most_channels = blocked ? 512 : 1024;
  const int64_t unit = whole / std::gcd(per, whole);
  int64_t tg = 1;
  if (unit * per <= most_channels) tg = blocked ? unit : most_channels / (unit * per) * unit;
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
  c.ok = (int64_t)c.vectors * c.segments <= kMaxSlots;
  c.lanes = std::min(c.vectors, kThreads);
  c.lines = kThreads / c.lanes;
  const int64_t blocks = samples * c.tiles;
  const int64_t most = (rows + c.lines * 8 - 1) / (c.lines * 8);
  int64_t chunks = std::max<int64_t>(1, std::min((kBlocks + blocks - 1) / blocks, most));
  c.chunk_rows = (uint32_t)((rows + chunks - 1) / chunks);
  c.chunks = (uint32_t)((rows + c.chunk_rows - 1) / c.chunk_rows);
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
thin_status launch_norm(const NormPlan& p, hipStream_t stream) {
  const uint32_t blocks = p.samples * p.tiles * p.chunks;
  const size_t lds = sizeof(Moments) * ((size_t)kThreads * SEG + p.vectors * SEG + p.tile_groups);
  if (p.chunks == 1) {
    hipLaunchKernelGGL((norm_whole_kernel<T, SEG>), dim3(blocks), dim3(kThreads), lds, stream, p);
    THIN_LAUNCH_CHECK("group_norm");
    return THIN_OK;
  }
  hipLaunchKernelGGL((norm_moments_kernel<T, SEG>), dim3(blocks), dim3(kThreads), lds, stream, p);
  THIN_LAUNCH_CHECK("group_norm_moments");
  hipLaunchKernelGGL((norm_apply_kernel<T>), dim3(blocks), dim3(kThreads), sizeof(Moments) * p.tile_groups, stream, p);
  THIN_LAUNCH_CHECK("group_norm_apply");
  return THIN_OK;
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" size_t thin_group_norm_workspace(const thin_desc* x, int32_t blocked, int64_t channels, int64_t groups) {
  if (!desc_valid(x) || !float_type(x->dtype) || x->rank < (blocked ? 5 : 2) || groups < 1 || channels < groups ||
      channels % groups || numel(x) == 0)
    return 0;
  int64_t rows = 1;
  for (int d = blocked ? 2 : 1; d < x->rank - 1; ++d) rows *= x->sizes[d];
  const Cut c = cut_of(x->sizes[0], rows, channels, groups, dtype_size(x->dtype), blocked != 0);
  return c.ok && c.chunks > 1 ? (size_t)x->sizes[0] * groups * c.chunks * 2 * sizeof(float) : 0;
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
  THIN_REQUIRE(same || !overlap(out, x), THIN_ERR_INVALID, "group_norm: the output overlaps x without being x");
  for (int i = 0; i < 2; ++i)
    THIN_REQUIRE(!params[i] || !overlap(out, params[i]), THIN_ERR_INVALID, "group_norm: the output overlaps a parameter");
  const int elem = dtype_size(x->dtype);
  THIN_REQUIRE(s.rows < (1ll << 31) && channels < (1ll << 31) && s.samples < (1ll << 31) &&
                   s.rows * (channels / groups) < (1ll << 31),
               THIN_ERR_UNSUPPORTED, "group_norm: tensor too large");
  const Cut c = cut_of(s.samples, s.rows, channels, groups, elem, blocked != 0);
  THIN_REQUIRE(c.ok, THIN_ERR_UNSUPPORTED, "group_norm: groups of %lld channels are not supported",
               (long long)(channels / groups));
  THIN_REQUIRE(s.samples * c.tiles * (int64_t)c.chunks < (1ll << 31), THIN_ERR_UNSUPPORTED, "group_norm: tensor too large");
  const size_t need = c.chunks > 1 ? (size_t)s.samples * groups * c.chunks * 2 * sizeof(float) : 0;
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "group_norm needs %zu bytes of workspace, got %zu", need, workspace_bytes);
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
  p.blocked = blocked ? 1 : 0;
  p.silu = silu ? 1 : 0;
  p.eps = (float)eps;
  return with_float_type(x->dtype, [&](auto zero) {
    using T = decltype(zero);
    switch (c.segments) {
      case 1: return launch_norm<T, 1>(p, stream);
      case 2: return launch_norm<T, 2>(p, stream);
      case 4: return launch_norm<T, 4>(p, stream);
      default:
        if constexpr (sizeof(T) == 2) return launch_norm<T, 8>(p, stream);
        else return THIN_ERR_UNSUPPORTED;
    }
  });
}
