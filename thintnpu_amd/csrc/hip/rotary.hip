// Rotary positions with several axes (time, height, width): pair i of a token's
// heads turns by positions[axes[i]] * freqs[i],
//
//   (a, b) -> (a cos - b sin, b cos + a sin)
//
// the pairs of a head being (i, i + P) or (2 i, 2 i + 1), dims from 2 P on copied.
//
// Bound by memory (each element is read and written once).  The angle is taken
// in 64 bits, as far positions need: turns = position * freq / 2 pi, a quarter
// turn at a time, so that 32 bits hold what is left.  A thread computes the
// angles of one piece of pairs of a token and turns that piece of several heads.
#include "rows.h"

#include <string.h>

namespace thin {
namespace {

struct RotaryTensor {
  const void* x;
  void* out;
  int64_t xb, xt, xh, ob, ot, oh;
};
struct RotaryPlan {
  RotaryTensor q, k;
  const void* positions;
  int64_t pa, pb, pt;
  const float* freqs;
  const int32_t* axes;
  int64_t freq_step, axis_step;
  uint32_t wide;  // positions of 64 bits
  uint32_t tokens, heads, all_heads, per_thread, dim, pairs, num_axes;
  uint32_t turn_pieces, pieces;  // of pairs, and with those of copied dims
  uint32_t last_turn, last_copy;  // where pieces begin at most (pair, dim)
  FastDiv by_pieces, by_chunks, by_tokens;
  uint32_t chunks;
  uint64_t threads;
  float sign;
};

// sin and cos of `turns` full turns: the nearest quarter is taken off in 64 bits,
// what is left is within an eighth turn, where the series to x^9 and x^8 is off by
// (pi/4)^11/11! < 2e-9 and (pi/4)^10/10! < 2.5e-8.
__device__ __forceinline__ void sin_cos(double turns, float& s, float& c) {
  turns -= __builtin_rint(turns);
  const double quarters = __builtin_rint(turns * 4.0);
  const float x = (float)(turns * 4.0 - quarters) * 1.57079632679f;
  const int n = (int)quarters;
  const float x2 = x * x;
  const float sx = x * __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, 2.75573192e-6f, -1.98412698e-4f),
                                                                           8.33333333e-3f), -1.66666667e-1f), 1.f);
  const float cx = __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, 2.48015873e-5f, -1.38888889e-3f),
                                                                       4.16666667e-2f), -0.5f), 1.f);
  const float a = n & 1 ? cx : sx, b = n & 1 ? sx : cx;
  s = n & 2 ? -a : a;
  c = (n + 1) & 2 ? -b : b;
}

// n of up to N elements from p on (N when n is); NT: streaming.
template <bool NT, typename T, int N>
__device__ __forceinline__ void load_some(const T* p, uint32_t n, float (&v)[N]) {
  typedef typename dev::Pack<T, N>::type pack;
  if (n >= (uint32_t)N) {
    pack w;
    if constexpr (NT) w = __builtin_nontemporal_load(reinterpret_cast<const pack*>(p));
    else w = *reinterpret_cast<const pack*>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)w[j];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (uint32_t)j < n ? (float)p[j] : 0.f;
  }
}
template <bool NT, typename T, int N>
__device__ __forceinline__ void store_some(T* p, uint32_t n, const float (&v)[N]) {
  typedef typename dev::Pack<T, N>::type pack;
  if (n >= (uint32_t)N) {
    pack w;
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = (T)v[j];
    if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<pack*>(p));
    else *reinterpret_cast<pack*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if ((uint32_t)j < n) p[j] = (T)v[j];
  }
}

// V pairs a piece (halves: V elements from each half; interleaved: 2 V elements).
// Heads go two at a time: their loads are issued before the first is stored (6400
// tokens of 8 x 2 x 16 heads of 64 dims: 85 us, 4.9 TB/s; 92 with one, 88 with four,
// 97 with eight at a time).
constexpr int kHeadsAhead = 2;
// The cosine of copied dims and of pairs of no axis: they stay, whatever they hold (an
// infinity times a sine of 0 is no number).
constexpr float kStays = 2.f;
template <typename T, int V, bool INTERLEAVED, bool NT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryPlan p) {
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.threads) return;
  const uint32_t r = p.by_pieces.div((uint32_t)id), piece = (uint32_t)id - r * p.pieces;
  const uint32_t row = p.by_chunks.div(r), chunk = r - row * p.chunks;  // row: (batch, token)
  const uint32_t b = p.by_tokens.div(row), t = row - b * p.tokens;
  const uint32_t first = chunk * p.per_thread, last = min(first + p.per_thread, p.all_heads);
  const auto head_of = [&](uint32_t h, const T*& x, T*& out) {
    const bool second = h >= p.heads;
    const RotaryTensor& a = second ? p.k : p.q;
    const uint32_t i = second ? h - p.heads : h;
    x = static_cast<const T*>(a.x) + b * a.xb + t * a.xt + i * a.xh;
    out = static_cast<T*>(a.out) + b * a.ob + t * a.ot + i * a.oh;
  };
  // A piece is two runs of V dims (interleaved: one of 2 V): of pairs, or, copied, of
  // the dims behind them.  The last ones begin early enough to be whole, and do some
  // of their neighbours' work too, but for in place.
  const bool turns = piece < p.turn_pieces;
  const uint32_t i0 = min(piece * V, p.last_turn);
  const uint32_t d0 = turns ? INTERLEAVED ? 2 * i0 : i0 : min(2 * p.pairs + (piece - p.turn_pieces) * 2 * V, p.last_copy);
  const uint32_t d1 = turns ? p.pairs + i0 : d0 + V, end = turns ? 2 * p.pairs : p.dim;
  // elements of the runs that there are
  const uint32_t n = INTERLEAVED ? end - d0 : turns ? p.pairs - i0 : end - d0;
  const uint32_t n1 = turns ? n : end > d1 ? end - d1 : 0;
  float s[V], c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s[j] = 0.f;
    c[j] = kStays;
    if (turns && i0 + j < p.pairs) {
      const int32_t axis = p.axes[(i0 + j) * p.axis_step];
      if ((uint32_t)axis < p.num_axes) {
        const int64_t at = axis * p.pa + b * p.pb + t * p.pt;
        const double position = p.wide ? (double)static_cast<const int64_t*>(p.positions)[at]
                                       : (double)static_cast<const int32_t*>(p.positions)[at];
        sin_cos(position * (double)p.freqs[(i0 + j) * p.freq_step] * 0.15915494309189535, s[j], c[j]);
        s[j] *= p.sign;
      }
    }
  }
  for (uint32_t h0 = first; h0 < last; h0 += kHeadsAhead) {
    // u, v: the first and the second of each pair, or (interleaved) the pairs' halves as they lie
    float u[kHeadsAhead][V], v[kHeadsAhead][V];
    const T* x;
    T* out;
#pragma unroll
    for (int k = 0; k < kHeadsAhead; ++k)
      if (h0 + k < last) {
        head_of(h0 + k, x, out);
        if constexpr (INTERLEAVED) {
          float both[2 * V];
          load_some<NT, T, 2 * V>(x + d0, n, both);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            u[k][j] = both[2 * j];
            v[k][j] = both[2 * j + 1];
          }
        } else {
          load_some<NT, T, V>(x + d0, n, u[k]);
          load_some<NT, T, V>(x + d1, n1, v[k]);
        }
      }
#pragma unroll
    for (int k = 0; k < kHeadsAhead; ++k)
      if (h0 + k < last) {
        head_of(h0 + k, x, out);
        float first_of[V], second_of[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool stays = c[j] == kStays;
          first_of[j] = stays ? u[k][j] : u[k][j] * c[j] - v[k][j] * s[j];
          second_of[j] = stays ? v[k][j] : v[k][j] * c[j] + u[k][j] * s[j];
        }
        if constexpr (INTERLEAVED) {
          float both[2 * V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            both[2 * j] = first_of[j];
            both[2 * j + 1] = second_of[j];
          }
          store_some<NT, T, 2 * V>(out + d0, n, both);
        } else {
          store_some<NT, T, V>(out + d0, n, first_of);
          store_some<NT, T, V>(out + d1, n1, second_of);
        }
      }
  }
}

// Threads that fill the card a few times over; past them a thread takes more
// heads with its angles, up to 16 (the same: 125 us with 4, 97 with 8, 87 with 16, 88
// with 32).
constexpr int64_t kEnough = 256 * 2048;
// Adjacent pairs of tensors from this many bytes on are read and written past the
// caches (420 MB: 78 us, 83 through them).  Halves are not: their runs end inside
// lines that the other half needs (336 MB, half of each head turned: 84 us, 101 past
// the caches).
constexpr int64_t kRotaryStreaming = (int64_t)64 << 20;

template <typename T, int V, bool INTERLEAVED>
thin_status launch(RotaryPlan& p, int64_t rows, hipStream_t stream) {
  p.turn_pieces = (p.pairs + V - 1) / V;
  p.pieces = p.turn_pieces + (p.dim - 2 * p.pairs + 2 * V - 1) / (2 * V);
  const uint32_t rest = p.dim - 2 * p.pairs;
  const bool apart = p.q.x != p.q.out && (!p.k.x || p.k.x != p.k.out);
  p.last_turn = apart && p.pairs >= V ? p.pairs - V : ~0u;
  p.last_copy = apart && rest >= 2 * V ? p.dim - 2 * V : ~0u;
  p.per_thread = 1;
  while (p.per_thread < 16 && p.per_thread < p.all_heads && rows * p.pieces * (p.all_heads / (2 * p.per_thread)) >= kEnough)
    p.per_thread *= 2;
  p.chunks = (p.all_heads + p.per_thread - 1) / p.per_thread;
  const int64_t threads = rows * p.chunks * p.pieces;
  THIN_REQUIRE(threads < (1ll << 31), THIN_ERR_UNSUPPORTED, "rotary_axes: tensor too large");
  p.threads = (uint64_t)threads;
  p.by_pieces = FastDiv::make(p.pieces);
  p.by_chunks = FastDiv::make(p.chunks);
  p.by_tokens = FastDiv::make(p.tokens);
  const dim3 grid((uint32_t)((threads + 255) / 256)), block(256);
  if (INTERLEAVED && rows * p.all_heads * p.dim * (int64_t)sizeof(T) >= kRotaryStreaming)
    hipLaunchKernelGGL((rotary_kernel<T, V, INTERLEAVED, INTERLEAVED>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((rotary_kernel<T, V, INTERLEAVED, false>), grid, block, 0, stream, p);
  THIN_LAUNCH_CHECK("rotary_axes");
  return THIN_OK;
}

// Pairs of a piece: as many as 16 bytes hold if they divide the pairs or are a small
// part of them; else fewer (2898 tokens of 29 x 8 heads, 45 pairs as halves: 85 us by
// four, 95 by eight; 27 adjacent: 59 by two, 67 by four).
template <typename T, int V, bool INTERLEAVED>
thin_status launch_pieces(RotaryPlan& p, int64_t rows, hipStream_t stream) {
  if constexpr (V > 1)
    if (p.pairs % V != 0 && p.pairs < 8 * V) return launch_pieces<T, V / 2, INTERLEAVED>(p, rows, stream);
  return launch<T, V, INTERLEAVED>(p, rows, stream);
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" thin_status thin_rotary_axes(const thin_desc* q, const thin_desc* k, const thin_desc* positions,
                                        const thin_desc* freqs, const thin_desc* axes, int32_t interleaved, int32_t inverse,
                                        const thin_desc* q_out, const thin_desc* k_out, hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(q) && desc_valid(positions) && desc_valid(freqs) && desc_valid(axes) && desc_valid(q_out) &&
                   !k == !k_out && (!k || (desc_valid(k) && desc_valid(k_out))),
               THIN_ERR_INVALID, "rotary_axes: invalid descriptor");
  THIN_REQUIRE(q->rank == 4 && float_type(q->dtype) && q_out->dtype == q->dtype && same_sizes(q, q_out), THIN_ERR_INVALID,
               "rotary_axes takes float16, bfloat16 or float32 q [batch, tokens, heads, dim], and out of its type and sizes");
  const int64_t B = q->sizes[0], T = q->sizes[1], H = q->sizes[2], D = q->sizes[3];
  THIN_REQUIRE(!k || (k->rank == 4 && k->dtype == q->dtype && k_out->dtype == q->dtype && same_sizes(k, k_out) &&
                      k->sizes[0] == B && k->sizes[1] == T && k->sizes[3] == D),
               THIN_ERR_INVALID, "rotary_axes: k does not fit q");
  THIN_REQUIRE(positions->rank == 3 && (positions->dtype == THIN_I32 || positions->dtype == THIN_I64) &&
                   positions->sizes[1] == B && positions->sizes[2] == T && positions->sizes[0] >= 1 &&
                   positions->sizes[0] <= 65536,
               THIN_ERR_INVALID, "rotary_axes takes int32 or int64 positions [axes, batch, tokens]");
  THIN_REQUIRE(freqs->rank == 1 && freqs->dtype == THIN_F32 && axes->rank == 1 && axes->dtype == THIN_I32 &&
                   axes->sizes[0] == freqs->sizes[0],
               THIN_ERR_INVALID, "rotary_axes takes float32 freqs and int32 axes [pairs]");
  const int64_t P = freqs->sizes[0];
  THIN_REQUIRE(2 * P <= D, THIN_ERR_INVALID, "rotary_axes: %lld pairs in heads of %lld dims", (long long)P, (long long)D);
  const int64_t all = H + (k ? k->sizes[2] : 0);
  if (B == 0 || T == 0 || all == 0 || D == 0) return THIN_OK;
  THIN_REQUIRE(D < (1ll << 16) && all < (1ll << 24) && T < (1ll << 30) && B < (1ll << 30) && B * T < (1ll << 31),
               THIN_ERR_UNSUPPORTED, "rotary_axes: tensor too large");
  const thin_desc* in[5] = {q, k, positions, freqs, axes};
  const thin_desc* outs[2] = {q_out, k_out};
  for (int i = 0; i < 2; ++i) {
    if (!outs[i]) continue;
    THIN_REQUIRE(in[i]->strides[3] == 1 && outs[i]->strides[3] == 1, THIN_ERR_UNSUPPORTED,
                 "rotary_axes: the dims of a head must be adjacent");
    THIN_REQUIRE(!repeats(outs[i]), THIN_ERR_INVALID, "rotary_axes: an output has a stride of 0");
    for (int j = 0; j < 5; ++j) {
      if (!in[j]) continue;
      const bool in_place = j == i && in[j]->data == outs[i]->data && memcmp(in[j]->strides, outs[i]->strides, 4 * 8) == 0;
      THIN_REQUIRE(in_place || !overlap(outs[i], in[j]), THIN_ERR_INVALID, "rotary_axes: an output overlaps an input");
    }
  }
  THIN_REQUIRE(!k || !overlap(q_out, k_out), THIN_ERR_INVALID, "rotary_axes: two outputs overlap");
  RotaryPlan p;
  memset(&p, 0, sizeof p);
  const auto tensor = [](const thin_desc* x, const thin_desc* o) {
    return RotaryTensor{x->data, o->data, x->strides[0], x->strides[1], x->strides[2], o->strides[0], o->strides[1], o->strides[2]};
  };
  p.q = tensor(q, q_out);
  if (k) p.k = tensor(k, k_out);
  p.positions = positions->data;
  p.pa = positions->strides[0]; p.pb = positions->strides[1]; p.pt = positions->strides[2];
  p.wide = positions->dtype == THIN_I64;
  p.freqs = static_cast<const float*>(freqs->data);
  p.axes = static_cast<const int32_t*>(axes->data);
  p.freq_step = freqs->strides[0];
  p.axis_step = axes->strides[0];
  p.tokens = (uint32_t)T;
  p.heads = (uint32_t)H;
  p.all_heads = (uint32_t)all;
  p.dim = (uint32_t)D;
  p.pairs = (uint32_t)P;
  p.num_axes = (uint32_t)positions->sizes[0];
  p.sign = inverse ? -1.f : 1.f;
  return with_float_type(q->dtype, [&](auto zero) {
    using E = decltype(zero);
    constexpr int V = sizeof(E) == 2 ? 8 : 4;  // 16 bytes
    if (interleaved) return launch_pieces<E, V / 2, true>(p, B * T, stream);
    return launch_pieces<E, V, false>(p, B * T, stream);
  });
}
