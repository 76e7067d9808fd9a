// Rows of scores: element types read as fp32, vectors at element alignment,
// and the order in which scores are ranked (NaN before everything, then from
// the highest down, +0 and -0 equal, the lower index first among equals).
// Shared by the expert routing and the token log probabilities.
#pragma once

#include "common.h"

#include <type_traits>

namespace thin {

// y = f(T()) for the descriptor's floating type.
template <typename F>
thin_status with_float_type(int32_t dtype, F&& f) {
  switch (dtype) {
    case THIN_F16: return f((_Float16)0);
    case THIN_BF16: return f((__bf16)0);
    default: return f(0.0f);
  }
}
inline bool float_type(int32_t dtype) { return dtype == THIN_F16 || dtype == THIN_BF16 || dtype == THIN_F32; }

// Elements [first, last) that a descriptor's sizes and strides reach from its
// data pointer.
inline int64_t extent(const thin_desc* d) {
  int64_t last = 0;
  for (int i = 0; i < d->rank; ++i) {
    if (d->sizes[i] == 0) return 0;
    last += (d->sizes[i] - 1) * d->strides[i];
  }
  return last + 1;
}
// True if the bytes two descriptors reach may have some in common.  Ranges that
// interleave (channel ranges of one wider tensor) have none where, modulo a
// stride that the outer dimensions are multiples of, the inner parts are apart.
inline bool overlap(const thin_desc* a, const thin_desc* b) {
  const int64_t delta = static_cast<const char*>(b->data) - static_cast<const char*>(a->data);
  const int64_t ea = dtype_size(a->dtype), eb = dtype_size(b->dtype), an = extent(a) * ea, bn = extent(b) * eb;
  if (!an || !bn || delta >= an || -delta >= bn) return false;
  for (int i = 0; i < a->rank; ++i) {
    const int64_t period = a->strides[i] * ea;
    if (period <= 0) continue;
    const auto inner = [&](const thin_desc* d, int64_t elem) {
      int64_t bytes = elem;
      for (int k = 0; k < d->rank; ++k)
        if (d->strides[k] * elem % period) bytes += (d->sizes[k] - 1) * d->strides[k] * elem;
      return bytes;
    };
    const int64_t ia = inner(a, ea), ib = inner(b, eb), at = ((delta % period) + period) % period;
    if (at >= ia && at + ib <= period) return false;
  }
  return true;
}
// True if elements of an output share memory by a stride of 0.
inline bool repeats(const thin_desc* d) {
  for (int i = 0; i < d->rank; ++i)
    if (d->sizes[i] > 1 && d->strides[i] == 0) return true;
  return false;
}
// HIP launches below 2^32 threads along a dimension.
inline bool launchable(int64_t blocks, int64_t threads) { return blocks * threads < (1ll << 32); }
// Workspaces hold 32-bit values.
inline bool workspace_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace thin

#if defined(__HIPCC__)
namespace thin {
namespace dev {

// N elements at element alignment: one wide load or store where the hardware
// takes unaligned addresses (global memory does).
template <typename T, int N>
struct Pack {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&v)[N]) {
  const typename Pack<T, N>::type w = *reinterpret_cast<const typename Pack<T, N>::type*>(p);
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = (float)w[j];
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&v)[N]) {
  typename Pack<T, N>::type w;
#pragma unroll
  for (int j = 0; j < N; ++j) w[j] = (T)v[j];
  *reinterpret_cast<typename Pack<T, N>::type*>(p) = w;
}

// Lane g's part of a row of n elements, PER each: the row's [g * PER, (g + 1) *
// PER), loaded from `from` on.  The last part is moved back to end with the row;
// its first `skip` elements are another lane's.  So every lane makes one wide
// load under no condition (200000 rows of 1000 bf16: 97 us, 146 with the ragged
// lane's elements loaded one by one).
// SHORT: the row may have fewer than PER elements.
template <int PER, bool SHORT>
struct Part {
  uint32_t from, skip, count;
  __device__ __forceinline__ Part(uint32_t g, uint32_t n)
      : from(min(g * PER, SHORT && n < PER ? 0u : n - PER)), skip(g * PER - from), count(min(n, (uint32_t)PER)) {}
  __device__ __forceinline__ bool own(int j) const {
    return (uint32_t)j >= skip && (!SHORT || (uint32_t)j < count);
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&v)[PER]) const {
    if (!SHORT || count == PER) {  // the same for all lanes
      load_pack<T, PER>(row + from, v);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = (float)row[min((uint32_t)j, count - 1)];
    }
  }
};

// Whole numbers in the order of the scores; 0 stands below every score.
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
  return x != x ? ~0ull : b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float key_score(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ double key_score(uint64_t k) {
  return __builtin_bit_cast(double, k >> 63 ? k ^ 0x8000000000000000ull : ~k);
}

// A 16-bit score and its index (< 65535) in one number, in the order of the
// scores, the lower index first among equals: no two are equal, and none is 0.
template <typename T>
__device__ __forceinline__ uint32_t place_key(float x, uint32_t index) {
  static_assert(sizeof(T) == 2, "16-bit scores");
  if constexpr (std::is_same<T, _Float16>::value) {
    const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)(x + 0.0f));  // x is a half: exact
    const uint32_t k = x != x ? 0xFFFFu : b ^ (b & 0x8000u ? 0xFFFFu : 0x8000u);
    return k << 16 | (0xFFFFu - index);
  } else {
    return (score_key(x) & 0xFFFF0000u) | (0xFFFFu - index);
  }
}
__device__ __forceinline__ uint32_t place_index(uint32_t k) { return 0xFFFFu - (k & 0xFFFFu); }
template <typename T>
__device__ __forceinline__ float place_score(uint32_t k) {
  const uint32_t b = k & 0x80000000u ? (k >> 16) ^ 0x8000u : ~k >> 16;
  return (float)__builtin_bit_cast(T, (uint16_t)b);
}

template <int O>
__device__ __forceinline__ uint32_t lane_xor_key(uint32_t k) { return lane_xor_bits<O>(k); }
template <int O>
__device__ __forceinline__ uint64_t lane_xor_key(uint64_t k) {
  return (uint64_t)lane_xor_bits<O>((uint32_t)(k >> 32)) << 32 | lane_xor_bits<O>((uint32_t)k);
}
template <int G, int O = G / 2, typename K>
__device__ __forceinline__ K group_max_key(K k) {
  if constexpr (O == 0) {
    return k;
  } else {
    const K other = lane_xor_key<O>(k);
    return group_max_key<G, O / 2>(k > other ? k : other);
  }
}

// Lanes of this lane's group of G whose predicate holds, bit 0 the group's first.
template <int G>
__device__ __forceinline__ uint64_t group_ballot(bool p) {
  const uint64_t all = __ballot(p);
  if constexpr (G == 64) return all;
  return (all >> (threadIdx.x & 63u & ~(uint32_t)(G - 1))) & ((1ull << G) - 1);
}

// Orders the LDS writes of a wavefront before the LDS reads that follow: the
// LDS executes a wave's instructions in order, so only the compiler has to.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The n best of the G * PER keys of a group, lane g holding elements
// g * PER + j, one after another: emit(i, element, key) runs on the lane that
// holds the i-th best.  Keys taken become 0.  Every lane of the group takes part.
template <int G, int PER, typename K, typename Emit>
__device__ __forceinline__ void take_best(K (&key)[PER], int n, uint32_t g, Emit emit) {
  K best = 0;
  int at = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (key[j] > best) {
      best = key[j];
      at = j;
    }
  for (int i = 0; i < n; ++i) {
    const K top = group_max_key<G>(best);
    const uint64_t holders = group_ballot<G>(best == top);
    if (g == (uint32_t)__builtin_ctzll(holders)) {
      emit(i, g * PER + at, top);
      best = 0;
      int next = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (j == at) key[j] = 0;
        if (key[j] > best) {
          best = key[j];
          next = j;
        }
      }
      at = next;
    }
  }
}


// The same for place_key()s: emit(i, key) runs on lane i % G, for G of them at a
// time.  Being unequal, the keys below the last one taken are found by a
// subtraction and a minimum (what is not below wraps), without removing any:
// 40 instructions for the next of 1024 by 64 lanes, take_best() 110.
template <int G, int PER, typename Emit>
__device__ __forceinline__ void take_places(const uint32_t (&key)[PER], int n, uint32_t g, Emit emit) {
  uint32_t best = 0, mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) best = max(best, key[j]);
  for (int i = 0; i < n; ++i) {
    const uint32_t top = group_max_key<G>(best);
    if (g == (uint32_t)i % G) mine = top;
    const uint32_t below = top - 1;
    uint32_t step = below;
#pragma unroll
    for (int j = 0; j < PER; ++j) step = min(step, below - key[j]);
    best = below - step;
    if ((uint32_t)i % G == G - 1 || i == n - 1) {
      const int at = i - (int)((uint32_t)i % G) + (int)g;
      if (at <= i) emit(at, mine);
    }
  }
}

}  // namespace dev
}  // namespace thin
#endif
