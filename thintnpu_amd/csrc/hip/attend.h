// Attention of query rows to keys and values of another length, shared by the
// cross attention (rows of a tensor) and the attention over the 8-bit cache
// (pages of e4m3 codes).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (s_j - m)),  s_j = q . k_j,
//   c = scale log2(e),               m = max_j s_j so far
//
// in one pass over the keys with the running maximum and sum.  A key-value head
// serves `group` query heads: its rows are (token, head of the group).
//
// Matrix layout.  The scores are taken transposed, S^T = K Q^T, 32 keys by 32
// rows: in the 32x32x16 result a lane holds one row (lane & 31) and 16 keys
// 8 (i / 4) + 4 (lane / 32) + i % 4.  So maxima, sums and rescaling are a lane's
// own but for one exchange of the halves, and the lane's exponentials are the B
// operand of O^T = V^T P^T as they stand: the operand wants 8 keys a lane, and
// any order of the keys will do if V^T comes in the same one.  V^T comes from
// row-major LDS by transposing reads (ds_read_b64_tr_b16: 16 lanes take a 4 x 16
// tile, lane i its column i).  The order within the dot products q . k is free
// too: step 2s + e of a half takes dims 32 s + 16 half + 8 e .. + 8, so that 16
// bytes of codes serve two steps.
#pragma once

#include "rows.h"

#include <string.h>

namespace thin {

// Sources of keys and values.
struct RowsOf {  // a tensor [batch, keys, heads, dim]
  const void* data;
  int64_t batch, key, head;  // strides in elements
};
struct PagesOf {  // codes [pages, heads, page, dim], scales [pages, heads]
  const uint8_t* codes;
  const float* scales;
  int64_t page, head, token;       // strides in elements
  int64_t scale_page, scale_head;
};

struct AttendPlan {
  const void* q;
  void* out;
  int64_t q_batch, q_token, q_head;
  int64_t o_batch, o_token, o_head;
  uint32_t batch, tokens, heads, group, rows, dim;  // heads: of the keys; rows = tokens * group
  uint32_t keys;                                    // as many as a sequence can have
  uint32_t row_blocks, splits;
  FastDiv by_group, by_splits, by_blocks, by_heads;
  float c;
  const int32_t* lengths;  // null: `keys`
  const int32_t* counts;   // null: `tokens`
  int64_t length_step, count_step;
  // rows
  RowsOf k, v;
  const uint8_t* mask;  // null: every key
  int64_t mask_batch, mask_key;
  // pages
  PagesOf kp, vp;
  const int32_t* table;
  int64_t table_batch, table_slot;
  uint32_t page_size, pages;
  FastDiv by_page;
  // partial results of splits: [batch, heads, row_blocks, splits, block rows] x {dim, m, l}
  float* sums;
  float* stats;
};

constexpr int kFewRows = 32;    // rows of one matrix tile: keys are split over the wavefronts
constexpr int kBlockRows = 128; // rows of a workgroup otherwise: 32 a wavefront

// Head widths that kernels exist for.
inline int padded_dim(int64_t d) {
  for (int w : {32, 64, 96, 128, 192, 256})
    if (d <= w) return w;
  return 0;
}

// Splits of a row's keys: until there are two workgroups a CU, none under
// kSplitKeys keys (shorter ones cost more to join than they give).
constexpr int64_t kSplitKeys = 256;
constexpr int64_t kWorkgroups = 512;
constexpr int64_t kMaxSplits = 128;
inline int64_t splits_of(int64_t units, int64_t keys) {
  const int64_t most = (keys + kSplitKeys - 1) / kSplitKeys, want = kWorkgroups / (units > 0 ? units : 1);
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n;
}
inline int64_t row_blocks_of(int64_t rows) { return rows <= kFewRows ? 1 : (rows + kBlockRows - 1) / kBlockRows; }
inline size_t attend_workspace(int64_t batch, int64_t heads, int64_t rows, int64_t keys, int64_t dim) {
  if (batch <= 0 || heads <= 0 || rows <= 0 || keys <= 0 || !padded_dim(dim)) return 0;
  const int64_t units = batch * heads * row_blocks_of(rows), splits = splits_of(units, keys);
  if (splits == 1) return 0;
  return (size_t)(units * splits * (rows <= kFewRows ? rows : kBlockRows) * (dim + 2) * 4);
}

// The part of a plan that both operators have.
inline void plan_attend(AttendPlan& p, const thin_desc* q, const thin_desc* out, int64_t heads, int64_t keys, float c,
                        void* workspace) {
  memset(&p, 0, sizeof p);
  p.q = q->data;
  p.out = out->data;
  p.q_batch = q->strides[0]; p.q_token = q->strides[1]; p.q_head = q->strides[2];
  p.o_batch = out->strides[0]; p.o_token = out->strides[1]; p.o_head = out->strides[2];
  p.batch = (uint32_t)q->sizes[0];
  p.tokens = (uint32_t)q->sizes[1];
  p.heads = (uint32_t)heads;
  p.group = (uint32_t)(q->sizes[2] / heads);
  p.rows = p.tokens * p.group;
  p.dim = (uint32_t)q->sizes[3];
  p.keys = (uint32_t)keys;
  p.c = c;
  const int64_t blocks = row_blocks_of(p.rows), units = (int64_t)p.batch * heads * blocks;
  const int64_t splits = splits_of(units, keys), block_rows = p.rows <= kFewRows ? p.rows : kBlockRows;
  p.row_blocks = (uint32_t)blocks;
  p.splits = (uint32_t)splits;
  p.by_group = FastDiv::make(p.group);
  p.by_splits = FastDiv::make(p.splits);
  p.by_blocks = FastDiv::make(p.row_blocks);
  p.by_heads = FastDiv::make(p.heads);
  if (splits > 1) {
    p.sums = static_cast<float*>(workspace);
    p.stats = p.sums + units * splits * block_rows * p.dim;
  }
}

}  // namespace thin

#if defined(__HIPCC__)
namespace thin {
namespace dev {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4e __attribute__((ext_vector_type(4), aligned(1)));  // at element alignment
typedef short s4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Matrix;
template <>
struct Matrix<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static constexpr float kShift = 0.f;
  static __device__ __forceinline__ f16v mul(v8 a, v8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t of_codes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
};
template <>
struct Matrix<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  // exponentials times 2^12 (the sum's too): 2^-26 of the largest is still a normal half
  static constexpr float kShift = 12.f;
  static __device__ __forceinline__ f16v mul(v8 a, v8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t of_codes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
};

// 16 codes as 16 numbers of 16 bits (exact: e4m3 has 3 bits and exponents -9 to 8).
template <typename T>
__device__ __forceinline__ void widen(u4 w, u4& a, u4& b) {
  a = u4{Matrix<T>::template of_codes<false>(w[0]), Matrix<T>::template of_codes<true>(w[0]),
         Matrix<T>::template of_codes<false>(w[1]), Matrix<T>::template of_codes<true>(w[1])};
  b = u4{Matrix<T>::template of_codes<false>(w[2]), Matrix<T>::template of_codes<true>(w[2]),
         Matrix<T>::template of_codes<false>(w[3]), Matrix<T>::template of_codes<true>(w[3])};
}
// Whether a NaN code (0x7F, 0xFF) is among 16.
__device__ __forceinline__ bool has_nan(u4 w) {
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) found |= ((w[i] & 0x7F7F7F7Fu) ^ 0x7F7F7F7Fu) - 0x01010101u;
  return found & 0x80808080u;
}

// Row strides of LDS tiles in elements of 16 bits.  K is read in 16-byte pieces
// of consecutive rows: a stride of an odd number of them meets every bank once.
// V is read in 32-byte pieces of four rows: an odd number of those does.
template <int DP>
struct Strides {
  static constexpr int K = DP + 8;
  static constexpr int V = DP + (DP / 32 % 2 ? 0 : 32);
};

// A sequence's part of the work.
struct Sequence {
  int32_t tokens;  // live query tokens
  int32_t before;  // PAGED: query t sees before + t + 1 keys
  int32_t length;  // keys that exist
};
template <bool PAGED>
__device__ __forceinline__ Sequence sequence_of(const AttendPlan& p, uint32_t b) {
  Sequence s;
  const int32_t n = p.counts ? p.counts[b * p.count_step] : (int32_t)p.tokens;
  s.tokens = max(0, min(n, (int32_t)p.tokens));
  const int32_t len = p.lengths ? p.lengths[b * p.length_step] : (int32_t)p.keys;
  s.before = 0;
  if (PAGED) s.before = max(len, 0) - s.tokens;
  s.length = max(0, min(len, (int32_t)p.keys));
  return s;
}
// Keys that row t sees; rows of no token see what costs no test.
template <bool PAGED>
__device__ __forceinline__ int32_t limit_of(const Sequence& s, int32_t t) {
  return PAGED ? max(0, min(s.length, s.before + t + 1)) : s.length;
}

// A split's keys [begin, end) of n, in steps of `step`.
struct Range {
  int32_t begin, end;
};
__device__ __forceinline__ Range range_of(int32_t n, uint32_t split, uint32_t splits, int32_t step) {
  const int32_t steps = (n + step - 1) / step;
  int32_t per = (steps + (int32_t)splits - 1) / (int32_t)splits;
  per = max(per, (int32_t)kSplitKeys / step);
  const int64_t at = (int64_t)split * per * step;
  Range r;
  r.begin = (int32_t)min(at, (int64_t)n);
  r.end = (int32_t)min(at + (int64_t)per * step, (int64_t)n);
  return r;
}
// The same for whoever joins them: how many have any keys.
__device__ __forceinline__ int32_t active_splits(int32_t n, uint32_t splits, int32_t step) {
  const int32_t steps = (n + step - 1) / step;
  int32_t per = (steps + (int32_t)splits - 1) / (int32_t)splits;
  per = max(per, (int32_t)kSplitKeys / step);
  return (steps + per - 1) / per;
}

// What a lane knows of one key of a tile: PAGED, its page and the page's scales.
struct KeyInfo {
  int32_t id;
  float ks, vs;
  bool seen;
};
template <bool PAGED>
__device__ __forceinline__ KeyInfo key_info(const AttendPlan& p, uint32_t b, uint32_t h, int32_t key, int32_t end) {
  KeyInfo i;
  i.id = 0;
  i.ks = i.vs = 0.f;
  i.seen = key < end;
  if constexpr (PAGED) {
    if (i.seen) {
      i.id = p.table[b * p.table_batch + p.by_page.div((uint32_t)key) * p.table_slot];
      i.seen = (uint32_t)i.id < p.pages;
      if (i.seen) {
        i.ks = p.kp.scales[i.id * p.kp.scale_page + h * p.kp.scale_head];
        i.vs = p.vp.scales[i.id * p.vp.scale_page + h * p.vp.scale_head];
      }
    }
  } else if (p.mask) {
    if (i.seen) i.seen = p.mask[b * p.mask_batch + key * p.mask_key] != 0;
  }
  return i;
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

__device__ __forceinline__ u4 load16(const void* p) { return *reinterpret_cast<const u4e*>(p); }
__device__ __forceinline__ const uint8_t* code_at(const PagesOf& c, int32_t id, uint32_t h, uint32_t token) {
  return c.codes + id * c.page + h * c.head + token * c.token;
}

// A lane's query row as the B operand of its steps; zeros for no row.
template <typename T, int DP>
__device__ __forceinline__ void load_query(const AttendPlan& p, uint32_t b, uint32_t h, uint32_t t, uint32_t g, bool live,
                                           uint32_t half, u4 (&q)[DP / 16]) {
  const T* row = static_cast<const T*>(p.q) + b * p.q_batch + t * p.q_token + (h * p.group + g) * p.q_head;
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    const uint32_t d = (i / 2) * 32 + half * 16 + (i % 2) * 8;
    q[i] = u4{0, 0, 0, 0};
    if (live && d < p.dim) q[i] = load16(row + d);
  }
}

// A lane's running softmax and its row's mix, 32 dims a vector: dim
// 32 i + 8 (j / 4) + 4 half + j % 4 is o[i][j].
template <int DP>
struct State {
  float m, l;  // l: of this half's keys
  f16v o[DP / 32];
  __device__ __forceinline__ State() : m(-__builtin_inff()), l(0.f) {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  }
};

// A row's exponentials are 2^(c s + offset_of(m)).  The offset is rounded, in
// proportion to m; what is taken from one maximum to another goes by the
// difference of the offsets as they are, so that the rounding is common to all.
__device__ __forceinline__ float offset_of(float m, float c, float shift) {
  return shift - (m == -__builtin_inff() ? 0.f : m) * c;
}
__device__ __forceinline__ float rescale_of(float from, float to, float c) {
  if (from == to) return 1.f;
  return from == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(offset_of(to, c, 0.f) - offset_of(from, c, 0.f));
}

// The next 32 * N keys' scores into the running softmax; s becomes the exponentials.
template <typename TV, int DP, int N>
__device__ __forceinline__ void soften(State<DP>& st, f16v (&s)[N], float c) {
  float top = s[0][0];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, s[n][j]);
  top = fmaxf(top, lane_xor<32>(top));
  const float m = fmaxf(st.m, top);
  if (__any(m > st.m)) {
    const float a = rescale_of(st.m, m, c);
    st.l *= a;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) st.o[i][j] *= a;
    st.m = m;
  }
  const float off = offset_of(st.m, c, 0.f) + Matrix<TV>::kShift;
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[n][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j], c, off));
      sum += s[n][j];
    }
  st.l += sum;
}

// Eight exponentials of a lane as the B operand: keys 16 kb + 4 half + {0..3, 8..11}.
template <typename TV>
__device__ __forceinline__ typename Matrix<TV>::v8 pack8(const f16v& s, int kb) {
  typename Matrix<TV>::v8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (TV)s[kb * 8 + j];
  return r;
}
// The same keys of V^T from LDS, for dims 32 i + (lane & 31).
template <typename TV, int STRIDE>
__device__ __forceinline__ typename Matrix<TV>::v8 values8(const TV* v, int row, int i, uint32_t lane) {
  const uint32_t at = (row + (lane >> 5) * 4 + ((lane >> 2) & 3)) * STRIDE + i * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  union {
    s4 part[2];
    typename Matrix<TV>::v8 all;
  } r;
  r.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(v + at));
  r.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(v + at + 8 * STRIDE));
  return r.all;
}

// o += V^T P^T over 32 * N keys of an LDS tile.
template <typename TV, int DP, int N>
__device__ __forceinline__ void mix(State<DP>& st, const f16v (&s)[N], const TV* v, uint32_t lane) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const typename Matrix<TV>::v8 p = pack8<TV>(s[n], kb);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
        st.o[i] = Matrix<TV>::mul(values8<TV, Strides<DP>::V>(v, n * 32 + kb * 16, i, lane), p, st.o[i]);
    }
}
// The same where a value is NaN and not every row sees every key: a key's value
// reaches the rows that see it alone.  One pass for each token of the wavefront,
// its keys' values alone, into its rows alone.
template <typename TV, int DP, int N>
__device__ __forceinline__ void mix_apart(State<DP>& st, const f16v (&s)[N], const TV* v, uint32_t lane, int32_t limit, int32_t k0) {
  int32_t done = -1;
  for (;;) {
    int32_t next = limit > done ? limit : 0x7FFFFFFF;  // the lowest limit not done
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) next = min(next, __shfl_xor(next, o, 64));
    if (next == 0x7FFFFFFF) break;
    done = next;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      f16v part;
#pragma unroll
      for (int j = 0; j < 16; ++j) part[j] = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          typename Matrix<TV>::v8 a = values8<TV, Strides<DP>::V>(v, n * 32 + kb * 16, i, lane);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int32_t key = k0 + n * 32 + kb * 16 + (int32_t)(lane >> 5) * 4 + (j & 3) + (j >> 2) * 8;
            if (key >= next) a[j] = (TV)0.f;
          }
          part = Matrix<TV>::mul(a, pack8<TV>(s[n], kb), part);
        }
      if (limit == next) {
#pragma unroll
        for (int j = 0; j < 16; ++j) st.o[i][j] += part[j];
      }
    }
  }
}

// Scores of unseen keys to -inf: bit k of `bits` is key k of the tile, the row
// sees keys below `limit`.
template <int N>
__device__ __forceinline__ void hide(f16v (&s)[N], uint64_t bits, int32_t k0, int32_t limit, uint32_t half) {
  const uint64_t mine = bits >> (half * 4);
  const int32_t left = limit - k0 - (int32_t)half * 4;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int key = n * 32 + (j / 4) * 8 + j % 4;
      if (!((mine >> key) & 1u) || key >= left) s[n][j] = -__builtin_inff();
    }
}

// PAGED: the scales of 16 keys each on scores and exponentials.
template <int N>
__device__ __forceinline__ void scale16(f16v (&s)[N], const KeyInfo& info, float KeyInfo::*which) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const float f = lane_value(info.*which, n * 32 + kb * 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[n][kb * 8 + j] *= f;
    }
}
// After the scales of the values: infinite ones leave unseen keys at zero.
template <int N>
__device__ __forceinline__ void hide_weights(f16v (&s)[N], uint64_t bits, int32_t k0, int32_t limit, uint32_t half) {
  const uint64_t mine = bits >> (half * 4);
  const int32_t left = limit - k0 - (int32_t)half * 4;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int key = n * 32 + (j / 4) * 8 + j % 4;
      if (!((mine >> key) & 1u) || key >= left) s[n][j] = 0.f;
    }
}

// A row's result: out, or its split's sums.
template <typename T, int DP>
__device__ __forceinline__ void store_row(const AttendPlan& p, uint32_t b, uint32_t h, uint32_t t, uint32_t g, uint64_t slot,
                                          uint32_t half, bool live, const State<DP>& st, float l) {
  if (p.splits == 1) {
    T* row = static_cast<T*>(p.out) + b * p.o_batch + t * p.o_token + (h * p.group + g) * p.o_head;
    const float r = live && l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t d = i * 32 + j * 8 + half * 4;
        if (d < p.dim) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = r == 0.f ? 0.f : st.o[i][j * 4 + k] * r;
          store_pack<T, 4>(row + d, v);
        }
      }
  } else {
    float* row = p.sums + slot * p.dim;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t d = i * 32 + j * 8 + half * 4;
        if (d < p.dim) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = st.o[i][j * 4 + k];
          store_pack<float, 4>(row + d, v);
        }
      }
    if (half == 0) {
      p.stats[slot * 2] = st.m;
      p.stats[slot * 2 + 1] = l;
    }
  }
}

// Where a workgroup works.  Workgroups are dealt to the 8 XCDs in turn; each XCD
// takes a run of neighbours, which read the same keys through its L2.  Row
// blocks go from the last (whose causal rows see the most keys) to the first.
struct Place {
  uint32_t b, h, block, split;
};
__device__ __forceinline__ Place place_of(const AttendPlan& p) {
  const uint32_t nb = gridDim.x, xcd = blockIdx.x & 7u, at = blockIdx.x >> 3;
  uint32_t i = xcd * (nb >> 3) + min(xcd, nb & 7u) + at, r;
  Place w;
  r = p.by_splits.div(i);
  w.split = i - r * p.splits;
  i = p.by_blocks.div(r);
  w.block = p.row_blocks - 1 - (r - i * p.row_blocks);
  w.b = p.by_heads.div(i);
  w.h = i - w.b * p.heads;
  return w;
}

// ---------------------------------------------------------------- many rows
// 128 rows a workgroup, 32 a wavefront; tiles of 64 keys go through registers
// (the next one's loads are in flight while a tile is worked on) to LDS, where
// unseen values become zeros and codes 16-bit numbers.
template <typename T, int DP, bool PAGED>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void tile_kernel(AttendPlan p) {
  typedef typename std::conditional<PAGED, __bf16, T>::type TV;
  constexpr int KT = 64, kPer = PAGED ? DP / 16 : DP / 8;        // pieces of a row
  constexpr int kPieces = KT * kPer, kMine = (kPieces + 255) / 256;
  constexpr int KS = Strides<DP>::K, VS = Strides<DP>::V;
  __shared__ __align__(16) uint16_t lds_k[KT * KS];
  __shared__ __align__(16) uint16_t lds_v[KT * VS];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, half = (tid >> 5) & 1u, wave = tid >> 6;
  const Place w = place_of(p);
  const Sequence seq = sequence_of<PAGED>(p, w.b);
  const uint32_t row = w.block * kBlockRows + wave * 32 + (lane & 31u), t = p.by_group.div(row), g = row - t * p.group;
  const bool mine = row < p.rows, live = mine && (int32_t)t < seq.tokens;
  const int32_t limit = live ? limit_of<PAGED>(seq, (int32_t)t) : 0x7FFFFFFF;
  // the workgroup's first and last live rows
  const int32_t t_first = (int32_t)p.by_group.div(w.block * kBlockRows);
  const int32_t t_last = min((int32_t)p.by_group.div(min(p.rows, (w.block + 1) * kBlockRows) - 1), seq.tokens - 1);
  const int32_t most = t_last < t_first ? 0 : limit_of<PAGED>(seq, t_last);
  const int32_t least = limit_of<PAGED>(seq, t_first);
  // this wavefront's
  const bool idle = !__any(live);
  int32_t wave_least = limit, wave_most = live ? limit : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    wave_least = min(wave_least, __shfl_xor(wave_least, o, 64));
    wave_most = max(wave_most, __shfl_xor(wave_most, o, 64));
  }
  const Range range = range_of(most, w.split, p.splits, KT);

  u4 q[DP / 16];
  load_query<T, DP>(p, w.b, w.h, t, g, live, half, q);
  State<DP> st;

  u4 rk[kMine], rv[kMine];
  KeyInfo next;
  const auto fetch = [&](int32_t k0) {
    next = key_info<PAGED>(p, w.b, w.h, k0 + (int32_t)lane, range.end);
    const uint64_t bits = __ballot(next.seen);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t piece = tid + i * 256, r = piece / kPer, col = piece - r * kPer;
      rk[i] = rv[i] = u4{0, 0, 0, 0};
      if constexpr (PAGED) {
        const int32_t id = __shfl(next.id, (int)(r & 63u), 64);
        if (r < (uint32_t)KT && ((bits >> r) & 1u) && col * 16 < p.dim) {
          const uint32_t key = (uint32_t)k0 + r, at = key - p.by_page.div(key) * p.page_size;
          rk[i] = load16(code_at(p.kp, id, w.h, at) + col * 16);
          rv[i] = load16(code_at(p.vp, id, w.h, at) + col * 16);
        }
      } else {
        if (((bits >> r) & 1u) && col * 8 < p.dim) {
          const int64_t key = k0 + (int32_t)r;
          rk[i] = load16(static_cast<const T*>(p.k.data) + w.b * p.k.batch + key * p.k.key + w.h * p.k.head + col * 8);
          rv[i] = load16(static_cast<const T*>(p.v.data) + w.b * p.v.batch + key * p.v.key + w.h * p.v.head + col * 8);
        }
      }
    }
  };
  if (range.begin < range.end) fetch(range.begin);
  for (int32_t k0 = range.begin; k0 < range.end; k0 += KT) {
    __syncthreads();  // the tile before is read
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t piece = tid + i * 256, r = piece / kPer, col = piece - r * kPer;
      if (kPieces % 256 == 0 || piece < (uint32_t)kPieces) {
        if constexpr (PAGED) {
          u4 a, b;
          widen<T>(rk[i], a, b);
          *reinterpret_cast<u4*>(lds_k + r * KS + col * 16) = a;
          *reinterpret_cast<u4*>(lds_k + r * KS + col * 16 + 8) = b;
          widen<TV>(rv[i], a, b);
          *reinterpret_cast<u4*>(lds_v + r * VS + col * 16) = a;
          *reinterpret_cast<u4*>(lds_v + r * VS + col * 16 + 8) = b;
          nan |= has_nan(rv[i]);
        } else {
          *reinterpret_cast<u4*>(lds_k + r * KS + col * 8) = rk[i];
          *reinterpret_cast<u4*>(lds_v + r * VS + col * 8) = rv[i];
        }
      }
    }
    const KeyInfo info = next;
    const uint64_t bits = __ballot(info.seen);
    bool apart = false;
    if (PAGED && k0 + KT > least) apart = __syncthreads_or(nan);
    else __syncthreads();
    if (k0 + KT < range.end) fetch(k0 + KT);
    if (idle || k0 >= wave_most) continue;

    f16v s[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[n][j] = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const uint32_t d = (i / 2) * 32 + half * 16 + (i % 2) * 8;
        const u4 k = *reinterpret_cast<const u4*>(lds_k + (n * 32 + (lane & 31u)) * KS + d);
        s[n] = Matrix<T>::mul(__builtin_bit_cast(typename Matrix<T>::v8, k), __builtin_bit_cast(typename Matrix<T>::v8, q[i]), s[n]);
      }
    }
    const bool whole = bits == ~0ull && k0 + KT <= wave_least;
    if constexpr (PAGED) scale16<2>(s, info, &KeyInfo::ks);
    if (!whole) hide<2>(s, bits, k0, limit, half);
    soften<TV, DP, 2>(st, s, p.c);
    if constexpr (PAGED) {
      scale16<2>(s, info, &KeyInfo::vs);
      if (!whole) hide_weights<2>(s, bits, k0, limit, half);
    }
    if (PAGED && apart) mix_apart<TV, DP, 2>(st, s, reinterpret_cast<const TV*>(lds_v), lane, limit, k0);
    else mix<TV, DP, 2>(st, s, reinterpret_cast<const TV*>(lds_v), lane);
  }
  const float l = st.l + lane_xor<32>(st.l);
  if (mine && (p.splits == 1 || range.begin < range.end)) {
    const uint64_t unit = ((uint64_t)w.b * p.heads + w.h) * p.row_blocks + w.block;
    store_row<T, DP>(p, w.b, w.h, t, g, (unit * p.splits + w.split) * kBlockRows + (row - w.block * kBlockRows), half, live, st, l);
  }
}

// ---------------------------------------------------------------- few rows
// Up to 32 rows of a head, as a token's or a few drafts' are: four wavefronts
// take tiles of 32 keys in turn, each on its own, and join at the end.  Keys go
// from memory to the operand's registers (a lane's 32 bytes, or 16 codes, are of
// one key), values through the wavefront's own part of LDS.
template <typename T, int DP, bool PAGED>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void few_kernel(AttendPlan p) {
  typedef typename std::conditional<PAGED, __bf16, T>::type TV;
  constexpr int KT = 32, W = 4, kPer = PAGED ? DP / 16 : DP / 8, kMine = KT * kPer / 64;
  constexpr int VS = Strides<DP>::V;
  constexpr int kDims = DP % 64 ? 32 : 64;
  constexpr int kTile = KT * VS * 2, kJoin = 32 * (kDims + 4) * 4;  // bytes of a wavefront's values, of its sums
  __shared__ __align__(16) char lds[W * (kTile > kJoin ? kTile : kJoin)];
  __shared__ float lds_m[W][32], lds_l[W][32], row_m[32], row_l[32];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, half = (tid >> 5) & 1u, wave = tid >> 6, col = lane & 31u;
  const Place w = place_of(p);
  const Sequence seq = sequence_of<PAGED>(p, w.b);
  const uint32_t t = p.by_group.div(col), g = col - t * p.group;
  const bool mine = col < p.rows, live = mine && (int32_t)t < seq.tokens;
  const int32_t limit = live ? limit_of<PAGED>(seq, (int32_t)t) : 0x7FFFFFFF;
  const int32_t most = seq.tokens > 0 ? limit_of<PAGED>(seq, seq.tokens - 1) : 0, least = limit_of<PAGED>(seq, 0);
  const Range range = range_of(most, w.split, p.splits, KT);
  TV* lds_v = reinterpret_cast<TV*>(lds + wave * kTile);

  u4 q[DP / 16];
  load_query<T, DP>(p, w.b, w.h, t, g, live, half, q);
  State<DP> st;

  constexpr int kKeys = PAGED ? DP / 32 : DP / 16;  // 16-byte pieces of a lane's key
  u4 rk[kKeys], rv[kMine];
  KeyInfo next;
  const auto fetch_keys = [&](int32_t k0) {
    const int32_t key = k0 + (int32_t)col;
    next = key_info<PAGED>(p, w.b, w.h, key, range.end);
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      rk[i] = u4{0, 0, 0, 0};
      if constexpr (PAGED) {
        const uint32_t d = i * 32 + half * 16;
        if (next.seen && d < p.dim) {
          const uint32_t at = (uint32_t)key - p.by_page.div((uint32_t)key) * p.page_size;
          rk[i] = load16(code_at(p.kp, next.id, w.h, at) + d);
        }
      } else {
        const uint32_t d = (i / 2) * 32 + half * 16 + (i % 2) * 8;
        if (next.seen && d < p.dim)
          rk[i] = load16(static_cast<const T*>(p.k.data) + w.b * p.k.batch + (int64_t)key * p.k.key + w.h * p.k.head + d);
      }
    }
  };
  const auto fetch_values = [&](int32_t k0) {
    const uint64_t bits = __ballot(next.seen);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t piece = lane + i * 64, r = piece / kPer, c = piece - r * kPer;
      const uint32_t key = (uint32_t)k0 + r;
      rv[i] = u4{0, 0, 0, 0};
      if constexpr (PAGED) {
        const int32_t id = __shfl(next.id, (int)r, 64);
        if (((bits >> r) & 1u) && c * 16 < p.dim) {
          rv[i] = load16(code_at(p.vp, id, w.h, key - p.by_page.div(key) * p.page_size) + c * 16);
        }
      } else {
        if (((bits >> r) & 1u) && c * 8 < p.dim)
          rv[i] = load16(static_cast<const T*>(p.v.data) + w.b * p.v.batch + (int64_t)key * p.v.key + w.h * p.v.head + c * 8);
      }
    }
  };
  int32_t k0 = range.begin + (int32_t)wave * KT;
  if (k0 < range.end) {
    fetch_keys(k0);
    fetch_values(k0);
  }
  for (; k0 < range.end; k0 += W * KT) {
    const KeyInfo info = next;
    const uint64_t bits = __ballot(info.seen);  // the halves alike
    f16v s[1];
#pragma unroll
    for (int j = 0; j < 16; ++j) s[0][j] = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      u4 a, b;
      if constexpr (PAGED) {
        widen<T>(rk[i], a, b);
      } else {
        a = rk[2 * i];
        b = rk[2 * i + 1];
      }
      typedef typename Matrix<T>::v8 v8;
      s[0] = Matrix<T>::mul(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, q[2 * i]), s[0]);
      s[0] = Matrix<T>::mul(__builtin_bit_cast(v8, b), __builtin_bit_cast(v8, q[2 * i + 1]), s[0]);
    }
    bool nan = false;
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t piece = lane + i * 64, r = piece / kPer, c = piece - r * kPer;
      if constexpr (PAGED) {
        u4 a, b;
        widen<TV>(rv[i], a, b);
        *reinterpret_cast<u4*>(lds_v + r * VS + c * 16) = a;
        *reinterpret_cast<u4*>(lds_v + r * VS + c * 16 + 8) = b;
        nan |= has_nan(rv[i]);
      } else {
        *reinterpret_cast<u4*>(lds_v + r * VS + c * 8) = rv[i];
      }
    }
    wave_lds_fence();
    if (k0 + W * KT < range.end) {
      fetch_keys(k0 + W * KT);
      fetch_values(k0 + W * KT);
    }
    const bool whole = bits == ~0ull && k0 + KT <= least;
    if constexpr (PAGED) scale16<1>(s, info, &KeyInfo::ks);
    if (!whole) hide<1>(s, bits, k0, limit, half);
    soften<TV, DP, 1>(st, s, p.c);
    if constexpr (PAGED) {
      scale16<1>(s, info, &KeyInfo::vs);
      if (!whole) hide_weights<1>(s, bits, k0, limit, half);
    }
    if (PAGED && k0 + KT > least && __any(nan)) mix_apart<TV, DP, 1>(st, s, lds_v, lane, limit, k0);
    else mix<TV, DP, 1>(st, s, lds_v, lane);
  }

  // join the wavefronts, kDims dims at a time
  float l = st.l + lane_xor<32>(st.l);
  if (half == 0) {
    lds_m[wave][col] = st.m;
    lds_l[wave][col] = l;
  }
  __syncthreads();
  float m = lds_m[0][col];
#pragma unroll
  for (int i = 1; i < W; ++i) m = fmaxf(m, lds_m[i][col]);
  const float a = rescale_of(st.m, m, p.c);
  l = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) l += lds_l[i][col] * rescale_of(lds_m[i][col], m, p.c);
  if (wave == 0 && half == 0) {
    row_m[col] = m;
    row_l[col] = l;
  }
  float* sums = reinterpret_cast<float*>(lds);
  const uint64_t unit = (uint64_t)w.b * p.heads + w.h;
  const bool empty = range.begin >= range.end;
#pragma unroll
  for (int part = 0; part < DP / kDims; ++part) {
#pragma unroll
    for (int i = 0; i < kDims / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = st.o[part * (kDims / 32) + i][j * 4 + k] * a;
        *reinterpret_cast<f4*>(sums + (wave * 32 + col) * (kDims + 4) + i * 32 + j * 8 + half * 4) = v;
      }
    __syncthreads();
    for (uint32_t at = tid; at < p.rows * (kDims / 4); at += 256) {
      const uint32_t r = at / (kDims / 4), c = (at % (kDims / 4)) * 4, d = part * kDims + c;
      if (d >= p.dim) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const f4 x = *reinterpret_cast<const f4*>(sums + (i * 32 + r) * (kDims + 4) + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += x[k];
      }
      const uint32_t rt = p.by_group.div(r), rg = r - rt * p.group;
      if (p.splits == 1) {
        const float total = row_l[r];
        const bool none = (int32_t)rt >= seq.tokens || total == 0.f;
        const float inv = 1.f / total;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = none ? 0.f : v[k] * inv;
        store_pack<T, 4>(static_cast<T*>(p.out) + w.b * p.o_batch + rt * p.o_token + (w.h * p.group + rg) * p.o_head + d, v);
      } else if (!empty) {
        const uint64_t slot = (unit * p.splits + w.split) * p.rows + r;
        store_pack<float, 4>(p.sums + slot * p.dim + d, v);
        if (d == 0) {
          p.stats[slot * 2] = row_m[r];
          p.stats[slot * 2 + 1] = row_l[r];
        }
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- splits
// One wavefront a row: its splits' sums at their highest maximum, four dims a
// lane (a row's dims past 256 do not exist).
template <typename T, bool PAGED>
__global__ __launch_bounds__(256) void join_kernel(AttendPlan p, uint32_t few) {
  const uint32_t lane = threadIdx.x & 63u, block_rows = few ? p.rows : kBlockRows;
  const uint64_t at = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (b, h, row)
  const uint64_t units = (uint64_t)p.batch * p.heads;
  if (at >= units * p.rows) return;
  const uint32_t unit = (uint32_t)(at / p.rows), row = (uint32_t)(at - (uint64_t)unit * p.rows);
  const uint32_t b = p.by_heads.div(unit), h = unit - b * p.heads;
  const uint32_t t = p.by_group.div(row), g = row - t * p.group;
  const Sequence seq = sequence_of<PAGED>(p, b);
  const uint32_t block = row / block_rows;
  const int32_t t_first = (int32_t)p.by_group.div(block * block_rows);
  const int32_t t_last = min((int32_t)p.by_group.div(min(p.rows, (block + 1) * block_rows) - 1), seq.tokens - 1);
  const int32_t most = t_last < t_first ? 0 : limit_of<PAGED>(seq, t_last);
  const int32_t n = (int32_t)t < seq.tokens ? active_splits(most, p.splits, few ? 32 : 64) : 0;
  const uint64_t first = ((uint64_t)unit * p.row_blocks + block) * p.splits * block_rows + (row - block * block_rows);
  float m = -__builtin_inff();
  for (int32_t i = (int32_t)lane; i < n; i += 64) m = fmaxf(m, p.stats[(first + (uint64_t)i * block_rows) * 2]);
  m = group_max<64>(m);
  float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t d = lane * 4;
  for (int32_t i = 0; i < n; ++i) {
    const uint64_t slot = first + (uint64_t)i * block_rows;
    const float f = rescale_of(p.stats[slot * 2], m, p.c);
    l += p.stats[slot * 2 + 1] * f;
    if (d < p.dim) {
      float x[4];
      load_pack<float, 4>(p.sums + slot * p.dim + d, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[k] * f;
    }
  }
  if (d < p.dim) {
    const float r = 1.f / l;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = n == 0 || l == 0.f ? 0.f : v[k] * r;
    store_pack<T, 4>(static_cast<T*>(p.out) + b * p.o_batch + t * p.o_token + (h * p.group + g) * p.o_head + d, v);
  }
}

}  // namespace dev

// Launches a plan whose operands are checked.
template <typename T, int DP, bool PAGED>
thin_status launch_attend_dim(const AttendPlan& p, hipStream_t stream) {
  const bool few = p.rows <= kFewRows;
  const uint32_t grid = p.batch * p.heads * p.row_blocks * p.splits;
  if (few) hipLaunchKernelGGL((dev::few_kernel<T, DP, PAGED>), dim3(grid), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((dev::tile_kernel<T, DP, PAGED>), dim3(grid), dim3(256), 0, stream, p);
  THIN_LAUNCH_CHECK("attend");
  if (p.splits > 1) {
    const uint64_t rows = (uint64_t)p.batch * p.heads * p.rows;
    hipLaunchKernelGGL((dev::join_kernel<T, PAGED>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, stream, p, few ? 1u : 0u);
    THIN_LAUNCH_CHECK("attend_join");
  }
  return THIN_OK;
}
template <typename T, bool PAGED>
thin_status launch_attend_type(const AttendPlan& p, hipStream_t stream) {
  switch (padded_dim(p.dim)) {
    case 32: return launch_attend_dim<T, 32, PAGED>(p, stream);
    case 64: return launch_attend_dim<T, 64, PAGED>(p, stream);
    case 96: return launch_attend_dim<T, 96, PAGED>(p, stream);
    case 128: return launch_attend_dim<T, 128, PAGED>(p, stream);
    case 192: return launch_attend_dim<T, 192, PAGED>(p, stream);
    default: return launch_attend_dim<T, 256, PAGED>(p, stream);
  }
}

}  // namespace thin
#endif
