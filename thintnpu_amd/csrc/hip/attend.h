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
//
// What is held in fewer bits: the weights alone, rounded once to the operands' type
// as the product with the values takes them (the matrix instructions for operands
// of 32 bits have a sixteenth of the rate).  Scores, maxima, totals, which take the
// unrounded weights, and sums have 32 bits.  Against 64 bits results are off by 1.1
// to 1.4 times what rounding them once to their type takes (2048 rows to 4096 states
// as bf16: 2.3e-3 and 1.7e-3 of them).
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
  uint32_t row_blocks, block_rows;
  uint32_t splits;  // many rows: of each row's keys
  uint32_t chunks;  // few rows: workgroups that the keys of all sequences are dealt to, or 0
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
  // partial results: [batch, heads, row_blocks, splits, block rows] or [chunks, rows] x {dim, m, l}
  float* sums;
  float* stats;
};

constexpr int kBlockRows = 128;  // rows of a workgroup of the kernel for many: 32 a wavefront

// Rows that the kernel for few takes.  Of a tensor, up to one matrix tile of 16: 24
// rows of 16 heads to 2 x 20000 states of 128 dims took 48 us in two tiles, 42 as
// many rows.  Of the cache, up to two: 24 rows of 16 x 8 heads to 4096 tokens took
// 35 us in two, 43 as many.
constexpr int few_rows(bool paged) { return paged ? 32 : 16; }

// Head widths that kernels exist for.
inline int padded_dim(int64_t d) {
  for (int w : {32, 64, 96, 128, 192, 256})
    if (d <= w) return w;
  return 0;
}

// Workgroups that a CU holds, by their registers; DP: padded_dim().
constexpr int few_workgroups(int DP, int rows, bool paged) {
  const int R = rows <= 16 ? 1 : 2;
  return DP * R <= 64 ? 4 : DP <= 128 && DP * R <= 128 ? 3 : DP <= 128 || (paged && R == 1) ? 2 : 1;
}
constexpr int tile_workgroups(int DP) { return DP <= 32 ? 4 : DP <= 64 ? 3 : DP <= 128 ? 2 : 1; }

constexpr int64_t kCus = 256;
constexpr int64_t kSplitKeys = 256;  // keys of a split or chunk at least (128 and 512 measured alike)
constexpr int64_t kMaxSplits = 128;

// Many rows: splits of every row's keys.  In rounds of the workgroups that the card
// holds, each as long as its keys and some 160 more, which beginning and end cost,
// and the join as much as 200.  (1024 rows of 3 x 4 heads over 8000 cached tokens, in
// a graph: 4 splits, 143 us; 2 take 152, 3 take 162.)
inline int64_t splits_of(int64_t units, int64_t keys, int64_t dim) {
  const int64_t most = (keys + kSplitKeys - 1) / kSplitKeys < kMaxSplits ? (keys + kSplitKeys - 1) / kSplitKeys : kMaxSplits;
  const int64_t at_a_time = kCus * tile_workgroups(padded_dim(dim));
  int64_t best = 1, least = 0;
  for (int64_t n = 1; n <= most && (n == 1 || units * n <= 8 * at_a_time); ++n) {
    const int64_t rounds = (units * n + at_a_time - 1) / at_a_time;
    const int64_t cost = rounds * ((keys + n - 1) / n + 160) + (n > 1 ? 200 : 0);
    if (n == 1 || cost < least) {
      best = n;
      least = cost;
    }
  }
  return best;
}

// Few rows: they are bound by memory and their sequences differ in length, so all
// keys of all sequences are dealt out in equal chunks, to as many workgroups as
// this: the card once or more, at least two to a head of a sequence (32 x 8 heads
// over 8192 cached tokens at most: 80 us, 156 by a workgroup each).  0: one
// workgroup to each, without a join, where that fills the card and the longest
// does not run on for long (32 x 16 heads to 1500 states: 45 us, 51 dealt out; 32
// x 8 over 2000 cached tokens 40, 30 dealt out: codes are fewer bytes), or where
// the join costs more than it gives (512 states: 10 us, 14 dealt out).
inline int64_t chunks_for(int64_t units, int64_t rows, int64_t keys, int64_t dim, bool paged) {
  const int64_t at_a_time = kCus * few_workgroups(padded_dim(dim), (int)rows, paged);
  // (sums of keys are taken in 32 bits, in units of 128)
  if (keys <= 512 || (keys <= 2048 && units >= kCus * (paged ? 2 : 1)) || units >= 4 * at_a_time ||
      units * (keys / 128 + 1) >= 1ll << 31)
    return 0;
  const int64_t n = (2 * units + at_a_time - 1) / at_a_time * at_a_time, useful = units * ((keys + kSplitKeys - 1) / kSplitKeys + 1);
  return n < useful ? n : useful;
}
inline int64_t row_blocks_of(int64_t rows, bool paged) { return rows <= few_rows(paged) ? 1 : (rows + kBlockRows - 1) / kBlockRows; }
inline size_t attend_workspace(int64_t batch, int64_t heads, int64_t rows, int64_t keys, int64_t dim, bool paged) {
  if (batch <= 0 || heads <= 0 || rows <= 0 || keys <= 0 || !padded_dim(dim)) return 0;
  const int64_t units = batch * heads * row_blocks_of(rows, paged);
  if (rows <= few_rows(paged)) return (size_t)(chunks_for(units, rows, keys, dim, paged) * rows * (dim + 2) * 4);
  const int64_t splits = splits_of(units, keys, dim);
  return splits == 1 ? 0 : (size_t)(units * splits * kBlockRows * (dim + 2) * 4);
}

// The part of a plan that both operators have.
inline void plan_attend(AttendPlan& p, const thin_desc* q, const thin_desc* out, int64_t heads, int64_t keys, bool paged,
                        float c, void* workspace) {
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
  const int64_t blocks = row_blocks_of(p.rows, paged), units = (int64_t)p.batch * heads * blocks;
  const bool few = p.rows <= few_rows(paged);
  const int64_t chunks = few ? chunks_for(units, p.rows, keys, p.dim, paged) : 0, splits = few ? 1 : splits_of(units, keys, p.dim);
  p.block_rows = few ? p.rows : kBlockRows;
  p.row_blocks = (uint32_t)blocks;
  p.splits = (uint32_t)splits;
  p.chunks = (uint32_t)chunks;
  p.by_group = FastDiv::make(p.group);
  p.by_splits = FastDiv::make(p.splits);
  p.by_blocks = FastDiv::make(p.row_blocks);
  p.by_heads = FastDiv::make(p.heads);
  if (splits > 1 || chunks) {
    p.sums = static_cast<float*>(workspace);
    p.stats = p.sums + (chunks ? chunks : units * splits) * p.block_rows * p.dim;
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
  static constexpr float kShift = 0.f;  // (a bf16 has the exponents of 32 bits)
  static __device__ __forceinline__ f16v mul(v8 a, v8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f4 mul16(v8 a, v8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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
  // exponentials times 2^8 (the sum's too): up to 2^12 with kSlack, and 2^-22 is
  // still a normal half
  static constexpr float kShift = 8.f;
  static __device__ __forceinline__ f16v mul(v8 a, v8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f4 mul16(v8 a, v8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ __forceinline__ uint32_t of_codes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
};

// 8 and 16 codes as numbers of 16 bits (exact: e4m3 has 3 bits and exponents -9 to 8).
template <typename T>
__device__ __forceinline__ u4 widen8(uint32_t lo, uint32_t hi) {
  return u4{Matrix<T>::template of_codes<false>(lo), Matrix<T>::template of_codes<true>(lo),
            Matrix<T>::template of_codes<false>(hi), Matrix<T>::template of_codes<true>(hi)};
}
template <typename T>
__device__ __forceinline__ void widen(u4 w, u4& a, u4& b) {
  a = widen8<T>(w[0], w[1]);
  b = widen8<T>(w[2], w[3]);
}
// Whether a NaN code (0x7F, 0xFF) is among 16.
__device__ __forceinline__ bool has_nan(u4 w) {
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) found |= ((w[i] & 0x7F7F7F7Fu) ^ 0x7F7F7F7Fu) - 0x01010101u;
  return found & 0x80808080u;
}
// Takes the NaN codes out of 16 of a key's values and notes the key at their dims:
// lowest[d] is the first key whose value is NaN there.  They reach the rows that see
// them alone, at the end: a weight of zero is no protection in a matrix product.
__device__ __forceinline__ void take_nan(u4& w, int32_t key, int32_t* lowest) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((w[i] >> (8 * j)) & 0x7Fu) == 0x7Fu) {
        atomicMin(lowest + i * 4 + j, key);
        w[i] &= ~(0xFFu << (8 * j));
      }
}

// Row strides of LDS tiles in elements of 16 bits.  K is read in 16-byte pieces
// of consecutive rows: a stride of an odd number of them meets every bank once.
// V is read in pieces of four rows: 64 bytes each for tiles of 32 rows, 32 bytes
// each for tiles of 16; an odd number of those does.
template <int DP>
struct Strides {
  static constexpr int K = DP + 8;
  static constexpr int V = DP + (DP / 32 % 2 ? 0 : 32);
  static constexpr int V16 = DP + 16;
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

// Sum over the lanes up to this one, by DPP.
__device__ __forceinline__ int32_t lanes_upto(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1, :2, :4, :8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15, :31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// Few rows, dealt out: chunk u of all sequences' is of sequence b, its `index`-th
// of `count`, of `size` keys each; `first` is the sequence's first.  Wavefronts
// find it for themselves, 64 sequences a round.
struct Chunk {
  int32_t size, first, index, count;
  uint32_t b;
  Sequence seq;
};
constexpr int32_t kChunkUnit = 128;  // keys that four wavefronts take at a time
template <bool PAGED>
__device__ __forceinline__ int32_t most_of(const Sequence& s) {
  return s.tokens > 0 ? limit_of<PAGED>(s, s.tokens - 1) : 0;
}
// BY: sequence u's, not chunk u.  False: there is none.
template <bool PAGED, bool BY>
__device__ __forceinline__ bool find_chunk(const AttendPlan& p, uint32_t lane, uint32_t u, Chunk& c) {
  const auto load = [&](uint32_t b) {
    Sequence s{0, 0, 0};
    if (b < p.batch) s = sequence_of<PAGED>(p, b);
    return s;
  };
  const Sequence first = load(lane);
  int32_t total = 0;  // in units
  for (uint32_t b0 = 0; b0 < p.batch; b0 += 64) {
    const int32_t n = most_of<PAGED>(b0 ? load(b0 + lane) : first);
    total += __builtin_amdgcn_readlane(lanes_upto((n + kChunkUnit - 1) / kChunkUnit), 63);
  }
  // Equal chunks.  Each head of a sequence may leave one unfilled, but most leave a
  // part of one: where they are many, the smallest that fit of what a quarter, a half
  // and all would take (32 x 8 heads over 8192 cached tokens at most: 80 us, 86 with
  // all).
  const int64_t units = (int64_t)p.batch * p.heads;
  for (int part = units * 7 > p.chunks ? 4 : 1; part; part >>= 1) {
    const int64_t room = (int64_t)p.chunks - units / part;
    c.size = max((int32_t)(((int64_t)total * p.heads + room - 1) / room) * kChunkUnit, (int32_t)kSplitKeys);
    if (part == 1) break;
    int64_t taken = 0;
    for (uint32_t b0 = 0; b0 < p.batch; b0 += 64) {
      const int32_t n = most_of<PAGED>(b0 ? load(b0 + lane) : first);
      taken += __builtin_amdgcn_readlane(lanes_upto((n + c.size - 1) / c.size), 63);
    }
    if (taken * p.heads <= p.chunks) break;
  }
  int32_t ahead = 0;
  for (uint32_t b0 = 0; b0 < p.batch; b0 += 64) {
    const Sequence s = b0 ? load(b0 + lane) : first;
    const int32_t n = (most_of<PAGED>(s) + c.size - 1) / c.size, upto = ahead + lanes_upto(n);
    const uint64_t found = BY ? (u - b0 < 64 ? 1ull << (u - b0) : 0ull) : __ballot(upto > (int32_t)u);
    if (found) {
      const int at = __builtin_ctzll(found);
      c.b = b0 + at;
      c.count = __builtin_amdgcn_readlane(n, at);
      c.first = __builtin_amdgcn_readlane(upto, at) - c.count;
      c.index = (int32_t)u - c.first;
      c.seq.tokens = __builtin_amdgcn_readlane(s.tokens, at);
      c.seq.before = __builtin_amdgcn_readlane(s.before, at);
      c.seq.length = __builtin_amdgcn_readlane(s.length, at);
      // the sequence's own chunks as equal as units allow
      const int32_t units = (most_of<PAGED>(c.seq) + kChunkUnit - 1) / kChunkUnit;
      if (c.count > 0) c.size = (units + c.count - 1) / c.count * kChunkUnit;
      return true;
    }
    ahead = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// The same address, known to be all lanes': a buffer descriptor that the compiler
// takes for a lane's own costs a loop over the lanes at each load.
__device__ __forceinline__ const uint8_t* scalar(const uint8_t* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ u4 load16(const void* p) { return *reinterpret_cast<const u4e*>(p); }
__device__ __forceinline__ const uint8_t* code_at(const PagesOf& c, int32_t id, uint32_t h, uint32_t token) {
  return c.codes + id * c.page + h * c.head + token * c.token;
}

// The maximum that a row's exponentials stand against is not raised wherever a score
// passes it, so sums are rescaled in few tiles.  Few rows: where one passes it by
// kSlack bits, so that an exponential is 2^kSlack at most.  Many rows: where the sum
// of a lane's 16 exponentials passes most_of_step(), so that no maxima of the step are
// taken but then, and in a row's first (300 rows of 8 x 8 heads to 8400 states: 72
// us; 77 with the step's maxima and kSlack, 101 with a slack of 0).
constexpr float kSlack = 4.f;
// With kShift that is 2^15, which a half holds.  Of pages 2^14: a weight there is an
// exponential times a multiple of its value's scale, which may be next to 2.
constexpr float most_of_step(bool paged) { return paged ? 64.f : 128.f; }

// Maxima are those of c s, rounded.  A row's exponentials are 2^(c s + offset_of(m))
// with the product in full: the maximum's rounding is common to all.
__device__ __forceinline__ float offset_of(float m) { return m == -__builtin_inff() ? 0.f : -m; }
__device__ __forceinline__ float rescale_of(float from, float to) {
  if (from == to) return 1.f;
  return from == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(offset_of(to) - offset_of(from));
}
// The scores' factor where some are -inf: 0 (a page's scale) times that is none.  A
// NaN stays one.
__device__ __forceinline__ float seen_factor(float c) { return c < 1.17549435e-38f ? 1.17549435e-38f : c; }

// V^T from LDS as the A operand, for dims 32 i + (lane & 31) and keys row + 4 half + {0..3, 8..11}.
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

// The values' scales go into the weights, as multiples of the largest that the row
// has seen so far (a power of two; what is summed is scaled along): so the weights
// fit a half, and what a row does not see does not make them small.
// A scale's power of two (of what is smaller, the least normal one) as bits, which
// compare as integers; 0 for 0 and what is not finite.
__device__ __forceinline__ uint32_t power_of(float vs) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, vs);
  return bits - 1u < 0x7F7FFFFFu ? max(bits & 0x7F800000u, 0x00800000u) : 0u;
}
__device__ __forceinline__ float inverse_of(uint32_t power) {  // 2^127's is not normal
  return __builtin_bit_cast(float, !power ? 0u : power == 0x7F000000u ? 0x00400000u : 0x7F000000u - power);
}

// Many rows: the weights take such a multiple f as a summand log2 f of their
// exponents, and the total its share back as 1 / f.  That holds for no f: an
// exponential times a far smaller one is 0, and has no share left to give back.  So
// below 2^-48 (half) and 2^-64 (bf16) the exponents take another multiple, and the
// weights the rest, as they stand in the operand: as halves they are zeros anyway.
// Totals lose less than 2^-62 a key so.  (A factor for each weight, as few rows have
// it, would be 16 more vector instructions a step where those are the bound.)
template <typename T>
struct Share;
template <>
struct Share<_Float16> {
  static constexpr float kLeast = 0x1p-48f;
  static __device__ __forceinline__ float of(float f) { return f < kLeast ? 1.f : f; }
  static __device__ __forceinline__ float rest(float f) { return f < kLeast ? 0.f : 1.f; }
};
template <>
struct Share<__bf16> {
  static constexpr float kLeast = 0x1p-64f;
  static __device__ __forceinline__ float of(float f) { return f < 0x1p-126f ? 1.f : f < kLeast ? f * 0x1p64f : f; }
  static __device__ __forceinline__ float rest(float f) { return f < 0x1p-126f ? 0.f : f < kLeast ? 0x1p-64f : 1.f; }
};

// A row's result: out, or its split's sums.  Dim 32 i + 8 (j / 4) + 4 half + j % 4
// of a row is o[i][j].
template <typename T, int DP>
__device__ __forceinline__ void store_row(const AttendPlan& p, uint32_t b, uint32_t h, uint32_t t, uint32_t g, uint64_t slot,
                                          uint32_t half, bool live, const f16v (&o)[DP / 32], float m, float l) {
  if (p.splits == 1) {
    T* row = static_cast<T*>(p.out) + b * p.o_batch + t * p.o_token + (h * p.group + g) * p.o_head;
    const bool none = !live || l == 0.f;
    const float r = 1.f / l;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t d = i * 32 + j * 8 + half * 4;
        if (d < p.dim) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = none ? 0.f : o[i][j * 4 + k] * r;
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
          for (int k = 0; k < 4; ++k) v[k] = o[i][j * 4 + k];
          store_pack<float, 4>(row + d, v);
        }
      }
    if (half == 0) {
      p.stats[slot * 2] = m;
      p.stats[slot * 2 + 1] = l;
    }
  }
}

// Where a workgroup works.  Workgroups are dealt to the 8 XCDs in turn.  Those of a
// head and split read the same keys: they go to one XCD's L2, and heads and splits
// to the XCDs in turn, so that sequences of unequal length are spread (in runs, an
// XCD with the longest sequence's heads worked on when the others had ended: chunks
// of prompts 310 us, 168 so, in a graph).  What is left of them goes to all XCDs.  Row blocks go
// from the last (whose causal rows see the most keys) to the first.
struct Place {
  uint32_t b, h, block, split;
};
__device__ __forceinline__ Place place_of(const AttendPlan& p) {
  const uint32_t groups = p.batch * p.heads * p.splits, whole = (groups >> 3) * p.row_blocks, xcd = blockIdx.x & 7u, at = blockIdx.x >> 3;
  const bool dealt = at < whole;
  const uint32_t i = dealt ? at : blockIdx.x - whole * 8, n = p.by_blocks.div(i);
  const uint32_t group = dealt ? n * 8 + xcd : (groups & ~7u) + n;
  Place w;
  w.block = p.row_blocks - 1 - (i - n * p.row_blocks);
  const uint32_t unit = p.by_splits.div(group);
  w.split = group - unit * p.splits;
  w.b = p.by_heads.div(unit);
  w.h = unit - w.b * p.heads;
  return w;
}

// ---------------------------------------------------------------- many rows
// 32 rows a wavefront, four wavefronts a workgroup, steps of 32 keys.  A step's
// keys and values go through registers to LDS (unseen ones as zeros, codes as
// 16-bit numbers), four steps each there.  Matrix instructions run beside the
// others if they do not wait for one another, so three steps overlap: the scores
// of step j + 1, the exponentials of step j and the mix of step j - 1, whose
// instructions take turns; the keys of step j + 3 and the values of step j + 1 are
// written meanwhile, and loads of one step more are in flight.  One barrier for two
// steps.  The exponentials do not wait for their step's maximum: they are taken
// against the maximum so far, and again where their sum shows that as too low.
// What bounds it: at 128 dims the matrix instructions and what is issued between
// them (2048 rows of 4 x 32 heads to 4096 states: 570 us, 960 TFLOP/s); at 32 and 64
// dims the softmax, whose 16 exponentials, 55 other vector instructions and, of codes,
// 16 widenings a step stand against 4 and 8 matrix instructions (300 rows of 8 x 8
// heads to 8400 states of 32 dims: 66 us; 1024 rows of 3 x 24 heads over 8000 cached
// tokens of 64: 129 us by itself, 440 TFLOP/s, and the join's 13).
// Rows: unseen states have -inf in the scores from the start (the accumulator's
// first value).  Pages: rows that do not see a whole step are masked afterwards.
template <typename T, int DP, bool PAGED>
__global__ __launch_bounds__(256, tile_workgroups(DP)) void tile_kernel(AttendPlan p) {
  typedef typename Matrix<T>::v8 v8;
  constexpr int KT = 32;
  constexpr int kPer = PAGED ? DP / 16 : DP / 8, kElems = PAGED ? 16 : 8;  // 16-byte pieces of a key, elements of one
  constexpr int kMine = (8 * kPer + 63) / 64;                             // a lane's of the 8 keys that its wavefront stages
  constexpr int KS = Strides<DP>::K, VS = Strides<DP>::V;
  __shared__ __align__(16) T lds_k[4][KT * KS];
  __shared__ __align__(16) T lds_v[4][KT * VS];
  __shared__ __align__(16) float lds_bias[4][PAGED ? 4 : KT];
  __shared__ int32_t lowest[PAGED ? DP : 1];  // keys with NaN values, where rows see different keys
  const uint32_t tid = threadIdx.x, lane = tid & 63u, half = (tid >> 5) & 1u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const Place w = place_of(p);
  const Sequence seq = sequence_of<PAGED>(p, w.b);
  const uint32_t row = w.block * kBlockRows + wave * 32 + (lane & 31u), t = p.by_group.div(row), g = row - t * p.group;
  const bool live = row < p.rows && (int32_t)t < seq.tokens;
  const int32_t limit = live ? limit_of<PAGED>(seq, (int32_t)t) : 0x7FFFFFFF;
  u4 q[DP / 16];  // as the B operand of its steps; zeros for no row
  {
    const T* x = static_cast<const T*>(p.q) + w.b * p.q_batch + t * p.q_token + (w.h * p.group + g) * p.q_head;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const uint32_t d = (i / 2) * 32 + half * 16 + (i % 2) * 8;
      q[i] = u4{0, 0, 0, 0};
      if (live && d < p.dim) q[i] = load16(x + d);
    }
  }
  // the workgroup's first and last live rows
  const int32_t t_first = (int32_t)p.by_group.div(w.block * kBlockRows);
  const int32_t t_last = min((int32_t)p.by_group.div(min(p.rows, (w.block + 1) * kBlockRows) - 1), seq.tokens - 1);
  const int32_t most = t_last < t_first ? 0 : limit_of<PAGED>(seq, t_last);
  const int32_t least = limit_of<PAGED>(seq, t_first);
  int32_t wave_least = limit;  // this wavefront's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) wave_least = min(wave_least, __shfl_xor(wave_least, o, 64));
  wave_least = __builtin_amdgcn_readfirstlane(wave_least);
  const Range range = range_of(most, w.split, p.splits, 64);
  int32_t steps = (range.end - range.begin + KT - 1) / KT;

  f16v o[DP / 32];
  float m = -__builtin_inff(), off = Matrix<T>::kShift, l = 0.f;  // l: of this half's keys
  bool fresh = true;  // some row has seen nothing yet
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  // PAGED: the largest of the values' scales that the row has seen, a power of two's
  // bits, and the last one over that, where the sums still stand in it
  uint32_t ref = 0;
  float moved = 1.f;
  bool moves = false;
  if constexpr (PAGED) {
    for (uint32_t d = tid; d < (uint32_t)DP; d += 256) lowest[d] = 0x7FFFFFFF;
    __syncthreads();  // the first stages note keys there
  }

  // Stage s: keys of step s and values of step s - 2, eight of each by a wavefront
  // (PAGED: of one page).  Loads go by a buffer descriptor of the step, so that a
  // lane's offsets stay what they are; an offset past the descriptor's end is a
  // zero.
  constexpr uint32_t kNowhere = 0x80000000u;
  u4 rk[kMine], rv[kMine];
  uint32_t k_off[kMine], v_off[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const uint32_t n = lane + i * 64, key = n / kPer, col = n - key * kPer;
    const bool have = n < 8u * kPer && col * kElems < p.dim;
    const int64_t k_step = PAGED ? p.kp.token : p.k.key * (int64_t)sizeof(T), v_step = PAGED ? p.vp.token : p.v.key * (int64_t)sizeof(T);
    k_off[i] = have ? key * (uint32_t)k_step + col * 16 : kNowhere;
    v_off[i] = have ? key * (uint32_t)v_step + col * 16 : kNowhere;
  }
  // rows: where the next stage's keys and values of the wavefront begin
  const int64_t k_move = p.k.key * (int64_t)(KT * sizeof(T)), v_move = p.v.key * (int64_t)(KT * sizeof(T));
  const uint8_t* k_at = static_cast<const uint8_t*>(p.k.data) +
                        (w.b * p.k.batch + w.h * p.k.head + (range.begin + (int32_t)wave * 8) * p.k.key) * (int64_t)sizeof(T);
  const uint8_t* v_at = static_cast<const uint8_t*>(p.v.data) +
                        (w.b * p.v.batch + w.h * p.v.head + (range.begin + (int32_t)wave * 8 - 2 * KT) * p.v.key) * (int64_t)sizeof(T);
  uint32_t bits_k = 0, bits_1 = 0, bits_v = 0;  // rows: the seen keys of steps s, s - 1 and s - 2
  uint32_t shown = 0;                           // rows: key lane % 32 of the next step
  uint32_t any_shown = 0;                       // rows: of all so far
  // PAGED: lane i knows group i % 2 of 16 keys of step i / 2 of a window of 32
  // steps; the next window's are looked up when one begins.
  struct Window {
    int32_t id;
    float c, vs;  // c: of the scores as the codes give them
  };
  const auto look_up_window = [&](int32_t first) {
    Window x{-1, 0.f, 0.f};
    const int32_t k = range.begin + (first + (int32_t)(lane >> 1)) * KT + (int32_t)(lane & 1u) * 16;
    if (k < range.end) {
      x.id = p.table[w.b * p.table_batch + p.by_page.div((uint32_t)k) * p.table_slot];
      if ((uint32_t)x.id >= p.pages) {
        x.id = -1;
      } else {
        x.c = p.c * p.kp.scales[x.id * p.kp.scale_page + w.h * p.kp.scale_head];
        x.vs = p.vp.scales[x.id * p.vp.scale_page + w.h * p.vp.scale_head];
      }
    }
    return x;
  };
  Window here{-1, 0.f, 0.f}, there{-1, 0.f, 0.f};
  float here_share = 0.f, here_back = 0.f;
  uint64_t here_tiny = 0;  // groups whose multiple is not in the exponents as a whole
  int32_t here_first = 0;  // the step that `here` begins with
  // The values' scales go into the weights as multiples of the largest up to the
  // window's end, of groups that all rows see part of: of these, what the exponents
  // and the totals take.  Groups behind them are some rows' only (the last two steps
  // at most that the wavefront's rows see): each row takes those as they come.
  const auto enter_window = [&](int32_t first) {
    here = there;
    here_first = first;
    uint32_t top = range.begin + (first + (int32_t)(lane >> 1)) * KT + (int32_t)(lane & 1u) * 16 < wave_least ? power_of(here.vs) : 0u;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, x, 64));
    top = (uint32_t)__builtin_amdgcn_readfirstlane((int)top);
    if (__any(top > ref)) {  // (all rows' is the same then)
      moved = __builtin_bit_cast(float, ref) * inverse_of(top);
      moves = true;
      ref = top;
    }
    const float f = here.vs * inverse_of(ref);
    here_share = __builtin_amdgcn_logf(Share<T>::of(f));
    here_back = __builtin_amdgcn_rcpf(Share<T>::of(f));
    here_tiny = __ballot(f < Share<T>::kLeast);
  };
  int32_t id_k = -1, id_1 = -1, id_v = -1;  // the pages of the wavefront's keys of steps s, s - 1 and s - 2
  // their places there; a step is two groups further, and pages are whole groups
  uint32_t at_k = 0, at_1 = 0, at_v = 0;
  if constexpr (PAGED) {
    at_k = (uint32_t)range.begin + wave * 8;
    at_k -= p.by_page.div(at_k) * p.page_size;
  }
  const uint8_t* k_codes = p.kp.codes + w.h * p.kp.head;
  const uint8_t* v_codes = p.vp.codes + w.h * p.vp.head;
  const auto look_up = [&](int32_t step) {
    if constexpr (!PAGED) {
      const int32_t k = range.begin + step * KT + (int32_t)(lane & 31u);
      shown = k < range.end;
      if (shown && p.mask) shown = p.mask[w.b * p.mask_batch + k * p.mask_key];
    }
  };
  const auto fetch = [&](int32_t stage) {
    if constexpr (PAGED) {
      id_v = id_1;
      id_1 = id_k;
      const int32_t at = stage - here_first;
      id_k = __builtin_amdgcn_readlane(at < 32 ? here.id : there.id, (at & 31) * 2 + (int32_t)(wave >> 1));
      const auto rsrc_of = [&](const uint8_t* codes, const PagesOf& x, int32_t id, uint32_t token) {
        return buffer_rsrc(scalar(codes + id * x.page + token * x.token), id >= 0 ? kNowhere : 0u);
      };
      const auto kr = rsrc_of(k_codes, p.kp, id_k, at_k), vr = rsrc_of(v_codes, p.vp, id_v, at_v);
      at_v = at_1;
      at_1 = at_k;
      at_k += p.page_size == 16 ? 0 : 32;
      if (at_k >= p.page_size) at_k -= p.page_size;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        rk[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_off[i], 0, 0));
        rv[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vr, v_off[i], 0, 0));
      }
    } else {
      bits_v = bits_1;
      bits_1 = bits_k;
      bits_k = (uint32_t)__ballot(shown != 0);
      any_shown |= bits_k;
      const uint32_t mine_k = (bits_k >> (wave * 8)) & 0xFFu, mine_v = (bits_v >> (wave * 8)) & 0xFFu;
      const auto kr = buffer_rsrc(k_at, kNowhere), vr = buffer_rsrc(v_at, kNowhere);
      k_at += k_move;
      v_at += v_move;
      if (mine_k == 0xFFu && mine_v == 0xFFu) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          rk[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_off[i], 0, 0));
          rv[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vr, v_off[i], 0, 0));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const uint32_t key = (lane + i * 64) / kPer;
          rk[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kr, (mine_k >> key) & 1u ? k_off[i] : kNowhere, 0, 0));
          rv[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vr, (mine_v >> key) & 1u ? v_off[i] : kNowhere, 0, 0));
        }
      }
    }
    look_up(stage + 1);
  };
  const auto store = [&](int32_t stage) {
    T* kt = lds_k[stage & 3] + wave * 8 * KS;
    T* vt = lds_v[(stage + 2) & 3] + wave * 8 * VS;
    const int32_t v0 = range.begin + (stage - 2) * KT;  // the values' step
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t n = lane + i * 64, key = n / kPer, col = n - key * kPer;
      if (8 * kPer % 64 && n >= 8u * kPer) continue;
      if constexpr (PAGED) {
        if (v0 + KT > least && has_nan(rv[i])) take_nan(rv[i], v0 + (int32_t)(wave * 8 + key), lowest + col * 16);
        u4 a, b;
        widen<T>(rk[i], a, b);
        *reinterpret_cast<u4*>(kt + key * KS + col * 16) = a;
        *reinterpret_cast<u4*>(kt + key * KS + col * 16 + 8) = b;
        widen<T>(rv[i], a, b);
        *reinterpret_cast<u4*>(vt + key * VS + col * 16) = a;
        *reinterpret_cast<u4*>(vt + key * VS + col * 16 + 8) = b;
      } else {
        *reinterpret_cast<u4*>(kt + key * KS + col * 8) = rk[i];
        *reinterpret_cast<u4*>(vt + key * VS + col * 8) = rv[i];
      }
    }
    if (!PAGED && wave == 0 && lane < 32) lds_bias[stage & 3][lane] = (bits_k >> lane) & 1u ? 0.f : -__builtin_inff();
  };
  const auto key_piece = [&](int slot, int i) {  // dims of step i of q . k
    return __builtin_bit_cast(v8, *reinterpret_cast<const u4*>(lds_k[slot] + (lane & 31u) * KS + half * 16 + (i / 2) * 32 + (i % 2) * 8));
  };
  const auto value_piece = [&](int slot, int i) {  // i: the step's 16 keys i / (DP / 32), dims i % (DP / 32)
    return values8<T, VS>(lds_v[slot], i / (DP / 32) * 16, i % (DP / 32), lane);
  };
  constexpr int kProducts = DP / 16;  // of a step, for the scores as for the mix
  // Scores of a step begin at 0, or at -inf for what is not seen.
  const auto first_scores = [&](int slot, bool all, const v8& kf) __attribute__((always_inline)) {
    f16v x;
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.f;
    if (PAGED || all) return Matrix<T>::mul(kf, __builtin_bit_cast(v8, q[0]), x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f4 y = *reinterpret_cast<const f4*>(lds_bias[slot] + j * 8 + half * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j * 4 + e] = y[e];
    }
    return Matrix<T>::mul(kf, __builtin_bit_cast(v8, q[0]), x);
  };

  // Step j: s holds its scores, `next` gets the next one's; before: the weights of
  // step j - 1, which are mixed, pr: its own.
  const auto advance = [&](int32_t j, f16v& s, f16v& next, const v8 (&before)[2], v8 (&pr)[2]) __attribute__((always_inline)) {
    const int32_t k0 = range.begin + j * KT;
    if (!(j & 1)) __syncthreads();
    constexpr int kAhead = kProducts < 4 ? kProducts : 4;
    const int k_slot = (j + 1) & 3, v_slot = (j + 3) & 3;
    v8 kf[kAhead], vf[2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = key_piece(k_slot, i);
    vf[0] = value_piece(v_slot, 0);
    vf[1] = value_piece(v_slot, 1);
    const bool all = bits_v == ~0u;  // of step j + 1
    store(j + 3);
    fetch(j + 4);
    float a = moved;  // what the sums so far are multiplied by, once step j - 1 is in
    bool raised = PAGED && moves;
    moved = 1.f;
    moves = false;
    float c[2] = {p.c, p.c}, share[2] = {0.f, 0.f}, back[2] = {1.f, 1.f};
    bool there_is[2] = {true, true}, unseen[2] = {false, false};
    if constexpr (PAGED) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int32_t at = (j - here_first) * 2 + n;
        there_is[n] = __builtin_amdgcn_readlane(here.id, at) >= 0;
        c[n] = lane_value(here.c, at);
        share[n] = lane_value(here_share, at);
        back[n] = lane_value(here_back, at);
      }
    }
    bool tiny = PAGED && ((here_tiny >> ((j - here_first) * 2)) & 3u);
    float add[2] = {PAGED ? off + share[0] : off, PAGED ? off + share[1] : off}, sum[2] = {0.f, 0.f};
    if constexpr (PAGED)
      if (!(there_is[0] && there_is[1] && k0 + KT <= wave_least)) {
        const int32_t left = limit - k0 - (int32_t)half * 4;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!there_is[i / 8] || i / 4 * 8 + i % 4 >= left) s[i] = -__builtin_inff();
        // nothing of scales that the row does not see
        float vs[2];
        uint32_t top = ref;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          unseen[n] = !there_is[n] || limit <= k0 + n * 16;
          vs[n] = lane_value(here.vs, (j - here_first) * 2 + n);
          if (!unseen[n]) top = max(top, power_of(vs[n]));
        }
        if (__any(top > ref)) {
          a *= __builtin_bit_cast(float, ref) * inverse_of(top);
          ref = top;
          raised = true;
        }
        tiny = false;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float f = vs[n] * inverse_of(ref);
          tiny = tiny || __any(!unseen[n] && f < Share<T>::kLeast);
          share[n] = unseen[n] ? 0.f : __builtin_amdgcn_logf(Share<T>::of(f));
          back[n] = unseen[n] ? 0.f : __builtin_amdgcn_rcpf(Share<T>::of(f));
          add[n] = unseen[n] ? 0.f : off + share[n];
          c[n] = seen_factor(unseen[n] ? 1.f : c[n]);
        }
      }
    const auto weigh = [&](int x) __attribute__((always_inline)) {  // elements x and x + 1
      float e[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x + i], c[x / 8], add[x / 8]));
        sum[x / 8] += e[i];
      }
      typename Matrix<T>::v2 both;
      both[0] = (T)e[0];
      both[1] = (T)e[1];
      uint32_t w = __builtin_bit_cast(uint32_t, both);
      asm volatile("" : "+v"(w), "+v"(sum[x / 8]));  // here, and not where they are used
      both = __builtin_bit_cast(typename Matrix<T>::v2, w);
      pr[x / 8][x % 8] = both[0];
      pr[x / 8][x % 8 + 1] = both[1];
    };
    // (After the last step, scores of what LDS holds, which nobody takes; before the
    // first, weights and values of 0.)
    next = first_scores(k_slot, all, kf[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      if (i) next = Matrix<T>::mul(kf[i % kAhead], __builtin_bit_cast(v8, q[i]), next);
      o[i % (DP / 32)] = Matrix<T>::mul(vf[i % 2], before[i / (DP / 32)], o[i % (DP / 32)]);
      if (i + kAhead < kProducts) kf[i % kAhead] = key_piece(k_slot, i + kAhead);
      if (i + 2 < kProducts) vf[i % 2] = value_piece(v_slot, i + 2);
#pragma unroll
      for (int x = i * 8 / kProducts * 2; x < (i + 1) * 8 / kProducts * 2; x += 2) weigh(x);
      __builtin_amdgcn_sched_barrier(0);
    }
    float total = PAGED ? sum[0] * back[0] + sum[1] * back[1] : sum[0] + sum[1];
    if (fresh || __any(total > most_of_step(PAGED) * __builtin_exp2f(Matrix<T>::kShift))) {
      float top[2] = {s[0], s[8]};
#pragma unroll
      for (int x = 1; x < 8; ++x) {
        top[0] = fmaxf(top[0], s[x]);
        top[1] = fmaxf(top[1], s[x + 8]);
      }
      // (a NaN is dropped: weights are NaN by themselves)
      const float highest = fmaxf(fmaxf(-__builtin_inff(), top[0] * c[0]), top[1] * c[1]);
      const float to = fmaxf(m, fmaxf(highest, lane_xor<32>(highest))), f = rescale_of(m, to);
      l *= f;
      a *= f;
      m = to;
      off = offset_of(to) + Matrix<T>::kShift;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        add[n] = !PAGED ? off : unseen[n] ? 0.f : off + share[n];
        sum[n] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < 16; x += 2) weigh(x);
      total = PAGED ? sum[0] * back[0] + sum[1] * back[1] : sum[0] + sum[1];
      raised = true;
      fresh = __any(m == -__builtin_inff());
    }
    l += total;
    if (raised) {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= a;
    }
    if constexpr (PAGED)
      if (tiny) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float rest = Share<T>::rest(lane_value(here.vs, (j - here_first) * 2 + n) * inverse_of(ref));
#pragma unroll
          for (int i = 0; i < 8; ++i) pr[n][i] = (T)((float)pr[n][i] * rest);
        }
      }
  };

  f16v s[2];
  v8 pr[2][2];
#pragma unroll
  for (int i = 0; i < 8; ++i) pr[1][0][i] = pr[1][1][i] = (T)0.f;
  if (steps > 0) {
    look_up(0);
    if constexpr (PAGED) {
      there = look_up_window(0);
      enter_window(0);
      there = look_up_window(32);
    }
    fetch(0);
    const bool all = bits_k == ~0u;
    store(0);
    fetch(1);
    store(1);
    fetch(2);
    store(2);
    fetch(3);
    __syncthreads();
    if (!__any(live)) {  // a wavefront without rows stages what the others take
      for (int32_t j = 0; j < steps; ++j) {
        if (!(j & 1)) __syncthreads();
        if (PAGED && j == here_first + 32) {
          enter_window(j);
          there = look_up_window(j + 32);
        }
        store(j + 3);
        fetch(j + 4);
      }
      steps = 0;
    }
    s[0] = first_scores(0, all, key_piece(0, 0));
#pragma unroll
    for (int i = 1; i < kProducts; ++i) s[0] = Matrix<T>::mul(key_piece(0, i), __builtin_bit_cast(v8, q[i]), s[0]);
    for (int32_t j = 0; j < steps; j += 2) {
      if (PAGED && j == here_first + 32) {
        enter_window(j);
        there = look_up_window(j + 32);
      }
      advance(j, s[0], s[1], pr[1], pr[0]);
      if (j + 1 < steps) advance(j + 1, s[1], s[0], pr[0], pr[1]);
    }
    __syncthreads();
    const auto finish = [&](const v8 (&last)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kProducts; ++i)
        o[i % (DP / 32)] = Matrix<T>::mul(value_piece((steps - 1) & 3, i), last[i / (DP / 32)], o[i % (DP / 32)]);
    };
    if (steps & 1) finish(pr[0]);
    else finish(pr[1]);
  }
  if constexpr (PAGED) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        o[i][j] *= __builtin_bit_cast(float, ref);
        if (limit > lowest[i * 32 + j / 4 * 8 + half * 4 + j % 4]) o[i][j] = __builtin_nanf("");
      }
  } else if (!any_shown) {  // nothing seen, and nothing of queries that are not finite
    m = -__builtin_inff();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
  }
  l += lane_xor<32>(l);
  if (row < p.rows && (p.splits == 1 || steps > 0)) {
    const uint64_t unit = ((uint64_t)w.b * p.heads + w.h) * p.row_blocks + w.block;
    store_row<T, DP>(p, w.b, w.h, t, g, (unit * p.splits + w.split) * kBlockRows + (row - w.block * kBlockRows), half, live, o, m, l);
  }
}

// ---------------------------------------------------------------- few rows
// Up to 16 R rows of a head, as a token's or a few drafts' are: bound by the keys'
// and values' way from memory.  Four wavefronts take tiles of 32 keys in turn,
// each on its own (no barrier in the loop), and join at the end.  Matrix tiles of
// 16 rows: S^T = K Q^T is two of 16 keys, a lane holding one row (lane & 15) and
// keys 4 (lane / 16) + 0..3 of each, which are the eight of its B operand.  Keys go
// from memory to the A operand's registers (a lane's bytes are of one key), values
// through the wavefront's own part of LDS.  A page holds whole groups of 16
// tokens, so that a matrix tile has one page and one scale, which stay scalar.
// Registers for the sums are half of what tiles of 32 rows take: 16 wavefronts
// a CU, each with its next 32 keys in flight.  (One row of 32 x 8 x 4 heads over 8192
// cached tokens at most: 68 us, 5.0 TB/s; of 64 x 16 heads to 1500 states at most: 63
// us, 3.9 TB/s; 6 x 5 of 2 x 4 over 60001 tokens: 25 us, 4.0 TB/s.)

// Step s of q . k takes dims dim_of() .. + 8 of quarter q of the lanes: 16 codes
// (32 bytes of 16-bit numbers) in one piece where the head is wide enough.
template <int DP>
__device__ __forceinline__ constexpr uint32_t dim_of(uint32_t s, uint32_t quarter) {
  return DP % 64 == 0 ? (s / 2) * 64 + quarter * 16 + (s % 2) * 8 : s * 32 + quarter * 8;
}

template <typename T, int DP, bool PAGED, int R>
__global__ __launch_bounds__(256, few_workgroups(DP, 16 * R, PAGED)) void few_kernel(AttendPlan p) {
  typedef typename Matrix<T>::v8 v8;
  constexpr int KT = 32, W = 4, kSteps = DP / 32;
  constexpr int kPer = PAGED ? DP / 16 : DP / 8, kMine = KT * kPer / 64;  // pieces of a value row, of a lane
  constexpr int VS = Strides<DP>::V16;
  constexpr int kDims = DP % 64 ? 32 : 64;
  constexpr int kTile = KT * VS * 2, kJoin = 16 * R * (kDims + 4) * 4;  // bytes of a wavefront's values, of its sums
  __shared__ __align__(16) char lds[W * (kTile > kJoin ? kTile : kJoin)];
  __shared__ float lds_m[W][16 * R], lds_l[W][16 * R], row_m[16 * R], row_l[16 * R];
  __shared__ int32_t lowest[PAGED ? DP : 1];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, col = lane & 15u, quarter = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  Place w;
  Range range;
  Sequence seq;
  if (p.chunks) {
    const uint32_t u = p.by_heads.div(blockIdx.x);
    Chunk c;
    if (!find_chunk<PAGED, false>(p, lane, u, c)) return;
    w.b = c.b;
    seq = c.seq;
    w.h = blockIdx.x - u * p.heads;
    range.begin = c.index * c.size;
    range.end = range.begin + c.size;
  } else {
    // Tensors, several rounds of workgroups: eight heads, whose keys lie side by side,
    // to one XCD (one row of 128 x 16 heads to 1500 states at most: 109 us, 120 in
    // turn; of 64 x 16, one round, 64.2 and 63.7).
    const bool beside = !PAGED && gridDim.x >= 2048 && blockIdx.x < (gridDim.x & ~63u);
    const uint32_t unit = beside ? (blockIdx.x & ~63u) + (blockIdx.x & 7u) * 8 + ((blockIdx.x >> 3) & 7u) : blockIdx.x;
    w.b = p.by_heads.div(unit);
    w.h = unit - w.b * p.heads;
    seq = sequence_of<PAGED>(p, w.b);
    range.begin = 0;
    range.end = 0x7FFFFFFF;
  }
  const int32_t most = most_of<PAGED>(seq), least = limit_of<PAGED>(seq, 0);
  range.end = min(range.end, most);
  T* lds_v = reinterpret_cast<T*>(lds + wave * kTile);

  u4 q[R][kSteps];
  int32_t limit[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = r * 16 + col, t = p.by_group.div(row), g = row - t * p.group;
    const bool live = row < p.rows && (int32_t)t < seq.tokens;
    limit[r] = live ? limit_of<PAGED>(seq, (int32_t)t) : 0;
    const T* x = static_cast<const T*>(p.q) + w.b * p.q_batch + t * p.q_token + (w.h * p.group + g) * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      q[r][s] = u4{0, 0, 0, 0};
      if (live && dim_of<DP>(s, quarter) < p.dim) q[r][s] = load16(x + dim_of<DP>(s, quarter));
    }
  }
  f4 o[R][DP / 16];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -__builtin_inff();
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[r][i] = f4{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t ref[R];  // the largest of the values' scales that a row has seen, a power of two's bits
  float inverse[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ref[r] = PAGED ? 0u : 0x3F800000u;
    inverse[r] = 0.f;
  }
  if constexpr (PAGED) {
    for (uint32_t d = tid; d < (uint32_t)DP; d += 256) lowest[d] = 0x7FFFFFFF;
    __syncthreads();
  }

  // PAGED: lane i knows the 16 keys i of the wavefront's next 32 tiles (i / 2 the tile, i % 2 its half)
  int32_t page_id = -1;
  float page_ks = 0.f, page_vs = 0.f;
  const auto look_up = [&](int32_t k0) {
    const int32_t key = k0 + (int32_t)(lane >> 1) * (W * KT) + (int32_t)(lane & 1u) * 16;
    page_id = -1;
    page_ks = page_vs = 0.f;
    if (key < range.end) {
      page_id = p.table[w.b * p.table_batch + p.by_page.div((uint32_t)key) * p.table_slot];
      if ((uint32_t)page_id >= p.pages) {
        page_id = -1;
      } else {
        page_ks = p.kp.scales[page_id * p.kp.scale_page + w.h * p.kp.scale_head];
        page_vs = p.vp.scales[page_id * p.vp.scale_page + w.h * p.vp.scale_head];
      }
    }
  };

  // what is loaded of the next tile
  u4 rk[2][PAGED ? (kSteps + 1) / 2 : kSteps];
  u4 rv[kMine];
  int32_t id[2] = {0, 0};
  bool seen = true;  // of key lane & 31
  const auto fetch = [&](int32_t k0, int32_t ahead) {  // `ahead` tiles behind the last look_up()
    if constexpr (PAGED) {
      const uint8_t* kb[2];
      const uint8_t* vb[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        id[n] = __builtin_amdgcn_readlane(page_id, ahead * 2 + n);
        const uint32_t key = (uint32_t)k0 + n * 16, at = key - p.by_page.div(key) * p.page_size;
        kb[n] = code_at(p.kp, id[n], w.h, at);
        vb[n] = code_at(p.vp, id[n], w.h, at);
      }
      const uint32_t key_off = col * (uint32_t)p.kp.token;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < (kSteps + 1) / 2; ++i) {
          rk[n][i] = u4{0, 0, 0, 0};
          if (id[n] >= 0) {
            if constexpr (DP % 64 == 0) {
              const uint32_t d = i * 64 + quarter * 16;
              if (d < p.dim) rk[n][i] = load16(kb[n] + key_off + d);
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t d = (2 * i + e) * 32 + quarter * 8;
                if (2 * i + e < kSteps && d < p.dim) {
                  typedef uint32_t u2e __attribute__((ext_vector_type(2), aligned(1)));
                  const u2e x = *reinterpret_cast<const u2e*>(kb[n] + key_off + d);
                  rk[n][i][2 * e] = x[0];
                  rk[n][i][2 * e + 1] = x[1];
                }
              }
            }
          }
        }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const uint32_t piece = lane + i * 64, r = piece / kPer, c = (piece - r * kPer) * 16;
        // the rows of one load are of the first half, of the second, or of both
        const uint32_t off = (r & 15u) * (uint32_t)p.vp.token + c;
        rv[i] = u4{0, 0, 0, 0};
        if (i * 64 + 63 < 16 * kPer) {
          if (id[0] >= 0 && c < p.dim) rv[i] = load16(vb[0] + off);
        } else if (i * 64 >= 16 * kPer) {
          if (id[1] >= 0 && c < p.dim) rv[i] = load16(vb[1] + off);
        } else {
          if ((r < 16 ? id[0] : id[1]) >= 0 && c < p.dim) rv[i] = load16((r < 16 ? vb[0] : vb[1]) + off);
        }
      }
    } else {
      const int32_t mine = k0 + (int32_t)(lane & 31u);
      seen = mine < range.end;
      if (p.mask && seen) seen = p.mask[w.b * p.mask_batch + mine * p.mask_key] != 0;
      const T* kb = static_cast<const T*>(p.k.data) + w.b * p.k.batch + w.h * p.k.head;
      const T* vb = static_cast<const T*>(p.v.data) + w.b * p.v.batch + w.h * p.v.head;
      // keys past the last read the last
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const T* row = kb + (int64_t)min(k0 + n * 16 + (int32_t)col, range.end - 1) * p.k.key;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint32_t d = dim_of<DP>(s, quarter);
          rk[n][s] = u4{0, 0, 0, 0};
          if (d < p.dim) rk[n][s] = load16(row + d);
        }
      }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const uint32_t piece = lane + i * 64, r = piece / kPer, c = (piece - r * kPer) * 8;
        rv[i] = u4{0, 0, 0, 0};
        if (c < p.dim) rv[i] = load16(vb + (int64_t)min(k0 + (int32_t)r, range.end - 1) * p.v.key + c);
      }
    }
  };

  int32_t k0 = range.begin + (int32_t)wave * KT, ahead = 0;
  if (k0 < range.end) {
    if (PAGED) look_up(k0);
    fetch(k0, 0);
  }
  for (; k0 < range.end; k0 += W * KT) {
    // scores
    f4 s[R][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        u4 a;
        if constexpr (PAGED) a = widen8<T>(rk[n][i / 2][i % 2 * 2], rk[n][i / 2][i % 2 * 2 + 1]);
        else a = rk[n][i];
#pragma unroll
        for (int r = 0; r < R; ++r)
          s[r][n] = Matrix<T>::mul16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, q[r][i]), s[r][n]);
      }
    }
    // which keys every live row sees
    uint32_t bits;
    if constexpr (PAGED) bits = (id[0] >= 0 ? 0xFFFFu : 0u) | (id[1] >= 0 ? 0xFFFF0000u : 0u);
    else bits = (uint32_t)__ballot(seen);
    const bool whole = bits == ~0u && k0 + KT <= least;
    // values to LDS
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t piece = lane + i * 64, r = piece / kPer, c = piece - r * kPer;
      if constexpr (PAGED) {
        if (!whole && has_nan(rv[i])) take_nan(rv[i], k0 + (int32_t)r, lowest + c * 16);
        u4 a, b;
        widen<T>(rv[i], a, b);
        *reinterpret_cast<u4*>(lds_v + r * VS + c * 16) = a;
        *reinterpret_cast<u4*>(lds_v + r * VS + c * 16 + 8) = b;
      } else {
        if (!whole && !((bits >> r) & 1u)) rv[i] = u4{0, 0, 0, 0};
        *reinterpret_cast<u4*>(lds_v + r * VS + c * 8) = rv[i];
      }
    }
    wave_lds_fence();
    const float ks0 = PAGED ? lane_value(page_ks, ahead * 2) : 1.f, ks1 = PAGED ? lane_value(page_ks, ahead * 2 + 1) : 1.f;
    const float vs0 = PAGED ? lane_value(page_vs, ahead * 2) : 1.f, vs1 = PAGED ? lane_value(page_vs, ahead * 2 + 1) : 1.f;
    if (k0 + W * KT < range.end) {
      if (PAGED && ++ahead == 32) {
        look_up(k0 + W * KT);
        ahead = 0;
      }
      fetch(k0 + W * KT, ahead);
    }
    // exponentials
    const float vs[2] = {vs0, vs1};
    v8 pr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float rc[2] = {p.c * ks0, p.c * ks1};
      float f[2] = {1.f, 1.f};  // the values' scales as multiples
      bool unseen[2] = {false, false};
      if (!whole) {
        const int32_t left = limit[r] - k0 - (int32_t)quarter * 4;
        const uint32_t mine = bits >> (quarter * 4);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((mine >> (j / 4 * 16 + j % 4)) & 1u) || j / 4 * 16 + j % 4 >= left) s[r][j / 4][j % 4] = -__builtin_inff();
        if constexpr (PAGED) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {  // nothing of scales that the row does not see
            unseen[n] = !((bits >> (n * 16)) & 1u) || limit[r] <= k0 + n * 16;
            rc[n] = seen_factor(unseen[n] ? 1.f : rc[n]);
          }
        }
      }
      uint32_t power = ref[r];
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (PAGED && !unseen[n]) power = max(power, power_of(vs[n]));
      float top = -__builtin_inff();
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float x = fmaxf(fmaxf(s[r][n][0], s[r][n][1]), fmaxf(s[r][n][2], s[r][n][3]));
        top = fmaxf(top, x * rc[n]);  // a NaN is dropped: weights are NaN by themselves
      }
      top = fmaxf(top, lane_xor<16>(top));
      top = fmaxf(top, lane_xor<32>(top));
      // (row by row, so that a later token's scale moves no rounding of another row)
      const bool low = top - m[r] > kSlack || (m[r] == -__builtin_inff() && top > m[r]);
      if (__any(low || (PAGED && power > ref[r]))) {
        const float to = low ? top : m[r], a = rescale_of(m[r], to);
        l[r] *= a;
        if (PAGED) inverse[r] = inverse_of(power);
        const float oa = PAGED ? a * (__builtin_bit_cast(float, ref[r]) * inverse[r]) : a;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[r][i] *= oa;
        m[r] = to;
        ref[r] = power;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
        if (PAGED) f[n] = unseen[n] ? 0.f : vs[n] * inverse[r];
      const float off = offset_of(m[r]) + Matrix<T>::kShift;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][n][j], rc[n], off));
          sum += e;
          pr[r][n * 4 + j] = (T)(PAGED ? e * f[n] : e);
        }
        l[r] += sum;
      }
    }
    // values, 16 dims a time
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const uint32_t at = (quarter * 4 + (col >> 2)) * VS + i * 16 + (col & 3u) * 4;
      union {
        s4 part[2];
        v8 all;
      } v;
      v.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(lds_v + at));
      v.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(lds_v + at + 16 * VS));
#pragma unroll
      for (int r = 0; r < R; ++r) o[r][i] = Matrix<T>::mul16(v.all, pr[r], o[r][i]);
    }
  }

  // join the wavefronts, kDims dims at a time
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += lane_xor<16>(l[r]);
    l[r] += lane_xor<32>(l[r]);
    if (quarter == 0) {
      lds_m[wave][r * 16 + col] = m[r];
      lds_l[wave][r * 16 + col] = l[r];
    }
  }
  __syncthreads();
  float a[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = r * 16 + col;
    float top = lds_m[0][row], sum = 0.f;
#pragma unroll
    for (int i = 1; i < W; ++i) top = fmaxf(top, lds_m[i][row]);
#pragma unroll
    for (int i = 0; i < W; ++i) sum += lds_l[i][row] * rescale_of(lds_m[i][row], top);
    a[r] = rescale_of(m[r], top) * __builtin_bit_cast(float, ref[r]);
    if (wave == 0 && quarter == 0) {
      row_m[row] = top;
      row_l[row] = sum;
    }
  }
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int part = 0; part < DP / kDims; ++part) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < kDims / 16; ++i) {
        f4 v = o[r][part * (kDims / 16) + i] * a[r];
        *reinterpret_cast<f4*>(sums + (wave * 16 * R + r * 16 + col) * (kDims + 4) + i * 16 + quarter * 4) = v;
      }
    __syncthreads();
    for (uint32_t at = tid; at < p.rows * (kDims / 4); at += 256) {
      const uint32_t r = at / (kDims / 4), c = (at % (kDims / 4)) * 4, d = part * kDims + c;
      if (d >= p.dim) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const f4 x = *reinterpret_cast<const f4*>(sums + (i * 16 * R + r) * (kDims + 4) + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += x[k];
      }
      const uint32_t rt = p.by_group.div(r), rg = r - rt * p.group;
      const bool live = (int32_t)rt < seq.tokens;
      if constexpr (PAGED) {
        const int32_t row_limit = live ? limit_of<PAGED>(seq, (int32_t)rt) : 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (row_limit > lowest[d + k]) v[k] = __builtin_nanf("");
      }
      if (!p.chunks) {
        const float total = row_l[r];
        const bool none = !live || total == 0.f;
        const float inv = 1.f / total;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = none ? 0.f : v[k] * inv;
        store_pack<T, 4>(static_cast<T*>(p.out) + w.b * p.o_batch + rt * p.o_token + (w.h * p.group + rg) * p.o_head + d, v);
      } else {
        const uint64_t slot = (uint64_t)blockIdx.x * p.rows + r;
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
// A row's splits at their highest maximum, by E threads: four dims a thread, and
// as many splits side by side as that leaves threads for (128 splits of 240 rows
// took 62 us by one wavefront a row, split after split, 9 by a workgroup each; 5
// splits of 19200 narrow rows 13.8 by a wavefront, 5.9 by 16 lanes).
template <typename T, bool PAGED, int E>
__global__ __launch_bounds__(256) void join_kernel(AttendPlan p) {
  __shared__ f4 part[256];
  constexpr int G = E < 64 ? E : 64;  // lanes that know of the row what all need
  const uint32_t lane = threadIdx.x & (G - 1u), mine = threadIdx.x % E;
  const uint64_t at = (uint64_t)blockIdx.x * (256 / E) + threadIdx.x / E;  // (b, h, row)
  if (E < 256 && at >= (uint64_t)p.batch * p.heads * p.rows) return;
  const uint32_t unit = (uint32_t)(at / p.rows), row = (uint32_t)(at - (uint64_t)unit * p.rows);
  const uint32_t b = p.by_heads.div(unit), h = unit - b * p.heads;
  const uint32_t t = p.by_group.div(row), g = row - t * p.group;
  Sequence seq;
  int32_t n;
  uint64_t first, step;  // its splits' places
  if (E >= 64 && p.chunks) {  // (a wavefront's rows are of one sequence)
    Chunk c;
    find_chunk<PAGED, true>(p, lane, b, c);
    seq = c.seq;
    n = c.count;
    first = ((uint64_t)c.first * p.heads + h) * p.rows + row;
    step = (uint64_t)p.heads * p.rows;
  } else {
    seq = sequence_of<PAGED>(p, b);
    const uint32_t block = row / kBlockRows;
    const int32_t t_first = (int32_t)p.by_group.div(block * kBlockRows);
    const int32_t t_last = min((int32_t)p.by_group.div(min(p.rows, (block + 1) * kBlockRows) - 1), seq.tokens - 1);
    n = active_splits(t_last < t_first ? 0 : limit_of<PAGED>(seq, t_last), p.splits, 64);
    first = ((uint64_t)unit * p.row_blocks + block) * p.splits * kBlockRows + (row - block * kBlockRows);
    step = kBlockRows;
  }
  if ((int32_t)t >= seq.tokens) n = 0;
  // the maximum and the total
  float m = -__builtin_inff(), l = 0.f;
  for (int32_t i = (int32_t)lane; i < n; i += G) m = fmaxf(m, p.stats[(first + (uint64_t)i * step) * 2]);
  m = group_max<G>(m);
  for (int32_t i = (int32_t)lane; i < n; i += G) {
    const float* stats = p.stats + (first + (uint64_t)i * step) * 2;
    l += stats[1] * rescale_of(stats[0], m);
  }
  l = group_sum<G>(l);
  const uint32_t quads = p.dim / 4, sides = E / quads, side = mine / quads, d = (mine - side * quads) * 4;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (side < sides) {
#pragma unroll 4
    for (int32_t i = (int32_t)side; i < n; i += (int32_t)sides) {
      const uint64_t slot = first + (uint64_t)i * step;
      float x[4];
      load_pack<float, 4>(p.sums + slot * p.dim + d, x);
      const float f = rescale_of(p.stats[slot * 2], m);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[k] * f;
    }
  }
  part[threadIdx.x] = v;
  if (E == 256) __syncthreads();
  else wave_lds_fence();
  if (side == 0) {
    for (uint32_t i = 1; i < sides; ++i) v += part[threadIdx.x + i * quads];
    const float r = 1.f / l;
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = n == 0 || l == 0.f ? 0.f : v[k] * r;
    store_pack<T, 4>(static_cast<T*>(p.out) + b * p.o_batch + t * p.o_token + (h * p.group + g) * p.o_head + d, o);
  }
}

}  // namespace dev

// Launches a plan whose operands are checked.
template <typename T, int DP, bool PAGED>
thin_status launch_attend_dim(const AttendPlan& p, hipStream_t stream) {
  const uint32_t units = p.batch * p.heads * p.row_blocks, rows = p.batch * p.heads * p.rows;
  const bool few = p.rows <= few_rows(PAGED);
  if (few && p.rows <= 16) {
    hipLaunchKernelGGL((dev::few_kernel<T, DP, PAGED, 1>), dim3(p.chunks ? p.chunks : units), dim3(256), 0, stream, p);
  } else if (few) {
    if constexpr (PAGED)
      hipLaunchKernelGGL((dev::few_kernel<T, DP, PAGED, 2>), dim3(p.chunks ? p.chunks : units), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((dev::tile_kernel<T, DP, PAGED>), dim3(units * p.splits), dim3(256), 0, stream, p);
  }
  THIN_LAUNCH_CHECK("attend");
  if (!p.chunks && p.splits == 1) return THIN_OK;
  // By the parts of a row, on the average; rows that fill the card take a wavefront or
  // 16 lanes (6400 rows of 12 parts of 32 dims: 42 us with the first launch, 33 so).
  if ((few ? p.chunks / units : p.splits) > 8 && rows < 2048)
    hipLaunchKernelGGL((dev::join_kernel<T, PAGED, 256>), dim3(rows), dim3(256), 0, stream, p);
  else if (DP <= 64 && !few)
    hipLaunchKernelGGL((dev::join_kernel<T, PAGED, 16>), dim3((rows + 15) / 16), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((dev::join_kernel<T, PAGED, 64>), dim3((rows + 3) / 4), dim3(256), 0, stream, p);
  THIN_LAUNCH_CHECK("attend_join");
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
