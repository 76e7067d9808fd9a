// Verification of drafted tokens against the target's probabilities.
//
//   draft i of a sequence stays while u_i q_i(x_i) < p_i(x_i), all before it
//   having stayed; then one more token comes from the target: from
//   max(p_n - q_n, 0) at the first draft n that fell, from p_n if none did, the
//   first whose distribution function passes r times the total.
//
// So the tokens are distributed as the target's own.  Products and sums are
// taken in 64 bits: u q is exact there, and the roundings of a sum over the
// vocabulary, in the order in which it is taken, move a border by little.  On the
// way to a sum that is compared with it: 17 of a tile (the element's own, 7 along a
// thread's, 6 over the lanes, 3 over the wavefronts), 6 and one for each 64 tiles
// ahead, 2 where a tile is taken apart from those, 28 within it; of the border, the
// total's 17 and 6 and one for each 64 tiles, and the product's.  Each is 2^-53 of
// the total at most: with all signs alike 79 up to 131072 tokens, 9e-15, and 205 of
// the longest rows, 2.3e-14 (sums in 32 bits: 1e-5).
//
// Bound by memory: of the target's and the draft's rows only one each is read
// whole.  Few rows, so each is cut into tiles over the card; a second launch
// finds the tile that holds the border and scans it again.  A row of one tile
// takes one launch.  (48 rows of 128000 in 32 bits, target and draft: 11.5 us, 4.3
// TB/s, and 7.8 of the second launch, a chain of loads and sums that takes 6.6 for
// two rows of 50001 too.)
#include "rows.h"

#include <string.h>

namespace thin {
namespace {

constexpr int kTile = 2048;        // elements of a workgroup at a time: 8 a thread
constexpr int64_t kMaxDrafts = 64; // one lane each
constexpr int64_t kMaxVocab = 1 << 23;
constexpr int kMostTiles = 4;      // of a workgroup

struct DraftPlan {
  const void* target;
  const void* draft;
  int64_t pb, pk, qb, qk;
  const int64_t* tokens;
  int64_t tb, tk;
  const int32_t* counts;
  int64_t count_step;
  const float* accept;
  int64_t ub, uk;
  const float* sample;
  int64_t sample_step;
  int64_t* out;
  int64_t ob, ok;
  int32_t* taken;
  int64_t taken_step;
  uint32_t drafts, vocab, tiles, per, groups;  // per: a workgroup's tiles; groups: of them, a row's
  FastDiv by_groups;
  double* sums;     // [batch, tiles, 2]: of what is left, of the target's row
  int32_t* stayed;  // [batch]
};

constexpr double kMost = 1.7976931348623157e308;  // of what is finite
// A probability; what is none counts as 0.
__device__ __forceinline__ double positive(double x) { return x > 0.0 && x <= kMost ? x : 0.0; }

// How many drafts stay; every lane of a wavefront gets it.
template <typename T>
__device__ __forceinline__ uint32_t stayed_of(const DraftPlan& p, uint32_t b, uint32_t lane, uint32_t& count) {
  const int32_t n = p.counts ? p.counts[b * p.count_step] : (int32_t)p.drafts;
  count = (uint32_t)max(0, min(n, (int32_t)p.drafts));
  bool stays = false;
  if (lane < count) {
    const int64_t x = p.tokens[b * p.tb + lane * p.tk];
    if (x >= 0 && x < (int64_t)p.vocab) {
      const double pt = positive((double)(float)static_cast<const T*>(p.target)[b * p.pb + lane * p.pk + x]);
      const double qt = p.draft ? (double)(float)static_cast<const T*>(p.draft)[b * p.qb + lane * p.qk + x] : 1.0;
      const double least = (double)p.accept[b * p.ub + lane * p.uk] * qt;
      stays = least >= -kMost && least < pt;  // (of a draft's own that is not finite, -inf too is none)
    }
  }
  const uint64_t fell = ~__ballot(stays);
  return fell ? (uint32_t)__builtin_ctzll(fell) : 64u;
}

// The row that the next token comes from.
template <typename T>
struct Rest {
  const T* p;
  const T* q;       // null: nothing is taken off but `without`
  int64_t without;  // a token that has no part, or -1
  uint32_t vocab;
  __device__ __forceinline__ Rest(const DraftPlan& a, uint32_t b, uint32_t stayed, uint32_t count)
      : p(static_cast<const T*>(a.target) + b * a.pb + stayed * a.pk), q(nullptr), without(-1), vocab(a.vocab) {
    if (stayed < count) {
      if (a.draft) q = static_cast<const T*>(a.draft) + b * a.qb + stayed * a.qk;
      else without = a.tokens[b * a.tb + stayed * a.tk];
    }
  }
  // Elements [at, at + 8): what is left of them, and the target's own.
  __device__ __forceinline__ void load(uint32_t at, double (&left)[8], double (&own)[8]) const {
    float x[8], y[8];
    const uint32_t n = at < vocab ? vocab - at : 0u;
    if (n >= 8) {
      dev::load_pack<T, 8>(p + at, x);
      if (q) dev::load_pack<T, 8>(q + at, y);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = (uint32_t)j < n ? (float)p[at + j] : 0.f;
        y[j] = q && (uint32_t)j < n ? (float)q[at + j] : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      own[j] = positive((double)x[j]);
      left[j] = (int64_t)(at + j) == without ? 0.0 : q ? (own[j] > 0.0 ? positive((double)x[j] - (double)y[j]) : 0.0) : own[j];
    }
  }
};

__device__ __forceinline__ double lane_double(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over the lanes up to this one, by DPP.
template <int CTRL, int ROWS>
__device__ __forceinline__ double plus_moved(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = plus_moved<0x111, 0xF>(v);  // row_shr:1, :2, :4, :8
  v = plus_moved<0x112, 0xF>(v);
  v = plus_moved<0x114, 0xF>(v);
  v = plus_moved<0x118, 0xF>(v);
  v = plus_moved<0x142, 0xA>(v);  // row_bcast:15, :31
  return plus_moved<0x143, 0xC>(v);
}
__device__ __forceinline__ double wave_total(double v) { return lane_double(wave_scan(v), 63); }

struct Shared {
  double left[kMostTiles][4], own[kMostTiles][4];
  uint32_t found, last;
};

// The first element of a tile whose sum, with `before` ahead of the tile, passes
// `edge`; where rounding leaves none, the tile's last that has a part.
template <typename T>
__device__ __forceinline__ uint32_t find_in_tile(const Rest<T>& rest, bool whole, uint32_t first, double before, double edge,
                                                 Shared& lds) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, at = first + threadIdx.x * 8;
  if (threadIdx.x == 0) {
    lds.found = 0xFFFFFFFFu;
    lds.last = 0;
  }
  double a[8], o[8], sum = 0.0;
  rest.load(at, a, o);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (whole) a[j] = o[j];
    sum += a[j];
  }
  const double scan = wave_scan(sum);
  if (lane == 63) lds.left[0][wave] = scan;
  __syncthreads();
  for (uint32_t i = 0; i < wave; ++i) before += lds.left[0][i];
  double run = before + (scan - sum);
  uint32_t found = 0xFFFFFFFFu, last = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    run += a[j];
    if (a[j] > 0.0) {
      last = at + j;
      if (run > edge) found = min(found, at + j);
    }
  }
  if (found != 0xFFFFFFFFu) atomicMin(&lds.found, found);
  if (last) atomicMax(&lds.last, last);
  __syncthreads();
  return lds.found != 0xFFFFFFFFu ? lds.found : lds.last;
}

// What a sequence's result takes, loaded before anything waits: drafts of this
// thread's places (K + 1 <= 65 of 256 threads) and the random number.
struct Given {
  int64_t token;
  float sample;
  __device__ __forceinline__ Given(const DraftPlan& p, uint32_t b) : token(-1), sample(p.sample[b * p.sample_step]) {
    if (threadIdx.x < p.drafts) token = p.tokens[b * p.tb + threadIdx.x * p.tk];
  }
  __device__ __forceinline__ double edge(double total) const {
    return (double)(sample > 0.f ? fminf(sample, 1.f) : 0.f) * total;
  }
  // The sequence's tokens, the last of them `next`.
  __device__ __forceinline__ void store(const DraftPlan& p, uint32_t b, uint32_t stayed, int64_t next) const {
    const uint32_t i = threadIdx.x;
    if (i <= p.drafts) p.out[b * p.ob + i * p.ok] = i < stayed ? token : i == stayed ? next : -1;
    if (i == 0) p.taken[b * p.taken_step] = (int32_t)stayed;
  }
};

template <typename T>
__global__ __launch_bounds__(256) void sums_kernel(DraftPlan p) {
  __shared__ Shared lds;
  const uint32_t b = p.by_groups.div(blockIdx.x), first = (blockIdx.x - b * p.groups) * p.per;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t count;
  const uint32_t stayed = stayed_of<T>(p, b, lane, count);
  const Rest<T> rest(p, b, stayed, count);
#pragma unroll
  for (uint32_t i = 0; i < (uint32_t)kMostTiles; ++i)
    if (i < p.per) {  // (past the row's end: zeros)
      double a[8], o[8], left = 0.0, own = 0.0;
      rest.load((first + i) * kTile + threadIdx.x * 8, a, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        left += a[j];
        own += o[j];
      }
      left = wave_total(left);
      own = wave_total(own);
      if (lane == 0) {
        lds.left[i][wave] = left;
        lds.own[i][wave] = own;
      }
    }
  __syncthreads();
  const uint32_t i = threadIdx.x & (kMostTiles - 1u);
  const double left = ((lds.left[i][0] + lds.left[i][1]) + lds.left[i][2]) + lds.left[i][3];
  const double own = ((lds.own[i][0] + lds.own[i][1]) + lds.own[i][2]) + lds.own[i][3];
  if (p.tiles > 1) {
    if (threadIdx.x < p.per && first + threadIdx.x < p.tiles) {
      double* sums = p.sums + ((uint64_t)b * p.tiles + first + threadIdx.x) * 2;
      sums[0] = left;
      sums[1] = own;
    }
    if (first == 0 && threadIdx.x == 0) p.stayed[b] = (int32_t)stayed;
    return;
  }
  const double all_left = ((lds.left[0][0] + lds.left[0][1]) + lds.left[0][2]) + lds.left[0][3];
  const double all_own = ((lds.own[0][0] + lds.own[0][1]) + lds.own[0][2]) + lds.own[0][3];
  __syncthreads();
  const Given given(p, b);
  const bool whole = !(all_left > 0.0);
  const double total = whole ? all_own : all_left;
  const uint32_t next = find_in_tile<T>(rest, whole, 0, 0.0, given.edge(total), lds);
  given.store(p, b, stayed, total > 0.0 ? (int64_t)next : -1);
}

// Where a row's border lies: the first tile whose sum passes it (where rounding
// leaves none, the last that has a part) and what is ahead of it.  64 tiles a
// round, by every wavefront for itself.
template <bool WHOLE>
__device__ __forceinline__ bool find_tile(const DraftPlan& p, const double* sums, const Given& given, uint32_t lane,
                                          uint32_t& tile, double& before, double& edge) {
  const auto part = [&](uint32_t i) { return i + lane < p.tiles ? sums[(i + lane) * 2 + (WHOLE ? 1 : 0)] : 0.0; };
  const double first = part(0), first_scan = wave_scan(first);
  double total = lane_double(first_scan, 63);
  for (uint32_t i = 64; i < p.tiles; i += 64) total += wave_total(part(i));
  if (!(total > 0.0)) return false;
  edge = given.edge(total);
  double ahead = 0.0;
  for (uint32_t i = 0; i < p.tiles; i += 64) {
    const double v = i ? part(i) : first, scan = i ? wave_scan(v) : first_scan;
    const uint64_t passed = __ballot(v > 0.0 && ahead + scan > edge), some = __ballot(v > 0.0);
    if (some) {
      const int l = passed ? __builtin_ctzll(passed) : 63 - __builtin_clzll(some);
      tile = i + l;
      before = lane_double(ahead + (scan - v), l);
      if (passed) break;
    }
    ahead += lane_double(scan, 63);
  }
  return true;
}

template <typename T>
__global__ __launch_bounds__(256) void find_kernel(DraftPlan p) {
  __shared__ Shared lds;
  const uint32_t b = blockIdx.x, lane = threadIdx.x & 63u;
  const double* sums = p.sums + (uint64_t)b * p.tiles * 2;
  const Given given(p, b);
  const uint32_t stayed = (uint32_t)p.stayed[b];
  const int32_t n = p.counts ? p.counts[b * p.count_step] : (int32_t)p.drafts;
  const uint32_t count = (uint32_t)max(0, min(n, (int32_t)p.drafts));
  const Rest<T> rest(p, b, stayed, count);
  uint32_t tile = 0;
  double before = 0.0, edge = 0.0;
  const bool some = find_tile<false>(p, sums, given, lane, tile, before, edge);
  const bool any = some || find_tile<true>(p, sums, given, lane, tile, before, edge);
  const uint32_t next = find_in_tile<T>(rest, !some, tile * kTile, before, edge, lds);
  given.store(p, b, stayed, any ? (int64_t)next : -1);
}

int64_t tiles_of(int64_t vocab) { return (vocab + kTile - 1) / kTile; }
// Tiles of a workgroup: one, or as many as leave enough workgroups, since each first
// finds out which row is the rest's (256 rows of 128000 as bf16: 42 us by four, 51 by one).
int64_t per_of(int64_t batch, int64_t vocab) {
  int64_t n = 1;
  while (n < kMostTiles && batch * ((tiles_of(vocab) + 2 * n - 1) / (2 * n)) >= 2048) n *= 2;
  return n;
}

template <typename T>
thin_status launch(const DraftPlan& p, int64_t batch, hipStream_t stream) {
  hipLaunchKernelGGL((sums_kernel<T>), dim3((uint32_t)(batch * p.groups)), dim3(256), 0, stream, p);
  THIN_LAUNCH_CHECK("verify_drafts");
  if (p.tiles > 1) {
    hipLaunchKernelGGL((find_kernel<T>), dim3((uint32_t)batch), dim3(256), 0, stream, p);
    THIN_LAUNCH_CHECK("verify_drafts_find");
  }
  return THIN_OK;
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" size_t thin_verify_drafts_workspace(int64_t batch, int64_t vocab) {
  if (batch <= 0 || vocab <= 0 || vocab > kMaxVocab) return 0;
  const int64_t tiles = tiles_of(vocab);
  return tiles == 1 ? 0 : (size_t)batch * (tiles * 16 + 8);
}

extern "C" thin_status thin_verify_drafts(const thin_desc* target, const thin_desc* draft, const thin_desc* tokens,
                                          const thin_desc* counts, const thin_desc* accept, const thin_desc* sample,
                                          const thin_desc* out, const thin_desc* taken, void* workspace,
                                          size_t workspace_bytes, hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(target) && desc_valid(tokens) && desc_valid(accept) && desc_valid(sample) && desc_valid(out) &&
                   desc_valid(taken) && (!draft || desc_valid(draft)) && (!counts || desc_valid(counts)),
               THIN_ERR_INVALID, "verify_drafts: invalid descriptor");
  THIN_REQUIRE(float_type(target->dtype) && target->rank == 3 && target->sizes[1] >= 1, THIN_ERR_INVALID,
               "verify_drafts takes float16, bfloat16 or float32 target probabilities [batch, drafts + 1, vocab]");
  const int64_t B = target->sizes[0], K = target->sizes[1] - 1, V = target->sizes[2];
  THIN_REQUIRE(!draft || (draft->dtype == target->dtype && draft->rank == 3 && draft->sizes[0] == B && draft->sizes[1] == K &&
                          draft->sizes[2] == V),
               THIN_ERR_INVALID, "verify_drafts takes draft probabilities [batch, drafts, vocab] of the target's type");
  THIN_REQUIRE(tokens->rank == 2 && tokens->dtype == THIN_I64 && tokens->sizes[0] == B && tokens->sizes[1] == K &&
                   accept->rank == 2 && accept->dtype == THIN_F32 && accept->sizes[0] == B && accept->sizes[1] == K &&
                   sample->rank == 1 && sample->dtype == THIN_F32 && sample->sizes[0] == B &&
                   (!counts || (counts->rank == 1 && counts->dtype == THIN_I32 && counts->sizes[0] == B)),
               THIN_ERR_INVALID,
               "verify_drafts takes int64 tokens and float32 accept [batch, drafts], float32 sample and int32 counts [batch]");
  THIN_REQUIRE(out->rank == 2 && out->dtype == THIN_I64 && out->sizes[0] == B && out->sizes[1] == K + 1 && taken->rank == 1 &&
                   taken->dtype == THIN_I32 && taken->sizes[0] == B,
               THIN_ERR_INVALID, "verify_drafts writes int64 tokens [batch, drafts + 1] and int32 taken [batch]");
  THIN_REQUIRE(V >= 1, THIN_ERR_INVALID, "verify_drafts needs a vocabulary");
  THIN_REQUIRE(K <= kMaxDrafts && V <= kMaxVocab, THIN_ERR_UNSUPPORTED,
               "verify_drafts takes up to %lld drafts of up to %lld tokens", (long long)kMaxDrafts, (long long)kMaxVocab);
  THIN_REQUIRE(V == 1 || (target->strides[2] == 1 && (!draft || draft->strides[2] == 1)), THIN_ERR_UNSUPPORTED,
               "verify_drafts: the probabilities of a row must be adjacent");
  if (B == 0) return THIN_OK;
  THIN_REQUIRE(B < (1ll << 24), THIN_ERR_UNSUPPORTED, "verify_drafts: tensor too large");
  const int64_t tiles = tiles_of(V);
  THIN_REQUIRE(launchable(B * tiles, 256), THIN_ERR_UNSUPPORTED, "verify_drafts: tensor too large");
  const thin_desc* outs[2] = {out, taken};
  for (const thin_desc* o : outs) {
    THIN_REQUIRE(!repeats(o), THIN_ERR_INVALID, "verify_drafts: an output has a stride of 0");
    for (const thin_desc* in : {target, draft, tokens, counts, accept, sample})
      THIN_REQUIRE(!in || !overlap(o, in), THIN_ERR_INVALID, "verify_drafts: an output overlaps an input");
  }
  THIN_REQUIRE(!overlap(out, taken), THIN_ERR_INVALID, "verify_drafts: two outputs overlap");
  const size_t need = thin_verify_drafts_workspace(B, V);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "verify_drafts needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  THIN_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, THIN_ERR_WORKSPACE,
               "verify_drafts: the workspace must be 8-byte aligned");
  DraftPlan p;
  memset(&p, 0, sizeof p);
  p.target = target->data;
  p.pb = target->strides[0];
  p.pk = target->strides[1];
  if (draft && K > 0) {
    p.draft = draft->data;
    p.qb = draft->strides[0];
    p.qk = draft->strides[1];
  }
  p.tokens = static_cast<const int64_t*>(tokens->data);
  p.tb = tokens->strides[0]; p.tk = tokens->strides[1];
  if (counts) {
    p.counts = static_cast<const int32_t*>(counts->data);
    p.count_step = counts->strides[0];
  }
  p.accept = static_cast<const float*>(accept->data);
  p.ub = accept->strides[0]; p.uk = accept->strides[1];
  p.sample = static_cast<const float*>(sample->data);
  p.sample_step = sample->strides[0];
  p.out = static_cast<int64_t*>(out->data);
  p.ob = out->strides[0]; p.ok = out->strides[1];
  p.taken = static_cast<int32_t*>(taken->data);
  p.taken_step = taken->strides[0];
  p.drafts = (uint32_t)K;
  p.vocab = (uint32_t)V;
  p.tiles = (uint32_t)tiles;
  p.per = (uint32_t)per_of(B, V);
  p.groups = (uint32_t)((tiles + p.per - 1) / p.per);
  p.by_groups = FastDiv::make(p.groups);
  if (tiles > 1) {
    p.sums = static_cast<double*>(workspace);
    p.stayed = reinterpret_cast<int32_t*>(p.sums + 2 * B * tiles);
  }
  return with_float_type(target->dtype, [&](auto zero) {
    using T = decltype(zero);
    return launch<T>(p, B, stream);
  });
}
