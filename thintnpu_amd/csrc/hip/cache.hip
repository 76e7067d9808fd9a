// A cache of keys and values in 8 bits: pages of e4m3 codes, a scale for each
// page and head.
//
//   write: s = the least 2^e with max |x| <= 448 2^e over a page's tokens,
//          code = e4m3(x / s); a page that holds earlier tokens keeps its scale
//          unless a new token needs a larger one, and then their codes become
//          e4m3(code s_old / s).
//
// A power of two costs e4m3 no precision (its steps go by the exponent), makes
// x / s exact, so that a code is one rounding of its value, and rounds an
// earlier token a second time only where it becomes subnormal.
//
// Attention over the pages: attend.h.
#include "attend.h"

#include <math.h>

namespace thin {
namespace {

constexpr float kTop = 448.f;  // the largest code
constexpr int kLeast = -110;   // scales from 2^-110: s and 1 / s are normal with every code

struct WritePlan {
  const void* k;
  const void* v;
  int64_t k_batch, k_token, k_head, v_batch, v_token, v_head;
  PagesOf kp, vp;
  float* k_scales;
  float* v_scales;
  uint8_t* k_codes;
  uint8_t* v_codes;
  const int32_t* table;
  int64_t table_batch, table_slot;
  const int32_t* lengths;
  const int32_t* counts;
  int64_t length_step, count_step;
  uint32_t batch, tokens, heads, dim, spans, page_size, slots, pages;
  FastDiv by_heads, by_spans, by_pieces;
  uint64_t units;
};

// 2^e, the least with amax <= 448 * 2^e = 1.75 * 2^(8 + e).
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __builtin_bit_cast(float, (uint32_t)(max(e, kLeast) + 127) << 23);
}

// x / s in codes; infinities become the largest code, NaN stays NaN.
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
  const auto fit = [](float x) { return x > kTop ? kTop : x < -kTop ? -kTop : x; };
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(fit(a), fit(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fit(c), fit(d), w, true);
}

// One wavefront for the new tokens of a page and head: 16 values a lane, once for
// their maximum, once for their codes (from L2: held in registers in between they
// took as long).  Bound by the chain of count, page, scale, values and codes, some 5
// us of it for one token of 48 sequences, and by memory behind that (6 x 8 heads of
// prompts of 2048 tokens at most, 128 dims, pages of 32: 14 us, 2.7 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void write_kernel(WritePlan p) {
  const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t lane = threadIdx.x & 63u;
  if (unit >= p.units) return;
  const uint32_t u = (uint32_t)(unit >> 1), value = (uint32_t)unit & 1u;
  const uint32_t r = p.by_heads.div(u), h = u - r * p.heads, b = p.by_spans.div(r), span = r - b * p.spans;
  const int32_t n = max(0, min(p.counts ? p.counts[b * p.count_step] : (int32_t)p.tokens, (int32_t)p.tokens));
  const int32_t begin = max(p.lengths[b * p.length_step], 0) - n;  // of the first new token
  const int64_t slot = max(begin, 0) / p.page_size + span;
  if (slot >= p.slots) return;
  const int64_t page_at = slot * p.page_size;
  const int64_t low = max(page_at, (int64_t)begin), high = min(page_at + p.page_size, (int64_t)begin + n);
  if (low >= high) return;
  const int32_t id = p.table[b * p.table_batch + slot * p.table_slot];
  if ((uint32_t)id >= p.pages) return;
  const PagesOf& to = value ? p.vp : p.kp;
  const uint32_t off = (uint32_t)(low - page_at), count = (uint32_t)(high - low);
  const int64_t token = value ? p.v_token : p.k_token;
  const T* x = static_cast<const T*>(value ? p.v : p.k) + b * (value ? p.v_batch : p.k_batch) +
               h * (value ? p.v_head : p.k_head) + (low - begin) * token;
  uint8_t* codes = (value ? p.v_codes : p.k_codes) + id * to.page + h * to.head;
  float* scale = (value ? p.v_scales : p.k_scales) + id * to.scale_page + h * to.scale_head;
  const float was = off ? *scale : 0.f;

  const uint32_t per = p.dim / 16, pieces = count * per;
  float amax = 0.f;
  for (uint32_t i = lane; i < pieces; i += 64) {
    const uint32_t t = p.by_pieces.div(i);
    float v[16];
    dev::load_pack<T, 16>(x + t * token + (i - t * per) * 16, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = __builtin_fabsf(v[j]);
      amax = a <= 3.4028235e38f ? fmaxf(amax, a) : amax;  // neither infinities nor NaN
    }
  }
  amax = dev::group_max<64>(amax);
  const bool keeps = off && was > 0.f && was <= 3.4028235e38f;
  float s = amax > 0.f ? scale_for(amax) : keeps ? was : 1.f;
  if (keeps && was >= s) s = was;
  // 1 / s is exact for powers of two, which all scales written here are
  const bool exact = (__builtin_bit_cast(uint32_t, s) & 0x7FFFFFu) == 0;
  const float inv = 1.f / s;
  if (off && s != was) {
    for (uint32_t i = lane; i < off * per; i += 64) {
      const uint32_t t = p.by_pieces.div(i);
      dev::u4e* at = reinterpret_cast<dev::u4e*>(codes + t * to.token + (i - t * per) * 16);
      dev::u4 w = *at;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], true);
        w[j] = code4(lo[0] * was / s, lo[1] * was / s, hi[0] * was / s, hi[1] * was / s);
      }
      *at = w;
    }
  }
  for (uint32_t i = lane; i < pieces; i += 64) {
    const uint32_t t = p.by_pieces.div(i);
    float v[16];
    dev::load_pack<T, 16>(x + t * token + (i - t * per) * 16, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = exact ? v[j] * inv : v[j] / s;
    dev::u4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = code4(v[j * 4], v[j * 4 + 1], v[j * 4 + 2], v[j * 4 + 3]);
    *reinterpret_cast<dev::u4e*>(codes + (off + t) * to.token + (i - t * per) * 16) = w;
  }
  if (lane == 0) *scale = s;
}

// What both operators ask of a cache for `heads` heads of `dim` dims.
thin_status check_cache(const char* name, const thin_desc* kc, const thin_desc* vc, const thin_desc* ks, const thin_desc* vs,
                        const thin_desc* table, const thin_desc* lengths, const thin_desc* counts, int64_t batch,
                        int64_t dim) {
  THIN_REQUIRE(kc->rank == 4 && kc->dtype == THIN_U8 && vc->dtype == THIN_U8 && same_sizes(kc, vc), THIN_ERR_INVALID,
               "%s takes k and v codes [pages, heads, page, dim] of bytes", name);
  const int64_t P = kc->sizes[0], H = kc->sizes[1], page = kc->sizes[2], D = kc->sizes[3];
  THIN_REQUIRE(D == dim, THIN_ERR_INVALID, "%s: a cache of %lld dims a head, rows of %lld", name, (long long)D, (long long)dim);
  THIN_REQUIRE(ks->rank == 2 && ks->dtype == THIN_F32 && ks->sizes[0] == P && ks->sizes[1] == H && vs->dtype == THIN_F32 &&
                   same_sizes(ks, vs),
               THIN_ERR_INVALID, "%s takes float32 scales [pages, heads]", name);
  THIN_REQUIRE(table->rank == 2 && table->dtype == THIN_I32 && table->sizes[0] == batch && lengths->rank == 1 &&
                   lengths->dtype == THIN_I32 && lengths->sizes[0] == batch &&
                   (!counts || (counts->rank == 1 && counts->dtype == THIN_I32 && counts->sizes[0] == batch)),
               THIN_ERR_INVALID, "%s takes int32 table [batch, slots], lengths [batch] and counts [batch]", name);
  THIN_REQUIRE(D >= 16 && D <= 256 && D % 16 == 0 && page >= 16 && page <= 1024 && page % 16 == 0, THIN_ERR_UNSUPPORTED,
               "%s takes heads of 16 to 256 dims and pages of 16 to 1024 tokens, multiples of 16, not %lld and %lld", name,
               (long long)D, (long long)page);
  THIN_REQUIRE(kc->strides[3] == 1 && vc->strides[3] == 1, THIN_ERR_UNSUPPORTED, "%s: the codes of a token must be adjacent",
               name);
  THIN_REQUIRE(kc->strides[2] < (1ll << 26) && vc->strides[2] < (1ll << 26), THIN_ERR_UNSUPPORTED,
               "%s: neighbouring tokens must be less than 2^26 bytes apart", name);
  THIN_REQUIRE(P < (1ll << 30) && table->sizes[1] < (1ll << 30) / page, THIN_ERR_UNSUPPORTED, "%s: tensor too large", name);
  return THIN_OK;
}

PagesOf pages_of(const thin_desc* codes, const thin_desc* scales) {
  return {static_cast<const uint8_t*>(codes->data), static_cast<const float*>(scales->data), codes->strides[0],
          codes->strides[1], codes->strides[2], scales->strides[0], scales->strides[1]};
}

}  // namespace
}  // namespace thin

using namespace thin;

extern "C" thin_status thin_cache_write(const thin_desc* k, const thin_desc* v, const thin_desc* k_cache,
                                        const thin_desc* v_cache, const thin_desc* k_scales, const thin_desc* v_scales,
                                        const thin_desc* table, const thin_desc* lengths, const thin_desc* counts,
                                        hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(k) && desc_valid(v) && desc_valid(k_cache) && desc_valid(v_cache) && desc_valid(k_scales) &&
                   desc_valid(v_scales) && desc_valid(table) && desc_valid(lengths) && (!counts || desc_valid(counts)),
               THIN_ERR_INVALID, "cache_write: invalid descriptor");
  THIN_REQUIRE(float_type(k->dtype) && v->dtype == k->dtype && k->rank == 4 && same_sizes(k, v), THIN_ERR_INVALID,
               "cache_write takes float16, bfloat16 or float32 k and v [batch, tokens, heads, dim] of one type");
  const int64_t B = k->sizes[0], T = k->sizes[1], H = k->sizes[2], D = k->sizes[3];
  const thin_status fits =
      check_cache("cache_write", k_cache, v_cache, k_scales, v_scales, table, lengths, counts, B, D);
  if (fits != THIN_OK) return fits;
  THIN_REQUIRE(k_cache->sizes[1] == H, THIN_ERR_INVALID, "cache_write: k of %lld heads, a cache of %lld", (long long)H,
               (long long)k_cache->sizes[1]);
  THIN_REQUIRE(k->strides[3] == 1 && v->strides[3] == 1, THIN_ERR_UNSUPPORTED,
               "cache_write: the dims of a head must be adjacent");
  const int64_t P = k_cache->sizes[0], page = k_cache->sizes[2], slots = table->sizes[1];
  if (numel(k) == 0 || P == 0 || slots == 0) return THIN_OK;
  THIN_REQUIRE(T < (1ll << 30) && B < (1ll << 30), THIN_ERR_UNSUPPORTED, "cache_write: tensor too large");
  const int64_t spans = (T + page - 2) / page + 1 < slots ? (T + page - 2) / page + 1 : slots;
  THIN_REQUIRE(H < (1ll << 30) && B * spans < (1ll << 30) && B * spans * H < (1ll << 30) &&
                   launchable((B * spans * H * 2 + 3) / 4, 256),
               THIN_ERR_UNSUPPORTED, "cache_write: tensor too large");
  const thin_desc* outs[4] = {k_cache, v_cache, k_scales, v_scales};
  for (int i = 0; i < 4; ++i) {
    THIN_REQUIRE(!repeats(outs[i]), THIN_ERR_INVALID, "cache_write: the cache has a stride of 0");
    for (const thin_desc* in : {k, v, table, lengths, counts})
      THIN_REQUIRE(!in || !overlap(outs[i], in), THIN_ERR_INVALID, "cache_write: the cache overlaps an input");
    for (int j = 0; j < i; ++j)
      THIN_REQUIRE(!overlap(outs[i], outs[j]), THIN_ERR_INVALID, "cache_write: two parts of the cache overlap");
  }
  WritePlan p;
  memset(&p, 0, sizeof p);
  p.k = k->data;
  p.v = v->data;
  p.k_batch = k->strides[0]; p.k_token = k->strides[1]; p.k_head = k->strides[2];
  p.v_batch = v->strides[0]; p.v_token = v->strides[1]; p.v_head = v->strides[2];
  p.kp = pages_of(k_cache, k_scales);
  p.vp = pages_of(v_cache, v_scales);
  p.k_codes = static_cast<uint8_t*>(k_cache->data);
  p.v_codes = static_cast<uint8_t*>(v_cache->data);
  p.k_scales = static_cast<float*>(k_scales->data);
  p.v_scales = static_cast<float*>(v_scales->data);
  p.table = static_cast<const int32_t*>(table->data);
  p.table_batch = table->strides[0];
  p.table_slot = table->strides[1];
  p.lengths = static_cast<const int32_t*>(lengths->data);
  p.length_step = lengths->strides[0];
  if (counts) {
    p.counts = static_cast<const int32_t*>(counts->data);
    p.count_step = counts->strides[0];
  }
  p.batch = (uint32_t)B;
  p.tokens = (uint32_t)T;
  p.heads = (uint32_t)H;
  p.dim = (uint32_t)D;
  p.spans = (uint32_t)spans;
  p.page_size = (uint32_t)page;
  p.slots = (uint32_t)slots;
  p.pages = (uint32_t)P;
  p.by_heads = FastDiv::make(p.heads);
  p.by_spans = FastDiv::make(p.spans);
  p.by_pieces = FastDiv::make(p.dim / 16);
  p.units = (uint64_t)B * spans * H * 2;
  return with_float_type(k->dtype, [&](auto zero) {
    using T_ = decltype(zero);
    hipLaunchKernelGGL((write_kernel<T_>), dim3((uint32_t)((p.units + 3) / 4)), dim3(256), 0, stream, p);
    THIN_LAUNCH_CHECK("cache_write");
    return THIN_OK;
  });
}

extern "C" size_t thin_cache_attention_workspace(const thin_desc* q, const thin_desc* k_cache, const thin_desc* table) {
  if (!desc_valid(q) || !desc_valid(k_cache) || !desc_valid(table) || q->rank != 4 || k_cache->rank != 4 ||
      table->rank != 2 || k_cache->sizes[1] <= 0)
    return 0;
  return attend_workspace(q->sizes[0], k_cache->sizes[1], q->sizes[1] * (q->sizes[2] / k_cache->sizes[1]),
                          table->sizes[1] * k_cache->sizes[2], q->sizes[3], true);
}

extern "C" thin_status thin_cache_attention(const thin_desc* q, const thin_desc* k_cache, const thin_desc* v_cache,
                                            const thin_desc* k_scales, const thin_desc* v_scales, const thin_desc* table,
                                            const thin_desc* lengths, const thin_desc* counts, float scale,
                                            const thin_desc* out, void* workspace, size_t workspace_bytes,
                                            hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(q) && desc_valid(k_cache) && desc_valid(v_cache) && desc_valid(k_scales) && desc_valid(v_scales) &&
                   desc_valid(table) && desc_valid(lengths) && desc_valid(out) && (!counts || desc_valid(counts)),
               THIN_ERR_INVALID, "cache_attention: invalid descriptor");
  THIN_REQUIRE((q->dtype == THIN_F16 || q->dtype == THIN_BF16) && out->dtype == q->dtype && q->rank == 4 && same_sizes(q, out),
               THIN_ERR_INVALID,
               "cache_attention takes float16 or bfloat16 q [batch, tokens, heads, dim], and out of its type and sizes");
  const int64_t B = q->sizes[0], T = q->sizes[1], H = q->sizes[2], D = q->sizes[3];
  const thin_status fits =
      check_cache("cache_attention", k_cache, v_cache, k_scales, v_scales, table, lengths, counts, B, D);
  if (fits != THIN_OK) return fits;
  const int64_t P = k_cache->sizes[0], Hk = k_cache->sizes[1], page = k_cache->sizes[2], S = table->sizes[1] * page;
  THIN_REQUIRE(Hk >= 1 && H % Hk == 0, THIN_ERR_INVALID, "cache_attention: %lld heads do not share %lld", (long long)H,
               (long long)Hk);
  THIN_REQUIRE(q->strides[3] == 1 && out->strides[3] == 1, THIN_ERR_UNSUPPORTED,
               "cache_attention: the dims of a head must be adjacent");
  const float c = scale * 1.4426950408889634f;
  THIN_REQUIRE(isnormal(c) && c > 0.f, THIN_ERR_INVALID, "cache_attention: the scale must be positive and finite");
  if (numel(q) == 0) return THIN_OK;
  const int64_t rows = T * (H / Hk), blocks = row_blocks_of(rows, true);
  THIN_REQUIRE(rows < (1ll << 30) && B < (1ll << 30) && launchable(B * Hk * blocks, 256) &&
                   launchable(B * Hk * rows, 256),
               THIN_ERR_UNSUPPORTED, "cache_attention: tensor too large");
  THIN_REQUIRE(!repeats(out), THIN_ERR_INVALID, "cache_attention: out has a stride of 0");
  for (const thin_desc* in : {q, k_cache, v_cache, k_scales, v_scales, table, lengths, counts})
    THIN_REQUIRE(!in || !overlap(out, in), THIN_ERR_INVALID, "cache_attention: out overlaps an input");
  const size_t need = attend_workspace(B, Hk, rows, S, D, true);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "cache_attention needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  THIN_REQUIRE(need == 0 || workspace_aligned(workspace), THIN_ERR_WORKSPACE,
               "cache_attention: the workspace must be 4-byte aligned");
  AttendPlan p;
  plan_attend(p, q, out, Hk, S, true, c, workspace);
  p.lengths = static_cast<const int32_t*>(lengths->data);
  p.length_step = lengths->strides[0];
  if (counts) {
    p.counts = static_cast<const int32_t*>(counts->data);
    p.count_step = counts->strides[0];
  }
  p.kp = pages_of(k_cache, k_scales);
  p.vp = pages_of(v_cache, v_scales);
  p.table = static_cast<const int32_t*>(table->data);
  p.table_batch = table->strides[0];
  p.table_slot = table->strides[1];
  p.page_size = (uint32_t)page;
  p.pages = (uint32_t)P;
  p.by_page = FastDiv::make(p.page_size);
  if (q->dtype == THIN_F16) return launch_attend_type<_Float16, true>(p, stream);
  return launch_attend_type<__bf16, true>(p, stream);
}
