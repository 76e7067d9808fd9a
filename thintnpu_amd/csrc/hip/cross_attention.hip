// Cross attention: queries to an encoder's states of another length, with a
// length or a mask for each sample and heads that share keys (attend.h has the
// kernels and their mathematics).
#include "attend.h"

#include <math.h>
#include <string.h>

using namespace thin;

extern "C" size_t thin_cross_attention_workspace(const thin_desc* q, const thin_desc* k) {
  if (!desc_valid(q) || !desc_valid(k) || q->rank != 4 || k->rank != 4 || k->sizes[2] <= 0) return 0;
  return attend_workspace(q->sizes[0], k->sizes[2], q->sizes[1] * (q->sizes[2] / k->sizes[2]), k->sizes[1], q->sizes[3],
                          false);
}

extern "C" thin_status thin_cross_attention(const thin_desc* q, const thin_desc* k, const thin_desc* v,
                                            const thin_desc* lengths, const thin_desc* mask, float scale,
                                            const thin_desc* out, void* workspace, size_t workspace_bytes,
                                            hipStream_t stream) {
  clear_error();
  THIN_REQUIRE(desc_valid(q) && desc_valid(k) && desc_valid(v) && desc_valid(out) && (!lengths || desc_valid(lengths)) &&
                   (!mask || desc_valid(mask)),
               THIN_ERR_INVALID, "cross_attention: invalid descriptor");
  THIN_REQUIRE((q->dtype == THIN_F16 || q->dtype == THIN_BF16) && k->dtype == q->dtype && v->dtype == q->dtype &&
                   out->dtype == q->dtype,
               THIN_ERR_INVALID, "cross_attention takes float16 or bfloat16 q, k, v and out of one type");
  THIN_REQUIRE(q->rank == 4 && k->rank == 4 && v->rank == 4, THIN_ERR_INVALID,
               "cross_attention takes q [batch, tokens, heads, dim], k and v [batch, states, heads, dim]");
  THIN_REQUIRE(same_sizes(q, out) && same_sizes(k, v), THIN_ERR_INVALID,
               "cross_attention: out has q's sizes, v has k's");
  const int64_t B = q->sizes[0], T = q->sizes[1], H = q->sizes[2], D = q->sizes[3], S = k->sizes[1], Hk = k->sizes[2];
  THIN_REQUIRE(k->sizes[0] == B && k->sizes[3] == D, THIN_ERR_INVALID, "cross_attention: k does not fit q");
  THIN_REQUIRE(Hk >= 1 && H % Hk == 0, THIN_ERR_INVALID, "cross_attention: %lld heads do not share %lld", (long long)H,
               (long long)Hk);
  THIN_REQUIRE(D >= 8 && D <= 256 && D % 8 == 0, THIN_ERR_UNSUPPORTED,
               "cross_attention takes heads of 8 to 256 dims, a multiple of 8, not %lld", (long long)D);
  THIN_REQUIRE(!lengths || (lengths->rank == 1 && lengths->dtype == THIN_I32 && lengths->sizes[0] == B), THIN_ERR_INVALID,
               "cross_attention takes int32 lengths [batch]");
  THIN_REQUIRE(!mask || (mask->rank == 2 && mask->dtype == THIN_U8 && mask->sizes[0] == B && mask->sizes[1] == S),
               THIN_ERR_INVALID, "cross_attention takes a mask [batch, states] of bytes");
  THIN_REQUIRE(q->strides[3] == 1 && k->strides[3] == 1 && v->strides[3] == 1 && out->strides[3] == 1, THIN_ERR_UNSUPPORTED,
               "cross_attention: the dims of a head must be adjacent");
  THIN_REQUIRE(S <= 1 || (k->strides[1] < (1ll << 25) && v->strides[1] < (1ll << 25)), THIN_ERR_UNSUPPORTED,
               "cross_attention: neighbouring states must be less than 2^25 elements apart");
  const float c = scale * 1.4426950408889634f;
  THIN_REQUIRE(isnormal(c) && c > 0.f, THIN_ERR_INVALID, "cross_attention: the scale must be positive and finite");
  if (numel(q) == 0) return THIN_OK;
  const int64_t rows = T * (H / Hk), blocks = row_blocks_of(rows, false);
  THIN_REQUIRE(rows < (1ll << 30) && S < (1ll << 30) && B < (1ll << 30) && launchable(B * Hk * blocks, 256) &&
                   launchable(B * Hk * rows, 256),
               THIN_ERR_UNSUPPORTED, "cross_attention: tensor too large");
  THIN_REQUIRE(!repeats(out), THIN_ERR_INVALID, "cross_attention: out has a stride of 0");
  for (const thin_desc* in : {q, k, v, lengths, mask})
    THIN_REQUIRE(!in || !overlap(out, in), THIN_ERR_INVALID, "cross_attention: out overlaps an input");
  const size_t need = attend_workspace(B, Hk, rows, S, D, false);
  THIN_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), THIN_ERR_WORKSPACE,
               "cross_attention needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  THIN_REQUIRE(need == 0 || workspace_aligned(workspace), THIN_ERR_WORKSPACE,
               "cross_attention: the workspace must be 4-byte aligned");
  AttendPlan p;
  plan_attend(p, q, out, Hk, S, false, c, workspace);
  if (lengths) {
    p.lengths = static_cast<const int32_t*>(lengths->data);
    p.length_step = lengths->strides[0];
  }
  p.k = {k->data, k->strides[0], k->strides[1], k->strides[2]};
  p.v = {v->data, v->strides[0], v->strides[1], v->strides[2]};
  if (mask) {
    p.mask = static_cast<const uint8_t*>(mask->data);
    p.mask_batch = mask->strides[0];
    p.mask_key = mask->strides[1];
  }
  if (q->dtype == THIN_F16) return launch_attend_type<_Float16, false>(p, stream);
  return launch_attend_type<__bf16, false>(p, stream);
}
