// thin_fused kernels of rotary positions, cross attention, the 8-bit cache and
// the verification of drafts on the PrivateUse1 backend: checks, outputs and
// workspace around the thin_hip C ABI.  None has a counterpart among the
// reference's operators (include/thin_hip.h names what each stands beside).
#include "thin_runtime.h"

#include <torch/library.h>

#include <cmath>
#include <tuple>
#include <vector>

namespace thin_decode {
using namespace thin_rt;

using Maybe = std::optional<at::Tensor>;

struct MaybeDesc {
  thin_desc d;
  const thin_desc* ptr = nullptr;
  MaybeDesc(const Maybe& t, const char* what) {
    if (!t || !t->defined()) return;
    inference(*t, what);
    d = desc(*t);
    ptr = &d;
  }
};
thin_desc operand(const at::Tensor& t, const char* what) {
  inference(t, what);
  return desc(t);
}
bool given(const Maybe& t) { return t && t->defined(); }
at::Tensor dense_like(const at::Tensor& x) {
  return at::empty(x.sizes(), x.options().memory_format(c10::MemoryFormat::Contiguous));
}
bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// ------------------------------------------------------------------ rotary positions
std::vector<at::Tensor> rotary_outputs(const at::Tensor& q, const Maybe& k) {
  TORCH_CHECK((half_type(q) || q.scalar_type() == at::kFloat) && q.dim() == 4,
              "rotary_axes takes float16, bfloat16 or float32 q [batch, tokens, heads, dim]");
  std::vector<at::Tensor> out{dense_like(q)};
  if (given(k)) out.push_back(dense_like(*k));
  return out;
}
std::vector<at::Tensor> rotary_axes(const at::Tensor& q, const at::Tensor& positions, const at::Tensor& freqs,
                                    const at::Tensor& axes, const Maybe& k, bool interleaved, bool inverse) {
  const char* what = "thin_fused.rotary_axes";
  const thin_desc qd = operand(q, what), pd = operand(positions, what), fd = operand(freqs, what), ad = operand(axes, what);
  MaybeDesc kd(k, what);
  select(q.device());
  std::vector<at::Tensor> out = rotary_outputs(q, k);
  const thin_desc qo = desc(out[0]);
  thin_desc ko{};
  if (kd.ptr) ko = desc(out[1]);
  check(thin_rotary_axes(&qd, kd.ptr, &pd, &fd, &ad, interleaved ? 1 : 0, inverse ? 1 : 0, &qo, kd.ptr ? &ko : nullptr,
                         stream()),
        "thin rotary_axes");
  after_launch();
  return out;
}
std::vector<at::Tensor> rotary_axes_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                         const Maybe& k, bool, bool) {
  return rotary_outputs(q, k);
}

// ------------------------------------------------------------------ cross attention
at::Tensor attended(const at::Tensor& q, const char* name) {
  TORCH_CHECK(half_type(q) && q.dim() == 4, name, " takes float16 or bfloat16 q [batch, tokens, heads, dim]");
  return dense_like(q);
}
float scale_of(const at::Tensor& q, std::optional<double> scale) {
  return scale ? (float)*scale : (float)(1.0 / std::sqrt((double)q.size(-1)));
}
at::Tensor cross_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Maybe& lengths,
                           const Maybe& mask, std::optional<double> scale) {
  const char* what = "thin_fused.cross_attention";
  const thin_desc qd = operand(q, what), kd = operand(k, what), vd = operand(v, what);
  MaybeDesc ld(lengths, what), md(mask, what);
  select(q.device());
  at::Tensor out = attended(q, "cross_attention");
  const thin_desc od = desc(out);
  const size_t bytes = thin_cross_attention_workspace(&qd, &kd);
  at::Tensor ws;
  if (bytes) ws = empty_bytes((int64_t)bytes);
  check(thin_cross_attention(&qd, &kd, &vd, ld.ptr, md.ptr, scale_of(q, scale), &od, bytes ? ws.data_ptr() : nullptr, bytes,
                             stream()),
        "thin cross_attention");
  after_launch();
  return out;
}
at::Tensor cross_attention_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const Maybe&, const Maybe&,
                                std::optional<double>) {
  return attended(q, "cross_attention");
}

// ------------------------------------------------------------------ cache
// The codes are bytes on this device.
void cache_write(const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache, at::Tensor& v_cache, at::Tensor& k_scales,
                 at::Tensor& v_scales, const at::Tensor& table, const at::Tensor& lengths, const Maybe& counts) {
  const char* what = "thin_fused.cache_write";
  const thin_desc kd = operand(k, what), vd = operand(v, what), kc = operand(k_cache, what), vc = operand(v_cache, what),
                  ks = operand(k_scales, what), vs = operand(v_scales, what), td = operand(table, what),
                  ld = operand(lengths, what);
  MaybeDesc cd(counts, what);
  select(k.device());
  check(thin_cache_write(&kd, &vd, &kc, &vc, &ks, &vs, &td, &ld, cd.ptr, stream()), "thin cache_write");
  after_launch();
}
void cache_write_meta(const at::Tensor&, const at::Tensor&, at::Tensor&, at::Tensor&, at::Tensor&, at::Tensor&,
                      const at::Tensor&, const at::Tensor&, const Maybe&) {}
at::Tensor cache_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& table,
                           const at::Tensor& lengths, const Maybe& counts, std::optional<double> scale) {
  const char* what = "thin_fused.cache_attention";
  const thin_desc qd = operand(q, what), kc = operand(k_cache, what), vc = operand(v_cache, what), ks = operand(k_scales, what),
                  vs = operand(v_scales, what), td = operand(table, what), ld = operand(lengths, what);
  MaybeDesc cd(counts, what);
  select(q.device());
  at::Tensor out = attended(q, "cache_attention");
  const thin_desc od = desc(out);
  const size_t bytes = thin_cache_attention_workspace(&qd, &kc, &td);
  at::Tensor ws;
  if (bytes) ws = empty_bytes((int64_t)bytes);
  check(thin_cache_attention(&qd, &kc, &vc, &ks, &vs, &td, &ld, cd.ptr, scale_of(q, scale), &od,
                             bytes ? ws.data_ptr() : nullptr, bytes, stream()),
        "thin cache_attention");
  after_launch();
  return out;
}
at::Tensor cache_attention_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                const at::Tensor&, const at::Tensor&, const at::Tensor&, const Maybe&,
                                std::optional<double>) {
  return attended(q, "cache_attention");
}

// ------------------------------------------------------------------ drafts
using Pair = std::tuple<at::Tensor, at::Tensor>;
Pair verify_outputs(const at::Tensor& target) {
  TORCH_CHECK((half_type(target) || target.scalar_type() == at::kFloat) && target.dim() == 3 && target.size(1) >= 1,
              "verify_drafts takes float16, bfloat16 or float32 target probabilities [batch, drafts + 1, vocab]");
  return {at::empty({target.size(0), target.size(1)}, target.options().dtype(at::kLong)),
          at::empty({target.size(0)}, target.options().dtype(at::kInt))};
}
Pair verify_drafts(const at::Tensor& target, const Maybe& draft, const at::Tensor& tokens, const at::Tensor& accept,
                   const at::Tensor& sample, const Maybe& counts) {
  const char* what = "thin_fused.verify_drafts";
  const thin_desc pd = operand(target, what), td = operand(tokens, what), ad = operand(accept, what), sd = operand(sample, what);
  MaybeDesc qd(draft, what), cd(counts, what);
  select(target.device());
  Pair out = verify_outputs(target);
  const thin_desc od = desc(std::get<0>(out)), nd = desc(std::get<1>(out));
  const size_t bytes = thin_verify_drafts_workspace(target.size(0), target.size(2));
  at::Tensor ws;
  if (bytes) ws = empty_bytes((int64_t)bytes);
  check(thin_verify_drafts(&pd, qd.ptr, &td, cd.ptr, &ad, &sd, &od, &nd, bytes ? ws.data_ptr() : nullptr, bytes, stream()),
        "thin verify_drafts");
  after_launch();
  return out;
}
Pair verify_drafts_meta(const at::Tensor& target, const Maybe&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const Maybe&) {
  return verify_outputs(target);
}

}  // namespace thin_decode

TORCH_LIBRARY_FRAGMENT(thin_fused, m) {
  m.def("rotary_axes(Tensor q, Tensor positions, Tensor freqs, Tensor axes, Tensor? k=None, bool interleaved=False, "
        "bool inverse=False) -> Tensor[]");
  m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? lengths=None, Tensor? mask=None, float? scale=None) -> Tensor");
  m.def("cache_write(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, "
        "Tensor(d!) v_scales, Tensor table, Tensor lengths, Tensor? counts=None) -> ()");
  m.def("cache_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, Tensor table, "
        "Tensor lengths, Tensor? counts=None, float? scale=None) -> Tensor");
  m.def("verify_drafts(Tensor target, Tensor? draft, Tensor tokens, Tensor accept, Tensor sample, Tensor? counts=None) "
        "-> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(thin_fused, PrivateUse1, m) {
  m.impl("rotary_axes", TORCH_FN(thin_decode::rotary_axes));
  m.impl("cross_attention", TORCH_FN(thin_decode::cross_attention));
  m.impl("cache_write", TORCH_FN(thin_decode::cache_write));
  m.impl("cache_attention", TORCH_FN(thin_decode::cache_attention));
  m.impl("verify_drafts", TORCH_FN(thin_decode::verify_drafts));
}

TORCH_LIBRARY_IMPL(thin_fused, AutogradPrivateUse1, m) {
  for (const char* name : {"rotary_axes", "cross_attention", "cache_write", "cache_attention", "verify_drafts"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(thin_fused, Meta, m) {
  m.impl("rotary_axes", TORCH_FN(thin_decode::rotary_axes_meta));
  m.impl("cross_attention", TORCH_FN(thin_decode::cross_attention_meta));
  m.impl("cache_write", TORCH_FN(thin_decode::cache_write_meta));
  m.impl("cache_attention", TORCH_FN(thin_decode::cache_attention_meta));
  m.impl("verify_drafts", TORCH_FN(thin_decode::verify_drafts_meta));
}
