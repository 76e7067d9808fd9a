// thin_fused kernels of group norm, expert blocks and token log probabilities
// on the PrivateUse1 backend: checks, outputs and workspace around the
// thin_hip C ABI.  None has a counterpart among the reference's operators
// (include/thin_hip.h names what each stands beside).
#include "thin_runtime.h"

#include <torch/library.h>

#include <tuple>

namespace thin_score {
using namespace thin_rt;

bool row_type(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat;
}
using Maybe = std::optional<at::Tensor>;

// Descriptor of an optional operand, or null.
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

// ------------------------------------------------------------------ group norm
int64_t norm_channels(const at::Tensor& x, std::optional<int64_t> channels) {
  TORCH_CHECK(row_type(x), "group_norm takes float16, bfloat16 or float32");
  TORCH_CHECK(x.dim() >= 2, "group_norm takes x [N, ..., C]");
  TORCH_CHECK(!channels || (x.dim() == 5 && x.size(4) == 16), "group_norm with channels takes NC1HWC0 [N, C1, H, W, 16]");
  return channels ? *channels : x.size(-1);
}
at::Tensor group_norm(const at::Tensor& x, int64_t groups, const Maybe& weight, const Maybe& bias, double eps, bool silu,
                      std::optional<int64_t> channels) {
  inference(x, "thin_fused.group_norm");
  const int64_t c = norm_channels(x, channels);
  const int blocked = channels ? 1 : 0;
  select(x.device());
  auto out = at::empty(x.sizes(), x.options().memory_format(c10::MemoryFormat::Contiguous));
  thin_desc xd = desc(x), od = desc(out);
  MaybeDesc w(weight, "thin_fused.group_norm"), b(bias, "thin_fused.group_norm");
  const size_t bytes = thin_group_norm_workspace(&xd, &od, blocked, c, groups);
  at::Tensor ws;
  if (bytes) ws = empty_bytes((int64_t)bytes);
  check(thin_group_norm(&xd, blocked, c, groups, w.ptr, b.ptr, eps, silu ? 1 : 0, &od, bytes ? ws.data_ptr() : nullptr,
                        bytes, stream()),
        "thin group_norm");
  after_launch();
  return out;
}
at::Tensor group_norm_meta(const at::Tensor& x, int64_t, const Maybe&, const Maybe&, double, bool,
                           std::optional<int64_t> channels) {
  norm_channels(x, channels);
  return at::empty(x.sizes(), x.options().memory_format(c10::MemoryFormat::Contiguous));
}

// ------------------------------------------------------------------ experts
using Pair = std::tuple<at::Tensor, at::Tensor>;
using Triple = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
using Quad = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

Pair route_outputs(const at::Tensor& logits, int64_t k) {
  TORCH_CHECK(row_type(logits) && logits.dim() == 2,
              "expert_route takes float16, bfloat16 or float32 logits [tokens, experts]");
  TORCH_CHECK(k >= 1, "expert_route chooses at least one expert");
  return {at::empty({logits.size(0), k}, logits.options().dtype(at::kFloat)),
          at::empty({logits.size(0), k}, logits.options().dtype(at::kInt))};
}
Pair expert_route(const at::Tensor& logits, int64_t k, const Maybe& bias, bool softmax, int64_t groups,
                  int64_t top_groups, bool renormalize, double scale) {
  inference(logits, "thin_fused.expert_route");
  select(logits.device());
  Pair out = route_outputs(logits, k);
  thin_desc ld = desc(logits), wd = desc(std::get<0>(out)), ed = desc(std::get<1>(out));
  MaybeDesc b(bias, "thin_fused.expert_route");
  check(thin_expert_route(&ld, b.ptr, softmax ? 1 : 0, groups, top_groups, renormalize ? 1 : 0, (float)scale, &wd, &ed,
                          stream()),
        "thin expert_route");
  after_launch();
  return out;
}
Pair expert_route_meta(const at::Tensor& logits, int64_t k, const Maybe&, bool, int64_t, int64_t, bool, double) {
  return route_outputs(logits, k);
}

Triple dispatch_outputs(const at::Tensor& x, const at::Tensor& experts, int64_t count) {
  TORCH_CHECK(row_type(x) && x.dim() == 2, "expert_dispatch takes float16, bfloat16 or float32 x [tokens, width]");
  TORCH_CHECK(experts.scalar_type() == at::kInt && experts.dim() == 2 && experts.size(0) == x.size(0),
              "expert_dispatch takes int32 experts [tokens, k]");
  TORCH_CHECK(count >= 1, "expert_dispatch needs at least one expert");
  return {at::empty({experts.numel(), x.size(1)}, x.options()), at::empty({count + 1}, experts.options()),
          at::empty(experts.sizes(), experts.options().memory_format(c10::MemoryFormat::Contiguous))};
}
Triple expert_dispatch(const at::Tensor& x, const at::Tensor& experts, int64_t count) {
  inference(x, "thin_fused.expert_dispatch");
  inference(experts, "thin_fused.expert_dispatch");
  select(x.device());
  Triple out = dispatch_outputs(x, experts, count);
  thin_desc xd = desc(x), ed = desc(experts), rd = desc(std::get<0>(out)), od = desc(std::get<1>(out)),
            sd = desc(std::get<2>(out));
  const size_t bytes = thin_expert_dispatch_workspace(experts.size(0), experts.size(1), count);
  at::Tensor ws;
  if (bytes) ws = empty_bytes((int64_t)bytes);
  check(thin_expert_dispatch(&xd, &ed, count, &rd, &od, &sd, bytes ? ws.data_ptr() : nullptr, bytes, stream()),
        "thin expert_dispatch");
  after_launch();
  return out;
}

at::Tensor combine_output(const at::Tensor& y, const at::Tensor& weights, const at::Tensor& slots) {
  TORCH_CHECK(row_type(y) && y.dim() == 2, "expert_combine takes float16, bfloat16 or float32 y [rows, width]");
  TORCH_CHECK(weights.scalar_type() == at::kFloat && slots.scalar_type() == at::kInt && slots.dim() == 2 &&
                  weights.sizes() == slots.sizes(),
              "expert_combine takes float32 weights and int32 slots [tokens, k]");
  return at::empty({slots.size(0), y.size(1)}, y.options());
}
at::Tensor expert_combine(const at::Tensor& y, const at::Tensor& weights, const at::Tensor& slots) {
  inference(y, "thin_fused.expert_combine");
  inference(weights, "thin_fused.expert_combine");
  inference(slots, "thin_fused.expert_combine");
  select(y.device());
  at::Tensor out = combine_output(y, weights, slots);
  thin_desc yd = desc(y), wd = desc(weights), sd = desc(slots), od = desc(out);
  check(thin_expert_combine(&yd, &wd, &sd, &od, stream()), "thin expert_combine");
  after_launch();
  return out;
}

// ------------------------------------------------------------------ log probabilities
Quad logprobs_outputs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top) {
  TORCH_CHECK(row_type(logits) && logits.dim() == 2,
              "token_logprobs takes float16, bfloat16 or float32 logits [rows, width]");
  TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.dim() == 1 && tokens.size(0) == logits.size(0),
              "token_logprobs takes int64 tokens [rows]");
  TORCH_CHECK(top >= 0, "token_logprobs: top must not be negative");
  const int64_t rows = logits.size(0);
  const auto f = logits.options().dtype(at::kFloat);
  return {at::empty({rows}, f), at::empty({rows}, f), at::empty({rows, top}, f),
          at::empty({rows, top}, logits.options().dtype(at::kLong))};
}
Quad token_logprobs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top) {
  inference(logits, "thin_fused.token_logprobs");
  inference(tokens, "thin_fused.token_logprobs");
  select(logits.device());
  Quad out = logprobs_outputs(logits, tokens, top);
  thin_desc ld = desc(logits), td = desc(tokens), pd = desc(std::get<0>(out)), hd = desc(std::get<1>(out)),
            ad = desc(std::get<2>(out)), id = desc(std::get<3>(out));
  const size_t bytes = thin_token_logprobs_workspace(logits.size(0), logits.size(1), top);
  at::Tensor ws;
  if (bytes) ws = empty_bytes((int64_t)bytes);
  check(thin_token_logprobs(&ld, &td, &pd, &hd, &ad, &id, bytes ? ws.data_ptr() : nullptr, bytes, stream()),
        "thin token_logprobs");
  after_launch();
  return out;
}

}  // namespace thin_score

TORCH_LIBRARY_FRAGMENT(thin_fused, m) {
  m.def("group_norm(Tensor x, int groups, Tensor? weight=None, Tensor? bias=None, float eps=1e-05, bool silu=False, "
        "int? channels=None) -> Tensor");
  m.def("expert_route(Tensor logits, int top_k, Tensor? bias=None, bool softmax=True, int groups=1, int top_groups=1, "
        "bool renormalize=True, float scale=1.0) -> (Tensor, Tensor)");
  m.def("expert_dispatch(Tensor x, Tensor experts, int num_experts) -> (Tensor, Tensor, Tensor)");
  m.def("expert_combine(Tensor y, Tensor weights, Tensor slots) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor tokens, int top=0) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(thin_fused, PrivateUse1, m) {
  m.impl("group_norm", TORCH_FN(thin_score::group_norm));
  m.impl("expert_route", TORCH_FN(thin_score::expert_route));
  m.impl("expert_dispatch", TORCH_FN(thin_score::expert_dispatch));
  m.impl("expert_combine", TORCH_FN(thin_score::expert_combine));
  m.impl("token_logprobs", TORCH_FN(thin_score::token_logprobs));
}

TORCH_LIBRARY_IMPL(thin_fused, AutogradPrivateUse1, m) {
  for (const char* name : {"group_norm", "expert_route", "expert_dispatch", "expert_combine", "token_logprobs"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(thin_fused, Meta, m) {
  m.impl("group_norm", TORCH_FN(thin_score::group_norm_meta));
  m.impl("expert_route", TORCH_FN(thin_score::expert_route_meta));
  m.impl("expert_dispatch", TORCH_FN(thin_score::dispatch_outputs));
  m.impl("expert_combine", TORCH_FN(thin_score::combine_output));
  m.impl("token_logprobs", TORCH_FN(thin_score::logprobs_outputs));
}
