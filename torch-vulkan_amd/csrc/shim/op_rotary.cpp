// torch_vulkan.rotary_embedding on the vk device (no reference counterpart): queries and keys turned by positions of several axes
// (frames, rows and columns of an image or a clip), differentiable.  It stands before the fused attention (op_attention.cpp),
// which reads its outputs in place.
#include <torch/csrc/autograd/custom_function.h>

#include "common.h"

namespace {

using namespace vkt;

struct Options {
  std::vector<int64_t> sections;
  bool interleaved;
};

// [B, H, S, D] in [B, S, H, D] memory.  Not a view: autograd would forbid in-place operations on one that leaves a function of ours.
at::Tensor bshd(const at::Tensor& like) {
  const int64_t H = like.size(1), S = like.size(2), D = like.size(3);
  return at::empty_strided(like.sizes(), {S * H * D, D, H * D, 1}, like.options());
}
at::Tensor unit_rows(const at::Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

// k may be undefined, and so is its result then.
std::tuple<at::Tensor, at::Tensor> turn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos, const at::Tensor& freqs, const Options& o, bool back) {
  const at::Tensor qo = bshd(q), ko = k.defined() ? bshd(k) : k;
  const bool has_k = k.defined() && k.size(1) > 0;
  if (q.size(0) == 0 || q.size(2) == 0 || q.size(3) == 0 || (q.size(1) == 0 && !has_k)) return {qo, ko};
  const bool swap = q.size(1) == 0;  // no queries: the keys alone
  const at::Tensor a = unit_rows(swap ? k : q), b = has_k && !swap ? unit_rows(k) : at::Tensor(), f = dense(freqs);
  hrt_rotary_args A{};
  A.q = dptr(a), A.q_out = dptr(swap ? ko : qo), A.pos = dptr(pos), A.freqs = dptr(f);
  const auto strides = [](const at::Tensor& t, int64_t* s) {
    const int64_t d[3] = {0, 1, 2};
    for (const int64_t i : d) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
  };
  strides(a, A.qs);
  A.Hq = static_cast<int32_t>(a.size(1));
  if (b.defined()) A.k = dptr(b), A.k_out = dptr(ko), A.Hk = static_cast<int32_t>(b.size(1)), strides(b, A.ks);
  A.B = q.size(0), A.S = q.size(2), A.D = static_cast<int32_t>(q.size(3));
  const bool batched = pos.dim() == 3 && pos.size(0) > 1;
  A.p_sb = batched ? pos.stride(0) : 0, A.p_ss = pos.size(-2) > 1 ? pos.stride(-2) : 0, A.p_sa = pos.size(-1) > 1 ? pos.stride(-1) : 0;
  A.pos_type = pos.scalar_type() == at::kInt ? 0 : pos.scalar_type() == at::kLong ? 1 : 2;
  int64_t end = 0;
  for (size_t i = 0; i < o.sections.size(); ++i) A.ends[i] = static_cast<int32_t>(end += o.sections[i]);
  A.axes = static_cast<int32_t>(o.sections.size()), A.P = static_cast<int32_t>(end);
  A.interleaved = o.interleaved, A.back = back;
  queue(typed("rotary", q.scalar_type()), A);
  return {qo, ko};
}

// Linear in q and k; the gradient is the opposite turn, differentiable in its turn.
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& pos,
                                                const at::Tensor& freqs, std::vector<int64_t> sections, bool interleaved, bool back) {
    const at::Tensor kd = k.value_or(at::Tensor());
    ctx->save_for_backward({pos, freqs});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["back"] = back;
    ctx->set_materialize_grads(false);
    const auto [qo, ko] = turn(q, kd, pos, freqs, {std::move(sections), interleaved}, back);
    return kd.defined() ? torch::autograd::variable_list{qo, ko} : torch::autograd::variable_list{qo};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(7);
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> sections = ctx->saved_data["sections"].toIntVector();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), back = !ctx->saved_data["back"].toBool();
    const at::Tensor gq = ctx->needs_input_grad(0) ? grads[0] : at::Tensor();
    const at::Tensor gk = grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : at::Tensor();
    if (!gq.defined() && !gk.defined()) return out;
    for (const at::Tensor* g : {&gq, &gk})
      if (g->defined()) no_tangent(*g, "rotary_embedding");
    note_gpu("torch_vulkan::rotary_embedding_backward");
    // one of the two alone goes as the queries
    const at::Tensor& one = gq.defined() ? gq : gk;
    const std::optional<at::Tensor> two = gq.defined() && gk.defined() ? std::optional<at::Tensor>(gk) : std::nullopt;
    torch::autograd::variable_list d;
    if (at::GradMode::is_enabled() && (one.requires_grad() || (two && two->requires_grad()))) {
      d = apply(one, two, saved[0], saved[1], sections, interleaved, back);
    } else {
      const auto [a, b] = turn(one, two.value_or(at::Tensor()), saved[0], saved[1], {sections, interleaved}, back);
      d = {a, b};
    }
    if (gq.defined()) out[0] = d[0];
    if (gk.defined()) out[1] = gq.defined() ? d[1] : d[0];
    return out;
  }
};

}  // namespace

namespace vkt {

std::vector<at::Tensor> rotary_embedding_vk(const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions, const at::Tensor& freqs,
                                            const std::vector<int64_t>& sections, bool interleaved) {
  const char* const who = "rotary_embedding";
  TORCH_CHECK(on_vk(q) && float_code(q.scalar_type()) >= 0 && q.dim() == 4, who, ": q must be a float32, bfloat16 or float16 vk tensor [B, H, S, D]");
  const int64_t B = q.size(0), S = q.size(2), D = q.size(3);
  if (present(k))
    TORCH_CHECK(on_vk(*k) && k->scalar_type() == q.scalar_type() && k->dim() == 4 && k->size(0) == B && k->size(2) == S && k->size(3) == D, who,
                ": k must be a vk tensor [", B, ", heads, ", S, ", ", D, "] in q's dtype, got ", k->sizes());
  TORCH_CHECK(D >= 1 && D <= 1024, who, ": D must be 1..1024, got ", D);
  const int64_t axes = static_cast<int64_t>(sections.size());
  TORCH_CHECK(axes >= 1 && axes <= HRT_ROTARY_AXES, who, ": sections must name the pairs of 1..", HRT_ROTARY_AXES, " axes");
  int64_t P = 0;
  for (const int64_t n : sections) {
    TORCH_CHECK(n >= 0 && n <= D, who, ": a section has 0 or more pairs, at most half of D in all");
    P += n;
  }
  TORCH_CHECK(P >= 1 && 2 * P <= D, who, ": sections must have at least one pair and at most ", D / 2, " in all, got ", P);
  TORCH_CHECK(on_vk(freqs) && freqs.scalar_type() == at::kDouble && freqs.dim() == 1 && freqs.size(0) == P, who, ": freqs must be a float64 vk tensor of ", P,
              " elements, one for each pair");
  const auto pt = positions.scalar_type();
  TORCH_CHECK(on_vk(positions) && (pt == at::kInt || pt == at::kLong || pt == at::kFloat), who, ": positions must be an int32, int64 or float32 vk tensor");
  TORCH_CHECK((positions.dim() == 2 || (positions.dim() == 3 && (positions.size(0) == B || positions.size(0) == 1))) && positions.size(-2) == S &&
                  positions.size(-1) == axes,
              who, ": positions must be [", S, ", ", axes, "] or [", B, ", ", S, ", ", axes, "], got ", positions.sizes());
  constexpr int64_t lim = int64_t(1) << 31;
  TORCH_CHECK(B * S < lim && q.size(1) <= 65536 && (!present(k) || k->size(1) <= 65536), who, ": too many tokens or heads");
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK(!grad || !(positions.requires_grad() || freqs.requires_grad()), who, ": positions and freqs take no gradient");
  no_tangent(q, who), no_tangent(positions, who), no_tangent(freqs, who);
  if (present(k)) no_tangent(*k, who);
  note_gpu("torch_vulkan::rotary_embedding");
  if (grad && (q.requires_grad() || (present(k) && k->requires_grad()))) return Rotary::apply(q, k, positions, freqs, sections, interleaved, false);
  const auto [qo, ko] = turn(q, k.value_or(at::Tensor()), positions, freqs, {sections, interleaved}, false);
  if (present(k)) return {qo, ko};
  return {qo};
}

}  // namespace vkt
