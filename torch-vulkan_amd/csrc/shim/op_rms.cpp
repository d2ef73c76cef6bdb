// torch_vulkan.rms_norm and rms_norm_int8 on the vk device (no reference counterpart): root-mean-square norm of rows, with the
// residual's addition, in the input's type (differentiable) or in 8 bits with a scale for each row, as int8_linear takes them
// (op_int8.cpp).  They stand beside layer_norm (op_rows.cpp).
#include <torch/csrc/autograd/custom_function.h>

#include "common.h"

namespace {

using namespace vkt;

// Tensors of one shape [..., D] as rows behind at most three outer dimensions, merged where all of them allow it; one that cannot be
// read so is copied.
struct Rows {
  std::vector<at::Tensor> t;
  int64_t rows = 1, D = 1, n1 = 1, n2 = 1;

  explicit Rows(std::vector<at::Tensor> in) : t(std::move(in)) {
    const at::Tensor* one = nullptr;
    for (at::Tensor& x : t) {
      if (!x.defined()) continue;
      if (x.size(-1) > 1 && x.stride(-1) != 1) x = x.contiguous();
      one = &x;
    }
    D = one->size(-1), rows = one->numel() / std::max<int64_t>(D, 1);
    if (!merge()) {
      for (at::Tensor& x : t)
        if (x.defined()) x = x.contiguous();
      merge();
    }
  }

  void put(size_t i, uint64_t* addr, int64_t* s3) const {
    if (!t[i].defined()) return;
    *addr = dptr(t[i]);
    for (int k = 0; k < 3; ++k) s3[k] = strides_[i][k];
  }

 private:
  std::vector<std::array<int64_t, 3>> strides_;

  bool merge() {
    const at::Tensor* one = nullptr;
    for (const at::Tensor& x : t)
      if (x.defined()) one = &x;
    std::vector<int64_t> size;                // outer dimensions, innermost first
    std::vector<std::vector<int64_t>> st(t.size());
    for (int64_t d = one->dim() - 2; d >= 0; --d) {
      const int64_t n = one->size(d);
      if (n == 1) continue;
      bool joins = !size.empty();
      for (size_t i = 0; i < t.size() && joins; ++i)
        if (t[i].defined()) joins = t[i].stride(d) == st[i].back() * size.back();
      if (joins) {
        size.back() *= n;
        continue;
      }
      size.push_back(n);
      for (size_t i = 0; i < t.size(); ++i) st[i].push_back(t[i].defined() ? t[i].stride(d) : 0);
    }
    if (size.size() > 3) return false;
    n2 = size.size() > 1 ? size[0] : 1, n1 = size.size() > 2 ? size[1] : 1;
    strides_.assign(t.size(), {0, 0, 0});
    for (size_t i = 0; i < t.size(); ++i) {
      if (size.size() == 1) strides_[i][0] = st[i][0];
      if (size.size() == 2) strides_[i][0] = st[i][1], strides_[i][2] = st[i][0];
      if (size.size() == 3) strides_[i][0] = st[i][2], strides_[i][1] = st[i][1], strides_[i][2] = st[i][0];
    }
    return true;
  }
};

struct Out {
  at::Tensor y, h, rstd, rest, q, scale;
};

// keep: also rstd, and what rounding took from h, for the backward pass.  coded: 8-bit rows in place of y.
Out forward_rows(const at::Tensor& x, const at::Tensor& w, const at::Tensor& r, double eps, bool keep, bool coded) {
  Out o;
  const auto f32 = x.options().dtype(at::kFloat);
  const at::IntArrayRef outer = x.sizes().slice(0, x.dim() - 1);
  if (coded) o.q = at::empty(x.sizes(), x.options().dtype(at::kChar)), o.scale = at::empty(outer, f32);
  else o.y = at::empty(x.sizes(), x.options());
  if (r.defined()) o.h = at::empty(x.sizes(), x.options());
  if (keep) o.rstd = at::empty({x.numel() / x.size(-1)}, f32);
  if (keep && r.defined() && x.scalar_type() != at::kFloat) o.rest = at::empty({x.numel() / x.size(-1), (x.size(-1) + 7) / 8 * 8}, x.options().dtype(at::kChar));
  if (x.numel() == 0) return o;
  const Rows in({x, r});
  const at::Tensor wd = w.defined() ? dense(w) : w;
  hrt_rms_args A{};
  in.put(0, &A.x, A.xs), in.put(1, &A.r, A.rs);
  if (wd.defined()) A.w = dptr(wd);
  if (coded) A.q = dptr(o.q), A.scale = dptr(o.scale);
  else A.y = dptr(o.y);
  if (o.h.defined()) A.h_out = dptr(o.h);
  if (keep) A.rstd = dptr(o.rstd);
  if (o.rest.defined()) A.h_rest = dptr(o.rest);
  A.rows = in.rows, A.D = in.D, A.n1 = in.n1, A.n2 = in.n2, A.eps = static_cast<float>(eps);
  queue(typed("rms_fwd", x.scalar_type()), A);
  return o;
}

// With a residual the backward pass reads h, and in 16 bits a byte a value that rounding h left, instead of both of its terms.
struct Norm : torch::autograd::Function<Norm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& w,
                                                const std::optional<at::Tensor>& r, double eps) {
    const at::Tensor wd = w.value_or(at::Tensor()), rd = r.value_or(at::Tensor());
    const Out o = forward_rows(x, wd, rd, eps, true, false);
    ctx->save_for_backward({rd.defined() ? o.h : x, o.rstd, wd, o.rest});
    ctx->set_materialize_grads(false);  // the gradient of an output that nothing uses is not read
    return rd.defined() ? torch::autograd::variable_list{o.y, o.h} : torch::autograd::variable_list{o.y};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm: its gradient is not differentiable (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &h = saved[0], &rstd = saved[1], &w = saved[2], &rest = saved[3];
    const at::Tensor gy = grads[0], gh = grads.size() > 1 ? grads[1] : at::Tensor();
    for (const at::Tensor* g : {&gy, &gh})
      if (g->defined()) no_tangent(*g, "rms_norm");
    torch::autograd::variable_list out(4);
    // needs_input_grad counts the tensors that are there
    const bool wants_x = ctx->needs_input_grad(0), wants_w = w.defined() && ctx->needs_input_grad(1);
    const bool wants_r = grads.size() > 1 && ctx->needs_input_grad(w.defined() ? 2 : 1);
    if ((!gy.defined() && !gh.defined()) || !(wants_x || wants_r || wants_w)) return out;
    note_gpu("torch_vulkan::rms_norm_backward");
    const auto like = [&](const at::Tensor& g) { return g.defined() && g.scalar_type() != h.scalar_type() ? g.to(h.scalar_type()) : g; };
    at::Tensor dx, dw, ws;
    if (wants_x || wants_r) dx = at::empty(h.sizes(), h.options());
    if (wants_w) dw = at::empty(w.sizes(), w.options());
    if (h.numel() == 0) {
      if (wants_w) dw.zero_();
    } else {
      const Rows in({like(gy), like(gh), h});
      const at::Tensor wd = w.defined() ? dense(w) : w;
      hrt_rms_bwd_args A{};
      in.put(0, &A.gy, A.gys), in.put(1, &A.gh, A.ghs), in.put(2, &A.h, A.hs);
      A.rstd = dptr(rstd), A.rows = in.rows, A.D = in.D, A.n1 = in.n1, A.n2 = in.n2;
      if (wd.defined()) A.w = dptr(wd);
      if (rest.defined()) A.h_rest = dptr(rest);
      if (dx.defined()) A.dx = dptr(dx);
      if (wants_w) {
        A.dw = dptr(dw);
        if (const int64_t n = hrt_rms_workspace(&A, float_code(h.scalar_type())); n > 0) ws = at::empty({n}, rstd.options()), A.ws = dptr(ws);
      }
      queue(typed("rms_bwd", h.scalar_type()), A);
    }
    if (wants_x) out[0] = dx;
    if (wants_r) out[2] = dx;  // x and the residual share one gradient
    out[1] = dw;
    return out;
  }
};

void check(const at::Tensor& x, const std::optional<at::Tensor>& w, const std::optional<at::Tensor>& r, double eps, const char* who) {
  TORCH_CHECK(on_vk(x) && float_code(x.scalar_type()) >= 0, who, ": x must be a float32, bfloat16 or float16 vk tensor");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, who, ": x must have a last dimension of at least one value, got ", x.sizes());
  if (present(w))
    TORCH_CHECK(on_vk(*w) && w->scalar_type() == x.scalar_type() && w->dim() == 1 && w->size(0) == x.size(-1), who, ": weight must be a vk tensor of ", x.size(-1),
                " elements in x's dtype");
  if (present(r))
    TORCH_CHECK(on_vk(*r) && r->scalar_type() == x.scalar_type() && r->sizes() == x.sizes(), who, ": residual must be a vk tensor of x's shape and dtype");
  TORCH_CHECK(eps >= 0 && eps <= 1e30, who, ": eps must be 0 or more, got ", eps);
  TORCH_CHECK(eps == 0 || static_cast<float>(eps) > 0, who, ": eps ", eps, " is 0 in float32: rows of zeros would be 0 / 0");
  constexpr int64_t lim = int64_t(1) << 31;
  TORCH_CHECK(x.size(-1) < lim && x.numel() / x.size(-1) < lim, who, ": too many rows or columns");
  no_tangent(x, who);
  if (present(w)) no_tangent(*w, who);
  if (present(r)) no_tangent(*r, who);
}

bool wants_grad(const at::Tensor& x, const std::optional<at::Tensor>& w, const std::optional<at::Tensor>& r) {
  return at::GradMode::is_enabled() && (x.requires_grad() || (present(w) && w->requires_grad()) || (present(r) && r->requires_grad()));
}

}  // namespace

namespace vkt {

std::vector<at::Tensor> rms_norm_vk(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual, double eps) {
  check(x, weight, residual, eps, "rms_norm");
  note_gpu("torch_vulkan::rms_norm");
  if (wants_grad(x, weight, residual)) return Norm::apply(x, weight, residual, eps);
  const Out o = forward_rows(x, weight.value_or(at::Tensor()), residual.value_or(at::Tensor()), eps, false, false);
  if (present(residual)) return {o.y, o.h};
  return {o.y};
}

std::vector<at::Tensor> rms_norm_int8_vk(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual, double eps) {
  check(x, weight, residual, eps, "rms_norm_int8");
  TORCH_CHECK(!wants_grad(x, weight, residual), "rms_norm_int8: has no gradient; train with rms_norm and int8_linear, which quantises its input, or call it under no_grad");
  note_gpu("torch_vulkan::rms_norm_int8");
  const Out o = forward_rows(x, weight.value_or(at::Tensor()), residual.value_or(at::Tensor()), eps, false, true);
  if (present(residual)) return {o.q, o.scale, o.h};
  return {o.q, o.scale};
}

}  // namespace vkt
