// 8-bit rows on the vk device (no reference counterpart): torch_vulkan.quantize_int8_rows and dequant_int8_rows, and
// int8_linear, whose operands are both 8-bit integers with one scale for each token and each output channel.  It stands
// beside dequant_int8_linear (op_quant.cpp) and mxfp4_linear (op_mx4.cpp), and like the latter passes gradients to its input and
// bias, for the adapters trained around a frozen base.
#include <torch/csrc/autograd/custom_function.h>

#include "common.h"

namespace {

using namespace vkt;

constexpr int64_t kMaxK = 131056;  // 2^14 K stays below 2^31
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

void check_rows(const at::Tensor& q, const at::Tensor& scale, const char* who, const char* name) {
  TORCH_CHECK(on_vk(q) && on_vk(scale), who, ": ", name, " and its scale must be on the vk device");
  TORCH_CHECK(q.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat, who, ": ", name, " must be int8 and its scale float32, got ",
              q.scalar_type(), " and ", scale.scalar_type());
  TORCH_CHECK(q.dim() >= 1 && scale.sizes() == q.sizes().slice(0, q.dim() - 1), who, ": ", name, "'s scale must have its shape without the last dimension, got ",
              q.sizes(), " and ", scale.sizes());
}

// x as a matrix of rows (sizes named: a -1 has no value where the last dimension is empty).
at::Tensor as_rows(const at::Tensor& x) {
  int64_t M = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) M *= x.size(i);
  return x.reshape({M, x.size(-1)});
}
at::Tensor unit_rows(const at::Tensor& x) { return x.size(1) <= 1 || x.stride(1) == 1 ? x : x.contiguous(); }

// x [rows, cols] into codes [rows, pitch] and scale [rows].
void quantize_rows(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale) {
  const at::Tensor r = unit_rows(x);
  queue(typed("i8_rows_quant", x.scalar_type()), hrt_i8_rows_args{dptr(r), dptr(codes), dptr(scale), r.size(0), r.size(1), r.stride(0), codes.size(1)});
}

void dequant_rows(const at::Tensor& q, const at::Tensor& scale, const at::Tensor& out) {
  queue(typed("i8_rows_dequant", out.scalar_type()), hrt_i8_rows_args{dptr(out), dptr(q), dptr(scale), q.size(0), q.size(1), q.size(1), q.stride(0)});
}

// 8-bit rows as the product reads them: whole 16-byte pieces on 16 bytes, a tile's row offsets in 31 bits; else a copy, its rows
// filled up with zeros.
at::Tensor product_rows(const at::Tensor& q) {
  const int64_t K = q.size(1);
  if (K % 16 == 0 && q.stride(1) == 1 && (q.size(0) <= 1 || (q.stride(0) % 16 == 0 && q.stride(0) < 8000000)) && dptr(q) % 16 == 0) return q;
  const at::Tensor c = at::empty({q.size(0), round16(K)}, q.options());
  if (K % 16 != 0) c.zero_();
  c.narrow(1, 0, K).copy_(q);
  return c;
}

int64_t pitch(const at::Tensor& q) { return q.size(0) > 1 ? q.stride(0) : q.size(1); }

struct Operands {
  at::Tensor x, x_scale, w, w_scale;  // x_scale undefined: x is yet to be quantised
  std::optional<at::Tensor> bias;
  at::ScalarType out;
};

// y [M, N] without autograd.
at::Tensor linear_rows(const Operands& o) {
  const int64_t M = o.x.size(0), K = o.x.size(1), N = o.w.size(0);
  const at::Tensor y = at::empty({M, N}, o.w.options().dtype(o.out));
  if (M == 0 || N == 0) return y;
  if (K == 0) return present(o.bias) ? y.copy_(*o.bias) : y.zero_();
  at::Tensor xq, xs, b;
  if (o.x_scale.defined()) {
    xq = product_rows(o.x), xs = dense(o.x_scale);
  } else if (hrt_i8_mm_quantises(M, K)) {  // quantised by the product itself
    xq = unit_rows(o.x);
  } else {
    xq = at::empty({M, round16(K)}, o.w.options()), xs = at::empty({M}, o.w_scale.options());
    quantize_rows(o.x, xq, xs);
  }
  const at::Tensor w = product_rows(o.w), ws = dense(o.w_scale);
  hrt_i8_mm_args A{};
  A.x = dptr(xq), A.x_scale = xs.defined() ? dptr(xs) : 0, A.w = dptr(w), A.w_scale = dptr(ws), A.y = dptr(y);
  if (present(o.bias)) b = dense(*o.bias), A.bias = dptr(b);
  A.M = M, A.N = N, A.K = w.size(1), A.x_sm = pitch(xq), A.w_sn = pitch(w);
  queue(typed("i8_mm", o.out), A);
  return y;
}

// The rows of a result in the shape of their tensor.  Not a view: nothing else holds the rows, and autograd would forbid in-place
// operations on a view that was made inside a function of ours.
at::Tensor in_shape(const at::Tensor& rows, at::IntArrayRef sizes) { return at::_unsafe_view(rows, sizes); }

struct Linear : torch::autograd::Function<Linear> {
  // (needs_input_grad counts the tensors that are there: those that may be missing come last)
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale,
                            const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& x_scale, at::ScalarType out) {
    ctx->save_for_backward({w, w_scale});
    ctx->saved_data["biased"] = present(bias);
    ctx->saved_data["sizes"] = x.sizes().vec();
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = w.size(0);
    return in_shape(linear_rows({as_rows(x), present(x_scale) ? x_scale->reshape({-1}) : at::Tensor(), w, w_scale, bias, out}), sizes);
  }

  // dx = g W and db = sum of g over the rows; the quantisation of x goes straight through, as if it had gone in unrounded.  Both depend
  // on g alone, and stay in the graph that is being made of the backward pass, if one is (create_graph).
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    no_tangent(grads[0], "int8_linear");
    torch::autograd::variable_list out(6);
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const at::Tensor g = as_rows(grads[0]), &w = saved[0], &scale = saved[1];
    const bool wants_x = ctx->needs_input_grad(0), wants_b = ctx->saved_data["biased"].toBool() && ctx->needs_input_grad(3);
    note_gpu("torch_vulkan::int8_linear_backward");
    if (at::GradMode::is_enabled() && g.requires_grad()) {
      if (wants_x) out[0] = at::mm(g, dequant_int8_rows_vk(w, scale, g.scalar_type())).view(sizes);
      if (wants_b) out[3] = g.sum(0);
      return out;
    }
    // the weights' values in g's type and the bias's sums in one launch, then the product
    const int64_t N = w.size(0), K = w.size(1);
    // so many rows that the sums' workgroups (64 columns each) would outlast the rest are summed by themselves: 16384 x 1024 34 us, so 16
    const bool product = wants_x && N > 0 && K > 0, sums = wants_b && N > 0 && g.size(0) > 0 && g.size(0) <= 8192;
    const at::Tensor rows = unit_rows(g);
    at::Tensor v, codes, s;
    hrt_i8_linear_back_args A{};
    A.M = g.size(0), A.N = N, A.K = K;
    if (product) {
      v = at::empty({N, K}, g.options()), codes = unit_rows(w), s = dense(scale);
      A.w = dptr(codes), A.w_scale = dptr(s), A.v = dptr(v), A.w_sn = codes.stride(0);
    }
    if (wants_b) out[3] = sums ? at::empty({N}, g.options()) : g.sum(0);
    if (sums) A.g = dptr(rows), A.db = dptr(out[3]), A.g_sm = pitch(rows);
    if (product || sums) queue(typed("i8_linear_back", g.scalar_type()), A);
    if (wants_x) out[0] = (product ? at::mm(rows, v) : at::zeros({g.size(0), K}, g.options())).view(sizes);
    return out;
  }
};

}  // namespace

namespace vkt {

std::tuple<at::Tensor, at::Tensor> quantize_int8_rows_vk(const at::Tensor& x) {
  TORCH_CHECK(on_vk(x) && float_code(x.scalar_type()) >= 0, "quantize_int8_rows: x must be a float32, bfloat16 or float16 vk tensor");
  TORCH_CHECK(x.dim() >= 1, "quantize_int8_rows: x must have at least one dimension");
  no_tangent(x, "quantize_int8_rows");
  const at::Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
  const at::Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (x.numel() == 0) {
    if (scale.numel() > 0) scale.zero_();
    return {codes, scale};
  }
  quantize_rows(as_rows(x), as_rows(codes), scale);
  note_gpu("torch_vulkan::quantize_int8_rows");
  return {codes, scale};
}

at::Tensor dequant_int8_rows_vk(const at::Tensor& q, const at::Tensor& scale, at::ScalarType out_dtype) {
  check_rows(q, scale, "dequant_int8_rows", "q");
  TORCH_CHECK(float_code(out_dtype) >= 0, "dequant_int8_rows: out_dtype must be float32, bfloat16 or float16, got ", out_dtype);
  TORCH_CHECK(!at::GradMode::is_enabled() || !scale.requires_grad(), "dequant_int8_rows: scale takes no gradient");
  no_tangent(scale, "dequant_int8_rows");
  const at::Tensor out = at::empty(q.sizes(), q.options().dtype(out_dtype));
  if (out.numel() == 0) return out;
  dequant_rows(unit_rows(as_rows(q)), dense(scale), as_rows(out));
  note_gpu("torch_vulkan::dequant_int8_rows");
  return out;
}

at::Tensor int8_linear_vk(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scale, const std::optional<at::Tensor>& bias,
                          const std::optional<at::Tensor>& x_scale, std::optional<at::ScalarType> out_dtype) {
  const char* const who = "int8_linear";
  const bool coded = on_vk(x) && x.scalar_type() == at::kChar;
  TORCH_CHECK(coded || (on_vk(x) && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf)), who,
              ": x must be a bfloat16, float16 or int8 vk tensor");
  TORCH_CHECK(coded == present(x_scale), who, ": x_scale belongs to an int8 x, and only to one");
  const at::ScalarType out = out_dtype.value_or(coded ? at::kBFloat16 : x.scalar_type());
  TORCH_CHECK(out == at::kBFloat16 || out == at::kHalf, who, ": out_dtype must be bfloat16 or float16, got ", out);
  TORCH_CHECK(coded || out == x.scalar_type(), who, ": out_dtype is x's own type unless x is int8");
  check_rows(weight, weight_scale, who, "weight");
  if (coded) check_rows(x, *x_scale, who, "x");
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1), who, ": weight must be [N, K] and x [..., K], got ", weight.sizes(), x.sizes());
  TORCH_CHECK(weight.size(1) <= kMaxK, who, ": K must be at most ", kMaxK, ", got ", weight.size(1));
  if (present(bias))
    TORCH_CHECK(on_vk(*bias) && bias->scalar_type() == out && bias->dim() == 1 && bias->size(0) == weight.size(0), who, ": bias must be a vk tensor of ",
                weight.size(0), " elements in the output's dtype");
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK(!grad || !(weight_scale.requires_grad() || (coded && x_scale->requires_grad())), who, ": scales take no gradient");
  no_tangent(x, who), no_tangent(weight_scale, who);
  if (present(bias)) no_tangent(*bias, who);
  if (coded) no_tangent(*x_scale, who);
  note_gpu("torch_vulkan::int8_linear");
  if (grad && (x.requires_grad() || (present(bias) && bias->requires_grad()))) return Linear::apply(x, weight, weight_scale, bias, x_scale, out);
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = weight.size(0);
  return in_shape(linear_rows({as_rows(x), coded ? x_scale->reshape({-1}) : at::Tensor(), weight, weight_scale, bias, out}), sizes);
}

}  // namespace vkt
