// Microscaled 4-bit floating point on the vk device (no reference counterpart): torch_vulkan.quantize_mxfp4 and
// dequant_mxfp4, and mxfp4_linear, the linear layer on frozen 4-bit weights, which stands beside the int8 one
// (op_quant.cpp) and also passes gradients to its input and bias, for the adapters trained around a frozen base.
// Weights are codes [N, ceil(K / 2)] and scale bytes [N, ceil(K / 32)], both uint8 (include/hrt_ops.h, hrt_mx4_args).
#include <torch/csrc/autograd/custom_function.h>

#include "common.h"

namespace {

using namespace vkt;

constexpr int64_t kBlock = 32;
int64_t blocks(int64_t cols) { return (cols + kBlock - 1) / kBlock; }

// Contiguous and on `align` bytes: what the kernels read whole words of.
at::Tensor dense_on(const at::Tensor& t, uint64_t align) {
  const at::Tensor c = dense(t);
  return dptr(c) % align == 0 ? c : c.clone();
}

void check_packed(const at::Tensor& codes, const at::Tensor& scale, int64_t cols, const char* who) {
  TORCH_CHECK(on_vk(codes) && on_vk(scale), who, ": codes and scale must be on the vk device");
  TORCH_CHECK(codes.scalar_type() == at::kByte && scale.scalar_type() == at::kByte, who, ": codes and scale must be uint8, got ",
              codes.scalar_type(), " and ", scale.scalar_type());
  TORCH_CHECK(codes.dim() >= 1 && scale.dim() == codes.dim() &&
                  codes.sizes().slice(0, codes.dim() - 1) == scale.sizes().slice(0, codes.dim() - 1),
              who, ": codes and scale must agree in all but the last dimension, got ", codes.sizes(), " and ", scale.sizes());
  TORCH_CHECK(cols >= 0 && codes.size(-1) == (cols + 1) / 2 && scale.size(-1) == blocks(cols), who, ": rows of ", cols,
              " values are ", (cols + 1) / 2, " bytes of codes and ", blocks(cols), " scales, got ", codes.size(-1), " and ",
              scale.size(-1));
}

// x as a matrix of rows (sizes named: a -1 has no value where the last dimension is empty).
at::Tensor as_rows(const at::Tensor& x) {
  int64_t M = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) M *= x.size(i);
  return x.reshape({M, x.size(-1)});
}

// x [rows, cols] with a unit column stride.
void quantize_rows(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale) {
  if (x.numel() == 0) return;
  queue(typed("mx4_quant", x.scalar_type()), hrt_mx4_args{dptr(x), dptr(codes), dptr(scale), x.size(0), x.size(1), x.stride(0)});
}

at::Tensor unit_rows(const at::Tensor& x) { return x.size(1) <= 1 || x.stride(1) == 1 ? x : x.contiguous(); }

// 16-bit rows with a unit column stride as the products read them: whole 16-byte words, a tile's row offsets in 31 bits.
at::Tensor whole_words(const at::Tensor& rows) {
  return rows.stride(0) % 8 != 0 || dptr(rows) % 16 != 0 || rows.stride(0) >= 4000000 ? rows.clone(at::MemoryFormat::Contiguous) : rows;
}

// y = x W^T + bias for x [M, K] without autograd.
at::Tensor linear_rows(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                       bool quantize) {
  const int64_t M = x.size(0), K = x.size(1), N = codes.size(0);
  if (K % kBlock != 0 || M == 0 || N == 0 || K == 0) {  // rows that end inside a block: the product of the values
    at::Tensor in = x;
    if (quantize) {
      const auto [c, s] = quantize_mxfp4_vk(x);
      in = dequant_mxfp4_vk(c, s, x.scalar_type(), K);
    }
    const at::Tensor w = dequant_mxfp4_vk(codes, scale, x.scalar_type(), K).t();
    return present(bias) ? at::addmm(*bias, in, w) : at::mm(in, w);
  }
  const at::Tensor w = dense_on(codes, 16), ws = dense_on(scale, 4);
  hrt_mx4_mm_args A{};
  A.w = dptr(w), A.w_scale = dptr(ws), A.M = M, A.N = N, A.K = K;
  at::Tensor b;
  if (present(bias)) b = dense(*bias), A.bias = dptr(b);
  at::Tensor rows = unit_rows(x), xc, xs;
  if (quantize) {
    xc = at::empty({M, K / 2}, codes.options());
    xs = at::empty({M, K / kBlock}, codes.options());
    quantize_rows(rows, xc, xs);
    A.x = dptr(xc), A.x_scale = dptr(xs);
  } else {
    rows = whole_words(rows);
    A.x = dptr(rows), A.x_sm = rows.stride(0);
  }
  const at::Tensor y = at::empty({M, N}, x.options());
  A.y = dptr(y);
  queue(typed("mx4_mm", x.scalar_type()), A);
  return y;
}

// g W for g [M, N], of rows of K values.
at::Tensor linear_back(const at::Tensor& g, const at::Tensor& codes, const at::Tensor& scale, int64_t K) {
  const int64_t M = g.size(0), N = g.size(1);
  if (K % kBlock != 0 || N % 8 != 0 || M == 0 || N == 0 || K == 0) return at::mm(g, dequant_mxfp4_vk(codes, scale, g.scalar_type(), K));
  const at::Tensor rows = whole_words(unit_rows(g)), w = dense_on(codes, 16), ws = dense(scale), y = at::empty({M, K}, g.options());
  hrt_mx4_mm_args A{};
  A.x = dptr(rows), A.x_sm = rows.stride(0), A.w = dptr(w), A.w_scale = dptr(ws), A.y = dptr(y), A.M = M, A.N = N, A.K = K;
  queue(typed("mx4_mm_back", g.scalar_type()), A);
  return y;
}

// The same, differentiable in g: its gradient is the forward product, without bias and on h as it is.
struct LinearBack : torch::autograd::Function<LinearBack> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& g, const at::Tensor& codes, const at::Tensor& scale,
                            int64_t K) {
    ctx->save_for_backward({codes, scale});
    return linear_back(g, codes, scale, K);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list h) {
    const auto saved = ctx->get_saved_variables();
    return {mxfp4_linear_vk(h[0], saved[0], saved[1], std::nullopt, false), {}, {}, {}};
  }
};

// The rows of a result in the shape of their tensor.  Not a view: nothing else holds the rows, and autograd would forbid in-place
// operations on a view that was made inside a function of ours.
at::Tensor in_shape(const at::Tensor& rows, at::IntArrayRef sizes) { return at::_unsafe_view(rows, sizes); }

struct Linear : torch::autograd::Function<Linear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale,
                            const std::optional<at::Tensor>& bias, bool quantize) {
    ctx->save_for_backward({codes, scale});
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->saved_data["biased"] = present(bias);
    std::vector<int64_t> out = x.sizes().vec();
    out.back() = codes.size(0);
    return in_shape(linear_rows(as_rows(x), codes, scale, bias, quantize), out);
  }

  // dx = g W and db = sum of g over the rows.  quantize: straight through, as if x had gone in unrounded.  Both depend on g, and
  // stay in the graph that is being made of the backward pass, if one is (create_graph).
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    no_tangent(grads[0], "mxfp4_linear");
    torch::autograd::variable_list out(5);
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const at::Tensor g = as_rows(grads[0]);
    if (ctx->needs_input_grad(0)) {
      const bool graph = at::GradMode::is_enabled() && g.requires_grad();
      out[0] = (graph ? LinearBack::apply(g, saved[0], saved[1], sizes.back()) : linear_back(g, saved[0], saved[1], sizes.back())).view(sizes);
    }
    if (ctx->saved_data["biased"].toBool() && ctx->needs_input_grad(3)) out[3] = g.sum(0);
    note_gpu("torch_vulkan::mxfp4_linear_backward");
    return out;
  }
};

}  // namespace

namespace vkt {

std::tuple<at::Tensor, at::Tensor> quantize_mxfp4_vk(const at::Tensor& x) {
  TORCH_CHECK(on_vk(x) && float_code(x.scalar_type()) >= 0, "quantize_mxfp4: x must be a float32, bfloat16 or float16 vk tensor");
  TORCH_CHECK(x.dim() >= 1, "quantize_mxfp4: x must have at least one dimension");
  no_tangent(x, "quantize_mxfp4");
  const int64_t cols = x.size(-1);
  std::vector<int64_t> sizes = x.sizes().vec();
  const auto bytes = x.options().dtype(at::kByte);
  sizes.back() = (cols + 1) / 2;
  const at::Tensor codes = at::empty(sizes, bytes);
  sizes.back() = blocks(cols);
  const at::Tensor scale = at::empty(sizes, bytes);
  if (x.numel() == 0) return {codes, scale};
  quantize_rows(unit_rows(as_rows(x)), codes, scale);
  note_gpu("torch_vulkan::quantize_mxfp4");
  return {codes, scale};
}

at::Tensor dequant_mxfp4_vk(const at::Tensor& codes, const at::Tensor& scale, at::ScalarType out_dtype, int64_t cols) {
  check_packed(codes, scale, cols, "dequant_mxfp4");
  TORCH_CHECK(float_code(out_dtype) >= 0, "dequant_mxfp4: out_dtype must be float32, bfloat16 or float16, got ", out_dtype);
  std::vector<int64_t> sizes = codes.sizes().vec();
  sizes.back() = cols;
  const at::Tensor out = at::empty(sizes, codes.options().dtype(out_dtype));
  if (out.numel() == 0) return out;
  const at::Tensor c = dense(codes), s = dense(scale);
  queue(typed("mx4_dequant", out_dtype), hrt_mx4_args{dptr(out), dptr(c), dptr(s), out.numel() / cols, cols, cols});
  note_gpu("torch_vulkan::dequant_mxfp4");
  return out;
}

at::Tensor mxfp4_linear_vk(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                           bool quantize_input) {
  TORCH_CHECK(on_vk(x) && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf),
              "mxfp4_linear: x must be a bfloat16 or float16 vk tensor");
  TORCH_CHECK(x.dim() >= 1 && codes.dim() == 2, "mxfp4_linear: x must have at least one dimension and codes two");
  check_packed(codes, scale, x.size(-1), "mxfp4_linear");
  if (present(bias))
    TORCH_CHECK(on_vk(*bias) && bias->scalar_type() == x.scalar_type() && bias->dim() == 1 && bias->size(0) == codes.size(0),
                "mxfp4_linear: bias must be a vk tensor of ", codes.size(0), " elements in x's dtype");
  no_tangent(x, "mxfp4_linear");
  if (present(bias)) no_tangent(*bias, "mxfp4_linear");
  note_gpu("torch_vulkan::mxfp4_linear");
  if (at::GradMode::is_enabled() && (x.requires_grad() || (present(bias) && bias->requires_grad())))
    return Linear::apply(x, codes, scale, bias, quantize_input);
  std::vector<int64_t> out = x.sizes().vec();
  out.back() = codes.size(0);
  return in_shape(linear_rows(as_rows(x), codes, scale, bias, quantize_input), out);
}

}  // namespace vkt
