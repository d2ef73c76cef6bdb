// torch.autocast(device_type="vk"): the policy the reference registers (csrc/shim.cpp:376-394), which is
// CUDA's: products and attention run in the autocast dtype, layer_norm / softmax / mse_loss in fp32,
// everything else passes through unchanged.  The 4-bit and 8-bit linear layers, attention with a relative position bias and the
// root-mean-square norm, which have no aten schema, follow linear, scaled_dot_product_attention and layer_norm.
#include <ATen/autocast_mode.h>
#include <torch/library.h>

#include "common.h"

TORCH_LIBRARY_IMPL(_, AutocastPrivateUse1, m) { m.fallback(torch::CppFunction::makeFallthrough()); }

TORCH_LIBRARY_IMPL(aten, AutocastPrivateUse1, m) {
  // lower precision
  KERNEL_PRIVATEUSEONE(mm, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(bmm, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(addmm, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(baddbmm, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(matmul, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(linear, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(conv1d, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(conv2d, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(conv3d, lower_precision_fp)
  KERNEL_PRIVATEUSEONE(scaled_dot_product_attention, lower_precision_fp)
  // fp32
  KERNEL_PRIVATEUSEONE(layer_norm, fp32)
  KERNEL_PRIVATEUSEONE(softmax, int, fp32)
  KERNEL_PRIVATEUSEONE(mse_loss, fp32)
}

namespace vkt {

namespace {
at::Tensor low(const at::Tensor& t) { return at::autocast::cached_cast(at::autocast::get_autocast_dtype(kDev), t, kDev); }
std::optional<at::Tensor> low(const std::optional<at::Tensor>& t) { return present(t) ? std::optional<at::Tensor>(low(*t)) : std::nullopt; }
at::Tensor full(const at::Tensor& t) { return at::autocast::cached_cast(at::kFloat, t, kDev); }
std::optional<at::Tensor> full(const std::optional<at::Tensor>& t) { return present(t) ? std::optional<at::Tensor>(full(*t)) : std::nullopt; }
}  // namespace

at::Tensor mxfp4_linear_autocast(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                                 bool quantize_input) {
  if (!at::autocast::is_autocast_enabled(kDev)) return mxfp4_linear_vk(x, codes, scale, bias, quantize_input);
  const c10::impl::ExcludeDispatchKeyGuard done(c10::DispatchKey::AutocastPrivateUse1);
  return mxfp4_linear_vk(low(x), codes, scale, low(bias), quantize_input);
}

at::Tensor int8_linear_autocast(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scale, const std::optional<at::Tensor>& bias,
                                const std::optional<at::Tensor>& x_scale, std::optional<at::ScalarType> out_dtype) {
  if (!at::autocast::is_autocast_enabled(kDev)) return int8_linear_vk(x, weight, weight_scale, bias, x_scale, out_dtype);
  const c10::impl::ExcludeDispatchKeyGuard done(c10::DispatchKey::AutocastPrivateUse1);
  // an output's type that is named stays: int8_linear refuses one that is not x's, unless x is int8
  const at::ScalarType t = out_dtype.value_or(at::autocast::get_autocast_dtype(kDev));
  return int8_linear_vk(low(x), weight, weight_scale, present(bias) ? std::optional<at::Tensor>(at::autocast::cached_cast(t, *bias, kDev)) : std::nullopt,
                        x_scale, t);
}

std::vector<at::Tensor> rms_norm_autocast(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual, double eps,
                                          bool int8) {
  const auto norm = int8 ? &rms_norm_int8_vk : &rms_norm_vk;
  if (!at::autocast::is_autocast_enabled(kDev)) return norm(x, weight, residual, eps);
  const c10::impl::ExcludeDispatchKeyGuard done(c10::DispatchKey::AutocastPrivateUse1);
  return norm(full(x), full(weight), full(residual), eps);
}

at::Tensor relative_bias_attention_autocast(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                            const std::optional<at::Tensor>& key_mask, bool causal, std::optional<double> scale,
                                            int64_t max_distance, int64_t query_offset) {
  if (!at::autocast::is_autocast_enabled(kDev))
    return relative_bias_attention_vk(q, k, v, table, key_mask, causal, scale, max_distance, query_offset);
  const c10::impl::ExcludeDispatchKeyGuard done(c10::DispatchKey::AutocastPrivateUse1);
  return relative_bias_attention_vk(low(q), low(k), low(v), low(table), key_mask, causal, scale, max_distance, query_offset);
}

}  // namespace vkt
