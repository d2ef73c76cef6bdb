// torch.autocast(device_type="vk"): the policy the reference registers (csrc/shim.cpp:376-394), which is
// CUDA's: products and attention run in the autocast dtype, layer_norm / softmax / mse_loss in fp32,
// everything else passes through unchanged.  The 4-bit linear layer and attention with a relative position bias, which have no
// aten schema, follow linear and scaled_dot_product_attention.
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
}  // namespace

at::Tensor mxfp4_linear_autocast(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                                 bool quantize_input) {
  if (!at::autocast::is_autocast_enabled(kDev)) return mxfp4_linear_vk(x, codes, scale, bias, quantize_input);
  const c10::impl::ExcludeDispatchKeyGuard done(c10::DispatchKey::AutocastPrivateUse1);
  return mxfp4_linear_vk(low(x), codes, scale, present(bias) ? std::optional<at::Tensor>(low(*bias)) : std::nullopt, quantize_input);
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
