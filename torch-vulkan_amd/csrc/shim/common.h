// Shared pieces of the "vk" PrivateUse1 shim, the upper half of the boundary: PyTorch calls the adapters
// declared in ops.h through the dispatcher registrations in register.cpp; an adapter decides whether the
// hrt kernels take the call, fills an include/hrt_ops.h argument block and queues it through the C ABI
// (include/hrt.h).  Interface counterpart in the reference: csrc/common.h:1-66.
#pragma once

#include <ATen/ATen.h>
#include <ATen/native/CPUFallback.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>
#include <string>
#include <string_view>

#include "hrt.h"
#include "hrt_ops.h"

namespace vkt {

constexpr c10::DeviceType kDev = c10::DeviceType::PrivateUse1;

// ---- the runtime ------------------------------------------------------------------------------------------
// runtime() initialises libhrt on first use (device selection, stream, kernel table) and throws with the
// runtime's message when that fails; every entry point that reaches the C ABI calls it first.
void runtime();
std::string runtime_error_text();
// Throws "vk: <what>: <runtime message>" unless rc == 0.
void expect_ok(int rc, const char* what);

// ---- kernels ------------------------------------------------------------------------------------------------
// Queue operator kernel `name` (it sizes its own grid) with an argument block; throws with the runtime's
// message when the kernel rejects its arguments.  Kernel ids are looked up once per name.
void queue(std::string_view name, const void* args, uint32_t len);
template <typename A>
inline void queue(std::string_view name, const A& args) {
  queue(name, &args, static_cast<uint32_t>(sizeof(A)));
}

// Float element kinds the kernels compute in: HRT_F32 / HRT_BF16 / HRT_F16, or -1; and the matching
// kernel-name suffix ("f32" / "bf16" / "f16"), or nullptr.
int float_code(at::ScalarType t);
const char* dtype_suffix(at::ScalarType t);
// "<op>_<suffix>", the registry's naming (e.g. "softmax_fwd_bf16").
std::string typed(std::string_view op, at::ScalarType t);

inline bool on_vk(const at::Tensor& t) { return t.defined() && t.device().type() == kDev; }
inline uint64_t dptr(const at::Tensor& t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }
inline at::Tensor dense(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
// Workspace that only makes an operator faster: `bytes` of device memory until the handle goes (kernels queued before
// may still use it: one stream), or an empty handle where there is no room and the operator goes on without; every
// empty one is counted.  By default (hrt_alloc_spare) nothing is given up for it: no idle slab, no wait for the GPU.
// reserve: room is made as for a tensor.
c10::DataPtr scratch(int64_t bytes, bool reserve = false);
inline uint64_t dptr(const c10::DataPtr& p) { return reinterpret_cast<uint64_t>(p.get()); }
uint64_t scratch_left_out();  // how many were empty
inline bool present(const std::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }
// Operators that call their kernels themselves would drop a forward-mode tangent without a word: they refuse one.
inline void no_tangent(const at::Tensor& t, const char* who) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), who, ": forward-mode differentiation is not supported");
}

// ---- accounting -------------------------------------------------------------------------------------------
// Per-operator counts of GPU launches and CPU fallbacks (with the fallback's host time), which the tests
// read through torch_vulkan.kernel_counts() / fallback_counts() (names as the reference's counters,
// csrc/shim.cpp:53-66).
void note_gpu(std::string_view op);
void note_cpu(std::string_view op, uint64_t ns);

// ---- the CPU fallback --------------------------------------------------------------------------------
// Boxed fallback for every operator without a vk kernel (csrc/shim.cpp:70-131): runs PyTorch's CPU
// kernel on host copies and returns vk results whenever an input was on vk.
void cpu_fallback_boxed(const c10::OperatorHandle& op, torch::jit::Stack* stack);

#define VKT_CPU(op, ...) at::native::call_fallback_fn<&vkt::cpu_fallback_boxed, at::_ops::op>::call(__VA_ARGS__)
#define VKT_CPU_SYMINT(op, ...) \
  at::native::call_fallback_fn_symint<&vkt::cpu_fallback_boxed, at::_ops::op>::call(__VA_ARGS__)

// ---- device copies used by several adapters -------------------------------------------------------
// Strided copy with float-kind conversion, or same-type raw copy; false = dtype pair not handled.
bool ew_copy(const at::Tensor& dst, const at::Tensor& src);
// Fill of a (possibly strided) tensor; false = dtype not handled.
bool ew_fill(const at::Tensor& dst, const at::Scalar& value);

// ---- switches --------------------------------------------------------------------------------------------
// Matrix-core gate of the GEMM adapter: on/off (VKT_NO_COOP), and the debug bisection window
// (set_coop_range: only matrix-core-eligible calls numbered [lo, hi) of the chosen kind use MFMA).
void set_coop_enabled(bool on);
bool coop_is_enabled();
uint32_t coop_caps();
void set_coop_range(uint64_t lo, uint64_t hi, int kind);
void reset_coop_calls();
uint64_t coop_calls();
// Fused attention policy: 0 off, 1 on, 2 auto (VKT_FUSED_ATTN / VKT_NO_FUSED_ATTN).
void set_fused_attention(int mode);

// Weight-only int8 (pybind `dequant_int8`) and the fused int8 linear (no reference counterpart).
at::Tensor dequant_int8_vk(const at::Tensor& q, const at::Tensor& scale, at::ScalarType out_dtype);
at::Tensor dequant_int8_linear_vk(const at::Tensor& x, const at::Tensor& q, const at::Tensor& scale,
                                  const std::optional<at::Tensor>& bias);

// Microscaled 4-bit floating point: packing, unpacking, and the linear layer on packed weights (differentiable in x and
// bias; no reference counterpart).
std::tuple<at::Tensor, at::Tensor> quantize_mxfp4_vk(const at::Tensor& x);
at::Tensor dequant_mxfp4_vk(const at::Tensor& codes, const at::Tensor& scale, at::ScalarType out_dtype, int64_t cols);
at::Tensor mxfp4_linear_vk(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                           bool quantize_input);
at::Tensor mxfp4_linear_autocast(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, const std::optional<at::Tensor>& bias,
                                 bool quantize_input);  // x and bias in the autocast dtype where autocast is on

// Fused attention with a learned relative position bias, differentiable (no reference counterpart).
at::Tensor relative_bias_attention_vk(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                      const std::optional<at::Tensor>& key_mask, bool causal, std::optional<double> scale,
                                      int64_t max_distance, int64_t query_offset);
at::Tensor relative_bias_attention_autocast(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                            const std::optional<at::Tensor>& key_mask, bool causal, std::optional<double> scale,
                                            int64_t max_distance, int64_t query_offset);  // the same of q, k, v and table


// 8-bit rows with one scale each, and the linear layer on them (differentiable in x and bias; no reference counterpart).
std::tuple<at::Tensor, at::Tensor> quantize_int8_rows_vk(const at::Tensor& x);
at::Tensor dequant_int8_rows_vk(const at::Tensor& q, const at::Tensor& scale, at::ScalarType out_dtype);
at::Tensor int8_linear_vk(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scale, const std::optional<at::Tensor>& bias,
                          const std::optional<at::Tensor>& x_scale, std::optional<at::ScalarType> out_dtype);
at::Tensor int8_linear_autocast(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scale, const std::optional<at::Tensor>& bias,
                                const std::optional<at::Tensor>& x_scale, std::optional<at::ScalarType> out_dtype);  // x and bias in the autocast dtype

// Root-mean-square norm, {y} or with a residual {y, h}; in 8 bits {q, scale} or {q, scale, h}.
std::vector<at::Tensor> rms_norm_vk(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual, double eps);
std::vector<at::Tensor> rms_norm_int8_vk(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual, double eps);
std::vector<at::Tensor> rms_norm_autocast(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual, double eps,
                                          bool int8);  // either of them, in fp32 where autocast is on

// Rotary positions of several axes, {q} or {q, k}.
std::vector<at::Tensor> rotary_embedding_vk(const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions, const at::Tensor& freqs,
                                            const std::vector<int64_t>& sections, bool interleaved);

}  // namespace vkt
