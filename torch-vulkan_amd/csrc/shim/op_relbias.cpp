// torch_vulkan.relative_bias_attention on the vk device (no reference counterpart): fused attention with a learned bias by
// bucketed relative position, a key mask and a causal form, differentiable in q, k, v and the bias table.  It stands beside
// F.scaled_dot_product_attention's fused kernels (op_attention.cpp), which take neither bias nor mask.
//
// q, k, v are [B, H, S, D] views read in place through their strides; rows that are not on 16 bytes or do not fill them
// (D % 8 != 0, f32: D % 4 != 0) cost a padded copy, and in training one of the output.  The output is [B, H, S, D] in
// [B, S, H, D] memory; gradients take their inputs' layouts where q, k and v are dense.
#include <torch/csrc/autograd/custom_function.h>

#include "common.h"

namespace {

using namespace vkt;

int64_t per16(at::ScalarType t) { return t == at::kFloat ? 4 : 8; }

// [B, H, S, D] in [B, S, H, D] memory.  Not a view: autograd would forbid in-place operations on one that leaves a function of ours.
at::Tensor bshd(const at::Tensor& like, int64_t S, int64_t D) {
  const int64_t H = like.size(1);
  return at::empty_strided({like.size(0), H, S, D}, {S * H * D, D, H * D, 1}, like.options());
}

// Whether the kernels read t [B, H, S, D] in place: rows of whole 16-byte pieces on 16-byte lines.
bool in_place(const at::Tensor& t) {
  const int64_t p = per16(t.scalar_type());
  if (t.size(3) % p != 0 || t.stride(3) != 1 || dptr(t) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) % p != 0 || t.stride(i) < 0)) return false;
  return t.size(2) <= 1 || t.stride(2) * (16 / p) < (int64_t(1) << 31) / 130;  // a stage's rows within 31-bit offsets
}

// t as the kernels read it, its rows padded with zeros to D columns.
at::Tensor rows_of(const at::Tensor& t, int64_t D) {
  if (t.size(3) == D && in_place(t)) return t;
  at::Tensor c = bshd(t, t.size(2), D);
  if (D > t.size(3)) c.zero_();
  c.narrow(3, 0, t.size(3)).copy_(t);
  return c;
}

void put(int64_t* s3, uint64_t* addr, const at::Tensor& t) {
  *addr = dptr(t);
  for (int i = 0; i < 3; ++i) s3[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

struct Options {
  bool causal;
  double scale;
  int64_t max_distance, offset;
};

hrt_attn_rel_args base_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& mask,
                            const Options& o) {
  hrt_attn_rel_args A{};
  put(&A.q_sb, &A.q, q);
  put(&A.k_sb, &A.k, k);
  put(&A.v_sb, &A.v, v);
  A.table = dptr(table);
  if (mask.defined()) A.mask = dptr(mask), A.mask_sb = mask.size(0) > 1 ? mask.stride(0) : 0;
  A.B = static_cast<int32_t>(q.size(0)), A.H = static_cast<int32_t>(q.size(1));
  A.Sq = static_cast<int32_t>(q.size(2)), A.Sk = static_cast<int32_t>(k.size(2)), A.D = static_cast<int32_t>(q.size(3));
  A.buckets = static_cast<int32_t>(table.size(0)), A.max_distance = static_cast<int32_t>(o.max_distance);
  A.causal = o.causal, A.q_off = o.offset, A.scale = static_cast<float>(o.scale);
  return A;
}

int64_t rows_in(const at::Tensor& q) { return q.size(0) * q.size(1) * q.size(2); }

// One block for what the backward needs beside o: lse, and for 16-bit types what o's rounding left, on 16
// bytes.
int64_t left_at(const at::Tensor& q) { return (rows_in(q) + 3) / 4 * 4; }
bool has_left(const at::Tensor& q) { return q.scalar_type() != at::kFloat; }

// o [B, H, Sq, D] (in [B, Sq, H, D] memory) and that block (train: with the second part), for rows as rows_of gives them.
std::tuple<at::Tensor, at::Tensor> forward_rows(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                                const at::Tensor& mask, const Options& opt, bool train) {
  const at::Tensor o = bshd(q, q.size(2), q.size(3));
  const bool left = train && has_left(q);
  const at::Tensor kept = at::empty({left ? left_at(q) + rows_in(q) * q.size(3) / 2 : rows_in(q)}, q.options().dtype(at::kFloat));
  hrt_attn_rel_args A = base_args(q, k, v, table, mask, opt);
  A.o = dptr(o), A.lse = dptr(kept);
  if (left) A.o_lo = dptr(kept) + 4 * left_at(q);
  c10::DataPtr part;
  if (const int64_t n = hrt_attn_rel_workspace(&A, float_code(q.scalar_type()), 0); n > 0) {
    part = scratch(n * 4);
    if (part) A.ws = dptr(part), A.ws_floats = n;
  }
  queue(typed("attn_rel_fwd", q.scalar_type()), A);
  return {o, kept};
}

struct Attention : torch::autograd::Function<Attention> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& table, const std::optional<at::Tensor>& key_mask, bool causal, double scale,
                            int64_t max_distance, int64_t offset) {
    const at::Tensor mask = key_mask.value_or(at::Tensor());
    const int64_t D = q.size(3), p = per16(q.scalar_type()), Dp = (D + p - 1) / p * p;
    if (q.numel() == 0 || k.size(2) == 0) {  // no rows, or no keys: zeros, and zero gradients
      ctx->save_for_backward({q, k, v, table});
      ctx->saved_data["D"] = int64_t(0);
      return at::zeros(q.sizes(), q.options());
    }
    const at::Tensor qr = rows_of(q, Dp), kr = rows_of(k, Dp), vr = rows_of(v, Dp), t = dense(table);
    const auto [o, kept] = forward_rows(qr, kr, vr, t, mask, {causal, scale, max_distance, offset}, true);
    ctx->save_for_backward({qr, kr, vr, t, mask, o, kept});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["max_distance"] = max_distance;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["D"] = D;
    return Dp == D ? o : bshd(o, o.size(2), D).copy_(o.narrow(3, 0, D));
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "relative_bias_attention: its gradient is not differentiable (create_graph)");
    no_tangent(grads[0], "relative_bias_attention");
    const auto saved = ctx->get_saved_variables();
    const int64_t D = ctx->saved_data["D"].toInt();
    if (D == 0) return {at::zeros_like(saved[0]), at::zeros_like(saved[1]), at::zeros_like(saved[2]), at::zeros_like(saved[3]), {}, {}, {}, {}, {}};
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &table = saved[3], &mask = saved[4], &o = saved[5], &kept = saved[6];
    const Options opt{ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), ctx->saved_data["max_distance"].toInt(),
                      ctx->saved_data["offset"].toInt()};
    const at::Tensor dout = rows_of(grads[0].scalar_type() == q.scalar_type() ? grads[0] : grads[0].to(q.scalar_type()), q.size(3));
    hrt_attn_rel_args A = base_args(q, k, v, table, mask, opt);
    put(&A.do_sb, &A.dout, dout);
    const bool wants_table = ctx->needs_input_grad(3), wants_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    // delta, and the partial sums of the table's gradient behind it
    const int64_t parts = wants_table ? hrt_attn_rel_workspace(&A, float_code(q.scalar_type()), 1) : 0;
    const at::Tensor work = at::empty({rows_in(q) + parts}, kept.options());
    A.o = dptr(o), A.lse = dptr(kept), A.delta = dptr(work);
    if (has_left(q)) A.o_lo = dptr(kept) + 4 * left_at(q);
    const bool like = q.is_non_overlapping_and_dense() && k.is_non_overlapping_and_dense() && v.is_non_overlapping_and_dense();
    if (like) A.flags = HRT_ATTN_GRAD_LIKE_INPUT;
    auto grad_for = [&](const at::Tensor& t) {
      return like ? at::empty_strided(t.sizes(), t.strides(), t.options()) : bshd(t, t.size(2), t.size(3));
    };
    torch::autograd::variable_list out(9);
    // dQ first: it also leaves delta for dK/dV
    at::Tensor dq, dtable;
    if (ctx->needs_input_grad(0)) dq = grad_for(q), A.dq = dptr(dq);
    if (wants_table) {
      dtable = at::empty_like(table);
      A.dtable = dptr(dtable), A.ws = dptr(work) + 4 * rows_in(q), A.ws_floats = parts;
      if (wants_kv) A.flags |= HRT_ATTN_REL_TABLE_LATER;
    }
    queue(typed("attn_rel_dq", q.scalar_type()), A);
    if (wants_kv) {
      const at::Tensor dk = grad_for(k), dv = grad_for(v);
      A.dk = dptr(dk), A.dv = dptr(dv);
      queue(typed("attn_rel_dkdv", q.scalar_type()), A);
      out[1] = dk.narrow(3, 0, D), out[2] = dv.narrow(3, 0, D);
    }
    if (dq.defined()) out[0] = dq.narrow(3, 0, D);
    out[3] = dtable;
    note_gpu("torch_vulkan::relative_bias_attention_backward");
    return out;
  }
};

}  // namespace

namespace vkt {

at::Tensor relative_bias_attention_vk(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                      const std::optional<at::Tensor>& key_mask, bool causal, std::optional<double> scale,
                                      int64_t max_distance, int64_t query_offset) {
  const char* const who = "relative_bias_attention";
  for (const at::Tensor* t : {&q, &k, &v, &table})
    TORCH_CHECK(on_vk(*t) && float_code(t->scalar_type()) >= 0 && t->scalar_type() == q.scalar_type(), who,
                ": q, k, v and table must be vk tensors of one type, float32, bfloat16 or float16");
  for (const at::Tensor* t : {&q, &k, &v, &table}) no_tangent(*t, who);
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, who, ": q, k and v must be [B, H, S, D], got ", q.sizes(), k.sizes(), v.sizes());
  const int64_t B = q.size(0), H = q.size(1), Sq = q.size(2), Sk = k.size(2), D = q.size(3);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(1) == H && k.size(3) == D, who,
              ": k and v must be [", B, ", ", H, ", Sk, ", D, "] (as many heads as q), got ", k.sizes(), v.sizes());
  TORCH_CHECK(D >= 1 && D <= 128, who, ": D must be 1..128, got ", D);
  constexpr int64_t lim = int64_t(1) << 31;
  TORCH_CHECK(Sq < lim && Sk < lim && B * H < lim, who, ": too long");
  TORCH_CHECK(table.dim() == 2 && table.size(1) == H, who, ": table must be [buckets, ", H, "], got ", table.sizes());
  uint16_t start[256];
  TORCH_CHECK(table.size(0) <= 512 && max_distance >= 0 && max_distance <= 1024 &&
                  hrt_attn_rel_buckets(static_cast<int32_t>(table.size(0)), static_cast<int32_t>(max_distance), causal, start) > 0,
              who, ": buckets must be 2..256 where causal, else even and 4..512, with max_distance above half of one direction's and at most 1024, got ",
              table.size(0), " buckets and max_distance ", max_distance);
  const double sc = scale.value_or(1.0 / std::sqrt(static_cast<double>(D)));
  TORCH_CHECK(sc >= 1e-20 && sc <= 1e20, who, ": scale must lie in 1e-20 .. 1e20, got ", sc);
  constexpr int64_t far = int64_t(1) << 40;
  TORCH_CHECK(query_offset >= -far && query_offset <= far, who, ": query_offset out of range, got ", query_offset);
  at::Tensor mask;
  if (present(key_mask)) {
    TORCH_CHECK(on_vk(*key_mask) && key_mask->scalar_type() == at::kBool && key_mask->dim() == 2 && key_mask->size(1) == Sk &&
                    (key_mask->size(0) == B || key_mask->size(0) == 1),
                who, ": key_mask must be a bool vk tensor [", B, " or 1, ", Sk, "], got ", key_mask->scalar_type(), key_mask->sizes());
    mask = Sk <= 1 || key_mask->stride(1) == 1 ? *key_mask : key_mask->contiguous();
  }
  const bool wants = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || table.requires_grad());
  note_gpu("torch_vulkan::relative_bias_attention");
  if (wants) {
    const std::optional<at::Tensor> m = mask.defined() ? std::optional<at::Tensor>(mask) : std::nullopt;
    return Attention::apply(q, k, v, table, m, causal, sc, max_distance, query_offset);
  }
  if (q.numel() == 0 || Sk == 0) return at::zeros(q.sizes(), q.options());
  const int64_t p = per16(q.scalar_type()), Dp = (D + p - 1) / p * p;
  const at::Tensor o =
      std::get<0>(forward_rows(rows_of(q, Dp), rows_of(k, Dp), rows_of(v, Dp), dense(table), mask, {causal, sc, max_distance, query_offset}, false));
  return Dp == D ? o : o.narrow(3, 0, D);
}

}  // namespace vkt
