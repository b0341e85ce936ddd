// Native host path of the latent cache's operators (include/pith_latent.h): part of torch_ops.cpp, which includes it behind its helpers. The same two
// layers: what is not of ordinary layout, or rejected by the library, goes to the Python body, nothing having been launched.
#pragma once

#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPGuard.h>

#include "pith_latent.h"

namespace {

bool on(const Tensor& t, const Tensor& like) { return t.is_cuda() && t.device() == like.device(); }
bool is_index(const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef shape) {
  return on(t, like) && t.scalar_type() == type && t.sizes() == shape && t.is_contiguous();
}
// [.., d] bf16 with unit stride along the features
bool rows_of(const Tensor& t, const Tensor& like, int64_t dim, int64_t d) {
  return on(t, like) && t.scalar_type() == at::kBFloat16 && t.dim() == dim && t.size(dim - 1) == d && t.stride(dim - 1) == 1;
}
// Token and head stride of a [T, H, d] tensor (of a dimension of one element: what a contiguous one has).
void token_strides(const Tensor& t, int64_t* ts, int64_t* hs) {
  *ts = t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
  *hs = t.size(1) > 1 ? t.stride(1) : t.size(2);
}

// A new tensor on the device of `like`, past the dispatcher: nothing between this op and the allocator wants to see it.
Tensor fresh(const Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) { return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt); }

bool checking_positions() {
  const char* e = std::getenv("PITHTRAIN_AMD_CHECK_POSITIONS");
  return e && e[0] == '1' && e[1] == 0;
}

bool latent_cache_args(pith_latent_cache& c, const Tensor& like, const Tensor& latent, const Tensor& k_pe, const OptTensor& scale) {
  const bool fp8 = latent.scalar_type() == at::kFloat8_e4m3fn;
  if (!on(latent, like) || !on(k_pe, like) || latent.dim() != 3 || latent.size(2) != PITH_LATENT_DIM || (!fp8 && latent.scalar_type() != at::kBFloat16)) return false;
  const int64_t pages = latent.size(0), page = latent.size(1);
  if (k_pe.scalar_type() != at::kBFloat16 || !has_shape(k_pe, {pages, page, PITH_LATENT_ROPE_DIM}) || latent.stride(2) != 1 || latent.stride(1) != PITH_LATENT_DIM ||
      k_pe.stride(2) != 1 || k_pe.stride(1) != PITH_LATENT_ROPE_DIM || fp8 != scale.has_value())
    return false;
  if (fp8) {
    if (!on(*scale, like) || scale->scalar_type() != at::kFloat || !has_shape(*scale, {pages, page}) || scale->stride(1) != 1) return false;
    c.scale = scale->data_ptr<float>();
    c.scale_ps = scale->stride(0);
  }
  c.latent = latent.data_ptr(); c.k_pe = k_pe.data_ptr();
  c.pages = pages; c.page_size = page;
  c.latent_ps = latent.stride(0); c.k_pe_ps = k_pe.stride(0);
  c.dtype = fp8 ? PITH_FP8_E4M3 : PITH_BF16;
  return true;
}

bool rotary_tables(const Tensor& cos, const Tensor& sin, const Tensor& like, int64_t* positions) {
  if (!on(cos, like) || !on(sin, like) || cos.scalar_type() != at::kBFloat16 || sin.scalar_type() != at::kBFloat16 || cos.dim() != 2 ||
      cos.size(1) != PITH_LATENT_ROPE_DIM || cos.sizes() != sin.sizes() || !cos.is_contiguous() || !sin.is_contiguous())
    return false;
  *positions = cos.size(0);
  return true;
}

bool page_table_args(const Tensor& table, const Tensor& like, int64_t b, const int32_t** ptr, int64_t* rs, int64_t* width) {
  if (!on(table, like) || table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != b || (table.size(1) > 1 && table.stride(1) != 1)) return false;
  *ptr = table.data_ptr<int32_t>();
  *width = table.size(1);
  *rs = b > 1 ? table.stride(0) : *width;
  return true;
}

void latent_append(const Tensor& kv_a, const Tensor& weight, const Tensor& cos, const Tensor& sin, const Tensor& pos, const Tensor& slots, const Tensor& latent,
                   const Tensor& k_pe, const OptTensor& scale, double eps) {
  if (kv_a.is_cuda() && !checking_positions()) {
    const c10::hip::HIPGuard guard(kv_a.device().index());
    pith_latent_append_args a = {};
    a.T = kv_a.size(0);
    if (rows_of(kv_a, kv_a, 2, PITH_LATENT_DIM + PITH_LATENT_ROPE_DIM) && on(weight, kv_a) && has_shape(weight, {PITH_LATENT_DIM}) && weight.is_contiguous() &&
        dtype_code(weight, &a.weight_dtype) && rotary_tables(cos, sin, kv_a, &a.P) && is_index(pos, kv_a, at::kLong, {a.T}) &&
        is_index(slots, kv_a, at::kLong, {a.T}) && latent_cache_args(a.cache, kv_a, latent, k_pe, scale)) {
      a.kv_a = kv_a.data_ptr(); a.weight = weight.data_ptr(); a.cos = cos.data_ptr(); a.sin = sin.data_ptr();
      a.position_ids = pos.data_ptr<int64_t>(); a.slots = slots.data_ptr<int64_t>();
      a.kv_a_rs = a.T > 1 ? kv_a.stride(0) : kv_a.size(1);
      a.eps = (float)eps;
      if (accepted(pith_latent_append(&a, stream_of(kv_a)))) return;
    }
  }
  py::gil_scoped_acquire gil;
  bodies()["latent_append"](kv_a, weight, cos, sin, pos, slots, latent, k_pe, scale, eps);
}

Two latent_gather(const Tensor& latent, const Tensor& k_pe, const OptTensor& scale, const Tensor& table, const Tensor& cu_rows, int64_t rows) {
  if (latent.is_cuda() && rows >= 0 && cu_rows.dim() == 1 && cu_rows.numel() > 0) {
    const c10::hip::HIPGuard guard(latent.device().index());
    pith_latent_gather_args a = {};
    a.B = cu_rows.numel() - 1;
    a.rows = rows;
    if (latent_cache_args(a.cache, latent, latent, k_pe, scale) && is_index(cu_rows, latent, at::kInt, {a.B + 1}) &&
        page_table_args(table, latent, a.B, &a.page_table, &a.table_rs, &a.table_width)) {
      Tensor out = fresh(latent, {rows, PITH_LATENT_DIM}, at::kBFloat16), pe = fresh(latent, {rows, PITH_LATENT_ROPE_DIM}, at::kBFloat16);
      a.cu_rows = cu_rows.data_ptr<int32_t>();
      a.latent_out = out.data_ptr(); a.k_pe_out = pe.data_ptr();
      a.latent_rs = PITH_LATENT_DIM; a.k_pe_rs = PITH_LATENT_ROPE_DIM;
      if (accepted(pith_latent_gather(&a, stream_of(latent)))) return {out, pe};
    }
  }
  return python_body<Two>("latent_gather", latent, k_pe, scale, table, cu_rows, rows);
}

bool absorb_args(pith_latent_absorb_args& a, const Tensor& x, const Tensor& weight, const Tensor& out, int64_t features) {
  if (!rows_of(x, x, 3, features) || !on(weight, x) || weight.scalar_type() != at::kBFloat16 || !weight.is_contiguous() || weight.dim() < 1 ||
      weight.size(-1) != PITH_LATENT_DIM || weight.numel() != x.size(1) * (PITH_LATENT_NOPE_DIM + PITH_LATENT_VALUE_DIM) * PITH_LATENT_DIM)
    return false;
  a.x = x.data_ptr(); a.weight = weight.data_ptr(); a.out = out.data_ptr();
  a.T = x.size(0); a.H = x.size(1);
  token_strides(x, &a.x_ts, &a.x_hs);
  token_strides(out, &a.out_ts, &a.out_hs);
  return true;
}

Two latent_absorb_query(const Tensor& q, const Tensor& weight, const Tensor& cos, const Tensor& sin, const Tensor& pos) {
  if (q.is_cuda() && q.dim() == 3 && !checking_positions()) {
    const c10::hip::HIPGuard guard(q.device().index());
    Tensor out = fresh(q, {q.size(0), q.size(1), PITH_LATENT_DIM}, q.scalar_type()), pe = fresh(q, {q.size(0), q.size(1), PITH_LATENT_ROPE_DIM}, q.scalar_type());
    pith_latent_absorb_args a = {};
    if (absorb_args(a, q, weight, out, PITH_LATENT_NOPE_DIM + PITH_LATENT_ROPE_DIM) && rotary_tables(cos, sin, q, &a.P) && is_index(pos, q, at::kLong, {a.T})) {
      a.q_pe = pe.data_ptr();
      token_strides(pe, &a.q_pe_ts, &a.q_pe_hs);
      a.cos = cos.data_ptr(); a.sin = sin.data_ptr(); a.position_ids = pos.data_ptr<int64_t>();
      if (accepted(pith_latent_absorb_query(&a, stream_of(q)))) return {out, pe};
    }
  }
  return python_body<Two>("latent_absorb_query", q, weight, cos, sin, pos);
}

Tensor latent_absorb_value(const Tensor& x, const Tensor& weight) {
  if (x.is_cuda() && x.dim() == 3) {
    const c10::hip::HIPGuard guard(x.device().index());
    Tensor out = fresh(x, {x.size(0), x.size(1), PITH_LATENT_VALUE_DIM}, x.scalar_type());
    pith_latent_absorb_args a = {};
    if (absorb_args(a, x, weight, out, PITH_LATENT_DIM) && accepted(pith_latent_absorb_value(&a, stream_of(x)))) return out;
  }
  return python_body<Tensor>("latent_absorb_value", x, weight);
}

Two latent_attention(const Tensor& q_latent, const Tensor& q_pe, const Tensor& latent, const Tensor& k_pe, const OptTensor& scale, const Tensor& table,
                     const Tensor& lengths, const Tensor& cu_q, double softmax_scale, const OptTensor& tree) {
  if (q_latent.is_cuda() && rows_of(q_latent, q_latent, 3, PITH_LATENT_DIM) && lengths.dim() == 1 && !(tree && checking_positions())) {
    const c10::hip::HIPGuard guard(q_latent.device().index());
    pith_latent_attn_args a = {};
    a.T = q_latent.size(0); a.H = q_latent.size(1); a.B = lengths.size(0);
    if (rows_of(q_pe, q_latent, 3, PITH_LATENT_ROPE_DIM) && q_pe.size(0) == a.T && q_pe.size(1) == a.H && latent_cache_args(a.cache, q_latent, latent, k_pe, scale) &&
        page_table_args(table, q_latent, a.B, &a.page_table, &a.table_rs, &a.table_width) && is_index(lengths, q_latent, at::kInt, {a.B}) &&
        is_index(cu_q, q_latent, at::kInt, {a.B + 1}) && (!tree || is_index(*tree, q_latent, at::kLong, {a.T}))) {
      Tensor o = fresh(q_latent, {a.T, a.H, PITH_LATENT_DIM}, at::kBFloat16), lse = fresh(q_latent, {a.H, a.T}, at::kFloat);
      a.q_latent = q_latent.data_ptr(); a.q_pe = q_pe.data_ptr(); a.o = o.data_ptr(); a.lse = lse.data_ptr<float>();
      a.lengths = lengths.data_ptr<int32_t>(); a.cu_q = cu_q.data_ptr<int32_t>();
      a.tree_mask = tree ? tree->data_ptr<int64_t>() : nullptr;
      token_strides(q_latent, &a.q_ts, &a.q_hs);
      token_strides(q_pe, &a.q_pe_ts, &a.q_pe_hs);
      token_strides(o, &a.o_ts, &a.o_hs);
      a.lse_hs = a.T;
      a.scale = (float)softmax_scale;
      a.workspace_bytes = pith_latent_attn_workspace_bytes(&a);
      Tensor ws = fresh(q_latent, {a.workspace_bytes}, at::kByte);
      a.workspace = ws.data_ptr();
      if (accepted(pith_latent_attn(&a, stream_of(q_latent)))) return {o, lse};
    }
  }
  return python_body<Two>("latent_attention", q_latent, q_pe, latent, k_pe, scale, table, lengths, cu_q, softmax_scale, tree);
}

// No gradients: a call that would have to record one, or to carry a forward-mode tangent on, is refused rather than cut off from the graph.
bool records(const Tensor& t) { return t.requires_grad(); }
bool records(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
bool records(double) { return false; }
bool records(int64_t) { return false; }
template <auto BODY>
struct ServingOp;
template <typename R, typename... Args, R (*BODY)(Args...)>
struct ServingOp<BODY> {
  template <const char* NAME>
  static R call(c10::DispatchKeySet keys, Args... args) {
    static const auto op = op_handle<R(Args...)>(NAME);
    TORCH_CHECK(!at::GradMode::is_enabled() || !(records(args) || ...), NAME, " has no backward: call it under torch.no_grad(), or detach what requires a gradient");
    TORCH_CHECK(!(tangent(args) || ...), NAME, " has no forward-mode derivative");
    at::AutoDispatchBelowAutograd guard;
    return op.redispatch(keys & c10::after_autograd_keyset, args...);
  }
};

constexpr char kLatentAppend[] = "pithtrain_amd::latent_append", kLatentGather[] = "pithtrain_amd::latent_gather",
               kLatentAbsorbQuery[] = "pithtrain_amd::latent_absorb_query", kLatentAbsorbValue[] = "pithtrain_amd::latent_absorb_value",
               kLatentAttention[] = "pithtrain_amd::latent_attention";

// Below autograd, also where no gradient is recorded: the tensors that append writes count as changed, so that a backward which saved one of them (or a view)
// notices. Those made in inference mode have no such count and are never saved.
void latent_append_counted(c10::DispatchKeySet keys, const Tensor& kv_a, const Tensor& weight, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                           const Tensor& slots, const Tensor& latent, const Tensor& k_pe, const OptTensor& scale, double eps) {
  static const auto op = op_handle<decltype(latent_append)>(kLatentAppend);
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    op.redispatch(keys & c10::after_ADInplaceOrView_keyset, kv_a, weight, cos, sin, pos, slots, latent, k_pe, scale, eps);
  }
  const auto changed = [](const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  changed(latent);
  changed(k_pe);
  if (scale) changed(*scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pithtrain_amd, m) {
  m.def("latent_append(Tensor kv_a, Tensor weight, Tensor cos, Tensor sin, Tensor position_ids, Tensor slots, Tensor(a!) latent, Tensor(b!) k_pe, "
        "Tensor(c!)? scale, float eps) -> ()");
  m.def("latent_gather(Tensor latent, Tensor k_pe, Tensor? scale, Tensor page_table, Tensor cu_rows, int rows) -> (Tensor, Tensor)");
  m.def("latent_absorb_query(Tensor q, Tensor weight, Tensor cos, Tensor sin, Tensor position_ids) -> (Tensor, Tensor)");
  m.def("latent_absorb_value(Tensor o_latent, Tensor weight) -> Tensor");
  m.def("latent_attention(Tensor q_latent, Tensor q_pe, Tensor latent, Tensor k_pe, Tensor? scale, Tensor page_table, Tensor lengths, Tensor cu_q, "
        "float softmax_scale, Tensor? tree_mask) -> (Tensor, Tensor)");
}

#define PITH_LATENT_IMPL(key)                              \
  TORCH_LIBRARY_IMPL(pithtrain_amd, key, m) {              \
    m.impl("latent_append", &latent_append);               \
    m.impl("latent_gather", &latent_gather);               \
    m.impl("latent_absorb_query", &latent_absorb_query);   \
    m.impl("latent_absorb_value", &latent_absorb_value);   \
    m.impl("latent_attention", &latent_attention);         \
  }
PITH_LATENT_IMPL(CUDA)
PITH_LATENT_IMPL(CPU)
#undef PITH_LATENT_IMPL

TORCH_LIBRARY_IMPL(pithtrain_amd, ADInplaceOrView, m) { m.impl("latent_append", &latent_append_counted); }

TORCH_LIBRARY_IMPL(pithtrain_amd, Autograd, m) {
  m.impl("latent_append", &ServingOp<&latent_append>::call<kLatentAppend>);
  m.impl("latent_gather", &ServingOp<&latent_gather>::call<kLatentGather>);
  m.impl("latent_absorb_query", &ServingOp<&latent_absorb_query>::call<kLatentAbsorbQuery>);
  m.impl("latent_absorb_value", &ServingOp<&latent_absorb_value>::call<kLatentAbsorbValue>);
  m.impl("latent_attention", &ServingOp<&latent_attention>::call<kLatentAttention>);
}
