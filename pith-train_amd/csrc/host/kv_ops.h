// Native host path of the key-value cache's operators and the planning of a step (include/pith_kv.h): part of torch_ops.cpp, which includes it behind
// latent_ops.h, whose helpers it shares. The same two layers: what is not of ordinary layout, or rejected by the library, goes to the Python body, nothing
// having been launched.
#pragma once

#include "pith_kv.h"

namespace {

// A page's part of the tensor is contiguous.
bool contiguous_pages(const Tensor& t) {
  int64_t expected = 1;
  for (int64_t i = t.dim() - 1; i > 0; --i) {
    if (t.size(i) != 1 && t.stride(i) != expected) return false;
    expected *= t.size(i);
  }
  return true;
}

bool kv_cache_args(pith_kv_cache& c, const Tensor& like, const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale) {
  const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  if (!on(k, like) || !on(v, like) || k.dim() != 4 || (!fp8 && k.scalar_type() != at::kBFloat16) || v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() ||
      !contiguous_pages(k) || !contiguous_pages(v) || fp8 != k_scale.has_value() || fp8 != v_scale.has_value())
    return false;
  if (fp8) {
    for (const Tensor* t : {&*k_scale, &*v_scale})
      if (!on(*t, like) || t->scalar_type() != at::kFloat || t->sizes() != k.sizes().slice(0, 3) || !contiguous_pages(*t)) return false;
    c.k_scale = k_scale->data_ptr<float>(); c.v_scale = v_scale->data_ptr<float>();
    c.k_scale_ps = k_scale->stride(0); c.v_scale_ps = v_scale->stride(0);
  }
  c.k = k.data_ptr(); c.v = v.data_ptr();
  c.pages = k.size(0); c.heads = k.size(1); c.page_size = k.size(2); c.dim = k.size(3);
  c.k_ps = k.stride(0); c.v_ps = v.stride(0);
  c.dtype = fp8 ? PITH_FP8_E4M3 : PITH_BF16;
  return true;
}

// cu_q, lengths and page table of B sequences.
template <typename A>
bool sequence_args(A& a, const Tensor& like, const Tensor& table, const Tensor& lengths, const OptTensor& cu_q) {
  a.B = lengths.dim() == 1 ? lengths.size(0) : -1;
  if (a.B < 0 || !is_index(lengths, like, at::kInt, {a.B}) || !page_table_args(table, like, a.B, &a.page_table, &a.table_rs, &a.table_width)) return false;
  if (cu_q ? !is_index(*cu_q, like, at::kInt, {a.B + 1}) : a.T != a.B) return false;
  a.lengths = lengths.data_ptr<int32_t>();
  a.cu_q = cu_q ? cu_q->data_ptr<int32_t>() : nullptr;
  return true;
}

// A part of `whole` as a tensor of its own: n elements from byte `at` on.
Tensor part_of(const Tensor& whole, int64_t at, int64_t n, at::ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

using Six = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

Six plan_step(const Tensor& counts, const Tensor& lengths, const Tensor& table, const Tensor& free_pages, const Tensor& free_count, int64_t page_size, int64_t tokens) {
  if (counts.is_cuda() && counts.dim() == 1 && free_pages.dim() == 1 && tokens >= 0) {
    const c10::hip::HIPGuard guard(counts.device().index());
    pith_plan_step_args a = {};
    a.B = counts.size(0); a.T = tokens; a.page_size = page_size; a.pool_size = free_pages.size(0);
    const int32_t* entries = nullptr;
    if (is_index(counts, counts, at::kInt, {a.B}) && is_index(lengths, counts, at::kInt, {a.B}) && page_table_args(table, counts, a.B, &entries, &a.table_rs, &a.table_width) &&
        is_index(free_pages, counts, at::kInt, {a.pool_size}) && is_index(free_count, counts, at::kInt, {1})) {
      // one allocation for all results and the workspace: six of them would take longer than the kernel, and a second one, for what the next step begins with, 0.6 of 6.3 us (a
      // result that is kept keeps all of them: 16 bytes a token and 12 a request, until the next step's take its place)
      a.workspace_bytes = pith_plan_step_workspace_bytes(&a);
      // (their parts begin at multiples of 16 bytes, which compiled graphs expect of a result)
      int64_t end = a.workspace_bytes;
      const auto place = [&](int64_t n, int64_t size) { return std::exchange(end, (end + n * size + 15) & ~(int64_t)15); };
      const int64_t at_positions = place(tokens, 8), at_slots = place(tokens, 8), at_cu = place(a.B + 1, 4), at_after = place(a.B, 4), at_granted = place(a.B, 4), at_count = place(1, 4);
      const Tensor whole = fresh(counts, {end}, at::kByte);
      const Tensor positions = part_of(whole, at_positions, tokens, at::kLong), slots = part_of(whole, at_slots, tokens, at::kLong), cu_q = part_of(whole, at_cu, a.B + 1, at::kInt),
                   after = part_of(whole, at_after, a.B, at::kInt), granted = part_of(whole, at_granted, a.B, at::kInt), count = part_of(whole, at_count, 1, at::kInt);
      a.workspace = whole.data_ptr();
      a.counts = counts.data_ptr<int32_t>(); a.lengths = lengths.data_ptr<int32_t>();
      a.page_table = table.data_ptr<int32_t>();
      a.free_pages = free_pages.data_ptr<int32_t>(); a.free_count = free_count.data_ptr<int32_t>();
      a.cu_q = cu_q.data_ptr<int32_t>(); a.position_ids = positions.data_ptr<int64_t>(); a.slots = slots.data_ptr<int64_t>();
      a.granted = granted.data_ptr<int32_t>(); a.lengths_out = after.data_ptr<int32_t>(); a.free_count_out = count.data_ptr<int32_t>();
      if (accepted(pith_plan_step(&a, stream_of(counts)))) return {cu_q, after, positions, slots, granted, count};
    }
  }
  return python_body<Six>("plan_step", counts, lengths, table, free_pages, free_count, page_size, tokens);
}

Tensor kv_append(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& q_weight, const OptTensor& k_weight, const Tensor& cos, const Tensor& sin,
                 const Tensor& pos, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_scale, const OptTensor& v_scale, double eps) {
  if (q.is_cuda() && q.dim() == 3 && !checking_positions()) {
    const c10::hip::HIPGuard guard(q.device().index());
    pith_kv_append_args a = {};
    a.T = q.size(0); a.H = q.size(1);
    bool ok = kv_cache_args(a.cache, q, k_cache, v_cache, k_scale, v_scale);
    const int64_t d = a.cache.dim;
    ok = ok && rows_of(q, q, 3, d) && rows_of(k, q, 3, d) && rows_of(v, q, 3, d) && k.size(0) == a.T && v.size(0) == a.T && k.size(1) == a.cache.heads &&
         v.size(1) == a.cache.heads && is_index(pos, q, at::kLong, {a.T}) && is_index(slots, q, at::kLong, {a.T}) && q_weight.has_value() == k_weight.has_value();
    for (const Tensor* t : {&cos, &sin}) ok = ok && on(*t, q) && t->scalar_type() == at::kBFloat16 && t->dim() == 2 && t->size(1) == d && t->is_contiguous();
    ok = ok && cos.size(0) == sin.size(0);
    if (ok && q_weight) {
      for (const Tensor* t : {&*q_weight, &*k_weight}) ok = ok && on(*t, q) && has_shape(*t, {d}) && t->is_contiguous() && t->scalar_type() == q_weight->scalar_type();
      ok = ok && dtype_code(*q_weight, &a.weight_dtype);
      a.q_weight = q_weight->data_ptr(); a.k_weight = k_weight->data_ptr();
    }
    if (ok) {
      Tensor out = fresh(q, q.sizes(), at::kBFloat16);
      a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.q_out = out.data_ptr();
      a.cos = cos.data_ptr(); a.sin = sin.data_ptr(); a.P = cos.size(0);
      a.position_ids = pos.data_ptr<int64_t>(); a.slots = slots.data_ptr<int64_t>();
      token_strides(q, &a.q_ts, &a.q_hs);
      token_strides(k, &a.k_ts, &a.k_hs);
      token_strides(v, &a.v_ts, &a.v_hs);
      token_strides(out, &a.q_out_ts, &a.q_out_hs);
      a.eps = (float)eps;
      if (accepted(pith_kv_append(&a, stream_of(q)))) return out;
    }
  }
  return python_body<Tensor>("kv_append", q, k, v, q_weight, k_weight, cos, sin, pos, slots, k_cache, v_cache, k_scale, v_scale, eps);
}

Two kv_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& table, const Tensor& lengths,
                 const OptTensor& cu_q, double softmax_scale, const OptTensor& tree) {
  if (q.is_cuda() && q.dim() == 3 && !(tree && checking_positions())) {
    const c10::hip::HIPGuard guard(q.device().index());
    pith_kv_attn_args a = {};
    a.T = q.size(0); a.H = q.size(1);
    bool ok = kv_cache_args(a.cache, q, k, v, k_scale, v_scale) && rows_of(q, q, 3, a.cache.dim) && (!tree || is_index(*tree, q, at::kLong, {a.T}));
    if (ok && lengths.dim() == 2) {  // tables of the heads
      a.B = lengths.size(0);
      ok = !tree && !cu_q && is_index(lengths, q, at::kInt, {a.B, a.cache.heads}) && on(table, q) && table.scalar_type() == at::kInt && table.dim() == 3 && table.size(0) == a.B &&
           table.size(1) == a.cache.heads && (table.size(2) == 1 || table.stride(2) == 1) && a.T == a.B;
      if (ok) {
        a.page_table = table.data_ptr<int32_t>(); a.lengths = lengths.data_ptr<int32_t>();
        a.table_width = table.size(2);
        a.table_hs = a.cache.heads > 1 ? table.stride(1) : a.table_width;
        a.table_rs = a.B > 1 ? table.stride(0) : a.table_width * a.cache.heads;
        a.head_tables = 1;
      }
    } else {
      ok = ok && sequence_args(a, q, table, lengths, cu_q);
    }
    if (ok) {
      Tensor o = fresh(q, q.sizes(), at::kBFloat16), lse = fresh(q, {a.H, a.T}, at::kFloat);
      a.q = q.data_ptr(); a.o = o.data_ptr(); a.lse = lse.data_ptr<float>();
      a.tree_mask = tree ? tree->data_ptr<int64_t>() : nullptr;
      token_strides(q, &a.q_ts, &a.q_hs);
      token_strides(o, &a.o_ts, &a.o_hs);
      a.lse_hs = a.T;
      a.scale = (float)softmax_scale;
      a.workspace_bytes = pith_kv_attn_workspace_bytes(&a);
      Tensor ws = fresh(q, {a.workspace_bytes}, at::kByte);
      a.workspace = ws.data_ptr();
      if (accepted(pith_kv_attn(&a, stream_of(q)))) return {o, lse};
    }
  }
  return python_body<Two>("kv_attention", q, k, v, k_scale, v_scale, table, lengths, cu_q, softmax_scale, tree);
}

bool bounds_beside(const Tensor& bounds, const Tensor& like) {
  return on(bounds, like) && bounds.scalar_type() == at::kBFloat16 && bounds.dim() == 4 && bounds.size(2) == 2 && contiguous_pages(bounds);
}

void kv_bounds(const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& bounds, const Tensor& table, const Tensor& lengths,
               const OptTensor& cu_q, int64_t tokens) {
  if (k.is_cuda()) {
    const c10::hip::HIPGuard guard(k.device().index());
    pith_kv_bounds_args a = {};
    a.T = tokens;
    if (kv_cache_args(a.cache, k, k, v, k_scale, v_scale) && bounds_beside(bounds, k) && bounds.size(0) == a.cache.pages && bounds.size(1) == a.cache.heads &&
        bounds.size(3) == a.cache.dim && sequence_args(a, k, table, lengths, cu_q)) {
      a.bounds = bounds.data_ptr();
      a.bounds_ps = bounds.stride(0);
      if (accepted(pith_kv_bounds(&a, stream_of(k)))) return;
    }
  }
  py::gil_scoped_acquire gil;
  bodies()["kv_bounds"](k, v, k_scale, v_scale, bounds, table, lengths, cu_q, tokens);
}

Two kv_select(const Tensor& q, const Tensor& bounds, const Tensor& table, const Tensor& lengths, const OptTensor& cu_q, int64_t page_size, int64_t keep) {
  if (q.is_cuda() && q.dim() == 3 && bounds_beside(bounds, q) && rows_of(q, q, 3, bounds.size(3)) && keep >= 1) {
    const c10::hip::HIPGuard guard(q.device().index());
    pith_kv_select_args a = {};
    a.T = q.size(0); a.H = q.size(1);
    a.pages = bounds.size(0); a.heads = bounds.size(1); a.dim = bounds.size(3);
    a.page_size = page_size; a.keep = keep;
    if (sequence_args(a, q, table, lengths, cu_q) && a.B > 0) {
      Tensor chosen = fresh(q, {a.T, a.heads, keep}, at::kInt), rows = fresh(q, {a.T, a.heads}, at::kInt);
      a.q = q.data_ptr(); a.bounds = bounds.data_ptr(); a.bounds_ps = bounds.stride(0);
      a.table_out = chosen.data_ptr<int32_t>(); a.lengths_out = rows.data_ptr<int32_t>();
      token_strides(q, &a.q_ts, &a.q_hs);
      a.workspace_bytes = pith_kv_select_workspace_bytes(&a);
      Tensor ws = fresh(q, {a.workspace_bytes}, at::kByte);
      a.workspace = ws.data_ptr();
      if (accepted(pith_kv_select(&a, stream_of(q)))) return {chosen, rows};
    }
  }
  return python_body<Two>("kv_select", q, bounds, table, lengths, cu_q, page_size, keep);
}

constexpr char kPlanStep[] = "pithtrain_amd::plan_step", kKVAppend[] = "pithtrain_amd::kv_append", kKVAttention[] = "pithtrain_amd::kv_attention",
               kKVBounds[] = "pithtrain_amd::kv_bounds", kKVSelect[] = "pithtrain_amd::kv_select";

// Below autograd: what an operator writes counts as changed (see latent_append_counted).
void count_changed(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
const Tensor* given(const OptTensor& t) { return t ? &*t : nullptr; }

Six plan_step_counted(c10::DispatchKeySet keys, const Tensor& counts, const Tensor& lengths, const Tensor& table, const Tensor& free_pages, const Tensor& free_count,
                      int64_t page_size, int64_t tokens) {
  static const auto op = op_handle<decltype(plan_step)>(kPlanStep);
  Six plan = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.redispatch(keys & c10::after_ADInplaceOrView_keyset, counts, lengths, table, free_pages, free_count, page_size, tokens);
  }();
  count_changed({&table, &free_pages});
  return plan;
}

Tensor kv_append_counted(c10::DispatchKeySet keys, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& q_weight, const OptTensor& k_weight,
                         const Tensor& cos, const Tensor& sin, const Tensor& pos, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache,
                         const OptTensor& k_scale, const OptTensor& v_scale, double eps) {
  static const auto op = op_handle<decltype(kv_append)>(kKVAppend);
  Tensor out = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.redispatch(keys & c10::after_ADInplaceOrView_keyset, q, k, v, q_weight, k_weight, cos, sin, pos, slots, k_cache, v_cache, k_scale, v_scale, eps);
  }();
  count_changed({&k_cache, &v_cache, given(k_scale), given(v_scale)});
  return out;
}

void kv_bounds_counted(c10::DispatchKeySet keys, const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& bounds,
                       const Tensor& table, const Tensor& lengths, const OptTensor& cu_q, int64_t tokens) {
  static const auto op = op_handle<decltype(kv_bounds)>(kKVBounds);
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    op.redispatch(keys & c10::after_ADInplaceOrView_keyset, k, v, k_scale, v_scale, bounds, table, lengths, cu_q, tokens);
  }
  count_changed({&bounds});
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pithtrain_amd, m) {
  m.def("plan_step(Tensor counts, Tensor lengths, Tensor(a!) page_table, Tensor(b!) free_pages, Tensor free_count, int page_size, int tokens) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("kv_append(Tensor q, Tensor k, Tensor v, Tensor? q_weight, Tensor? k_weight, Tensor cos, Tensor sin, Tensor position_ids, Tensor slots, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, float eps) -> Tensor");
  m.def("kv_attention(Tensor q, Tensor k, Tensor v, Tensor? k_scale, Tensor? v_scale, Tensor page_table, Tensor lengths, Tensor? cu_q, float softmax_scale, "
        "Tensor? tree_mask) -> (Tensor, Tensor)");
  m.def("kv_bounds(Tensor k, Tensor v, Tensor? k_scale, Tensor? v_scale, Tensor(a!) bounds, Tensor page_table, Tensor lengths, Tensor? cu_q, int tokens) -> ()");
  m.def("kv_select(Tensor q, Tensor bounds, Tensor page_table, Tensor lengths, Tensor? cu_q, int page_size, int keep) -> (Tensor, Tensor)");
}

#define PITH_KV_IMPL(key)                      \
  TORCH_LIBRARY_IMPL(pithtrain_amd, key, m) {  \
    m.impl("plan_step", &plan_step);           \
    m.impl("kv_append", &kv_append);           \
    m.impl("kv_attention", &kv_attention);     \
    m.impl("kv_bounds", &kv_bounds);           \
    m.impl("kv_select", &kv_select);           \
  }
PITH_KV_IMPL(CUDA)
PITH_KV_IMPL(CPU)
#undef PITH_KV_IMPL

TORCH_LIBRARY_IMPL(pithtrain_amd, ADInplaceOrView, m) {
  m.impl("plan_step", &plan_step_counted);
  m.impl("kv_append", &kv_append_counted);
  m.impl("kv_bounds", &kv_bounds_counted);
}

TORCH_LIBRARY_IMPL(pithtrain_amd, Autograd, m) {
  m.impl("plan_step", &ServingOp<&plan_step>::call<kPlanStep>);
  m.impl("kv_append", &ServingOp<&kv_append>::call<kKVAppend>);
  m.impl("kv_attention", &ServingOp<&kv_attention>::call<kKVAttention>);
  m.impl("kv_bounds", &ServingOp<&kv_bounds>::call<kKVBounds>);
  m.impl("kv_select", &ServingOp<&kv_select>::call<kKVSelect>);
}
