// PyTorch operator library over the C ABI (include/sgld_b200.h): registers
//   torch.ops.sglang_decode.plan_build, .decode, .decode_shared_prefix, .merge,
//   .prompt_attention and .norm_rope
// so the decode path is visible to torch's operator registry (schemas with mutation
// annotations, Meta kernels for tracing) while every launch still goes through the
// torch-free C entry points of libsgld_sm100.so.  Argument checks, strides, pointers and
// the current CUDA stream are read here, in C++, so a decode step costs Python one
// operator call per launch group.
//
// The ops replace the reference's Triton launches: plan_build <- planning/builder.py:6-28,
// decode <- runtime/engine.py:62-73, merge <- kernels/merge.py:7-30.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>

#include <algorithm>
#include <cstring>
#include <string>

#include "sgld_b200.h"

namespace {

void check_status(int rc, const char* what) {
  if (rc == SGLD_OK) return;
  const std::string msg = std::string(what) + ": " + sgld_last_error();
  if (rc == SGLD_ERR_INVALID_ARGUMENT || rc == SGLD_ERR_UNSUPPORTED) TORCH_CHECK_VALUE(false, msg);
  TORCH_CHECK(false, msg);
}

int32_t dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return SGLD_DTYPE_F16;
    case at::kBFloat16: return SGLD_DTYPE_BF16;
    case at::kFloat8_e4m3fn: return SGLD_DTYPE_E4M3;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t.scalar_type());
  }
  return -1;
}

sgld_plan_geometry geometry_of(at::IntArrayRef g) {
  TORCH_CHECK_VALUE(g.size() == 5, "geometry is (batch_capacity, max_splits, max_context, groups, workers)");
  return sgld_plan_geometry{static_cast<int32_t>(g[0]), static_cast<int32_t>(g[1]), static_cast<int32_t>(g[2]),
                            static_cast<int32_t>(g[3]), static_cast<int32_t>(g[4])};
}

// The plan is one contiguous int32 storage, laid out as sgld_plan_buffers_in_storage says.
sgld_plan_buffers plan_of(const at::Tensor& storage, const sgld_plan_geometry& g) {
  TORCH_CHECK_VALUE(storage.scalar_type() == at::kInt && storage.is_cuda() && storage.is_contiguous(),
                    "the plan storage must be a contiguous int32 CUDA tensor");
  const size_t words = sgld_plan_storage_words(&g);
  TORCH_CHECK_VALUE(words > 0 && static_cast<size_t>(storage.numel()) >= words, "the plan storage holds ",
                    storage.numel(), " int32 words; the geometry needs ", words);
  sgld_plan_buffers b;
  check_status(sgld_plan_buffers_in_storage(storage.data_ptr<int32_t>(), &g, &b), "sgld_plan_buffers_in_storage");
  return b;
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool finite_positive(double x) { return x > 0.0 && x <= 3.0e38; }

void plan_build(const at::Tensor& plan, at::IntArrayRef geometry, int64_t force_mode,
                const std::optional<at::Tensor>& rules, int64_t n_rules, const std::optional<at::Tensor>& counters) {
  const c10::cuda::CUDAGuard guard(plan.device());
  const sgld_plan_geometry g = geometry_of(geometry);
  const sgld_plan_buffers p = plan_of(plan, g);
  const int32_t* r = rules.has_value() && n_rules > 0 ? rules->data_ptr<int32_t>() : nullptr;
  int32_t* c = counters.has_value() ? counters->data_ptr<int32_t>() : nullptr;
  const int32_t nc = counters.has_value() ? static_cast<int32_t>(counters->numel()) : 0;
  check_status(sgld_plan_build(&p, &g, static_cast<int32_t>(force_mode), r, static_cast<int32_t>(n_rules), c, nc,
                               stream_of(plan)),
               "sgld_plan_build");
}

// The engine's argument checks: the reference's runtime/engine.py:35-61, plus the additions
// (fewer Q rows than the capacity, fp8 K/V, logit cap, the fused KV-cache write).  Query
// heads and head_dim come from `out` ([capacity, query_heads, head_dim], the engine's output
// buffer), kv_heads from the geometry.  Every failure raises ValueError in Python.
void check_decode_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
                       const std::optional<at::Tensor>& indptr, const at::Tensor& out, const sgld_plan_geometry& g,
                       int64_t page_size, double logit_cap, double k_scale, double v_scale,
                       const std::optional<at::Tensor>& k_new, const std::optional<at::Tensor>& v_new,
                       const std::optional<at::Tensor>& new_loc) {
  const bool kv_fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  const bool q16 = q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16;
  TORCH_CHECK_VALUE(q16 && v.scalar_type() == k.scalar_type() && (k.scalar_type() == q.scalar_type() || kv_fp8),
                    "BF16/FP16 Q/K/V of identical dtype are required (or fp8 e4m3 K/V)");
  TORCH_CHECK_VALUE(out.dim() == 3 && out.size(0) == g.batch_capacity, "out must be [capacity, query_heads, head_dim]");
  const int64_t hq = out.size(1), d = out.size(2), hkv = g.groups;
  TORCH_CHECK_VALUE(!kv_fp8 || d == 128, "fp8 K/V are supported for head_dim 128");
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(1) == hq && q.size(2) == d && q.size(0) >= 1 &&
                        q.size(0) <= g.batch_capacity,
                    "Q must be [rows <= capacity, query_heads, head_dim]");
  TORCH_CHECK_VALUE(out.scalar_type() == q.scalar_type(), "Q dtype differs from the engine's output dtype");
  for (const at::Tensor* t : {&q, &k, &v, &pages})
    TORCH_CHECK_VALUE(t->device() == out.device(), "all tensors must live on the engine's device");
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt, "page table / kv_indices must be int32");
  if (!indptr.has_value()) {
    TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(),
                      "paged KV must have matching [page,token,head,dim] shapes");
    TORCH_CHECK_VALUE(k.size(1) == page_size && k.size(2) == hkv && k.size(3) == d,
                      "KV geometry differs from the capture configuration");
    const int64_t max_pages = (g.max_context + page_size - 1) / page_size;
    TORCH_CHECK_VALUE(pages.dim() == 2 && pages.size(0) == g.batch_capacity && pages.size(1) == max_pages,
                      "page table capacity mismatch");
  } else {
    TORCH_CHECK_VALUE(k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == hkv && k.size(2) == d,
                      "CSR KV must be [token,head,dim]");
    TORCH_CHECK_VALUE(page_size == 1 && pages.dim() == 1, "CSR integration uses one-token physical pages");
    TORCH_CHECK_VALUE(indptr->scalar_type() == at::kInt && indptr->dim() == 1 && indptr->device() == out.device(),
                      "kv_indptr must be a 1-D int32 tensor");
  }
  TORCH_CHECK_VALUE(finite_positive(k_scale), "k_scale must be a finite value > 0");
  TORCH_CHECK_VALUE(finite_positive(v_scale), "v_scale must be a finite value > 0");
  TORCH_CHECK_VALUE(logit_cap >= 0.0 && logit_cap <= 3.0e38, "logit_cap must be a finite value >= 0 (0 disables it)");
  if (!new_loc.has_value()) {
    TORCH_CHECK_VALUE(!k_new.has_value() && !v_new.has_value(), "k_new / v_new need new_loc");
    return;
  }
  const int64_t rows = q.size(0);
  for (const std::optional<at::Tensor>* t : {&k_new, &v_new})
    TORCH_CHECK_VALUE(t->has_value() && (*t)->scalar_type() == q.scalar_type() && (*t)->device() == out.device() &&
                          (*t)->dim() == 3 && (*t)->size(0) == rows && (*t)->size(1) == hkv && (*t)->size(2) == d,
                      "k_new / v_new must be [q rows, kv_heads, head_dim] in Q's dtype");
  const at::Tensor& loc = *new_loc;
  TORCH_CHECK_VALUE((loc.scalar_type() == at::kLong || loc.scalar_type() == at::kInt) &&
                        loc.device() == out.device() && loc.dim() == 1 && loc.size(0) == rows && loc.stride(0) == 1,
                    "new_loc must be a contiguous 1-D int64/int32 tensor, one slot per Q row");
}

// The C arguments of a checked decode call.
// K/V: paged [pages, page_size, Hkv, D] or CSR [tokens, Hkv, D] (indptr given).
sgld_decode_args decode_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
                             const std::optional<at::Tensor>& indptr, const at::Tensor& out, const at::Tensor& partial,
                             const at::Tensor& lse, const at::Tensor& counter, const at::Tensor& status,
                             const sgld_plan_geometry& g, int64_t page_size, double scale, double logit_cap,
                             double k_scale, double v_scale, const std::optional<at::Tensor>& k_new,
                             const std::optional<at::Tensor>& v_new, const std::optional<at::Tensor>& new_loc) {
  sgld_decode_args a;
  std::memset(&a, 0, sizeof(a));
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.pages = pages.data_ptr<int32_t>();
  for (int i = 0; i < 3; ++i) a.q_stride[i] = q.stride(i);
  if (indptr.has_value()) {
    a.indptr = indptr->data_ptr<int32_t>();
    const int64_t ks[4] = {k.stride(0), 0, k.stride(1), k.stride(2)};
    const int64_t vs[4] = {v.stride(0), 0, v.stride(1), v.stride(2)};
    std::memcpy(a.k_stride, ks, sizeof(ks));
    std::memcpy(a.v_stride, vs, sizeof(vs));
  } else {
    for (int i = 0; i < 4; ++i) a.k_stride[i] = k.stride(i), a.v_stride[i] = v.stride(i);
    a.pt_stride[0] = pages.stride(0);
    a.pt_stride[1] = pages.stride(1);
  }
  a.kv_extent = k.size(0) == v.size(0) ? k.size(0) : 0;
  a.dtype = dtype_code(q);
  a.kv_dtype = dtype_code(k);
  a.query_heads = static_cast<int32_t>(out.size(1));
  a.kv_heads = g.groups;
  a.head_dim = static_cast<int32_t>(out.size(2));
  a.page_size = static_cast<int32_t>(page_size);
  a.scale = static_cast<float>(scale);
  a.logit_cap = static_cast<float>(logit_cap);
  a.k_scale = static_cast<float>(k_scale);
  a.v_scale = static_cast<float>(v_scale);
  a.q_rows = static_cast<int32_t>(q.size(0));
  if (new_loc.has_value()) {
    a.k_new = k_new->data_ptr();
    a.v_new = v_new->data_ptr();
    a.new_loc = new_loc->data_ptr();
    for (int i = 0; i < 3; ++i) a.knew_stride[i] = k_new->stride(i), a.vnew_stride[i] = v_new->stride(i);
    a.new_loc_int32 = new_loc->scalar_type() == at::kInt ? 1 : 0;
  }
  a.counter = counter.data_ptr<int32_t>();
  a.partial = partial.data_ptr<float>();
  a.lse = lse.data_ptr<float>();
  a.status = status.data_ptr<int32_t>();
  return a;
}

void decode(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
            const std::optional<at::Tensor>& indptr, at::Tensor out, at::Tensor partial, at::Tensor lse,
            at::Tensor counter, at::Tensor status, const at::Tensor& plan, at::IntArrayRef geometry, int64_t page_size,
            double scale, double logit_cap, double k_scale, double v_scale, const std::optional<at::Tensor>& k_new,
            const std::optional<at::Tensor>& v_new, const std::optional<at::Tensor>& new_loc) {
  const c10::cuda::CUDAGuard guard(out.device());
  const sgld_plan_geometry g = geometry_of(geometry);
  check_decode_call(q, k, v, pages, indptr, out, g, page_size, logit_cap, k_scale, v_scale, k_new, v_new, new_loc);
  const sgld_plan_buffers p = plan_of(plan, g);
  const sgld_decode_args a = decode_args(q, k, v, pages, indptr, out, partial, lse, counter, status, g, page_size, scale,
                                         logit_cap, k_scale, v_scale, k_new, v_new, new_loc);
  check_status(sgld_decode_persistent(&a, &p, &g, stream_of(out)), "sgld_decode_persistent");
}

// The same with the shared prefix: `prefix` names token slots (CSR) or pages (paged).
void decode_shared_prefix(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
                          const std::optional<at::Tensor>& indptr, at::Tensor out, at::Tensor partial, at::Tensor lse,
                          at::Tensor counter, at::Tensor status, const at::Tensor& plan, at::IntArrayRef geometry,
                          int64_t page_size, double scale, double logit_cap, const std::optional<at::Tensor>& k_new,
                          const std::optional<at::Tensor>& v_new, const std::optional<at::Tensor>& new_loc,
                          const at::Tensor& prefix, const std::optional<at::Tensor>& prefix_length, at::Tensor workspace) {
  const c10::cuda::CUDAGuard guard(out.device());
  const sgld_plan_geometry g = geometry_of(geometry);
  check_decode_call(q, k, v, pages, indptr, out, g, page_size, logit_cap, 1.0, 1.0, k_new, v_new, new_loc);
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type(), "a shared prefix needs K/V of Q's dtype");
  TORCH_CHECK_VALUE(k.size(0) == v.size(0), "K and V must have the same extent");
  TORCH_CHECK_VALUE(prefix.scalar_type() == at::kInt && prefix.device() == out.device() && prefix.dim() == 1 &&
                        (prefix.size(0) <= 1 || prefix.stride(0) == 1),
                    "prefix must be a contiguous 1-D int32 tensor of token slots (CSR) or pages");
  TORCH_CHECK_VALUE(prefix.size(0) * page_size < (int64_t{1} << 31), "prefix names 2^31 tokens or more");
  TORCH_CHECK_VALUE(!prefix_length.has_value() ||
                        (prefix_length->scalar_type() == at::kInt && prefix_length->device() == out.device() &&
                         prefix_length->numel() == 1),
                    "prefix_length must be an int32 tensor of one element on the engine's device");
  TORCH_CHECK_VALUE(workspace.device() == out.device() && workspace.is_contiguous(), "workspace must be contiguous");
  const sgld_plan_buffers p = plan_of(plan, g);
  sgld_decode_args a = decode_args(q, k, v, pages, indptr, out, partial, lse, counter, status, g, page_size, scale, logit_cap,
                                   1.0, 1.0, k_new, v_new, new_loc);
  if (pages.numel() == 0) a.pages = nullptr;   // no request may have own tokens: nothing is read for them
  sgld_prefix_args x;
  std::memset(&x, 0, sizeof(x));
  x.index = prefix.size(0) > 0 ? prefix.data_ptr<int32_t>() : nullptr;
  x.length = prefix_length.has_value() ? prefix_length->data_ptr<int32_t>() : nullptr;
  x.capacity = static_cast<int32_t>(prefix.size(0) * page_size);
  x.workspace = workspace.data_ptr();
  x.workspace_bytes = static_cast<size_t>(workspace.nbytes());
  check_status(sgld_decode_shared_prefix(&a, &x, &p, &g, stream_of(out)), "sgld_decode_shared_prefix");
}

void merge(const at::Tensor& partial, const at::Tensor& lse, const at::Tensor& counts, const at::Tensor& error,
           at::Tensor out) {
  const c10::cuda::CUDAGuard guard(partial.device());
  TORCH_CHECK_VALUE(partial.dim() == 4, "partial is [batch, heads, splits, head_dim]");
  check_status(sgld_merge_splits(partial.data_ptr<float>(), lse.data_ptr<float>(), counts.data_ptr<int32_t>(),
                                 error.data_ptr<int32_t>(), out.data_ptr(), dtype_code(out),
                                 static_cast<int32_t>(partial.size(0)), static_cast<int32_t>(partial.size(1)),
                                 static_cast<int32_t>(partial.size(3)), static_cast<int32_t>(partial.size(2)),
                                 stream_of(partial)),
               "sgld_merge_splits");
}

bool index_like(const at::Tensor& t, int64_t n, const at::Device& device) {
  return (t.scalar_type() == at::kLong || t.scalar_type() == at::kInt) && t.device() == device && t.dim() == 1 &&
         t.size(0) == n && (n <= 1 || t.stride(0) == 1);
}

// Do two tensors share memory (as far as their layouts tell)?  `same_is_fine`: not if they are the
// same elements in the same order.
bool shares_memory(const at::Tensor& a, const at::Tensor& b, bool same_is_fine = false) {
  const at::MemOverlapStatus s = at::get_overlap_status(a, b);
  if (s == at::MemOverlapStatus::Full)
    return !(same_is_fine && a.data_ptr() == b.data_ptr() && a.strides() == b.strides());
  return s == at::MemOverlapStatus::Partial;
}

bool repeats_memory(const at::Tensor& t) { return at::has_internal_overlap(t) == at::MemOverlap::Yes; }

void strides_of(const at::Tensor& t, int64_t* s) {
  for (int64_t i = 0; i < t.dim(); ++i) s[i] = t.stride(i);
}

// q [T, Hq, D], k (and v) [T, Hkv, D]; the caches are [slots, Hkv, D] or [pages, page_size, Hkv, D].
void norm_rope(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions, const at::Tensor& table,
               const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight, double eps,
               bool interleaved, at::Tensor q_out, const std::optional<at::Tensor>& k_out,
               const std::optional<at::Tensor>& v, const std::optional<at::Tensor>& k_cache,
               const std::optional<at::Tensor>& v_cache, const std::optional<at::Tensor>& slots, double k_scale,
               double v_scale, const std::optional<at::Tensor>& status) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(q.device());
  const auto dtype = q.scalar_type();
  const auto device = q.device();
  TORCH_CHECK_VALUE(dtype == at::kHalf || dtype == at::kBFloat16, "q must be fp16 or bf16");
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2),
                    "q and k must be [tokens, heads, head_dim] with the same tokens and head_dim");
  const int64_t tokens = q.size(0), d = q.size(2);
  const auto like = [&](const at::Tensor& t, at::IntArrayRef sizes) {
    return t.scalar_type() == dtype && t.device() == device && t.sizes() == sizes;
  };
  TORCH_CHECK_VALUE(like(k, k.sizes()), "k must have q's dtype and device");
  TORCH_CHECK_VALUE(like(q_out, q.sizes()), "q_out must have q's shape, dtype and device");
  TORCH_CHECK_VALUE(!k_out.has_value() || like(*k_out, k.sizes()), "k_out must have k's shape, dtype and device");
  TORCH_CHECK_VALUE(!repeats_memory(q_out) && !shares_memory(q_out, q, true) && !shares_memory(q_out, k) &&
                        (!v.has_value() || !shares_memory(q_out, *v)),
                    "q_out may be q itself, but must not share memory with q, k or v otherwise");
  TORCH_CHECK_VALUE(!k_out.has_value() ||
                        (!repeats_memory(*k_out) && !shares_memory(*k_out, k, true) && !shares_memory(*k_out, q) &&
                         !shares_memory(*k_out, q_out) && (!v.has_value() || !shares_memory(*k_out, *v))),
                    "k_out may be k itself, but must not share memory with q, k, v or q_out otherwise");
  TORCH_CHECK_VALUE(index_like(positions, tokens, device), "positions must be a contiguous int64/int32 tensor, one per token");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kFloat && table.device() == device && table.dim() == 2 &&
                        table.stride(1) == 1,
                    "table must be fp32 [positions, rotary] with unit stride along its rows");
  sgld_norm_rope_args a;
  std::memset(&a, 0, sizeof(a));
  for (const std::optional<at::Tensor>* w : {&q_weight, &k_weight}) {
    if (!w->has_value()) continue;
    const at::Tensor& t = **w;
    TORCH_CHECK_VALUE(t.device() == device && t.dim() == 1 && t.size(0) == d && t.stride(0) == 1 &&
                          (t.scalar_type() == dtype || t.scalar_type() == at::kFloat),
                      "norm weights must be contiguous [head_dim] in q's dtype or fp32");
    a.weight_f32 = t.scalar_type() == at::kFloat ? 1 : 0;
  }
  TORCH_CHECK_VALUE(!q_weight.has_value() || !k_weight.has_value() || q_weight->scalar_type() == k_weight->scalar_type(),
                    "q_weight and k_weight must have one dtype");
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.positions = positions.data_ptr();
  a.positions_int32 = positions.scalar_type() == at::kInt ? 1 : 0;
  a.table = table.data_ptr<float>();
  a.table_stride = table.stride(0);
  a.table_rows = table.size(0);
  a.rotary = static_cast<int32_t>(table.size(1));
  a.q_weight = q_weight.has_value() ? q_weight->data_ptr() : nullptr;
  a.k_weight = k_weight.has_value() ? k_weight->data_ptr() : nullptr;
  a.q_out = q_out.data_ptr();
  strides_of(q, a.q_stride);
  strides_of(k, a.k_stride);
  strides_of(q_out, a.qo_stride);
  if (k_out.has_value()) {
    a.k_out = k_out->data_ptr();
    strides_of(*k_out, a.ko_stride);
  }
  a.page_size = 1;
  if (slots.has_value()) {
    TORCH_CHECK_VALUE(v.has_value() && k_cache.has_value() && v_cache.has_value(),
                      "the cache write needs v, k_cache, v_cache and slots");
    TORCH_CHECK_VALUE(like(*v, k.sizes()), "v must have k's shape, dtype and device");
    TORCH_CHECK_VALUE(index_like(*slots, tokens, device), "slots must be a contiguous int64/int32 tensor, one per token");
    const at::Tensor &kc = *k_cache, &vc = *v_cache;
    const bool paged = kc.dim() == 4;
    TORCH_CHECK_VALUE((paged || kc.dim() == 3) && kc.sizes() == vc.sizes() && kc.size(-2) == k.size(1) && kc.size(-1) == d,
                      "the caches must be [slots, kv_heads, head_dim] or [pages, page_size, kv_heads, head_dim]");
    TORCH_CHECK_VALUE(kc.device() == device && vc.device() == device && kc.scalar_type() == vc.scalar_type() &&
                          (kc.scalar_type() == dtype || kc.scalar_type() == at::kFloat8_e4m3fn),
                      "the caches must be of q's dtype or fp8 e4m3, on q's device");
    TORCH_CHECK_VALUE(finite_positive(k_scale) && finite_positive(v_scale), "k_scale / v_scale must be finite values > 0");
    a.v = v->data_ptr();
    strides_of(*v, a.v_stride);
    a.k_cache = kc.data_ptr();
    a.v_cache = vc.data_ptr();
    for (int i = 0; i < 4; ++i) {
      a.kc_stride[i] = paged ? kc.stride(i) : (i == 0 ? kc.stride(0) : i == 1 ? 0 : kc.stride(i - 1));
      a.vc_stride[i] = paged ? vc.stride(i) : (i == 0 ? vc.stride(0) : i == 1 ? 0 : vc.stride(i - 1));
    }
    a.page_size = paged ? static_cast<int32_t>(kc.size(1)) : 1;
    a.cache_slots = kc.size(0) * a.page_size;
    a.cache_fp8 = kc.scalar_type() == at::kFloat8_e4m3fn ? 1 : 0;
    a.slots = slots->data_ptr();
    a.slots_int32 = slots->scalar_type() == at::kInt ? 1 : 0;
    a.k_scale = static_cast<float>(k_scale);
    a.v_scale = static_cast<float>(v_scale);
  } else {
    TORCH_CHECK_VALUE(!v.has_value() && !k_cache.has_value() && !v_cache.has_value(), "v, k_cache and v_cache need slots");
    TORCH_CHECK_VALUE(k_out.has_value(), "k_out is needed where no cache is written");
  }
  if (status.has_value()) {
    TORCH_CHECK_VALUE(status->scalar_type() == at::kInt && status->device() == device && status->numel() >= 1,
                      "status must be an int32 tensor on q's device");
    a.status = status->data_ptr<int32_t>();
  }
  a.tokens = tokens;
  a.query_heads = static_cast<int32_t>(q.size(1));
  a.kv_heads = static_cast<int32_t>(k.size(1));
  a.head_dim = static_cast<int32_t>(d);
  a.interleaved = interleaved ? 1 : 0;
  a.dtype = dtype_code(q);
  a.eps = static_cast<float>(eps);
  if (tokens == 0) return;   // empty tensors have no address to check
  check_status(sgld_norm_rope(&a, stream_of(q)), "sgld_norm_rope");
}

// q [T, Hq, D]; k, v [N, Hkv, D]; kv_indices picks their rows.  Split results, where a call needs
// them, live in a temporary of the caching allocator on the current stream.
void prompt_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& indptr,
                      const std::optional<at::Tensor>& kv_indptr, const std::optional<at::Tensor>& kv_indices,
                      at::Tensor out, const std::optional<at::Tensor>& lse, double scale, double logit_cap,
                      int64_t window_left, const std::optional<at::Tensor>& status) {
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(q.device());
  const auto device = q.device();
  TORCH_CHECK_VALUE(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q must be fp16 or bf16");
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.size(2) == q.size(2),
                    "q must be [tokens, query_heads, head_dim], k and v [rows, kv_heads, head_dim]");
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK_VALUE(t->scalar_type() == q.scalar_type() && t->device() == device, "k and v must have q's dtype and device");
  TORCH_CHECK_VALUE(out.scalar_type() == q.scalar_type() && out.device() == device && out.sizes() == q.sizes(),
                    "out must have q's shape, dtype and device");
  TORCH_CHECK_VALUE(!repeats_memory(out) && !shares_memory(out, q) && !shares_memory(out, k) && !shares_memory(out, v),
                    "out must not share memory with q, k or v");
  const auto is_pointers = [&](const at::Tensor& t) {
    return t.scalar_type() == at::kInt && t.device() == device && t.dim() == 1 && t.size(0) >= 1 &&
           (t.size(0) == 1 || t.stride(0) == 1);
  };
  TORCH_CHECK_VALUE(is_pointers(indptr), "indptr must be a contiguous int32 tensor of sequences + 1 offsets on q's device");
  TORCH_CHECK_VALUE(!kv_indptr.has_value() || (is_pointers(*kv_indptr) && kv_indptr->size(0) == indptr.size(0)),
                    "kv_indptr must be like indptr");
  TORCH_CHECK_VALUE(!kv_indices.has_value() || kv_indptr.has_value(), "kv_indices need kv_indptr");
  TORCH_CHECK_VALUE(!kv_indices.has_value() ||
                        (kv_indices->scalar_type() == at::kInt && kv_indices->device() == device && kv_indices->dim() == 1 &&
                         (kv_indices->size(0) <= 1 || kv_indices->stride(0) == 1)),
                    "kv_indices must be a contiguous 1-D int32 tensor on q's device");
  TORCH_CHECK_VALUE(!lse.has_value() || (lse->scalar_type() == at::kFloat && lse->device() == device && lse->dim() == 2 &&
                                         lse->size(0) == q.size(0) && lse->size(1) == q.size(1) && lse->is_contiguous()),
                    "lse must be a contiguous fp32 [tokens, query_heads] tensor on q's device");
  TORCH_CHECK_VALUE(!status.has_value() || (status->scalar_type() == at::kInt && status->device() == device && status->numel() >= 1),
                    "status must be an int32 tensor on q's device");
  TORCH_CHECK_VALUE(finite_positive(scale), "scale must be a finite value > 0");
  TORCH_CHECK_VALUE(window_left >= -1, "window_left must be >= 0, or -1 for none");
  TORCH_CHECK_VALUE(q.size(0) < (int64_t{1} << 31) && indptr.size(0) < (int64_t{1} << 31), "too many tokens or sequences");
  sgld_prompt_args a;
  std::memset(&a, 0, sizeof(a));
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.lse = lse.has_value() ? lse->data_ptr<float>() : nullptr;
  a.q_indptr = indptr.data_ptr<int32_t>();
  a.kv_indptr = kv_indptr.has_value() ? kv_indptr->data_ptr<int32_t>() : nullptr;
  // An empty index list stays one (it names no row): it has no address of its own.
  static const int32_t none = 0;
  a.kv_indices = kv_indices.has_value() ? (kv_indices->size(0) > 0 ? kv_indices->data_ptr<int32_t>() : &none) : nullptr;
  a.kv_indices_count = kv_indices.has_value() ? kv_indices->size(0) : 0;
  a.status = status.has_value() ? status->data_ptr<int32_t>() : nullptr;
  strides_of(q, a.q_stride);
  strides_of(k, a.k_stride);
  strides_of(v, a.v_stride);
  strides_of(out, a.out_stride);
  a.kv_extent = k.size(0);
  a.tokens = static_cast<int32_t>(q.size(0));
  a.seqs = static_cast<int32_t>(indptr.size(0) - 1);
  a.query_heads = static_cast<int32_t>(q.size(1));
  a.kv_heads = static_cast<int32_t>(k.size(1));
  a.head_dim = static_cast<int32_t>(q.size(2));
  a.dtype = dtype_code(q);
  a.window_left = static_cast<int32_t>(std::min<int64_t>(window_left, INT32_MAX / 2));
  a.scale = static_cast<float>(scale);
  a.logit_cap = static_cast<float>(logit_cap);
  const size_t bytes = sgld_prompt_workspace_bytes(&a);
  at::Tensor workspace;
  if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  check_status(sgld_prompt_attention(&a, bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)),
               "sgld_prompt_attention");
}

void plan_build_meta(const at::Tensor&, at::IntArrayRef, int64_t, const std::optional<at::Tensor>&, int64_t,
                     const std::optional<at::Tensor>&) {}
void decode_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                 const std::optional<at::Tensor>&, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                 const at::Tensor&, at::IntArrayRef, int64_t, double, double, double, double,
                 const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&) {}
void merge_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor) {}
void prompt_attention_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                           const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, at::Tensor,
                           const std::optional<at::Tensor>&, double, double, int64_t, const std::optional<at::Tensor>&) {}
void decode_shared_prefix_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                               const std::optional<at::Tensor>&, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                               at::Tensor, const at::Tensor&, at::IntArrayRef, int64_t, double, double,
                               const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                               const std::optional<at::Tensor>&, const at::Tensor&, const std::optional<at::Tensor>&,
                               at::Tensor) {}
void norm_rope_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, double, bool, at::Tensor,
                    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, double, double,
                    const std::optional<at::Tensor>&) {}

}  // namespace

TORCH_LIBRARY(sglang_decode, m) {
  m.def("plan_build(Tensor(a!) plan, int[] geometry, int force_mode, Tensor? rules, int n_rules, "
        "Tensor(b!)? counters) -> ()");
  m.def("decode(Tensor q, Tensor(a!) k, Tensor(b!) v, Tensor pages, Tensor? indptr, Tensor(c!) out, "
        "Tensor(d!) partial, Tensor(e!) lse, Tensor(f!) counter, Tensor(g!) status, Tensor plan, int[] geometry, "
        "int page_size, float scale, float logit_cap, float k_scale, float v_scale, Tensor? k_new, Tensor? v_new, "
        "Tensor? new_loc) -> ()");
  m.def("merge(Tensor partial, Tensor lse, Tensor counts, Tensor error, Tensor(a!) out) -> ()");
  m.def("prompt_attention(Tensor q, Tensor k, Tensor v, Tensor indptr, Tensor? kv_indptr, Tensor? kv_indices, "
        "Tensor(a!) out, Tensor(b!)? lse, float scale, float logit_cap, int window_left, Tensor(c!)? status) -> ()");
  m.def("decode_shared_prefix(Tensor q, Tensor(a!) k, Tensor(b!) v, Tensor pages, Tensor? indptr, Tensor(c!) out, "
        "Tensor(d!) partial, Tensor(e!) lse, Tensor(f!) counter, Tensor(g!) status, Tensor plan, int[] geometry, "
        "int page_size, float scale, float logit_cap, Tensor? k_new, Tensor? v_new, Tensor? new_loc, Tensor prefix, "
        "Tensor? prefix_length, Tensor(h!) workspace) -> ()");
  m.def("norm_rope(Tensor q, Tensor k, Tensor positions, Tensor table, Tensor? q_weight, Tensor? k_weight, float eps, "
        "bool interleaved, Tensor(a!) q_out, Tensor(b!)? k_out, Tensor? v, Tensor(c!)? k_cache, Tensor(d!)? v_cache, "
        "Tensor? slots, float k_scale, float v_scale, Tensor(e!)? status) -> ()");
}

TORCH_LIBRARY_IMPL(sglang_decode, CUDA, m) {
  m.impl("plan_build", &plan_build);
  m.impl("decode", &decode);
  m.impl("merge", &merge);
  m.impl("norm_rope", &norm_rope);
  m.impl("prompt_attention", &prompt_attention);
  m.impl("decode_shared_prefix", &decode_shared_prefix);
}

TORCH_LIBRARY_IMPL(sglang_decode, Meta, m) {
  m.impl("plan_build", &plan_build_meta);
  m.impl("decode", &decode_meta);
  m.impl("merge", &merge_meta);
  m.impl("norm_rope", &norm_rope_meta);
  m.impl("prompt_attention", &prompt_attention_meta);
  m.impl("decode_shared_prefix", &decode_shared_prefix_meta);
}
