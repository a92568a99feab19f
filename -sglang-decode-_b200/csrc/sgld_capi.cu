// C ABI entry points (include/sgld_b200.h): host-side argument checks, then one
// asynchronous launch each.  No allocation, no synchronisation, no host readback.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>

#include "sgld_attend.cuh"
#include "sgld_internal.cuh"

namespace {

thread_local std::string g_last_error;

int fail(int code, const std::string& msg) {
  g_last_error = msg;
  return code;
}

int cuda_fail(cudaError_t e, const char* where) {
  g_last_error = std::string(where) + ": " + cudaGetErrorString(e);
  return SGLD_ERR_CUDA;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int bit_length(int64_t x) {
  int n = 0;
  while (x > 0) {
    ++n;
    x >>= 1;
  }
  return n;
}

// Capacity contract of the reference's DecodeConfig (config.py:27-38), minus the
// group-size whitelist (any integer group 1..16 is supported here).
int check_geometry(const sgld_plan_geometry* g) {
  if (g == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "geometry is NULL");
  if (g->batch_capacity <= 0 || g->max_splits <= 0 || g->max_context <= 0 || g->groups <= 0 ||
      g->workers <= 0)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "geometry fields must be positive");
  const int64_t records = static_cast<int64_t>(g->batch_capacity) * g->max_splits;
  if (records > sgld::kMaxRecords)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "record capacity batch_capacity*max_splits exceeds 4096");
  if (records * g->groups >= (int64_t{1} << 31))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "task capacity must stay below 2^31");
  if (g->workers > sgld::kMaxPlanWorkers)
    return fail(SGLD_ERR_UNSUPPORTED, "workers above 4096 are not supported");
  return SGLD_OK;
}

int plan_buckets(const sgld_plan_geometry* g) {
  const int64_t tiles = (static_cast<int64_t>(g->max_context) + sgld::kBlockKV - 1) / sgld::kBlockKV;
  return bit_length(tiles - 1) + 1;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static bool tried = false;
  if (!tried) {
    tried = true;
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// 4D map {D, Hkv, page_size, pages} over a paged K or V tensor with element strides
// (head, token-in-page, page); boxes of {64 dims, 1 head, box_rows tokens, 1 page}
// land in shared memory with the 128-byte swizzle.
bool encode_paged_map(CUtensorMap* map, const void* base, int32_t dtype, int64_t d, int64_t hkv, int64_t ps,
                      int64_t pages, const int64_t* stride, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(hkv), static_cast<cuuint64_t>(ps),
                        static_cast<cuuint64_t>(pages)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(stride[2]) * 2, static_cast<cuuint64_t>(stride[1]) * 2,
                           static_cast<cuuint64_t>(stride[0]) * 2};
  for (cuuint64_t st : strides)
    if (st == 0 || st % 16 != 0 || st >= (cuuint64_t{1} << 40)) return false;
  cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type =
      dtype == SGLD_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = enc(map, type, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

// 3D map {D, Hq, rows} over Q with element strides (head, request); boxes of {64 dims,
// 16 heads, 1 request} land in shared memory with the 128-byte swizzle.  Heads past Hq and
// requests past `rows` read as zeros.
bool encode_q_map(CUtensorMap* map, const void* base, int32_t dtype, int64_t d, int64_t hq, int64_t rows,
                  const int64_t* stride) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr || (reinterpret_cast<uintptr_t>(base) & 15u) != 0 || stride[2] != 1) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(hq), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride[1]) * 2, static_cast<cuuint64_t>(stride[0]) * 2};
  for (cuuint64_t st : strides)
    if (st == 0 || st % 16 != 0 || st >= (cuuint64_t{1} << 40)) return false;
  cuuint32_t box[3] = {64, 16, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      dtype == SGLD_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = enc(map, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

// Kernel choice.  SGLD_DECODE_KERNEL=tcgen05 selects the tcgen05 kernel wherever it applies,
// =small the small-batch kernel wherever it applies, =mma the persistent mma.sync kernel
// everywhere; unset, the measured-faster kernel for the geometry: the small-batch kernel when
// the whole task capacity is at most kSmallTaskCapacity, else the persistent mma.sync kernel.
constexpr int64_t kSmallTaskCapacity = 1024;

bool kernel_env_is(const char* name) {
  const char* v = std::getenv("SGLD_DECODE_KERNEL");
  return v != nullptr && std::strcmp(v, name) == 0;
}
bool kernel_env_unset() {
  const char* v = std::getenv("SGLD_DECODE_KERNEL");
  return v == nullptr || v[0] == 0;
}
bool use_tc_kernel() { return kernel_env_is("tcgen05"); }

bool tma_disabled_by_env() {
  const char* v = std::getenv("SGLD_DISABLE_TMA");
  return v != nullptr && v[0] == '1';
}

// Norm + rotation: below this many (token, head step) units every warp takes one step, so that the
// whole call is in flight at once; above it four, which reads the rotation once for four steps.
constexpr int64_t kFewRopeSteps = 148 * 64;

// SGLD_ATTEND_STALL=tasks:ns makes waits of the tcgen05 attention kernel run out, for tests: its issuer stops
// after that many tasks in every CTA (-1: never), and waits expire after that many ns, not 4 s.
void set_wait_limits(sgld::AttendLaunch& a) {
  a.stall = -1;
  a.wait_ns = 4000000000ull;
  const char* v = std::getenv("SGLD_ATTEND_STALL");
  int stall = 0;
  unsigned long long ns = 0;
  if (v != nullptr && std::sscanf(v, "%d:%llu", &stall, &ns) == 2) a.stall = stall < -1 ? -1 : stall, a.wait_ns = ns;
}

int check_plan_pointers(const sgld_plan_buffers* p) {
  if (p == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "plan buffers are NULL");
  const void* ptrs[] = {p->lengths, p->splits, p->active, p->counts, p->offsets, p->chunk,
                        p->request, p->split, p->begin, p->end, p->weight, p->order,
                        p->pack_first, p->pack_count, p->record_count, p->num_packs, p->mode,
                        p->error, p->static_head, p->static_next, p->arrivals};
  for (const void* q : ptrs)
    if (q == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "a plan buffer pointer is NULL");
  return SGLD_OK;
}

}  // namespace

namespace sgld {
// Record `msg` as this host thread's sgld_last_error() message and return `code`.
int set_last_error(int code, const char* msg) { return fail(code, msg); }
}  // namespace sgld

extern "C" {

int32_t sgld_abi_version(void) { return SGLD_ABI_VERSION; }

const char* sgld_last_error(void) { return g_last_error.c_str(); }

size_t sgld_layer_workspace_bytes(int32_t batch_capacity, int32_t query_heads, int32_t kv_heads,
                                  int32_t head_dim, int32_t max_splits) {
  if (batch_capacity <= 0 || query_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_splits <= 0)
    return 0;
  const size_t slots = static_cast<size_t>(batch_capacity) * query_heads * max_splits;
  return 2 * sizeof(int32_t)                                   /* claim counter + spare */
         + slots * head_dim * sizeof(float)                    /* partial */
         + slots * sizeof(float)                               /* lse */
         + sizeof(int32_t);                                    /* status */
}

size_t sgld_plan_storage_words(const sgld_plan_geometry* g) {
  if (g == nullptr || g->batch_capacity <= 0 || g->max_splits <= 0 || g->groups <= 0 || g->workers <= 0) return 0;
  const size_t b = static_cast<size_t>(g->batch_capacity), e = b * g->max_splits, t = e * g->groups;
  return 5 * b + 2 + 6 * e + 3 * t + 4 + static_cast<size_t>(g->workers) + b * g->groups;   // sizes as listed below
}

int sgld_plan_buffers_in_storage(int32_t* storage, const sgld_plan_geometry* g, sgld_plan_buffers* out) {
  if (storage == nullptr || out == nullptr || sgld_plan_storage_words(g) == 0)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "storage, geometry or output is NULL or empty");
  const size_t b = static_cast<size_t>(g->batch_capacity), e = b * g->max_splits, t = e * g->groups;
  int32_t* cur = storage;
  auto take = [&cur](size_t n) {
    int32_t* p = cur;
    cur += n;
    return p;
  };
  out->lengths = take(b);
  out->splits = take(b);
  out->active = take(1);
  out->counts = take(b);
  out->offsets = take(b + 1);
  out->chunk = take(b);
  out->request = take(e);
  out->split = take(e);
  out->begin = take(e);
  out->end = take(e);
  out->weight = take(e);
  out->order = take(e);
  out->pack_first = take(t);
  out->pack_count = take(t);
  out->record_count = take(1);
  out->num_packs = take(1);
  out->mode = take(1);
  out->error = take(1);
  out->static_head = take(static_cast<size_t>(g->workers));
  out->static_next = take(t);
  out->arrivals = take(b * g->groups);
  return SGLD_OK;
}

int sgld_plan_build(const sgld_plan_buffers* plan, const sgld_plan_geometry* geometry,
                    int32_t force_mode, const int32_t* rules, int32_t n_rules,
                    int32_t* layer_counters, int32_t n_counter_words, void* stream) {
  int rc = check_geometry(geometry);
  if (rc) return rc;
  if ((rc = check_plan_pointers(plan))) return rc;
  if (force_mode < -1 || force_mode > 4) return fail(SGLD_ERR_INVALID_ARGUMENT, "force_mode must be -1..4");
  if (n_rules < 0 || (n_rules > 0 && rules == nullptr))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "rules pointer/count mismatch");
  if (n_counter_words < 0 || (n_counter_words > 0 && layer_counters == nullptr))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "counter pointer/count mismatch");
  sgld::PlanLaunch a;
  a.p = *plan;
  a.bcap = geometry->batch_capacity;
  a.smax = geometry->max_splits;
  a.maxctx = geometry->max_context;
  a.groups = geometry->groups;
  a.workers = geometry->workers;
  a.buckets = plan_buckets(geometry);
  a.force = force_mode;
  a.rules = rules;
  a.n_rules = n_rules;
  a.counters = layer_counters;
  a.n_counters = n_counter_words;
  if (a.buckets > sgld::kMaxBuckets) return fail(SGLD_ERR_UNSUPPORTED, "max_context too large");
  cudaError_t e = sgld::launch_plan(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "sgld_plan_build launch");
  return SGLD_OK;
}

}  // extern "C"

namespace sgld {

// Every host-side check of sgld_decode_persistent, with nothing enqueued: shapes, dtypes,
// pointers (scratch included), strides and capacities.  SGLD_OK when a launch may follow.
int validate_decode(const sgld_decode_args* args, const sgld_plan_buffers* plan,
                    const sgld_plan_geometry* geometry, bool own_tokens) {
  if (args == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "decode args are NULL");
  int rc = check_geometry(geometry);
  if (rc) return rc;
  if ((rc = check_plan_pointers(plan))) return rc;
  const sgld_decode_args& d = *args;
  if (!d.q || !d.k || !d.v || !d.out || (own_tokens && !d.pages) || !d.counter || !d.partial || !d.lse || !d.status)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "a tensor or scratch pointer is NULL");
  if (!aligned16(d.partial))   // the epilogue and the merge move partial rows as float4
    return fail(SGLD_ERR_INVALID_ARGUMENT, "partial must be 16-byte aligned");
  if (!(d.logit_cap >= 0.f) || d.logit_cap > 3.0e38f)   // rejects NaN, negatives and infinity
    return fail(SGLD_ERR_INVALID_ARGUMENT, "logit_cap must be a finite value >= 0 (0 disables it)");
  if (!(d.k_scale >= 0.f) || d.k_scale > 3.0e38f || !(d.v_scale >= 0.f) || d.v_scale > 3.0e38f)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "k_scale / v_scale must be finite values >= 0 (0 reads as 1)");
  const bool kv_fp8 = d.kv_dtype == SGLD_DTYPE_E4M3;
  if (!kv_fp8 && d.kv_dtype != d.dtype)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "kv_dtype must equal dtype or be SGLD_DTYPE_E4M3");
  if (d.dtype != SGLD_DTYPE_F16 && d.dtype != SGLD_DTYPE_BF16)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "dtype must be fp16 or bf16");
  if (d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256)
    return fail(SGLD_ERR_UNSUPPORTED, "supported head dimensions: 64, 128, 256");
  if (kv_fp8 && d.head_dim != 128) return fail(SGLD_ERR_UNSUPPORTED, "fp8 K/V: head_dim 128 only");
  if (d.kv_heads <= 0 || d.query_heads <= 0 || d.query_heads % d.kv_heads)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "query heads must be a positive multiple of KV heads");
  const int group = d.query_heads / d.kv_heads;
  if (group > 16) return fail(SGLD_ERR_UNSUPPORTED, "GQA group sizes above 16 are not supported");
  if (d.kv_heads != geometry->groups)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "kv_heads must equal the plan's groups");
  if (d.page_size <= 0) return fail(SGLD_ERR_INVALID_ARGUMENT, "page_size must be positive");
  const bool csr = d.indptr != nullptr;
  if (csr && d.page_size != 1) return fail(SGLD_ERR_INVALID_ARGUMENT, "CSR indexing uses page_size 1");
  if (!(d.scale == d.scale)) return fail(SGLD_ERR_INVALID_ARGUMENT, "scale is NaN");
  const int32_t q_rows = d.q_rows == 0 ? geometry->batch_capacity : d.q_rows;
  if (q_rows < 0 || q_rows > geometry->batch_capacity)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "q_rows must be 0 (capacity) or 1..batch_capacity");
  const bool kv_write = d.new_loc != nullptr;
  if (!kv_write && (d.k_new != nullptr || d.v_new != nullptr))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "k_new / v_new need new_loc");
  if (kv_write && (d.k_new == nullptr || d.v_new == nullptr))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "the KV-cache write needs k_new, v_new and new_loc");

  return SGLD_OK;
}

// The calling thread's current CUDA context (a CUcontext), or nullptr when the driver
// entry point is unavailable.  Caches keyed by device ordinal compare it to notice a
// device reset (a new primary context reuses the ordinal but not the old addresses).
void* current_context() {
  using GetCurrent = CUresult (*)(CUcontext*);
  static GetCurrent fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return static_cast<GetCurrent>(nullptr);
    return reinterpret_cast<GetCurrent>(p);
  }();
  CUcontext ctx = nullptr;
  if (fn == nullptr || fn(&ctx) != CUDA_SUCCESS) return nullptr;
  return ctx;
}

}  // namespace sgld

extern "C" {

}  // extern "C"

namespace {

// Fill the kernel parameter block of a validated call and choose the kernel; returns an
// SGLD_KERNEL_* value.
// allow_small: the small-batch kernel, which merges the splits itself, may be chosen.
int prepare_launch(const sgld_decode_args& d, const sgld_plan_buffers* plan, const sgld_plan_geometry* geometry,
                   sgld::DecodeLaunch& a, bool allow_small = true) {
  const bool kv_fp8 = d.kv_dtype == SGLD_DTYPE_E4M3;
  const int group = d.query_heads / d.kv_heads;
  const bool csr = d.indptr != nullptr;
  const int32_t q_rows = d.q_rows == 0 ? geometry->batch_capacity : d.q_rows;
  std::memset(&a, 0, sizeof(a));
  a.d = d;
  a.p = *plan;
  a.bcap = geometry->batch_capacity;
  a.smax = geometry->max_splits;
  a.workers = geometry->workers;
  a.group_size = group;
  a.csr = csr ? 1 : 0;
  if (csr) a.d.k_stride[1] = 0, a.d.v_stride[1] = 0;
  // 16-byte copies need 16-byte aligned rows: strides in whole 16-byte chunks of elements.
  const int64_t per_chunk = kv_fp8 ? 16 : 8;
  bool fast_kv = aligned16(d.k) && aligned16(d.v) && d.k_stride[3] == 1 && d.v_stride[3] == 1;
  for (int i = 0; i < 3; ++i)
    fast_kv = fast_kv && (a.d.k_stride[i] % per_chunk == 0) && (a.d.v_stride[i] % per_chunk == 0);
  a.kv_fp8 = kv_fp8 ? 1 : 0;
  if (a.d.k_scale == 0.f) a.d.k_scale = 1.f;
  if (a.d.v_scale == 0.f) a.d.v_scale = 1.f;
  a.q_rows = q_rows;
  a.fast_kv = fast_kv ? 1 : 0;
  a.fast_q = (aligned16(d.q) && d.q_stride[2] == 1 && d.q_stride[0] % 8 == 0 && d.q_stride[1] % 8 == 0) ? 1 : 0;
  const int ps = d.page_size;
  const bool pageable_tma = !csr && fast_kv && ps % 32 == 0 && d.kv_extent > 0 &&
                            d.kv_extent < (int64_t{1} << 31) && !tma_disabled_by_env();
  // The tcgen05 kernel: head_dim 128, 16-bit K/V in 16-byte rows, Q loadable by a TMA box.
  if (!kv_fp8 && d.head_dim == 128 && fast_kv && a.fast_q && use_tc_kernel() &&
      encode_q_map(&a.qmap, d.q, d.dtype, d.head_dim, d.query_heads, q_rows, d.q_stride)) {
    if (pageable_tma &&
        encode_paged_map(&a.kmap, d.k, d.dtype, d.head_dim, d.kv_heads, ps, d.kv_extent, d.k_stride, 32) &&
        encode_paged_map(&a.vmap, d.v, d.dtype, d.head_dim, d.kv_heads, ps, d.kv_extent, d.v_stride, 32)) {
      a.tma_kv = 1;
      a.box_rows = 32;
      return SGLD_KERNEL_TCGEN05_TMA;
    }
    return SGLD_KERNEL_TCGEN05;
  }
  // Small-batch kernel: one CTA per task of the capacity (head_dim 128, 16-bit K/V, group <= 8).
  const int64_t task_capacity = static_cast<int64_t>(geometry->batch_capacity) * geometry->max_splits * d.kv_heads;
  if (allow_small && !kv_fp8 && d.head_dim == 128 && group <= 8 && fast_kv && a.fast_q && task_capacity <= (int64_t{1} << 20) &&
      (kernel_env_is("small") || (kernel_env_unset() && task_capacity <= kSmallTaskCapacity)))
    return SGLD_KERNEL_SMALL;
  // mma.sync kernel.  Paged KV by tensor-map TMA: a box of 32 tokens never crosses a page
  // because stages start 32-token aligned and 32 divides the page size.  Smaller pages stay
  // on the multi-warp cp.async path, which measured faster than 8- or 16-row boxes.  So do
  // D <= 128 kernels with a group of at most 8: they carry 10 cp.async producer warps,
  // which outrun a single thread issuing boxes (C4, page 64: 982 vs 1080 us).
  const bool wide_cp_async = d.head_dim <= 128 && group <= 8;
  if (!kv_fp8 && pageable_tma && !wide_cp_async) {
    const int box_rows = 32;
    if (encode_paged_map(&a.kmap, d.k, d.dtype, d.head_dim, d.kv_heads, ps, d.kv_extent, d.k_stride, box_rows) &&
        encode_paged_map(&a.vmap, d.v, d.dtype, d.head_dim, d.kv_heads, ps, d.kv_extent, d.v_stride, box_rows)) {
      a.tma_kv = 1;
      a.box_rows = box_rows;
      return SGLD_KERNEL_MMA_SYNC_TMA;
    }
  }
  return SGLD_KERNEL_MMA_SYNC;
}

}  // namespace

extern "C" {

int sgld_decode_kernel_kind(const sgld_decode_args* args, const sgld_plan_buffers* plan,
                            const sgld_plan_geometry* geometry) {
  const int rc = sgld::validate_decode(args, plan, geometry);
  if (rc) return -rc;
  sgld::DecodeLaunch a;
  return prepare_launch(*args, plan, geometry, a);
}

}  // extern "C"

namespace {

// The launches of a decode call; with `prefix`, its attention after the KV-cache write and the
// merge of both parts in the place of the split merge.
int run_decode(const sgld_decode_args& d, const sgld_plan_buffers* plan, const sgld_plan_geometry* geometry,
               const sgld::AttendLaunch* prefix, bool prefix_tc, cudaStream_t st) {
  const bool kv_fp8 = d.kv_dtype == SGLD_DTYPE_E4M3;
  const int32_t q_rows = d.q_rows == 0 ? geometry->batch_capacity : d.q_rows;
  const bool kv_write = d.new_loc != nullptr;
  const int ps = d.page_size;
  sgld::DecodeLaunch a;
  const int kind = prepare_launch(d, plan, geometry, a, prefix == nullptr);
  cudaError_t e;
  if (kv_write) {   // the step's KV-cache write, chained right before the decode
    sgld::KVWrite kw = {};
    kw.k_new = d.k_new;
    kw.v_new = d.v_new;
    kw.new_loc = d.new_loc;
    kw.k = const_cast<void*>(d.k);
    kw.v = const_cast<void*>(d.v);
    for (int i = 0; i < 4; ++i) kw.k_stride[i] = a.d.k_stride[i], kw.v_stride[i] = a.d.v_stride[i];
    for (int i = 0; i < 3; ++i) kw.kn_stride[i] = d.knew_stride[i], kw.vn_stride[i] = d.vnew_stride[i];
    kw.slots = d.kv_extent > 0 ? d.kv_extent * ps : 0;
    kw.rows = q_rows;
    kw.page_size = ps;
    kw.kv_heads = d.kv_heads;
    kw.head_dim = d.head_dim;
    kw.loc_int32 = d.new_loc_int32 != 0 ? 1 : 0;
    kw.dtype = d.dtype;
    kw.pool_fp8 = kv_fp8 ? 1 : 0;
    kw.k_scale = a.d.k_scale;
    kw.v_scale = a.d.v_scale;
    kw.status = d.status;
    e = sgld::launch_kv_write(kw, st, true);
    if (e != cudaSuccess) return cuda_fail(e, "sgld_decode_persistent KV-cache write launch");
  }
  if (prefix != nullptr) {
    e = prefix_tc ? sgld::launch_attend_tc(*prefix, st) : sgld::launch_attend_mma(*prefix, st);
    if (e != cudaSuccess) return cuda_fail(e, "sgld_decode_shared_prefix prefix launch");
  }
  if (prefix != nullptr && d.pages == nullptr) e = cudaSuccess;   // no own tokens: the prefix alone
  else if (kind == SGLD_KERNEL_TCGEN05 || kind == SGLD_KERNEL_TCGEN05_TMA) e = sgld::launch_decode_tc(a, st);
  else if (kind == SGLD_KERNEL_SMALL) e = sgld::launch_decode_small(a, st);
  else e = sgld::launch_decode(a, st);
  if (e != cudaSuccess) return cuda_fail(e, "sgld_decode_persistent launch");
  if (kind == SGLD_KERNEL_SMALL) return SGLD_OK;   // the small-batch kernel merges the splits itself
  if (prefix != nullptr) {
    e = sgld::launch_merge_prefix(*prefix, d, *plan, geometry->batch_capacity, geometry->max_splits, st);
    if (e != cudaSuccess) return cuda_fail(e, "sgld_decode_shared_prefix merge launch");
    return SGLD_OK;
  }
  e = sgld::launch_merge(d.partial, d.lse, plan->counts, plan->error, d.out, d.dtype, geometry->batch_capacity,
                         d.query_heads, d.head_dim, geometry->max_splits, st, true, d.counter);
  if (e != cudaSuccess) return cuda_fail(e, "sgld_decode_persistent merge launch");
  return SGLD_OK;
}

}  // namespace

extern "C" {

int sgld_decode_persistent(const sgld_decode_args* args, const sgld_plan_buffers* plan,
                           const sgld_plan_geometry* geometry, void* stream) {
  const int rc = sgld::validate_decode(args, plan, geometry);
  if (rc) return rc;
  return run_decode(*args, plan, geometry, nullptr, false, static_cast<cudaStream_t>(stream));
}

int sgld_merge_splits(const float* partial, const float* lse, const int32_t* counts,
                      const int32_t* error, void* out, int32_t dtype, int32_t batch_capacity,
                      int32_t query_heads, int32_t head_dim, int32_t max_splits, void* stream) {
  if (!partial || !lse || !counts || !error || !out)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "a merge pointer is NULL");
  if (dtype != SGLD_DTYPE_F16 && dtype != SGLD_DTYPE_BF16)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "dtype must be fp16 or bf16");
  if (batch_capacity <= 0 || query_heads <= 0 || max_splits <= 0 || batch_capacity > 65535 ||
      query_heads > 65535)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "merge geometry out of range");
  if (head_dim <= 0 || head_dim % 4 != 0 || head_dim > 4096)
    return fail(SGLD_ERR_UNSUPPORTED, "head_dim must be a multiple of 4 up to 4096");
  if (!aligned16(partial)) return fail(SGLD_ERR_INVALID_ARGUMENT, "partial must be 16-byte aligned");
  cudaError_t e = sgld::launch_merge(partial, lse, counts, error, out, dtype, batch_capacity, query_heads,
                                     head_dim, max_splits, static_cast<cudaStream_t>(stream), false, nullptr);
  if (e != cudaSuccess) return cuda_fail(e, "sgld_merge_splits launch");
  return SGLD_OK;
}

}  // extern "C"

namespace {

int sm_count() {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) {
    cudaGetLastError();
    return 148;
  }
  return sms;
}

// 2D map {columns, rows} over a K or V pool of `rows` token rows, `pitch` elements apart, boxes of 64
// columns x box_rows rows with the 128-byte swizzle.
bool encode_rows_map(CUtensorMap* map, const void* base, int32_t dtype, int64_t cols, int64_t rows, int64_t pitch,
                     int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch) * 2};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type =
      dtype == SGLD_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 3D map {D, Hq, tokens} over Q; a box is one tile: 64 dims, the group's heads, 128 / group tokens.
bool encode_query_map(CUtensorMap* map, const sgld::AttendLaunch& a) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.query_heads),
                        static_cast<cuuint64_t>(a.tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.q_stride[1]) * 2, static_cast<cuuint64_t>(a.q_stride[0]) * 2};
  for (cuuint64_t st : strides)
    if (st == 0 || st % 16 != 0 || st >= (cuuint64_t{1} << 40)) return false;
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(128 / a.group)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      a.dtype == SGLD_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, type, 3, const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The pool as rows of tokens: token-major (heads side by side in a row) or head-major (a head's
// rows after another's).  False where neither describes it.
bool pool_maps(const sgld::AttendLaunch& a, const void* base, const int64_t* stride, CUtensorMap* box, int32_t* head_col,
               int32_t* head_row, int32_t* map_rows) {
  const int64_t pitch = a.page_size > 1 ? stride[1] : stride[0], hs = a.kv_heads > 1 ? stride[2] : 0, d = a.head_dim;
  if (pitch <= 0 || pitch % 8 != 0 || pitch >= (int64_t{1} << 38) || hs % 8 != 0 || hs < 0) return false;
  int64_t cols = d, rows = a.kv_extent;
  *head_col = *head_row = 0;
  if (hs * (a.kv_heads - 1) + d <= pitch) {
    cols = hs * (a.kv_heads - 1) + d;
    *head_col = static_cast<int32_t>(hs);
  } else if (hs % pitch == 0 && pitch >= d && hs / pitch < (int64_t{1} << 31)) {
    rows = (a.kv_heads - 1) * (hs / pitch) + a.kv_extent;
    *head_row = static_cast<int32_t>(hs / pitch);
  } else {
    return false;
  }
  if (cols >= (int64_t{1} << 31) || rows >= (int64_t{1} << 31) - 128 || rows <= 0) return false;
  *map_rows = static_cast<int32_t>(rows);
  return encode_rows_map(box, base, a.dtype, cols, rows, pitch, a.box_rows);
}

// Row alignment and, where the tcgen05 kernel applies, its tensor maps (true).
bool prepare_attend(sgld::AttendLaunch& a) {
  set_wait_limits(a);
  // The stride of an extent of one is never used: any value may stand there.
  if (a.tokens == 1) a.q_stride[0] = a.out_stride[0] = static_cast<int64_t>(a.query_heads) * a.head_dim;
  if (a.query_heads == 1) a.q_stride[1] = a.out_stride[1] = a.head_dim;
  if (a.kv_extent == 1) a.k_stride[0] = a.v_stride[0] = static_cast<int64_t>(a.kv_heads) * a.head_dim;
  if (a.kv_heads == 1) a.k_stride[2] = a.v_stride[2] = a.head_dim;
  bool ok = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && a.q_stride[2] == 1 && a.k_stride[3] == 1 &&
            a.v_stride[3] == 1 && a.q_stride[0] % 8 == 0 && a.q_stride[1] % 8 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && a.k_stride[i] % 8 == 0 && a.v_stride[i] % 8 == 0;
  if (a.out != nullptr)
    ok = ok && aligned16(a.out) && a.out_stride[2] == 1 && a.out_stride[0] % 8 == 0 && a.out_stride[1] % 8 == 0;
  a.aligned = ok ? 1 : 0;
  if (!ok || a.head_dim > 128 || a.kv_extent <= 0 || !encode_query_map(&a.qmap, a)) return false;
  // Rows copied one by one are addressed by 32-bit offsets in units of 16 bytes.
  for (const int64_t* st : {a.k_stride, a.v_stride}) {
    const int64_t pitch = a.page_size > 1 ? st[1] : st[0];
    if (pitch < 0 || pitch / 8 * a.kv_extent >= (int64_t{1} << 32) - 1) return false;
  }
  if (a.page_size > 1 && (a.k_stride[0] != a.k_stride[1] * a.page_size || a.v_stride[0] != a.v_stride[1] * a.page_size))
    return false;
  // Rows that a box may take together: a block's without indices, else the page's largest power
  // of two; below 8 a box saves little over copying the rows one by one.
  a.box_rows = 128;
  if (a.kv_indices != nullptr) {
    a.box_rows = a.page_size & -a.page_size;
    if (a.box_rows > 128) a.box_rows = 128;
    if (a.box_rows < 8) a.box_rows = 0;
  }
  if (a.box_rows > 0 &&
      !(pool_maps(a, a.k, a.k_stride, &a.kmap, &a.k_head_col, &a.k_head_row, &a.map_rows_k) &&
        pool_maps(a, a.v, a.v_stride, &a.vmap, &a.v_head_col, &a.v_head_row, &a.map_rows_v)))
    a.box_rows = 0;
  return true;
}

// Splits of the keys: as many as keep every SM at work, where the tasks (tiles x KV heads) alone
// do not.  The cost of s splits is the rounds of tasks times the key blocks of one, plus two
// blocks' worth of a task's fixed time; each split also costs a partial result, so ties go low.
int choose_splits(int64_t tasks, int64_t keys, int sms) {
  const int64_t blocks = (keys + 127) / 128;
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int s = 1; s <= 64 && s <= blocks; ++s) {
    const int64_t rounds = (tasks * s + sms - 1) / sms, cost = rounds * ((blocks + s - 1) / s + 2);
    if (cost < best_cost) best = s, best_cost = cost;
  }
  return best;
}

size_t split_bytes(int64_t rows, int64_t heads, int64_t d, int splits) {
  return static_cast<size_t>(rows) * heads * splits * (d + 1) * sizeof(float);
}

int prompt_launch(const sgld_prompt_args* args, sgld::AttendLaunch& a, bool& tc) {
  if (args == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "prompt args are NULL");
  const sgld_prompt_args& p = *args;
  if (p.tokens < 0 || p.seqs < 0 || p.kv_extent < 0 || p.kv_indices_count < 0)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "tokens, seqs and extents must be >= 0");
  if (p.dtype != SGLD_DTYPE_F16 && p.dtype != SGLD_DTYPE_BF16)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "dtype must be fp16 or bf16");
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return fail(SGLD_ERR_UNSUPPORTED, "supported head dimensions: 64, 128, 256");
  if (p.kv_heads <= 0 || p.query_heads <= 0 || p.query_heads % p.kv_heads || p.query_heads > 65535)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "query heads must be a positive multiple of KV heads");
  if (p.query_heads / p.kv_heads > 16) return fail(SGLD_ERR_UNSUPPORTED, "GQA group sizes above 16 are not supported");
  if (!(p.scale > 0.f) || p.scale > 3.0e38f) return fail(SGLD_ERR_INVALID_ARGUMENT, "scale must be a finite value > 0");
  if (!(p.logit_cap >= 0.f) || p.logit_cap > 3.0e38f)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "logit_cap must be a finite value >= 0 (0 disables it)");
  if (p.window_left < -1) return fail(SGLD_ERR_INVALID_ARGUMENT, "window_left must be >= 0, or -1 for none");
  if (p.kv_extent >= (int64_t{1} << 31) || p.kv_indices_count >= (int64_t{1} << 31))
    return fail(SGLD_ERR_UNSUPPORTED, "more than 2^31 - 1 key rows");
  std::memset(&a, 0, sizeof(a));
  tc = false;
  if (p.tokens == 0 || p.seqs == 0) return SGLD_OK;
  if (!p.q || !p.out || !p.q_indptr || (p.kv_extent > 0 && (!p.k || !p.v)))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "a tensor pointer is NULL");
  if (p.kv_indices != nullptr && p.kv_indptr == nullptr)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "kv_indices need kv_indptr");
  a.q = p.q;
  a.k = p.k;
  a.v = p.v;
  a.out = p.out;
  a.lse = p.lse;
  a.q_indptr = p.q_indptr;
  a.kv_indptr = p.kv_indptr != nullptr ? p.kv_indptr : p.q_indptr;
  a.kv_indices = p.kv_indices;
  a.status = p.status;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = p.q_stride[i], a.out_stride[i] = p.out_stride[i];
  const int64_t ks[4] = {p.k_stride[0], 0, p.k_stride[1], p.k_stride[2]}, vs[4] = {p.v_stride[0], 0, p.v_stride[1], p.v_stride[2]};
  std::memcpy(a.k_stride, ks, sizeof(ks));
  std::memcpy(a.v_stride, vs, sizeof(vs));
  a.kv_count = p.kv_indices != nullptr ? p.kv_indices_count : p.kv_extent;
  a.kv_extent = p.kv_extent;
  a.tokens = p.tokens;
  a.seqs = p.seqs;
  a.query_heads = p.query_heads;
  a.kv_heads = p.kv_heads;
  a.group = p.query_heads / p.kv_heads;
  a.head_dim = p.head_dim;
  a.page_size = 1;
  a.dtype = p.dtype;
  a.causal = 1;
  // A window that no key of the call can leave is none: the kernels subtract it from key positions in 32 bits,
  // and those of queries before key 0 are negative.
  a.window_left = p.window_left < a.kv_count ? p.window_left : -1;
  a.scale = p.scale;
  a.logit_cap = p.logit_cap;
  tc = prepare_attend(a);
  // Split the keys only where the tiles leave SMs idle; the tasks hold one tile of 64 rows or, on
  // the tcgen05 kernel, two of 128.
  const int step = tc ? 2 * (128 / a.group) : 64 / a.group, sms = sm_count();
  const int64_t tiles = a.tokens / step + a.seqs, tasks = tiles * a.kv_heads;
  if (tasks > (int64_t{1} << 30)) return fail(SGLD_ERR_UNSUPPORTED, "too many tokens for one call");
  int64_t keys = a.kv_count / a.seqs;
  if (a.window_left >= 0 && keys > a.window_left + static_cast<int64_t>(step)) keys = a.window_left + step;
  a.splits = tasks * 2 <= sms ? choose_splits(tasks, keys, sms) : 1;
  return SGLD_OK;
}

int prefix_splits(int32_t batch, int32_t query_heads, int32_t kv_heads, int32_t head_dim, int32_t capacity) {
  const int group = query_heads / kv_heads, step = head_dim <= 128 ? 2 * (128 / group) : 64 / group;
  return choose_splits(static_cast<int64_t>((batch + step - 1) / step) * kv_heads, capacity, sm_count());
}

}  // namespace

extern "C" {

size_t sgld_prompt_workspace_bytes(const sgld_prompt_args* args) {
  sgld::AttendLaunch a;
  bool tc;
  if (prompt_launch(args, a, tc) != SGLD_OK || a.splits <= 1) return 0;
  return split_bytes(a.tokens, a.query_heads, a.head_dim, a.splits);
}

int sgld_prompt_kernel_kind(const sgld_prompt_args* args) {
  sgld::AttendLaunch a;
  bool tc;
  const int rc = prompt_launch(args, a, tc);
  return rc ? -rc : tc ? SGLD_KERNEL_TCGEN05_TMA : SGLD_KERNEL_MMA_SYNC;
}

int sgld_prompt_attention(const sgld_prompt_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  sgld::AttendLaunch a;
  bool tc;
  const int rc = prompt_launch(args, a, tc);
  if (rc) return rc;
  if (args->tokens == 0 || args->seqs == 0) return SGLD_OK;
  if (a.splits > 1) {
    if (workspace == nullptr || !aligned16(workspace) ||
        workspace_bytes < split_bytes(a.tokens, a.query_heads, a.head_dim, a.splits))
      return fail(SGLD_ERR_INVALID_ARGUMENT, "the workspace is smaller than sgld_prompt_workspace_bytes or not 16-byte aligned");
    a.partial = static_cast<float*>(workspace);
    a.partial_lse = a.partial + static_cast<int64_t>(a.tokens) * a.query_heads * a.splits * a.head_dim;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = tc ? sgld::launch_attend_tc(a, st) : sgld::launch_attend_mma(a, st);
  if (e != cudaSuccess) return cuda_fail(e, "sgld_prompt_attention launch");
  if (a.splits > 1) {
    e = sgld::launch_merge_prompt(a, a.out, a.lse, st);
    if (e != cudaSuccess) return cuda_fail(e, "sgld_prompt_attention merge launch");
  }
  return SGLD_OK;
}

size_t sgld_prefix_workspace_bytes(int32_t batch_capacity, int32_t query_heads, int32_t kv_heads, int32_t head_dim,
                                   int32_t capacity) {
  if (batch_capacity <= 0 || kv_heads <= 0 || query_heads <= 0 || query_heads % kv_heads || query_heads / kv_heads > 16 ||
      head_dim <= 0 || capacity < 0)
    return 0;
  return split_bytes(batch_capacity, query_heads, head_dim,
                     prefix_splits(batch_capacity, query_heads, kv_heads, head_dim, capacity));
}

int sgld_decode_shared_prefix(const sgld_decode_args* args, const sgld_prefix_args* prefix,
                              const sgld_plan_buffers* plan, const sgld_plan_geometry* geometry, void* stream) {
  const int rc = sgld::validate_decode(args, plan, geometry, args != nullptr && args->pages != nullptr);
  if (rc) return rc;
  if (prefix == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "prefix args are NULL");
  const sgld_decode_args& d = *args;
  if (d.kv_dtype == SGLD_DTYPE_E4M3) return fail(SGLD_ERR_UNSUPPORTED, "a shared prefix needs 16-bit K/V");
  if (!(d.scale > 0.f) || d.scale > 3.0e38f) return fail(SGLD_ERR_INVALID_ARGUMENT, "scale must be a finite value > 0");
  if (d.k_scale != 0.f && d.k_scale != 1.f) return fail(SGLD_ERR_UNSUPPORTED, "a shared prefix takes no k_scale / v_scale");
  if (d.v_scale != 0.f && d.v_scale != 1.f) return fail(SGLD_ERR_UNSUPPORTED, "a shared prefix takes no k_scale / v_scale");
  if (prefix->capacity < 0 || (prefix->capacity > 0 && prefix->index == nullptr))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "prefix index / capacity mismatch");
  if (d.kv_extent <= 0 || d.kv_extent * d.page_size >= (int64_t{1} << 31))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "a shared prefix needs kv_extent, below 2^31 token slots");
  const bool csr = d.indptr != nullptr;
  if (!csr && d.page_size > 1 && d.kv_extent > 1 &&
      (d.k_stride[0] != d.page_size * d.k_stride[1] || d.v_stride[0] != d.page_size * d.v_stride[1]))
    return fail(SGLD_ERR_UNSUPPORTED, "a shared prefix needs the pool's pages one after another");
  if (prefix->capacity % d.page_size != 0)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "the prefix capacity must be whole pages");
  // A workspace made for another capacity may hold fewer splits than this one would take.
  const size_t one = split_bytes(geometry->batch_capacity, d.query_heads, d.head_dim, 1);
  if (prefix->workspace == nullptr || !aligned16(prefix->workspace) || prefix->workspace_bytes < one)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "the workspace is smaller than one split's results or not 16-byte aligned");
  int splits = prefix_splits(geometry->batch_capacity, d.query_heads, d.kv_heads, d.head_dim, prefix->capacity);
  if (static_cast<size_t>(splits) > prefix->workspace_bytes / one) splits = static_cast<int>(prefix->workspace_bytes / one);
  sgld::AttendLaunch a;
  std::memset(&a, 0, sizeof(a));
  a.q = d.q;
  a.k = d.k;
  a.v = d.v;
  a.partial = static_cast<float*>(prefix->workspace);
  a.partial_lse = a.partial + static_cast<int64_t>(geometry->batch_capacity) * d.query_heads * splits * d.head_dim;
  a.kv_indices = prefix->index;
  a.kv_length = prefix->length;
  a.active = plan->active;
  a.status = d.status;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = d.q_stride[i];
  for (int i = 0; i < 4; ++i) a.k_stride[i] = d.k_stride[i], a.v_stride[i] = d.v_stride[i];
  if (csr) a.k_stride[1] = a.v_stride[1] = 0;
  if (d.page_size > 1) {                          // (the stride of a single page is never used)
    a.k_stride[0] = d.page_size * d.k_stride[1];
    a.v_stride[0] = d.page_size * d.v_stride[1];
  }
  a.kv_count = prefix->capacity;
  a.kv_extent = d.kv_extent * d.page_size;
  a.tokens = d.q_rows == 0 ? geometry->batch_capacity : d.q_rows;
  a.seqs = 1;
  a.query_heads = d.query_heads;
  a.kv_heads = d.kv_heads;
  a.group = d.query_heads / d.kv_heads;
  a.head_dim = d.head_dim;
  a.page_size = d.page_size;
  a.dtype = d.dtype;
  a.splits = splits;
  a.window_left = -1;
  a.scale = d.scale;
  a.logit_cap = d.logit_cap;
  const bool tc = prepare_attend(a);
  return run_decode(d, plan, geometry, &a, tc, static_cast<cudaStream_t>(stream));
}

int sgld_norm_rope(const sgld_norm_rope_args* args, void* stream) {
  if (args == nullptr) return fail(SGLD_ERR_INVALID_ARGUMENT, "norm_rope args are NULL");
  sgld_norm_rope_args a = *args;
  if (a.tokens < 0 || a.query_heads <= 0 || a.kv_heads <= 0 || a.query_heads > 65535 || a.kv_heads > 65535)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "tokens must be >= 0 and the head counts positive");
  if (a.dtype != SGLD_DTYPE_F16 && a.dtype != SGLD_DTYPE_BF16)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "dtype must be fp16 or bf16");
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256)
    return fail(SGLD_ERR_UNSUPPORTED, "supported head dimensions: 64, 128, 256");
  if (a.rotary <= 0 || a.rotary > a.head_dim || a.rotary % 16 != 0)
    return fail(SGLD_ERR_UNSUPPORTED, "rotary must be a multiple of 16 up to head_dim");
  const bool cached = a.slots != nullptr;
  if (cached ? (!a.v || !a.k_cache || !a.v_cache) : (a.v || a.k_cache || a.v_cache))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "the cache write needs v, k_cache, v_cache and slots");
  if (!cached && !a.k_out) return fail(SGLD_ERR_INVALID_ARGUMENT, "k_out may be NULL only with a cache write");
  if (cached && (a.page_size <= 0 || a.cache_slots < 0))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "page_size must be positive and cache_slots >= 0");
  if (!(a.eps >= 0.f) || a.eps > 3.0e38f) return fail(SGLD_ERR_INVALID_ARGUMENT, "eps must be a finite value >= 0");
  if (a.cache_fp8 && (!(a.k_scale > 0.f) || a.k_scale > 3.0e38f || !(a.v_scale > 0.f) || a.v_scale > 3.0e38f))
    return fail(SGLD_ERR_INVALID_ARGUMENT, "k_scale / v_scale must be finite values > 0");
  if (a.table_rows < 0) return fail(SGLD_ERR_INVALID_ARGUMENT, "table_rows must be >= 0");
  if (a.tokens == 0) return SGLD_OK;
  if (!a.q || !a.k || !a.positions || !a.table || !a.q_out)
    return fail(SGLD_ERR_INVALID_ARGUMENT, "a tensor pointer is NULL");
  const int heads_per_step = 256 / a.head_dim;
  const int64_t k_steps = (a.kv_heads + heads_per_step - 1) / heads_per_step;
  const int64_t steps = (a.query_heads + heads_per_step - 1) / heads_per_step + k_steps * (cached ? 2 : 1);
  if (a.tokens > (int64_t{1} << 31) / steps) return fail(SGLD_ERR_UNSUPPORTED, "too many tokens for one call");
  bool vec = aligned16(a.q) && aligned16(a.k) && aligned16(a.q_out) && aligned16(a.table) && aligned16(a.q_weight) &&
             aligned16(a.k_weight) && a.table_stride % 4 == 0;
  const auto rows_ok = [](const int64_t* s, int n) {
    bool ok = s[n - 1] == 1;
    for (int i = 0; i < n - 1; ++i) ok = ok && s[i] % 8 == 0;
    return ok;
  };
  vec = vec && rows_ok(a.q_stride, 3) && rows_ok(a.k_stride, 3) && rows_ok(a.qo_stride, 3);
  if (a.k_out != nullptr) vec = vec && aligned16(a.k_out) && rows_ok(a.ko_stride, 3);
  if (cached)
    vec = vec && aligned16(a.v) && aligned16(a.k_cache) && aligned16(a.v_cache) && rows_ok(a.v_stride, 3) &&
          rows_ok(a.kc_stride, 4) && rows_ok(a.vc_stride, 4);
  const bool few = a.tokens * steps < kFewRopeSteps;
  cudaError_t e = sgld::launch_norm_rope(a, vec, few, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "sgld_norm_rope launch");
  return SGLD_OK;
}

}  // extern "C"
