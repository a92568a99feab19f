// Attention of packed query rows over long keys, on mma.sync: the form for every stride and for
// head_dim 256 (sgld_attend_tc.cu holds the tcgen05 form for 16-byte aligned rows and head_dim
// 64 / 128), and the merge of split results.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - m),   s_j = scale * q . k_j  (soft-capped)
//
// over the keys j that the row sees, in one pass with a running maximum m and sum.  One CTA of
// four warps takes 64 rows of one KV head and walks its keys in blocks of 64 (32 for head_dim 256),
// each block copied to shared memory as it is; a warp holds 16 rows, scores and output in
// registers.  Scores, maxima, sums and outputs are fp32; the weights p are rounded to 16 bits for
// the second product, as its operands must be, while their sum keeps the fp32 values.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "sgld_attend.cuh"
#include "sgld_internal.cuh"
#include "sgld_ptx.cuh"

namespace sgld {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRows = 64;       // rows of a tile
constexpr int kThreads = 128;

template <int D>
constexpr int key_block() { return D == 256 ? 32 : 64; }
template <int D>
constexpr int pitch() { return D + 8; }      // shared rows, padded: ldmatrix without bank conflicts
template <int D>
constexpr int smem_bytes() { return (kRows + 2 * key_block<D>()) * pitch<D>() * 2; }

// One row of D elements into shared memory; slot < 0 (or src == nullptr) writes zeros.
template <typename T, int D>
__device__ __forceinline__ void copy_chunk(T* dst, const T* src, int64_t stride, int c, bool aligned) {
  if (src == nullptr) {
    *reinterpret_cast<uint4*>(dst + c * 8) = make_uint4(0u, 0u, 0u, 0u);
  } else if (aligned) {
    *reinterpret_cast<uint4*>(dst + c * 8) = *reinterpret_cast<const uint4*>(src + c * 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[c * 8 + i] = src[(c * 8 + i) * stride];
  }
}

// (Two blocks an SM named for head_dim 256, where the compiler would otherwise spill for three: 856 us for 4096
// tokens of 8 / 2 heads, against 1209.  The others choose for themselves: 373 and 708 us, 16 / 4 heads of 64 / 128,
// against 399 and 718 with three.)
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, D == 256 ? 2 : 0) attend_mma_kernel(const __grid_constant__ AttendLaunch a) {
  constexpr int kB = key_block<D>(), kP = pitch<D>(), kNb = kB / 8, kDb = D / 8;
  constexpr float kBias = WeightBias<T>::value;
  extern __shared__ __align__(16) unsigned char smem[];
  T* qs = reinterpret_cast<T*>(smem);
  T* ks = qs + kRows * kP;
  T* vs = ks + kB * kP;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int G = a.group, step = kRows / G;
  int chunk = 0;
  int64_t before = 0;
  const AttendTask t = find_task(a, step, kB, blockIdx.x, chunk, before);   // every warp finds the same task
  if (!t.valid) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = (t.last - t.first) * G;
  const bool aligned = a.aligned != 0;
  for (int i = threadIdx.x; i < kRows * (D / 8); i += kThreads) {
    const int r = i / (D / 8), c = i % (D / 8);
    const T* src = r < rows ? static_cast<const T*>(a.q) + static_cast<int64_t>(t.first + r / G) * a.q_stride[0] +
                                  static_cast<int64_t>(t.head * G + r % G) * a.q_stride[1]
                            : nullptr;
    copy_chunk<T, D>(qs + r * kP, src, a.q_stride[2], c, aligned);
  }
  // This thread's two rows of its warp's 16.
  int lo[2], hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + lane / 4 + 8 * h, row = t.first + r / G;
    lo[h] = first_key(a, t, row);
    hi[h] = r < rows ? last_key(a, t, row) : -1;
  }
  float o[kDb][4];
#pragma unroll
  for (int i = 0; i < kDb; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float c_scale = a.scale * kLog2e, over_cap = a.logit_cap > 0.f ? a.scale / a.logit_cap : 0.f,
              cap_log2e = a.logit_cap * kLog2e;

  for (int j0 = t.lo; j0 < t.hi; j0 += kB) {
    __syncthreads();
    for (int i = threadIdx.x; i < kB * (D / 8); i += kThreads) {
      const int r = i / (D / 8), c = i % (D / 8), j = j0 + r;
      const int64_t slot = j < t.hi ? key_slot(a, t.kv_begin, j) : -1;
      const T *kp = nullptr, *vp = nullptr;
      if (slot >= 0) {
        const int64_t page = slot / a.page_size, in = slot - page * a.page_size;
        kp = static_cast<const T*>(a.k) + page * a.k_stride[0] + in * a.k_stride[1] + t.head * a.k_stride[2];
        vp = static_cast<const T*>(a.v) + page * a.v_stride[0] + in * a.v_stride[1] + t.head * a.v_stride[2];
      }
      copy_chunk<T, D>(ks + r * kP, kp, a.k_stride[3], c, aligned);
      copy_chunk<T, D>(vs + r * kP, vp, a.v_stride[3], c, aligned);
    }
    __syncthreads();
    float s[kNb][4];
#pragma unroll
    for (int n = 0; n < kNb; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int d = 0; d < D; d += 16) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4(smem_addr(qs + (warp * 16 + (lane & 15)) * kP + d + (lane >> 4) * 8), a0, a1, a2, a3);
#pragma unroll
      for (int n = 0; n < kNb; n += 2) {
        uint32_t b0, b1, b2, b3;   // keys 8n..8n+7 (b0, b1) and 8n+8.. (b2, b3), dims d and d + 8
        ldsm_x4(smem_addr(ks + (n * 8 + (lane & 7) + (lane >> 4) * 8) * kP + d + ((lane >> 3) & 1) * 8), b0, b1, b2, b3);
        Mma<T>::run(s[n], a0, a1, a2, a3, b0, b1);
        Mma<T>::run(s[n + 1], a0, a1, a2, a3, b2, b3);
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kNb; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = e >> 1, j = j0 + n * 8 + (lane & 3) * 2 + (e & 1);
        float x = a.logit_cap > 0.f ? capped_log2(s[n][e], over_cap, cap_log2e) : s[n][e] * c_scale;
        if (j < lo[h] || j > hi[h]) x = -INFINITY;
        s[n][e] = x;
        top[h] = fmaxf(top[h], x);
      }
    }
    float ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      const float mn = fmaxf(m[h], top[h]);
      ref[h] = mn == -INFINITY ? 0.f : mn;
      const float w = ex2(m[h] - ref[h]);
      m[h] = mn;
      l[h] *= w;
#pragma unroll
      for (int i = 0; i < kDb; ++i) o[i][2 * h] *= w, o[i][2 * h + 1] *= w;
    }
#pragma unroll
    for (int n = 0; n < kNb; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - (ref[e >> 1] - kBias));
        l[e >> 1] += s[n][e];
      }
    }
#pragma unroll
    for (int n = 0; n < kNb; n += 2) {       // 16 keys a step
      const uint32_t a0 = Mma<T>::pack(s[n][0], s[n][1]), a1 = Mma<T>::pack(s[n][2], s[n][3]);
      const uint32_t a2 = Mma<T>::pack(s[n + 1][0], s[n + 1][1]), a3 = Mma<T>::pack(s[n + 1][2], s[n + 1][3]);
#pragma unroll
      for (int i = 0; i < kDb; i += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(smem_addr(vs + (n * 8 + (lane & 15)) * kP + i * 8 + (lane >> 4) * 8), b0, b1, b2, b3);
        Mma<T>::run(o[i], a0, a1, a2, a3, b0, b1);
        Mma<T>::run(o[i + 1], a0, a1, a2, a3, b2, b3);
      }
    }
  }

  uint32_t again[2];
  float e2[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = warp * 16 + lane / 4 + 8 * h, row = t.first + r / G, head = t.head * G + r % G;
    const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
    e2[h] = l[h] == 0.f ? -INFINITY : m[h] - kBias + lg2(l[h]);
    const int64_t at = static_cast<int64_t>(row) * a.query_heads + head;
    bool odd = false;
    if (r < rows) {
#pragma unroll
      for (int i = 0; i < kDb; ++i) {
        const float x = o[i][2 * h] * inv, y = o[i][2 * h + 1] * inv;
        odd = odd || !(fabsf(x) <= 3.0e38f) || !(fabsf(y) <= 3.0e38f);
        const int d = i * 8 + (lane & 3) * 2;
        if (a.partial != nullptr) {
          *reinterpret_cast<float2*>(a.partial + (at * a.splits + t.split) * D + d) = make_float2(x, y);
        } else {
          T* out = static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.out_stride[0] + static_cast<int64_t>(head) * a.out_stride[1];
          if (aligned) {
            *reinterpret_cast<uint32_t*>(out + d) = Mma<T>::pack(x, y);
          } else {
            out[d * a.out_stride[2]] = from_float<T>(x);
            out[(d + 1) * a.out_stride[2]] = from_float<T>(y);
          }
        }
      }
      if ((lane & 3) == 0) {
        if (a.partial != nullptr) a.partial_lse[at * a.splits + t.split] = e2[h] * kLn2;
        else if (a.lse != nullptr) a.lse[at] = e2[h] * kLn2;
      }
    }
    again[h] = __ballot_sync(0xffffffffu, odd);
    again[h] = __ballot_sync(0xffffffffu, (lane & 3) == 0 && (again[h] >> lane & 0xfu) != 0);   // one lane of each such row
  }
  if ((again[0] | again[1]) == 0) return;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + lane / 4 + 8 * h;
    if (again[h] != 0) form_again<T, D, 1>(a, t, again[h], t.first + r / G, t.head * G + r % G, h == 0 ? e2[0] : e2[1], nullptr);
  }
}

template <typename T, int D>
cudaError_t launch(const AttendLaunch& a, cudaStream_t stream) {
  constexpr int bytes = smem_bytes<D>();
  const cudaError_t e = cudaFuncSetAttribute(attend_mma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  const int step = kRows / a.group;
  const int64_t tiles = a.tokens / step + a.seqs;      // at least the tiles of any cut into sequences
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.splits * a.kv_heads));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attend_mma_kernel<T, D>, a);
}

template <typename T>
cudaError_t launch_dim(const AttendLaunch& a, cudaStream_t stream) {
  if (a.head_dim == 64) return launch<T, 64>(a, stream);
  if (a.head_dim == 128) return launch<T, 128>(a, stream);
  return launch<T, 256>(a, stream);
}

// ---------------------------------------------------------------- merge of split results
// One warp per (row, query head): the LSE-weighted sum of the row's split results, all of `second` (the
// prefix, or a prompt's splits) and then `first` (a decode's counts[row] slots of first_max; absent
// for the prompt attention, and for a decode without an index of own tokens, whose rows with counts
// are NaN), each in split order.  A slot whose LSE is -inf saw no key: its values do not count.  A row is a chain of two memory round trips (its count, its slots), which bound the
// kernel, not the bytes: values are loaded together with their LSEs, four slots at a time, at 64
// registers for 32 warps an SM (16384 rows of nine prefix slots and one own: 23 us; with eight slots at a
// time and their values only after the LSEs, at 96 registers, 34).
struct MergeLaunch {
  const float* first;
  const float* first_lse;
  const int32_t* counts;
  const float* second;
  const float* second_lse;
  const int32_t* error;
  const int32_t* active;
  void* out;
  float* lse;
  int32_t* claim;
  int32_t* status;           // bit 512: a row has own tokens but no index names them
  int64_t out_stride[3];
  int32_t first_max, second_max, rows, rows_second, heads, head_dim;
  const int32_t* q_indptr;   // rows at or past q_indptr[seqs] are left as they are
  int32_t seqs;
};

constexpr int kMergeWarps = 4;
constexpr int kBatch = 4;        // slots loaded at a time

struct Running {
  float m, l;
  float4 acc;
};

__device__ __forceinline__ void merge_slots(Running& r, const float* part, const float* lse, int n, int d_dim) {
  for (int s0 = 0; s0 < n; s0 += kBatch) {
    float e[kBatch];
    float4 p[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      e[u] = -INFINITY;
      p[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + u < n) {
        e[u] = __ldcg(lse + s0 + u) * kLog2e;
        p[u] = __ldcg(reinterpret_cast<const float4*>(part + static_cast<int64_t>(s0 + u) * d_dim));
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (e[u] == -INFINITY) continue;
      const float mn = fmaxf(r.m, e[u]);
      const float w0 = ex2(r.m - mn), w1 = ex2(e[u] - mn);
      r.acc.x = r.acc.x * w0 + p[u].x * w1;
      r.acc.y = r.acc.y * w0 + p[u].y * w1;
      r.acc.z = r.acc.z * w0 + p[u].z * w1;
      r.acc.w = r.acc.w * w0 + p[u].w * w1;
      r.l = r.l * w0 + w1;
      r.m = mn;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kMergeWarps * 32, 8) merge_shared_kernel(const __grid_constant__ MergeLaunch a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (a.claim != nullptr && blockIdx.x == 0 && threadIdx.x < 2) a.claim[threadIdx.x] = 0;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5);
  if (at >= static_cast<int64_t>(a.rows) * a.heads) return;
  const int row = static_cast<int>(at / a.heads), head = static_cast<int>(at - static_cast<int64_t>(row) * a.heads);
  const int lane = threadIdx.x & 31;
  if (a.q_indptr != nullptr && (row < a.q_indptr[0] || row >= a.q_indptr[a.seqs])) return;
  const bool err = a.error != nullptr && *a.error != 0;
  const bool shared = row < a.rows_second && (a.active == nullptr || row < *a.active);
  int n = a.counts != nullptr ? a.counts[row] : 0;
  const bool lost = n > 0 && a.first == nullptr;
  if (lost) {
    if (head == 0 && lane == 0) atomicOr(a.status, 512);
    n = 0;
  }
  for (int d = lane * 4; d < a.head_dim; d += 128) {
    Running r{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if (shared)
      merge_slots(r, a.second + at * a.second_max * a.head_dim + d, a.second_lse + at * a.second_max, a.second_max, a.head_dim);
    if (n > 0)
      merge_slots(r, a.first + at * a.first_max * a.head_dim + d, a.first_lse + at * a.first_max, n, a.head_dim);
    const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
    float v[4] = {r.acc.x * inv, r.acc.y * inv, r.acc.z * inv, r.acc.w * inv};
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.out_stride[0] + static_cast<int64_t>(head) * a.out_stride[1];
    if (err || lost) v[0] = v[1] = v[2] = v[3] = __int_as_float(0x7fc00000);
    if (a.out_stride[2] == 1 && (reinterpret_cast<uintptr_t>(out + d) & 7) == 0) {
      *reinterpret_cast<uint2*>(out + d) = make_uint2(Mma<T>::pack(v[0], v[1]), Mma<T>::pack(v[2], v[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[(d + i) * a.out_stride[2]] = from_float<T>(v[i]);
    }
    if (d == 0 && a.lse != nullptr) a.lse[at] = r.l == 0.f ? -INFINITY : (r.m + lg2(r.l)) * kLn2;
  }
}

cudaError_t launch_merge_shared(const MergeLaunch& a, int dtype, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.rows) * a.heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + kMergeWarps - 1) / kMergeWarps));
  cfg.blockDim = dim3(kMergeWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return dtype == SGLD_DTYPE_BF16 ? cudaLaunchKernelEx(&cfg, merge_shared_kernel<__nv_bfloat16>, a)
                                  : cudaLaunchKernelEx(&cfg, merge_shared_kernel<__half>, a);
}

}  // namespace

cudaError_t launch_attend_mma(const AttendLaunch& a, cudaStream_t stream) {
  return a.dtype == SGLD_DTYPE_BF16 ? launch_dim<__nv_bfloat16>(a, stream) : launch_dim<__half>(a, stream);
}

cudaError_t launch_merge_prompt(const AttendLaunch& a, void* out, float* lse, cudaStream_t stream) {
  MergeLaunch m = {};
  m.second = a.partial;
  m.second_lse = a.partial_lse;
  m.out = out;
  m.lse = lse;
  for (int i = 0; i < 3; ++i) m.out_stride[i] = a.out_stride[i];
  m.second_max = a.splits;
  m.rows = m.rows_second = a.tokens;
  m.heads = a.query_heads;
  m.head_dim = a.head_dim;
  m.q_indptr = a.q_indptr;
  m.seqs = a.seqs;
  return launch_merge_shared(m, a.dtype, stream);
}

cudaError_t launch_merge_prefix(const AttendLaunch& a, const sgld_decode_args& d, const sgld_plan_buffers& p, int bcap,
                                int smax, cudaStream_t stream) {
  MergeLaunch m = {};
  m.first = d.pages != nullptr ? d.partial : nullptr;
  m.first_lse = d.lse;
  m.counts = p.counts;
  m.first_max = smax;
  m.second = a.partial;
  m.second_lse = a.partial_lse;
  m.second_max = a.splits;
  m.error = p.error;
  m.active = p.active;
  m.out = d.out;
  m.claim = d.counter;
  m.status = d.status;
  m.out_stride[0] = static_cast<int64_t>(d.query_heads) * d.head_dim;
  m.out_stride[1] = d.head_dim;
  m.out_stride[2] = 1;
  m.rows = bcap;
  m.rows_second = a.tokens;
  m.heads = d.query_heads;
  m.head_dim = d.head_dim;
  return launch_merge_shared(m, d.dtype, stream);
}

}  // namespace sgld
