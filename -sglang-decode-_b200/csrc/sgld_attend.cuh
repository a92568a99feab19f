// Attention of many query rows over long keys: shared by the prompt attention (causal, packed
// sequences) and the prefix part of the shared-prefix decode (every request's query rows over
// one run of keys).
//
// Rows.  The G query heads of a KV head share its keys, so they are packed into the rows of one
// tile: row r of a tile holds token t0 + r / G and query head kvh * G + r % G.  A short prompt or
// a decode batch thus fills a tile of the matrix units that one head alone would leave empty.
//
// Work.  A task is (tile of tokens of one sequence, KV head, split of its keys).  Sequences are
// read from device pointers, so a task index is turned into its task on the GPU.  Tasks are
// numbered from the longest to the shortest (causal tiles see 1 to all keys), so that those taken
// last are short and the SMs end together.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "sgld_internal.cuh"
#include "sgld_ptx.cuh"

namespace sgld {

struct alignas(64) AttendLaunch {
  CUtensorMap qmap;            // 3D {D, Hq, tokens}, box {64, G, 128 / G}                (tcgen05 kernel)
  CUtensorMap kmap, vmap;      // 2D {columns, rows} of the K / V pool, box {64, box_rows}
  const void* q;
  const void* k;
  const void* v;
  void* out;                   // [tokens, Hq, D] in `dtype`; nullptr: partials
  float* lse;                  // [tokens, Hq] natural log; may be nullptr
  float* partial;              // [tokens, Hq, splits, D] fp32
  float* partial_lse;          // [tokens, Hq, splits]
  const int32_t* q_indptr;     // [seqs + 1]; nullptr: one sequence of all tokens
  const int32_t* kv_indptr;    // [seqs + 1]; nullptr: one sequence of kv_count keys
  const int32_t* kv_indices;   // key rows (page_size 1) or pages; nullptr: key j of a sequence is row begin + j
  const int32_t* kv_length;    // [1] keys of the one sequence, at most kv_count; nullptr: kv_count
  const int32_t* active;       // [1] rows in use, at most tokens; nullptr: tokens
  int32_t* status;
  int64_t q_stride[3];         // elements: (token, head, dim)
  int64_t k_stride[4];         // (page, token-in-page, head, dim)
  int64_t v_stride[4];
  int64_t out_stride[3];
  int64_t kv_count;            // entries that indices may address: keys, or pages * page_size
  int64_t kv_extent;           // token slots of the pool
  int32_t k_head_col, k_head_row, v_head_col, v_head_row;   // column / row of a head in the 2D maps
  int32_t map_rows_k, map_rows_v;                           // rows of the maps: the row that reads as zeros
  int32_t tokens, seqs, query_heads, kv_heads, group, head_dim, page_size, dtype;
  int32_t splits, causal, window_left;
  int32_t box_rows;            // consecutive pool rows of a box: 128 without indices, 8 .. 128 rows of a
                               // page, 0 where every row is copied by itself
  int32_t aligned;             // every row 16-byte aligned with unit stride along D
  float scale, logit_cap;
  int32_t stall;               // tasks after which the tcgen05 kernel's issuer stops in every CTA (tests); -1: never
  uint64_t wait_ns;            // after which its waits expire
};

cudaError_t launch_attend_mma(const AttendLaunch& a, cudaStream_t stream);
cudaError_t launch_attend_tc(const AttendLaunch& a, cudaStream_t stream);
// The split results of a prompt call into `out` (a.out_stride) and, where given, `lse`.
cudaError_t launch_merge_prompt(const AttendLaunch& a, void* out, float* lse, cudaStream_t stream);
// A decode's split slots and the prefix partials of `a` into the decode's output; zeroes the
// decode's claim words as launch_merge does.
cudaError_t launch_merge_prefix(const AttendLaunch& a, const sgld_decode_args& d, const sgld_plan_buffers& p, int bcap,
                                int smax, cudaStream_t stream);

struct AttendTask {
  int32_t first, last;   // token rows [first, last) of the task
  int32_t shift;         // key position that token row r sees last: r + shift (causal)
  int32_t kv_begin;      // index of the sequence's key 0
  int32_t kv_len;        // keys of the sequence
  int32_t lo, hi;        // keys [lo, hi) of the task, its split included
  int32_t head, split, valid;
};

// Up to this many sequences, tiles are numbered from the most keys to the fewest; finding one then takes
// a search over all sequences.  More sequences are taken one after another.
constexpr int kSortedSeqs = 128;

// Rows and keys of a sequence, cut to the tensors they address.
__device__ __forceinline__ void sequence_bounds(const AttendLaunch& a, int s, int& q0, int& q1, int& k0, int& k1) {
  q0 = min(max(a.q_indptr[s], 0), a.tokens);
  q1 = min(max(a.q_indptr[s + 1], q0), a.tokens);
  k0 = static_cast<int>(min(static_cast<int64_t>(max(a.kv_indptr[s], 0)), a.kv_count));
  k1 = static_cast<int>(min(static_cast<int64_t>(max(a.kv_indptr[s + 1], k0)), a.kv_count));
}

// The first tile of a sequence (rows n, keys m) that sees at least `keys` keys, where no tile counts
// as seeing more than `most`; its number of tiles if there is none.
__device__ __forceinline__ int first_tile(int n, int m, int step, int keys, int most) {
  const int tiles = (n + step - 1) / step;
  if (keys <= 0) return 0;
  if (keys > most || keys > m) return tiles;
  const int x = keys - (m - n);                      // tokens up to the one that sees key keys - 1
  return min(tiles, max(0, (x + step - 1) / step - 1));
}

// Rows and keys of up to kSortedSeqs sequences, lane l holding those of l, l + 32, ...
struct SequenceSizes {
  int n[kSortedSeqs / 32], m[kSortedSeqs / 32];
};

// Tiles of all sequences that see more than 128 (level - 1) keys; whole warp.
__device__ __forceinline__ int tiles_from(const SequenceSizes& z, int seqs, int step, int level, int most) {
  int count = 0;
#pragma unroll
  for (int i = 0; i < kSortedSeqs / 32; ++i) {
    if (i * 32 >= seqs) break;
    count += (z.n[i] + step - 1) / step - first_tile(z.n[i], z.m[i], step, level > 0 ? (level - 1) * 128 + 1 : 0, most);
  }
  return __reduce_add_sync(0xffffffffu, count);
}

// Sequence and tile of tile number `tile` (whole warp; every lane gets them); false past the last.
// `chunk` and `before` are a cursor of the unsorted order: pass 0, 0 first.  Tiles may come in any order,
// as the hardware may hand out waiting blocks in any: ascending ones go on from the cursor, one that
// lies before it starts over.
__device__ __forceinline__ bool find_tile(const AttendLaunch& a, int step, int64_t tile, int& chunk, int64_t& before,
                                          int& q0, int& q1, int& k0, int& k1, int& index) {
  const int lane = threadIdx.x & 31;
  if (a.q_indptr == nullptr) {
    q0 = 0;
    q1 = a.active != nullptr ? min(max(*a.active, 0), a.tokens) : a.tokens;
    k0 = 0;
    k1 = static_cast<int>(a.kv_length != nullptr ? min(static_cast<int64_t>(max(*a.kv_length, 0)), a.kv_count) : a.kv_count);
    const int n = (q1 + step - 1) / step;
    if (tile >= n) return false;
    index = static_cast<int>(n - 1 - tile);
    return true;
  }
  if (a.seqs == 1) {                                 // the same order without a search
    sequence_bounds(a, 0, q0, q1, k0, k1);
    const int n = (q1 - q0 + step - 1) / step;
    if (tile >= n) return false;
    index = static_cast<int>(n - 1 - tile);
    return true;
  }
  if (a.seqs <= kSortedSeqs) {
    // Level n holds the tiles of n blocks of 128 keys: the highest level whose tiles and all above
    // are more than `tile`, then the place within it, sequence by sequence.
    const int most = a.window_left >= 0 ? min(a.window_left, 0x3fffffff) + step : 0x7fffffff;
    SequenceSizes z;
    int top = 0;
#pragma unroll
    for (int i = 0; i < kSortedSeqs / 32; ++i) {
      z.n[i] = z.m[i] = 0;
      if (i * 32 + lane < a.seqs) {
        sequence_bounds(a, i * 32 + lane, q0, q1, k0, k1);
        z.n[i] = q1 - q0;
        z.m[i] = k1 - k0;
      }
      if (z.n[i] > 0) top = max(top, (min(z.m[i], most) + 127) / 128);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (tile >= tiles_from(z, a.seqs, step, 0, most)) return false;
    int low = 0, high = top;                         // tiles_from(low) > tile
    while (low < high) {
      const int mid = (low + high + 1) >> 1;
      if (tiles_from(z, a.seqs, step, mid, most) > tile) low = mid;
      else high = mid - 1;
    }
    int rank = static_cast<int>(tile) - tiles_from(z, a.seqs, step, low + 1, most);
#pragma unroll
    for (int i = 0; i < kSortedSeqs / 32; ++i) {
      if (i * 32 >= a.seqs) break;
      const int from = first_tile(z.n[i], z.m[i], step, low > 0 ? (low - 1) * 128 + 1 : 0, most);
      const int to = first_tile(z.n[i], z.m[i], step, low * 128 + 1, most);
      int sum = to - from;
#pragma unroll
      for (int bit = 1; bit < 32; bit <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, bit);
        if (lane >= bit) sum += x;
      }
      const int total = __shfl_sync(0xffffffffu, sum, 31);
      if (rank < total) {
        const int owner = __ffs(__ballot_sync(0xffffffffu, rank < sum)) - 1;
        index = __shfl_sync(0xffffffffu, from + sum - 1 - rank, owner);
        sequence_bounds(a, i * 32 + owner, q0, q1, k0, k1);
        return true;
      }
      rank -= total;
    }
    return false;
  }
  if (tile < before) chunk = 0, before = 0;
  while (chunk < a.seqs) {
    const int s = chunk + lane;
    int n = 0;
    q0 = q1 = k0 = k1 = 0;
    if (s < a.seqs) {
      sequence_bounds(a, s, q0, q1, k0, k1);
      n = (q1 - q0 + step - 1) / step;
    }
    int sum = n;
#pragma unroll
    for (int bit = 1; bit < 32; bit <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, bit);
      if (lane >= bit) sum += x;
    }
    const int total = __shfl_sync(0xffffffffu, sum, 31);
    if (tile < before + total) {
      const int at = static_cast<int>(tile - before);
      const int owner = __ffs(__ballot_sync(0xffffffffu, at < sum)) - 1;
      index = __shfl_sync(0xffffffffu, sum - 1 - at, owner);
      q0 = __shfl_sync(0xffffffffu, q0, owner);
      q1 = __shfl_sync(0xffffffffu, q1, owner);
      k0 = __shfl_sync(0xffffffffu, k0, owner);
      k1 = __shfl_sync(0xffffffffu, k1, owner);
      return true;
    }
    before += total;
    chunk += 32;
  }
  return false;
}

// Task number `task` (KV head fastest, then split, then tile); whole warp.  32-bit arithmetic: the
// launch bounds the tasks, and a 64-bit division costs as much as all the rest.
__device__ __forceinline__ AttendTask find_task(const AttendLaunch& a, int step, int block, uint32_t task, int& chunk,
                                                int64_t& before) {
  AttendTask t;
  const uint32_t rest = task / static_cast<uint32_t>(a.kv_heads), tile = rest / static_cast<uint32_t>(a.splits);
  t.head = static_cast<int>(task - rest * static_cast<uint32_t>(a.kv_heads));
  t.split = static_cast<int>(rest - tile * static_cast<uint32_t>(a.splits));
  int q0 = 0, q1 = 0, k0 = 0, k1 = 0, index = 0;
  t.valid = find_tile(a, step, tile, chunk, before, q0, q1, k0, k1, index) ? 1 : 0;
  t.first = q0 + index * step;
  t.last = min(t.first + step, q1);
  t.kv_begin = k0;
  t.kv_len = k1 - k0;
  t.shift = t.kv_len - (q1 - q0) - q0;      // token row r sits at key position r + shift
  t.lo = 0;
  t.hi = t.kv_len;
  if (a.causal) {
    t.hi = max(0, min(t.kv_len, t.last + t.shift));
    if (a.window_left >= 0) t.lo = min(t.hi, max(0, t.first + t.shift - a.window_left));
  }
  if (a.splits > 1) {                       // whole blocks of keys per split
    const uint32_t blocks = (t.hi - t.lo + block - 1) / block;     // at most 2^26, and 64 splits
    const int b0 = static_cast<int>(blocks * t.split / static_cast<uint32_t>(a.splits));
    const int b1 = static_cast<int>(blocks * (t.split + 1) / static_cast<uint32_t>(a.splits));
    const int lo = t.lo;
    t.lo = min(t.hi, lo + b0 * block);
    t.hi = min(t.hi, lo + b1 * block);
  }
  return t;
}

// Does token row `row` of task t see key j?  (j within the task's keys.)
__device__ __forceinline__ int last_key(const AttendLaunch& a, const AttendTask& t, int row) {
  return a.causal ? min(t.hi - 1, row + t.shift) : t.hi - 1;
}
__device__ __forceinline__ int first_key(const AttendLaunch& a, const AttendTask& t, int row) {
  return a.causal && a.window_left >= 0 ? max(t.lo, row + t.shift - a.window_left) : t.lo;
}

// Token slot of key j of a sequence, or -1 when its index lies outside the pool.
__device__ __forceinline__ int64_t key_slot(const AttendLaunch& a, int kv_begin, int j) {
  int64_t slot;
  if (a.kv_indices == nullptr) {
    slot = static_cast<int64_t>(kv_begin) + j;
  } else if (a.page_size == 1) {
    slot = a.kv_indices[static_cast<int64_t>(kv_begin) + j];
  } else {
    const int at = kv_begin + j, page = at / a.page_size;
    slot = static_cast<int64_t>(a.kv_indices[page]) * a.page_size + (at - page * a.page_size);
    if (a.kv_indices[page] < 0) slot = -1;
  }
  return slot >= 0 && slot < a.kv_extent ? slot : -1;
}

// Weights are formed as 2^(s - m + kWeightBias), m the reference maximum in log2 units.  fp16 keeps 11
// bits down to 2^-14 only: lifted by 2^7, weights keep them down to 2^-21 of the largest, and stay
// below 2^15 where the reference may lag by 2^8.  bf16 has the exponents of fp32.
template <typename T>
struct WeightBias {
  static constexpr float value = 0.f;
};
template <>
struct WeightBias<__half> {
  static constexpr float value = 7.f;
};

// Soft cap, in log2 units: cap * log2(e) * tanh(u), u = s * scale / cap.  1 - 2 / (1 + e^2u) is exact to
// 2^-22 of the cap, not of a small result: below 1/2, where scores of a few units under a cap of
// 30 or 50 lie, tanh(u) = u P(u^2) instead, P of degree 4 with the least largest relative error
// (Remez exchange, rounded to fp32: 1e-7).
constexpr float kTanhPoly = 0.5f;
constexpr float kTanh0 = 1.000000000e+00f, kTanh1 = -3.333306909e-01f, kTanh2 = 1.332477927e-01f, kTanh3 = -5.298607424e-02f,
                kTanh4 = 1.713500731e-02f;
__device__ __forceinline__ float capped_log2(float s, float scale_over_cap, float cap_log2e) {
  const float u = s * scale_over_cap, z = u * u;
  if (fabsf(u) < kTanhPoly) {
    const float p = fmaf(fmaf(fmaf(fmaf(kTanh4, z, kTanh3), z, kTanh2), z, kTanh1), z, kTanh0);
    return cap_log2e * u * p;
  }
  const float e = ex2(u * 2.8853900817779268f);                        // exp(2 u)
  return cap_log2e * (1.f - __fdividef(2.f, 1.f + e));
}

// ---------------------------------------------------------------- results that are not finite
// The matrix form multiplies masked values by a weight of zero, which is NaN where such a value (a
// later token's, say) is not finite.  form_again mends a warp's rows that came out so, a lane each.
//
// What a value of such a row is follows from the values that the row sees: NaN beside a NaN or beside both
// infinities, an infinity beside that infinity (each weight is positive), and only where all of them
// are finite it has to be summed again.  Most rows of a sequence with a bad value see it, so the first
// question is asked of all rows together: the keys that all of them see are searched once, from the
// newest (a bad token is mostly followed by bad ones) until NaNs settle every value in question.
// Rows that need the sum are those beside a bad value that they do not see: one or two tiles of a
// sequence for each dim.  One NaN among the first keys of 32 / 8 heads: 0.26 ms for
// 1024 tokens (57 when each row walked its own keys one by one), 3.7 for 8192.  The last of 16000 tokens NaN, 16 / 4
// heads, so that the 63 before it in its tile are summed again: 29 ms.
//
// A row of V or K is D / 8 lanes of 16 bytes; a warp reads 256 / D keys at a time.
struct Kinds {             // bit i: the lane's dim i has a NaN, a plus or a minus infinity
  uint32_t nan = 0, up = 0, down = 0;
};

template <typename T>
__device__ __forceinline__ uint4 load_dims(const T* row, int64_t stride, bool aligned) {
  if (aligned) return *reinterpret_cast<const uint4*>(row);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t lo = *reinterpret_cast<const uint16_t*>(row + (2 * i) * stride);
    const uint16_t hi = *reinterpret_cast<const uint16_t*>(row + (2 * i + 1) * stride);
    w[i] = lo | static_cast<uint32_t>(hi) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void to_dims(const uint4& w, float (&x)[8]) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t bits = static_cast<uint16_t>(words[i >> 1] >> (16 * (i & 1)));
    x[i] = to_float<T>(*reinterpret_cast<const T*>(&bits));
  }
}

// A step is done: waits that stand behind it start over.
__device__ __forceinline__ void take_time(uint64_t* beat) {
  if (beat != nullptr && (threadIdx.x & 31) == 0)
    atomicMax(reinterpret_cast<unsigned long long*>(beat), static_cast<unsigned long long>(global_timer_ns()));
}

// Element offset of key j's row in K or V, or -1 where it reads as zeros.
__device__ __forceinline__ int64_t row_offset(const AttendLaunch& a, const int64_t* stride, int64_t slot) {
  if (slot < 0) return -1;
  if (a.page_size == 1) return slot * stride[0];
  const int64_t page = slot / a.page_size;
  return page * stride[0] + (slot - page * a.page_size) * stride[1];
}

// The values that are not finite in V of keys [from, to), newest first, until `want` of the lane's dims are
// all known to hold a NaN; whole warp, the same in all lanes of a dim.
template <typename T, int D, int R>
__device__ __forceinline__ void find_kinds(const AttendLaunch& a, const AttendTask& t, int from, int to, uint32_t want,
                                           Kinds& k, uint64_t* beat) {
  constexpr int kLanes = D / 8, kSub = 32 / kLanes, kAhead = 4;
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u, kExp2 = kExp | kExp << 16;
  const int lane = threadIdx.x & 31, sub = lane / kLanes;
  const int64_t stride = a.v_stride[3];
  const bool aligned = R > 1 || a.aligned != 0;       // (always in the tcgen05 kernel)
  const T* v = static_cast<const T*>(a.v) + t.head * a.v_stride[2] + (lane % kLanes) * 8 * stride;
  for (int end = to; end > from; end -= 32) {
    if (__all_sync(0xffffffffu, (k.nan & want) == want)) return;
    const int64_t mine = end - 1 - lane >= from ? row_offset(a, a.v_stride, key_slot(a, t.kv_begin, end - 1 - lane)) : -1;
    for (int u = 0; u < kLanes; u += kAhead) {
      uint4 w[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, mine, (u + i) * kSub + sub);
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        if (at >= 0) w[i] = load_dims<T>(v + at, stride, aligned);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        uint32_t bad = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) bad |= __vcmpeq2(words[x] & kExp2, kExp2);
        if (bad == 0) continue;
        for (int x = 0; x < 8; ++x) {
          const uint32_t h = (x < 4 ? (x < 2 ? w[i].x : w[i].y) : (x < 6 ? w[i].z : w[i].w)) >> (16 * (x & 1));
          if ((h & kExp) != kExp) continue;
          if ((h & 0x7fffu) != kExp) k.nan |= 1u << x;
          else if (h & 0x8000u) k.down |= 1u << x;
          else k.up |= 1u << x;
        }
      }
    }
#pragma unroll
    for (int bit = kLanes; bit < 32; bit <<= 1) {
      k.nan |= __shfl_xor_sync(0xffffffffu, k.nan, bit);
      k.up |= __shfl_xor_sync(0xffffffffu, k.up, bit);
      k.down |= __shfl_xor_sync(0xffffffffu, k.down, bit);
    }
    take_time(beat);
  }
}

// The lane's dims of sum_j p_j v_j / sum_j p_j for up to R rows at once, by one warp; row i: token row[i], query
// head head[i], keys [from[i], to[i]) (from >= to: no such row).  p_j = 2^(s_j - e2), e2 the row's log2-sum-exp, so that
// the p_j sum to about one and no partial sum exceeds the largest value.  Rows share the loads, whose latency
// bounds it: four in the tcgen05 kernel, one in the mma.sync kernel, which has no registers for more.
template <typename T, int D, int R>
__device__ __forceinline__ void sum_again(const AttendLaunch& a, const AttendTask& t, const int (&row)[R],
                                          const int (&head)[R], const int (&from)[R], const int (&to)[R],
                                          const float (&e2)[R], float (&acc)[R][8], uint64_t* beat) {
  constexpr int kLanes = D / 8, kSub = 32 / kLanes, kAhead = 4;
  const int lane = threadIdx.x & 31, sub = lane / kLanes, d0 = (lane % kLanes) * 8;
  const int64_t ks = a.k_stride[3], vs = a.v_stride[3];
  const bool aligned = R > 1 || a.aligned != 0;
  float q[R][8], sum[R];
  int first = 0x7fffffff, end = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    sum[i] = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) q[i][x] = acc[i][x] = 0.f;
    if (from[i] >= to[i]) continue;
    first = min(first, from[i]);
    end = max(end, to[i]);
    to_dims<T>(load_dims<T>(static_cast<const T*>(a.q) + static_cast<int64_t>(row[i]) * a.q_stride[0] +
                                static_cast<int64_t>(head[i]) * a.q_stride[1] + d0 * a.q_stride[2], a.q_stride[2], aligned), q[i]);
  }
  const T* k = static_cast<const T*>(a.k) + t.head * a.k_stride[2] + d0 * ks;
  const T* v = static_cast<const T*>(a.v) + t.head * a.v_stride[2] + d0 * vs;
  const float scale = a.scale * 1.4426950408889634f, cap = a.logit_cap, over_cap = cap > 0.f ? a.scale / cap : 0.f;
  for (int j0 = first; j0 < end; j0 += 32) {
    const int64_t slot = j0 + lane < end ? key_slot(a, t.kv_begin, j0 + lane) : -1;
    const int64_t my_k = row_offset(a, a.k_stride, slot), my_v = row_offset(a, a.v_stride, slot);
    for (int u = 0; u < kLanes; u += kAhead) {
      uint4 kw[kAhead], vw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t at_k = __shfl_sync(0xffffffffu, my_k, (u + i) * kSub + sub);
        const int64_t at_v = __shfl_sync(0xffffffffu, my_v, (u + i) * kSub + sub);
        kw[i] = vw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (at_k >= 0) {
          kw[i] = load_dims<T>(k + at_k, ks, aligned);
          vw[i] = load_dims<T>(v + at_v, vs, aligned);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int j = j0 + (u + i) * kSub + sub;
        float kx[8], vx[8], sc[R];
        to_dims<T>(kw[i], kx);
        to_dims<T>(vw[i], vx);
        // (A value that is not finite counts for no row: those that see it do not ask for its dim.)
#pragma unroll
        for (int y = 0; y < 8; ++y) vx[y] = fabsf(vx[y]) <= 3.4028235e38f ? vx[y] : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          sc[r] = 0.f;
#pragma unroll
          for (int y = 0; y < 8; ++y) sc[r] = fmaf(q[r][y], kx[y], sc[r]);
        }
#pragma unroll
        for (int bit = kLanes / 2; bit >= 1; bit >>= 1) {
#pragma unroll
          for (int r = 0; r < R; ++r) sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], bit);
        }
        if (cap > 0.f) {
#pragma unroll
          for (int r = 0; r < R; ++r) sc[r] = capped_log2(sc[r], over_cap, cap * 1.4426950408889634f);
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) sc[r] *= scale;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = ex2(sc[r] - e2[r]), p = j >= from[r] && j < to[r] ? w : 0.f;
          sum[r] += p;
#pragma unroll
          for (int y = 0; y < 8; ++y) acc[r][y] = fmaf(p, vx[y], acc[r][y]);
        }
      }
    }
    take_time(beat);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int bit = kLanes; bit < 32; bit <<= 1) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], bit);
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[r][x] += __shfl_xor_sync(0xffffffffu, acc[r][x], bit);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) acc[r][x] /= sum[r];
  }
}

// `odd`: the lanes whose row (token `row`, query head `head`, log2-sum-exp `e2`) has a stored result that is not finite.
// `beat` (shared memory, or nullptr): the time of the last step, for waits that stand behind this one.
template <typename T, int D, int R>
__device__ __noinline__ void form_again(const AttendLaunch& a, const AttendTask& t, uint32_t odd, int row, int head, float e2,
                                        uint64_t* beat) {
  constexpr int kLanes = D / 8;
  const int lane = threadIdx.x & 31, d0 = (lane % kLanes) * 8;
  __syncwarp();                 // other lanes stored pieces of these rows: their stores come first
  // (A sum that is not finite comes from a score that is NaN, and with it the whole row stays so.)
  odd = __ballot_sync(0xffffffffu, (odd >> lane & 1u) != 0 && (e2 == -INFINITY || fabsf(e2) <= 3.4028235e38f));
  const bool mine = (odd >> lane & 1u) != 0 && e2 != -INFINITY;
  const auto bad_dims = [&](int64_t at_row, int at_head) -> uint32_t {   // of a row's stored result
    const int64_t at = at_row * a.query_heads + at_head;
    uint32_t bad = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const float y = a.partial != nullptr
                          ? a.partial[(at * a.splits + t.split) * D + d0 + x]
                          : to_float<T>(static_cast<const T*>(a.out)[at_row * a.out_stride[0] + at_head * a.out_stride[1] +
                                                                     (d0 + x) * a.out_stride[2]]);
      bad |= (fabsf(y) <= 3.4028235e38f ? 0u : 1u) << x;
    }
    return bad;
  };
  // The keys that all of these rows see, and the dims that any of them asks for.
  int from = __reduce_max_sync(0xffffffffu, mine ? first_key(a, t, row) : 0);
  int to = __reduce_min_sync(0xffffffffu, mine ? last_key(a, t, row) + 1 : 0x7fffffff);
  if (from >= to) from = to = t.lo;                   // (none: each row looks through its own)
  uint32_t any = 0;
  for (uint32_t rest = odd; rest != 0; rest &= rest - 1) {
    const int who = __ffs(rest) - 1;
    any |= bad_dims(__shfl_sync(0xffffffffu, row, who), __shfl_sync(0xffffffffu, head, who));
  }
  Kinds common;
  bool searched = false;
  while (odd != 0) {
    int rows[R], heads[R], lo[R], hi[R];
    float e[R], acc[R][8] = {};
    uint32_t want[R];
    Kinds k[R];
    bool sum = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      want[i] = 0;
      lo[i] = hi[i] = rows[i] = heads[i] = 0;
      e[i] = 0.f;
      if (odd == 0) continue;
      const int who = __ffs(odd) - 1;
      odd &= odd - 1;
      rows[i] = __shfl_sync(0xffffffffu, row, who);
      heads[i] = __shfl_sync(0xffffffffu, head, who);
      e[i] = __shfl_sync(0xffffffffu, e2, who);
      want[i] = bad_dims(rows[i], heads[i]);
      if (e[i] == -INFINITY) continue;                // a row without a weight is zero
      if (!searched) find_kinds<T, D, R>(a, t, from, to, any, common, beat);
      searched = true;
      k[i] = common;
      lo[i] = first_key(a, t, rows[i]);
      hi[i] = last_key(a, t, rows[i]) + 1;
      if (from < to) {
        find_kinds<T, D, R>(a, t, lo[i], from, want[i], k[i], beat);
        find_kinds<T, D, R>(a, t, to, hi[i], want[i], k[i], beat);
      } else {
        find_kinds<T, D, R>(a, t, lo[i], hi[i], want[i], k[i], beat);
      }
      if (__any_sync(0xffffffffu, (want[i] & ~(k[i].nan | k[i].up | k[i].down)) != 0)) sum = true;
      else hi[i] = lo[i];
    }
    if (sum) sum_again<T, D, R>(a, t, rows, heads, lo, hi, e, acc, beat);
    if (lane >= kLanes) continue;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t at = static_cast<int64_t>(rows[i]) * a.query_heads + heads[i];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint32_t bit = 1u << x;
        if (!(want[i] & bit)) continue;
        const float y = e[i] == -INFINITY ? 0.f
                        : (k[i].nan & bit) || ((k[i].up & bit) && (k[i].down & bit)) ? __int_as_float(0x7fc00000)
                        : (k[i].up & bit) ? INFINITY : (k[i].down & bit) ? -INFINITY : acc[i][x];
        if (a.partial != nullptr) {
          a.partial[(at * a.splits + t.split) * D + d0 + x] = y;
        } else {
          static_cast<T*>(a.out)[static_cast<int64_t>(rows[i]) * a.out_stride[0] + static_cast<int64_t>(heads[i]) * a.out_stride[1] +
                                 (d0 + x) * a.out_stride[2]] = from_float<T>(y);
        }
      }
    }
  }
}

}  // namespace sgld
