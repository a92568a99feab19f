// Attention of packed query rows over long keys on the 5th-generation tensor cores: head_dim 64
// and 128, 16-byte aligned rows.  (Other layouts: sgld_attend.cu, which states the formula.)
//
// One persistent CTA per SM.  A task gives it two tiles of 128 query rows (rows are packed as
// token x query head of one KV head) and a run of keys, walked in blocks of 128:
//
//   loaders (3 warps)   find the tasks, copy Q once and K, V block by block into a ring of
//                       shared tiles: TMA boxes where the keys are consecutive rows (packed keys,
//                       pages), else row by row (cache slots; the last block of a run).
//   MMA issuer (1 warp) S = Q K^T (128 x 128 x D) into tensor memory, and one block later
//                       O += P V with P read from tensor memory, the two tiles in turn: while one
//                       tile's scores are in its softmax, the tensor cores work on the other's.
//   softmax (2 x 4 warps, one group a tile)  a thread owns one row: it loads the 128 scores of its
//                       row, takes their maximum, writes p = 2^(s - m) back over them as 16-bit
//                       pairs and keeps the row's sum; no value crosses lanes.  m moves only when
//                       a block exceeds it by 2^8 (p stays in range): the thread then
//                       scales its row of O in tensor memory, which the pipeline allows because
//                       S of this block is issued after O of the last.  At the task's end it
//                       divides its row of O by the sum and stores it.
//
// Bounds: a pair of blocks costs 4 x 128 x 128 x D multiply-adds on the tensor cores (2048
// cycles at D = 128) and 2 x 128 x 128 exponentials on the special function units (2048 cycles at
// 16 a cycle), so the two run at the same pace and overlap; K and V come through L2.  Measured: 3550
// cycles, a tile's chain of softmax (2000) and P V, Q K and their latencies (1280) with two tiles in
// flight, which is what tensor memory holds (S 2 x 128 + O 2 x 128 columns): two causal prompts of
// 8K tokens, 32 / 8 heads, D 128: 1003-1048 us with the power cap's clock, 1.03-1.07 PFLOP/s.
//
// Precision: scores, maxima, sums and O are fp32; p is rounded to 16 bits for the second product
// (its operand type), the sum keeps the fp32 values.
//
// Every wait is bounded (4 s); a role whose wait expires sets a status bit and makes the others' waits
// expire, the copies and MMAs in flight are awaited, the rows of all tasks that the CTA had taken and
// may not have stored are set to NaN (give_up), and tensor memory is freed on every path.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "sgld_attend.cuh"
#include "sgld_internal.cuh"
#include "sgld_ptx.cuh"

namespace sgld {
namespace {

constexpr uint64_t kDrainLimitNs = 4000000000ull;   // of the waits for a CTA's own copies and MMAs at its end
constexpr uint64_t kFailed = ~0ull;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleLog2 = 8.f;
constexpr int kRows = 128;                 // rows of a tile (MMA M) and keys of a block (MMA N)
constexpr int kMmaWarp = 0, kLoaderWarp = 1, kLoaders = 3, kSoftmaxWarp = 4, kWarps = 12, kThreads = kWarps * 32;
constexpr int kTaskRing = 4;
// Tasks that a CTA has taken and may not have stored: the one that the slowest softmax warp is at, the ring's,
// one found and not published, one claimed.
constexpr int kTaken = 8;
static_assert(kTaken >= kTaskRing + 3, "tasks not stored are among the last taken");
constexpr int kTmemCols = 512;             // S at 0 and 128 (P over S), O at 256 and 256 + D
constexpr uint32_t kTmem = 0;              // all of tensor memory is allocated: it starts at column 0
// Registers a thread: 384 x 168 at launch; the softmax groups take 208, the others keep 88.
constexpr int kRegsSoftmax = 208, kRegsOther = 88;

template <int D>
struct Layout {
  static constexpr int kTile = kRows * D * 2;            // one Q, K or V tile
  static constexpr int kStages = D == 128 ? 5 : 10;      // K and V tiles in the ring
  static constexpr int kOffRing = 2 * kTile;
  static constexpr int kOffMisc = kOffRing + kStages * kTile;
  static constexpr int kBytes = kOffMisc + 1024 + 1024;  // misc, and slack to align the base to 1 KB
};

// What a wait looks at once it does not succeed at once.
struct alignas(16) Clock {
  uint64_t beat;               // time of form_again's last step: waits behind it go on; kFailed: all expire
  uint64_t limit;              // ns since `beat` and since the wait began
};

struct Misc {
  uint64_t kv_full[10], kv_empty[10];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_ready[2][2], o_full[2], o_free[2];   // p_ready: [tile][half of the keys]
  uint64_t tfull[kTaskRing], tempty[kTaskRing];
  uint64_t drain;
  uint64_t claimed;
  alignas(16) uint64_t claim[2];
  AttendTask task[kTaskRing];
  uint32_t tmem_base;
  Clock clock, drain_clock;
  int64_t issued[kLoaders];    // ring tiles that each loader has arrived for, at its end
  uint32_t taken[kTaken], n_taken, lost;   // the last tasks taken; lost: a claim without an answer
};
static_assert(sizeof(Misc) <= 1024, "misc area too small");
static_assert(Layout<128>::kBytes <= 232448 && Layout<64>::kBytes <= 232448, "shared memory budget exceeded");

enum : int { kStatusWait = 1 };

// A wait expires when clock.limit has passed since it began and since the last step of form_again in this
// CTA (with bad values in a long sequence those steps can take longer, and end by themselves), or when
// another has expired.  One block of assembly: as C++ the compiler lays the loop out between the
// instructions of the roles' own loops, and the kernel is 3 to 12% slower for it (the forms differed,
// the work did not).
__device__ __forceinline__ bool bounded_wait(const Clock& clock, uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 start, now, beat, limit;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 start, %%globaltimer;\n\t"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "ld.volatile.shared::cta.v2.u64 {beat, limit}, [%3];\n\t"
      "mov.u64 now, %%globaltimer;\n\t"
      "max.u64 beat, beat, start;\n\t"          // kFailed: now - beat wraps to now + 1
      "sub.u64 now, now, beat;\n\t"
      "setp.lt.u64 q, now, limit;\n\t"
      "@q bra AGAIN;\n\t"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity), "r"(smem_addr(&clock))
      : "memory");
  return ok != 0;
}

// Bounded wait of a whole warp, which it reconverges.
__device__ __forceinline__ bool warp_wait(Misc& ms, uint64_t* bar, uint32_t parity, int* status) {
  const bool ok = __all_sync(0xffffffffu, bounded_wait(ms.clock, bar, parity));
  if (!ok && (threadIdx.x & 31) == 0) {
    atomicMax(reinterpret_cast<unsigned long long*>(&ms.clock.beat), static_cast<unsigned long long>(kFailed));
    if (status != nullptr) atomicOr(status, kStatusWait);
  }
  return ok;
}

// The same at a role's end, for what the CTA itself has in flight, also after a failure.
__device__ __forceinline__ bool drain_wait(Misc& ms, uint64_t* bar, uint32_t parity, int* status) {
  const bool ok = __all_sync(0xffffffffu, bounded_wait(ms.drain_clock, bar, parity));
  if (!ok && status != nullptr && (threadIdx.x & 31) == 0) atomicOr(status, kStatusWait);
  return ok;
}

// A counter into a ring of n barriers and its phase.
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++i == n) {
      i = 0;
      phase ^= 1u;
    }
  }
};

// Blocks of 128 keys of each tile of a task (tile 1 is empty when the task has one tile).
__device__ __forceinline__ void tile_blocks(const AttendLaunch& a, const AttendTask& t, int tokens, int (&n)[2]) {
  const int hi0 = a.causal ? min(t.hi, min(t.first + tokens, t.last) + t.shift) : t.hi;
  n[0] = max(0, hi0 - t.lo + kRows - 1) / kRows;
  n[1] = t.first + tokens < t.last ? max(0, t.hi - t.lo + kRows - 1) / kRows : 0;
}

template <typename T, int D, bool kCap>
struct Attend {
  using L = Layout<D>;
  static constexpr int kHalf = kRows * 128;        // bytes of one 64-dim half of a tile
  static constexpr float kBias = WeightBias<T>::value;

  // ------------------------------------------------------------------ loaders (3 warps)
  // A block's K and V come by TMA boxes, which loader 0 issues, or row by row: an index per row
  // (cache slots), or the last block of a run, whose missing rows are zeros.  Rows are copied with
  // 16-byte cp.async by all three: four gathered rows a TMA copy (tile::gather4) measured 2.2 times
  // slower, at some 50 cycles a copy.
  static constexpr int kRowLanes = D / 8;               // lanes of a row
  static constexpr int kRowsPerCopy = 32 / kRowLanes;
  static constexpr int kCopies = kRows / kRowsPerCopy;  // of a tile; loader w issues w, w + 3, ...
  static constexpr int kMine = (kCopies + kLoaders - 1) / kLoaders;
  static constexpr int kHeld = 32 / kRowsPerCopy;       // copies whose rows one register of the lanes holds
  static_assert(kMine <= 2 * kHeld, "two registers hold the rows of a tile");

  // The pool rows of the block at key j that this lane holds (of copies w + 3 l: lane 's row of the
  // first kHeld in slot[0], of the others in slot[1]), or the first row of box `lane` in slot[0]; values
  // outside [0, kv_extent) read as zeros.  Looked up one block ahead and not looked at here, so that
  // the loads are in flight during the copies of this block.
  __device__ static void look_up(const AttendLaunch& a, const AttendTask& t, int w, int j, int (&slot)[2], int& boxes) {
    const int lane = threadIdx.x & 31;
    boxes = a.box_rows > 0 && j + kRows <= t.hi && (a.kv_indices == nullptr || (t.kv_begin + j) % a.box_rows == 0)
                ? kRows / a.box_rows : 0;
    slot[0] = slot[1] = -1;
    if (boxes > 0) {
      if (lane < boxes) slot[0] = static_cast<int>(key_slot(a, t.kv_begin, j + lane * a.box_rows));
      return;
    }
    const int left = min(kRows, t.hi - j);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = (w + kLoaders * (u * kHeld + lane / kRowsPerCopy)) * kRowsPerCopy + lane % kRowsPerCopy;
      if (r < left)
        slot[u] = a.kv_indices != nullptr && a.page_size == 1 ? __ldg(a.kv_indices + t.kv_begin + j + r)
                                                              : static_cast<int>(key_slot(a, t.kv_begin, j + r));
    }
  }

  // One tile by boxes: loader 0 announces its bytes and issues the copies; every thread arrives.
  __device__ static void load_boxes(const CUtensorMap* box, int w, int boxes, int box_rows, int slot, int col, int base,
                                    int map_rows, uint32_t dst, uint64_t* full) {
    const int lane = threadIdx.x & 31;
    if (w == 0 && lane == 0) mbar_arrive_expect_tx(full, L::kTile);
    else mbar_arrive(full);
    __syncwarp();
    if (w != 0) return;
    for (int i = 0; i < boxes; ++i) {
      const int s = __shfl_sync(0xffffffffu, slot, i), r = s >= 0 ? base + s : map_rows;   // past the map: zeros
      if (lane == 0) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * kHalf + i * box_rows * 128, box, col + c * 64, r, full);
      }
    }
    __syncwarp();
  }

  // This loader's rows of one tile; each thread arrives when its own copies have landed.  `at`: the held
  // rows' offsets from `head` in 16-byte units, all ones where a row reads as zeros; `whole`: none
  // does.  Four instructions a copy: the loaders share their issue slots with the softmax.
  __device__ static void load_rows(const T* head, int w, const uint32_t (&at)[2], bool whole, uint32_t dst, uint64_t* full) {
    const int lane = threadIdx.x & 31, c = lane % kRowLanes, sub = lane / kRowLanes;
    const uint4* src = reinterpret_cast<const uint4*>(head) + c;
    // Rows of copies 4 apart share their place in the swizzle.
    uint32_t d[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = (w + kLoaders * k) * kRowsPerCopy + sub;
      d[k] = dst + (c >> 3) * kHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    }
    constexpr int kFour = 4 * kLoaders * kRowsPerCopy * 128;
    static_assert((4 * kLoaders * kRowsPerCopy) % 8 == 0, "four copies on, the swizzle repeats");
    if (whole) {
#pragma unroll
      for (int l = 0; l < kMine; ++l) {
        const uint32_t x = __shfl_sync(0xffffffffu, at[l / kHeld], (l % kHeld) * kRowsPerCopy + sub);
        if ((l + 1) * kLoaders <= kCopies || w + l * kLoaders < kCopies) cp_async_16(d[l & 3] + (l >> 2) * kFour, src + x);
      }
    } else {
#pragma unroll
      for (int l = 0; l < kMine; ++l) {
        const uint32_t x = __shfl_sync(0xffffffffu, at[l / kHeld], (l % kHeld) * kRowsPerCopy + sub);
        const bool in = x != 0xffffffffu;
        if ((l + 1) * kLoaders <= kCopies || w + l * kLoaders < kCopies)
          cp_async_16_fill(d[l & 3] + (l >> 2) * kFour, in ? src + x : src, in ? 16u : 0u);
      }
    }
    cp_async_arrive_noinc(full);
  }

  // Ask the hardware for the next block of the grid that has not been launched: this CTA runs it as its
  // next task instead.
  __device__ static void claim_task(Misc& ms, int& asked) {
    ++asked;
    if ((threadIdx.x & 31) == 0) {
      fence_proxy_async_smem();                 // the last answer has been read
      mbar_arrive_expect_tx(&ms.claimed, 16);
      asm volatile(
          "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
              smem_addr(ms.claim)),
          "r"(smem_addr(&ms.claimed))
          : "memory");
    }
    __syncwarp();
  }
  // The answer: the block's number, or -1 when none is left.
  __device__ static int64_t answer(Misc& ms) {
    const volatile uint64_t* r = ms.claim;
    const uint64_t lo = r[0], hi = r[1];
    uint32_t given, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 c;\n\tmov.b128 c, {%2, %3};\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, c;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, c;\n\t}"
        : "=r"(given), "=r"(x)
        : "l"(lo), "l"(hi));
    __syncwarp();
    return given != 0 ? static_cast<int64_t>(x) : -1;
  }
  __device__ static bool next_task(Misc& ms, int& asked, uint32_t& phase, int64_t& task, int* status) {
    if (!warp_wait(ms, &ms.claimed, phase, status)) return false;
    --asked;
    phase ^= 1u;
    task = answer(ms);
    return true;
  }
  __device__ static void note_task(Misc& ms, int64_t task) {
    if ((threadIdx.x & 31) == 0) ms.taken[ms.n_taken++ % kTaken] = static_cast<uint32_t>(task);
  }

  // Tasks (loader 0) and copies until the last task; `issued` counts the ring tiles, `q_issued`
  // the Q loads, `asked` a claim without its answer.
  __device__ static void load_tasks(const AttendLaunch& a, unsigned char* smem, Misc& ms, int w, int64_t& issued,
                                    int64_t& q_issued, int& asked, uint32_t& cph) {
    const int lane = threadIdx.x & 31;
    int* status = a.status;
    const int tokens = kRows / a.group;                     // of one tile
    const uint32_t q_bytes = static_cast<uint32_t>(tokens * a.group * D * 2);
    Ring kv, tr;
    uint32_t qph = 0;
    int chunk = 0;
    int64_t before = 0;
    int64_t task = blockIdx.x;
    while (true) {
      AttendTask t;
      if (w == 0) {
        t.valid = 0;
        if (task >= 0) t = find_task(a, 2 * tokens, kRows, static_cast<uint32_t>(task), chunk, before);
        // Blocks past the last task wait to be launched: take them all, which is quicker.
        while (!t.valid && task >= 0) {
          claim_task(ms, asked);
          if (!next_task(ms, asked, cph, task, status)) return;
        }
        if (t.valid) note_task(ms, task);
        if (!warp_wait(ms, &ms.tempty[tr.i], tr.phase ^ 1u, status)) return;
        if (lane == 0) {
          ms.task[tr.i] = t;
          mbar_arrive(&ms.tfull[tr.i]);
        }
      } else {
        if (!warp_wait(ms, &ms.tfull[tr.i], tr.phase, status)) return;
        t = ms.task[tr.i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&ms.tempty[tr.i]);
      }
      tr.next(kTaskRing);
      if (!t.valid) return;
      int n[2];
      tile_blocks(a, t, tokens, n);
      const int blocks = max(n[0], n[1]);
      if (blocks == 0) {
        if (w == 0) {
          claim_task(ms, asked);
          if (!next_task(ms, asked, cph, task, status)) return;
        }
        continue;
      }
      int slot[2], next[2], boxes, next_boxes = 0;
      look_up(a, t, w, t.lo, slot, boxes);
      for (int b = 0; b < blocks; ++b) {
        if (b == blocks - 1 && w == 0) claim_task(ms, asked);      // late: the SM that is done first takes the next
        if (b + 1 < blocks) look_up(a, t, w, t.lo + (b + 1) * kRows, next, next_boxes);   // in flight during the waits
        if (b == 0 && w == 0) {                             // Q right before the first K
          if (!warp_wait(ms, &ms.q_empty, qph ^ 1u, status)) return;
          qph ^= 1u;
          if (lane == 0) {
            const int tiles = t.first + tokens < t.last ? 2 : 1;
            mbar_arrive_expect_tx(&ms.q_full, q_bytes * tiles);
            for (int g = 0; g < tiles; ++g)
              for (int c = 0; c < D / 64; ++c)
                tma_load_3d(smem_addr(smem) + g * L::kTile + c * kHalf, &a.qmap, c * 64, t.head * a.group,
                            t.first + g * tokens, &ms.q_full);
          }
          ++q_issued;
          __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {                       // K, then V
          if (!warp_wait(ms, &ms.kv_empty[kv.i], kv.phase ^ 1u, status)) return;
          ++issued;
          const uint32_t dst = smem_addr(smem + L::kOffRing + kv.i * L::kTile);
          if (boxes > 0) {
            load_boxes(x == 0 ? &a.kmap : &a.vmap, w, boxes, a.box_rows, slot[0],
                       t.head * (x == 0 ? a.k_head_col : a.v_head_col), t.head * (x == 0 ? a.k_head_row : a.v_head_row),
                       x == 0 ? a.map_rows_k : a.map_rows_v, dst, &ms.kv_full[kv.i]);
          } else {
            const int64_t* st = x == 0 ? a.k_stride : a.v_stride;
            const uint32_t pitch = static_cast<uint32_t>((a.page_size > 1 ? st[1] : st[0]) / 8);
            uint32_t at[2];
            bool whole = true;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const bool in = static_cast<uint32_t>(slot[u]) < static_cast<uint32_t>(a.kv_extent);
              at[u] = in ? static_cast<uint32_t>(slot[u]) * pitch : 0xffffffffu;
              whole = whole && (in || u * kHeld + lane / kRowsPerCopy >= kMine ||
                                w + kLoaders * (u * kHeld + lane / kRowsPerCopy) >= kCopies);
            }
            load_rows(static_cast<const T*>(x == 0 ? a.k : a.v) + t.head * st[2], w, at, __all_sync(0xffffffffu, whole), dst,
                      &ms.kv_full[kv.i]);
          }
          kv.next(L::kStages);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) slot[u] = next[u];
        boxes = next_boxes;
      }
      if (w == 0 && !next_task(ms, asked, cph, task, status)) return;
    }
  }

  // The copies in flight land before the CTA ends, also where another role gave up.
  __device__ static void loader(const AttendLaunch& a, unsigned char* smem, Misc& ms, int w) {
    int64_t issued = 0, q_issued = 0;
    int asked = 0;
    uint32_t cph = 0;
    load_tasks(a, smem, ms, w, issued, q_issued, asked, cph);
    const int lane = threadIdx.x & 31;
    if (asked > 0) {
      const bool ok = drain_wait(ms, &ms.claimed, cph, a.status);
      const int64_t task = ok ? answer(ms) : -1;
      if (task >= 0) note_task(ms, task);
      if (!ok && lane == 0) ms.lost = 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // A loader whose wait expired may have left before the others: it arrives for the tiles that they
    // have issued (fewer than the ring holds, as a stage is filled again only after all arrived for it).
    if (lane == 0) ms.issued[w] = issued;
    asm volatile("bar.sync 1, %0;" ::"n"(kLoaders * 32) : "memory");
    int64_t most = 0;
    for (int i = 0; i < kLoaders; ++i) most = max(most, ms.issued[i]);
    for (int64_t i = issued; i < most; ++i) mbar_arrive(&ms.kv_full[i % L::kStages]);
    __syncwarp();
    for (int i = 0; i < L::kStages && i < most; ++i) {
      const int64_t last = most - 1 - (most - 1 - i) % L::kStages;          // the last tile put into stage i
      drain_wait(ms, &ms.kv_full[i], static_cast<uint32_t>(last / L::kStages) & 1u, a.status);
    }
    if (q_issued > 0) drain_wait(ms, &ms.q_full, static_cast<uint32_t>(q_issued - 1) & 1u, a.status);
  }

  // ------------------------------------------------------------------ MMA issuer (1 warp)
  // The whole warp walks the tasks and lane 0 issues: code that one lane alone runs cannot keep
  // the descriptors in uniform registers, and moving them there for each MMA made the issue itself
  // the bound (90 to 160 cycles an MMA, which takes 64).
  __device__ static void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 lane;\n\tmov.u32 lane, %%laneid;\n\tsetp.eq.u32 q, lane, 0;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  }
  __device__ static void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 lane;\n\tmov.u32 lane, %%laneid;\n\tsetp.eq.u32 q, lane, 0;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
  }
  __device__ static void commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .u32 lane;\n\tmov.u32 lane, %%laneid;\n\tsetp.eq.u32 q, lane, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
        : "memory");
  }

  // `q` and `k` / `v`: descriptors of the tile's first step; later steps add to the address field.
  __device__ static void issue_qk(uint64_t q, uint64_t k, int g) {
    constexpr uint32_t bf = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc = mma_idesc(bf, 0u, 0u, kRows, kRows);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const uint32_t step = ((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
      mma_ss(kTmem + g * kRows, q + (g * (L::kTile >> 4) + step), k + step, idesc, ks > 0 ? 1u : 0u);
    }
  }

  // Keys 64 h .. 64 h + 63 of the block.
  __device__ static void issue_pv(uint64_t v, int g, int h, uint32_t first) {
    constexpr uint32_t bf = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc = mma_idesc(bf, 0u, 1u, D, kRows);
#pragma unroll
    for (int i = 0; i < kRows / 32; ++i) {
      const int ks = h * (kRows / 32) + i;
      mma_ts(kTmem + 256 + g * D, kTmem + g * kRows + ks * 8, v + ((ks * 2048) >> 4), idesc, ks == 0 ? first ^ 1u : 1u);
    }
  }

  // Every MMA and its commits have completed when this returns: the barriers and tensor memory
  // that they touch are given up after it.
  __device__ static void mma_issuer(const AttendLaunch& a, unsigned char* smem, Misc& ms) {
    mma_tasks(a, smem, ms);
    __syncwarp();
    commit(&ms.drain);
    drain_wait(ms, &ms.drain, 0, a.status);
  }

  __device__ static void mma_tasks(const AttendLaunch& a, unsigned char* smem, Misc& ms) {
    const int lane = threadIdx.x & 31;
    int* status = a.status;
    const int tokens = kRows / a.group;
    const uint64_t qdesc = smem_desc(smem_addr(smem), 16, 1024, 2);
    const uint64_t kdesc = smem_desc(smem_addr(smem + L::kOffRing), 16, 1024, 2);
    const uint64_t vdesc = smem_desc(smem_addr(smem + L::kOffRing), kHalf, 1024, 2);
    Ring kv, tr;
    uint32_t qph = 0, pph[2] = {0, 0}, oph[2] = {1, 1};
    for (int done = 0; done != a.stall; ++done) {
      if (!warp_wait(ms, &ms.tfull[tr.i], tr.phase, status)) return;
      const AttendTask t = ms.task[tr.i];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ms.tempty[tr.i]);
      tr.next(kTaskRing);
      if (__shfl_sync(0xffffffffu, t.valid, 0) == 0) return;
      int n[2];
      tile_blocks(a, t, tokens, n);
      n[0] = __shfl_sync(0xffffffffu, n[0], 0);
      n[1] = __shfl_sync(0xffffffffu, n[1], 0);
      const int blocks = max(n[0], n[1]);
      if (blocks == 0) continue;
      if (!warp_wait(ms, &ms.q_full, qph, status) || !warp_wait(ms, &ms.kv_full[kv.i], kv.phase, status)) return;
      qph ^= 1u;
      fence_proxy_async_smem();               // row copies arrive through the generic proxy
      tc_fence_after();
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (n[g] > 0) {
          issue_qk(qdesc, kdesc + kv.i * (L::kTile >> 4), g);
          commit(&ms.s_full[g]);
        }
      }
      commit(&ms.kv_empty[kv.i]);
      kv.next(L::kStages);
      if (blocks == 1) commit(&ms.q_empty);
      for (int b = 0; b < blocks; ++b) {
        const Ring v = kv;                    // V of this block, then K of the next
        kv.next(L::kStages);
        if (!warp_wait(ms, &ms.kv_full[v.i], v.phase, status)) return;
        if (b + 1 < blocks && !warp_wait(ms, &ms.kv_full[kv.i], kv.phase, status)) return;
        fence_proxy_async_smem();
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (b < n[g]) {
            if (b == 0) {
              if (!warp_wait(ms, &ms.o_free[g], oph[g], status)) return;
              oph[g] ^= 1u;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!warp_wait(ms, &ms.p_ready[g][h], pph[g], status)) return;
              tc_fence_after();
              issue_pv(vdesc + v.i * (L::kTile >> 4), g, h, b == 0 ? 1u : 0u);
            }
            pph[g] ^= 1u;
            if (b == n[g] - 1) commit(&ms.o_full[g]);
          }
          if (b + 1 < n[g]) {
            issue_qk(qdesc, kdesc + kv.i * (L::kTile >> 4), g);
            commit(&ms.s_full[g]);
          }
        }
        commit(&ms.kv_empty[v.i]);
        if (b + 1 < blocks) {
          commit(&ms.kv_empty[kv.i]);
          kv.next(L::kStages);
          if (b + 2 == blocks) commit(&ms.q_empty);
        }
      }
    }
  }

  // ------------------------------------------------------------------ softmax (one thread a row)
  // The four lanes of a quad exchange 16-byte pieces: lane i comes with pieces 0..3 of row i and
  // leaves with piece i of rows 0..3, so that a quad's store covers 64 consecutive bytes.
  __device__ static void quad_transpose(uint4 (&x)[4]) {
    const int i = threadIdx.x & 3;
#pragma unroll
    for (int bit = 1; bit <= 2; bit <<= 1) {
      const bool up = (i & bit) != 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k & bit) continue;
        uint4& lo = x[k];
        uint4& hi = x[k | bit];
        uint4 send = up ? lo : hi;
        send.x = __shfl_xor_sync(0xffffffffu, send.x, bit);
        send.y = __shfl_xor_sync(0xffffffffu, send.y, bit);
        send.z = __shfl_xor_sync(0xffffffffu, send.z, bit);
        send.w = __shfl_xor_sync(0xffffffffu, send.w, bit);
        if (up) lo = send;
        else hi = send;
      }
    }
  }

  // 32 columns (from d0) of the warp's rows, scaled by inv, to the output or the partials; `row`: the four
  // rows of the lane's quad there (nullptr: not stored).  `check` turns NaN where a value is not finite.
  __device__ static void store_rows(const AttendLaunch& a, unsigned char* const (&row)[4], int d0, const uint32_t (&o)[32],
                                    float inv, float& check) {
    const int lane = threadIdx.x & 31;
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      x[i] = __uint_as_float(o[i]) * inv;
      check = fmaf(x[i], 0.f, check);
    }
    if (a.partial != nullptr) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p[i] = make_uint4(__float_as_uint(x[16 * h + 4 * i]), __float_as_uint(x[16 * h + 4 * i + 1]),
                            __float_as_uint(x[16 * h + 4 * i + 2]), __float_as_uint(x[16 * h + 4 * i + 3]));
        quad_transpose(p);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (row[k] != nullptr) *reinterpret_cast<uint4*>(row[k] + d0 * 4 + h * 64 + (lane & 3) * 16) = p[k];
      }
    } else {
      uint4 p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = make_uint4(Mma<T>::pack(x[8 * i], x[8 * i + 1]), Mma<T>::pack(x[8 * i + 2], x[8 * i + 3]),
                          Mma<T>::pack(x[8 * i + 4], x[8 * i + 5]), Mma<T>::pack(x[8 * i + 6], x[8 * i + 7]));
      quad_transpose(p);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (row[k] != nullptr) *reinterpret_cast<uint4*>(row[k] + d0 * 2 + (lane & 3) * 16) = p[k];
    }
  }

  // A row's scores to their soft-capped values in log2 units (capped_log2).  Where all of a warp's
  // arguments are small, the common case, the polynomial alone: FMA units, two scores an
  // instruction, instead of two special function values a score.
  __device__ static void cap_scores(uint32_t (&s)[4][32], float over_cap, float cap_log2e) {
    float largest = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) largest = fmaxf(largest, fabsf(__uint_as_float(s[i >> 5][i & 31])));
    if (__all_sync(0xffffffffu, largest * over_cap < kTanhPoly)) {     // (a NaN stays one either way)
      const uint64_t in = pair(over_cap, over_cap), out = pair(cap_log2e, cap_log2e);
#pragma unroll
      for (int i = 0; i < kRows; i += 2) {
        const uint64_t u = mul2(pair(s[i >> 5][i & 31], s[i >> 5][(i & 31) + 1]), in), z = mul2(u, u);
        uint64_t p = fma2(pair(kTanh4, kTanh4), z, pair(kTanh3, kTanh3));
        p = fma2(p, z, pair(kTanh2, kTanh2));
        p = fma2(p, z, pair(kTanh1, kTanh1));
        p = fma2(p, z, pair(kTanh0, kTanh0));
        unpair(mul2(mul2(u, out), p), s[i >> 5][i & 31], s[i >> 5][(i & 31) + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const float u = __uint_as_float(s[i >> 5][i & 31]) * over_cap, z = u * u;
        const float p = fmaf(fmaf(fmaf(fmaf(kTanh4, z, kTanh3), z, kTanh2), z, kTanh1), z, kTanh0) * u;
        float d;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(1.f + ex2(u * 2.8853900817779268f)));
        s[i >> 5][i & 31] = __float_as_uint(cap_log2e * (fabsf(u) < kTanhPoly ? p : fmaf(-2.f, d, 1.f)));
      }
    }
  }

  __device__ static void signal(uint64_t* bar) {
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  }
  // The values are computed before what follows.
  __device__ static void keep(uint32_t (&p)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) asm volatile("" : "+r"(p[i]), "+r"(p[i + 1]), "+r"(p[i + 2]), "+r"(p[i + 3]));
  }

  // p = 2^(s c - ref) of 32 scores as 16-bit pairs, and their sum onto `sum`.  All on the special
  // function units: a quarter of them as polynomials on the FMA units, which cost 12 cycles a
  // value there against 8, made the kernel 8% slower.
  __device__ static void weights(const uint32_t (&s)[32], uint64_t c2, uint64_t r2, uint32_t (&p)[16], uint64_t (&sum)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      uint32_t x0, x1;
      unpair(fma2(pair(s[2 * i], s[2 * i + 1]), c2, r2), x0, x1);
      const float e0 = ex2(__uint_as_float(x0)), e1 = ex2(__uint_as_float(x1));
      sum[i & 1] = add2(sum[i & 1], pair(e0, e1));
      p[i] = Mma<T>::pack(e0, e1);
    }
  }

  __device__ static float largest(const uint32_t (&s)[32]) {
    float t[2] = {fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])), fmaxf(__uint_as_float(s[2]), __uint_as_float(s[3]))};
#pragma unroll
    for (int i = 4; i < 32; i += 4) {
      t[0] = fmaxf(fmaxf(t[0], __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
      t[1] = fmaxf(fmaxf(t[1], __uint_as_float(s[i + 2])), __uint_as_float(s[i + 3]));
    }
    return fmaxf(t[0], t[1]);
  }

  // Scale this thread's row of O, and its sum, to the reference maximum `to`.  O holds all
  // earlier blocks: the commit of the scores covers every MMA issued before them.
  __device__ static void rescale(uint32_t o_addr, float to, float& m, float& l) {
    const float w = to == -INFINITY ? 1.f : ex2(m - to);
    m = to;
    l *= w;
#pragma unroll 1
    for (int q = 0; q < D / 32; ++q) {
      uint32_t o[32];
      tmem_ld32(o_addr + q * 32, o);
      tmem_wait32(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w);
      tmem_st32_nowait(o_addr + q * 32, o);
    }
  }

  // One block of a row whose scores are all seen, with the reference m of the blocks before: the
  // weights are formed while the maximum is found, which the special function units leave room
  // for, and the first half is signalled once m is known to hold.  False (nothing signalled): m
  // must move.
  __device__ static bool block_ahead(Misc& ms, uint32_t s_addr, float c, float m, int g, bool live, float& l,
                                     uint32_t (&s)[4][32]) {
    const float ref = (m == -INFINITY ? 0.f : m) - kBias;
    const uint64_t c2 = pair(c, c), r2 = pair(-ref, -ref);
    uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
    uint32_t p0[16], p1[16];
    weights(s[0], c2, r2, p0, sum);
    weights(s[1], c2, r2, p1, sum);
    const float mx = fmaxf(fmaxf(largest(s[0]), largest(s[1])), fmaxf(largest(s[2]), largest(s[3]))) * c;
    // (Rows that are not stored may hold anything.)
    if (__any_sync(0xffffffffu, live && mx > m + kRescaleLog2)) return false;
    tmem_st16_nowait(s_addr, p0);
    tmem_st16_nowait(s_addr + 16, p1);
    weights(s[2], c2, r2, p0, sum);
    keep(p0);                                  // hides the wait for the stores before
    signal(&ms.p_ready[g][0]);
    tmem_st16_nowait(s_addr + 32, p0);
    weights(s[3], c2, r2, p1, sum);
    tmem_st16_nowait(s_addr + 48, p1);
    signal(&ms.p_ready[g][1]);
    uint32_t a0, a1;
    unpair(add2(sum[0], sum[1]), a0, a1);
    l += __uint_as_float(a0) + __uint_as_float(a1);
    return true;
  }

  // Any other block: the maximum first.
  __device__ static void block_after(Misc& ms, uint32_t s_addr, uint32_t o_addr, float c, int g, bool live, bool first, float& m, float& l,
                                     const uint32_t (&s)[4][32]) {
    const float mx = fmaxf(fmaxf(largest(s[0]), largest(s[1])), fmaxf(largest(s[2]), largest(s[3]))) * c;
    if (first) m = mx;
    else if (__any_sync(0xffffffffu, live && mx > m + kRescaleLog2)) rescale(o_addr, fmaxf(m, mx), m, l);
    const float ref = (m == -INFINITY ? 0.f : m) - kBias;
    const uint64_t c2 = pair(c, c), r2 = pair(-ref, -ref);
    uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t p[16];
      weights(s[q], c2, r2, p, sum);
      if (q == 2) {
        keep(p);
        signal(&ms.p_ready[g][0]);
      }
      tmem_st16_nowait(s_addr + q * 16, p);
    }
    signal(&ms.p_ready[g][1]);
    uint32_t a0, a1;
    unpair(add2(sum[0], sum[1]), a0, a1);
    l += __uint_as_float(a0) + __uint_as_float(a1);
  }

  __device__ static void softmax(const AttendLaunch& a, Misc& ms, int g) {
    int* status = a.status;
    const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, r = warp * 32 + lane;
    const int G = a.group, tokens = kRows / G;
    const uint32_t taddr = kTmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t s_addr = taddr + g * kRows, o_addr = taddr + 256 + g * D;
    const float c = kCap ? 1.f : a.scale * kLog2e;
    const float over_cap = kCap ? a.scale / a.logit_cap : 0.f, cap_log2e = a.logit_cap * kLog2e;
    Ring tr;
    uint32_t sph = 0, oph = 0;
    while (true) {
      if (!warp_wait(ms, &ms.tfull[tr.i], tr.phase, status)) return;
      const AttendTask t = ms.task[tr.i];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ms.tempty[tr.i]);
      tr.next(kTaskRing);
      if (!t.valid) return;
      int n[2];
      tile_blocks(a, t, tokens, n);
      const int blocks = n[g];
      const int row = t.first + g * tokens + r / G, head = t.head * G + r % G;
      const bool live = r < tokens * G && row < t.last;
      // Keys this row sees; rows that are not stored see all, so that they ask for no masking.
      const int lo = live ? first_key(a, t, row) : 0, hi = live ? last_key(a, t, row) : 0x3fffffff;
      float m = -INFINITY, l = 0.f;
      for (int b = 0; b < blocks; ++b) {
        if (!warp_wait(ms, &ms.s_full[g], sph, status)) return;
        sph ^= 1u;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(s_addr + q * 32, s[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_wait32(s[q]);
        const int j0 = t.lo + b * kRows;
        if (kCap) cap_scores(s, over_cap, cap_log2e);
        const bool masked = __any_sync(0xffffffffu, j0 < lo || j0 + kRows - 1 > hi);
        if (masked) {
          const int from = lo - j0, to = hi - j0;
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            if (i > to) s[i >> 5][i & 31] = 0xff800000u;
          if (__any_sync(0xffffffffu, from > 0)) {           // a window's lower edge
#pragma unroll
            for (int i = 0; i < kRows; ++i)
              if (i < from) s[i >> 5][i & 31] = 0xff800000u;
          }
        }
        if (b == 0 || masked || !block_ahead(ms, s_addr, c, m, g, live, l, s))
          block_after(ms, s_addr, o_addr, c, g, live, b == 0, m, l, s);
      }
      const int64_t at = static_cast<int64_t>(row) * a.query_heads + head;
      if (blocks > 0) {
        if (!warp_wait(ms, &ms.o_full[g], oph, status)) return;
        oph ^= 1u;
        tc_fence_after();
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float e2 = l == 0.f ? -INFINITY : m - kBias + lg2(l);
      bool odd = false;
      unsigned char* dst = nullptr;
      if (live)
        dst = a.partial != nullptr
                  ? reinterpret_cast<unsigned char*>(a.partial + (at * a.splits + t.split) * D)
                  : static_cast<unsigned char*>(a.out) + (static_cast<int64_t>(row) * a.out_stride[0] +
                                                          static_cast<int64_t>(head) * a.out_stride[1]) * 2;
      if (g == 0 || t.first + tokens < t.last) {
        unsigned char* rows[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          rows[k] = reinterpret_cast<unsigned char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), (lane & ~3) + k));
        float check = 0.f;
#pragma unroll 1
        for (int d0 = 0; d0 < D; d0 += 64) {
          uint32_t o[2][32];
          if (blocks > 0) {
            tmem_ld32(o_addr + d0, o[0]);
            tmem_ld32(o_addr + d0 + 32, o[1]);
            tmem_wait32(o[0]);
            tmem_wait32(o[1]);
            if (d0 + 64 == D) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&ms.o_free[g]);      // the next task's O may be written
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[0][i] = o[1][i] = 0u;
          }
          store_rows(a, rows, d0, o[0], inv, check);
          store_rows(a, rows, d0 + 32, o[1], inv, check);
        }
        odd = !(check == 0.f);
        if (live) {
          if (a.partial != nullptr) a.partial_lse[at * a.splits + t.split] = e2 * kLn2;
          else if (a.lse != nullptr) a.lse[at] = e2 * kLn2;
        }
      }
      const uint32_t again = __ballot_sync(0xffffffffu, odd && live);
      if (again != 0) form_again<T, D, 4>(a, t, again, row, head, e2, &ms.clock.beat);
    }
  }

  // After an expired wait, by the softmax warps: NaN for the rows (and split results) of the last tasks
  // taken, as no other CTA will run them.  Some may have been stored in full: they are NaN all the same.
  // Where the hardware did not answer a claim, the task is not known, and every row of the call is set.
  __device__ static void give_up(const AttendLaunch& a, const Misc& ms) {
    const int warp = (threadIdx.x >> 5) - kSoftmaxWarp, lane = threadIdx.x & 31;
    const int tokens = kRows / a.group;
    const float nan = __int_as_float(0x7fc00000);
    const uint32_t n = ms.lost ? gridDim.x : min(ms.n_taken, static_cast<uint32_t>(kTaken));
    int chunk = 0;
    int64_t before = 0;
    for (uint32_t i = 0; i < n; ++i) {
      const AttendTask t = find_task(a, 2 * tokens, kRows, ms.lost ? i : ms.taken[i], chunk, before);
      if (!t.valid) continue;
      for (int r = warp; r < (t.last - t.first) * a.group; r += kWarps - kSoftmaxWarp) {
        const int row = t.first + r / a.group, head = t.head * a.group + r % a.group;
        const int64_t at = static_cast<int64_t>(row) * a.query_heads + head;
        for (int d = lane; d < D; d += 32) {
          if (a.partial != nullptr)
            a.partial[(at * a.splits + t.split) * D + d] = nan;
          else
            static_cast<T*>(a.out)[static_cast<int64_t>(row) * a.out_stride[0] + static_cast<int64_t>(head) * a.out_stride[1] + d] =
                from_float<T>(nan);
        }
        if (lane == 0 && a.partial != nullptr) a.partial_lse[at * a.splits + t.split] = nan;
        else if (lane == 0 && a.lse != nullptr) a.lse[at] = nan;
      }
    }
  }
};

template <typename T, int D, bool kCap>
__global__ void __launch_bounds__(kThreads, 1) attend_tc_kernel(const __grid_constant__ AttendLaunch a) {
  using A = Attend<T, D, kCap>;
  using L = Layout<D>;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  Misc& ms = *reinterpret_cast<Misc*>(smem + L::kOffMisc);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    ms.clock = Clock{0, a.wait_ns};
    ms.drain_clock = Clock{0, kDrainLimitNs};
    ms.n_taken = ms.lost = 0;
    for (int i = 0; i < L::kStages; ++i) mbar_init(&ms.kv_full[i], kLoaders * 32), mbar_init(&ms.kv_empty[i], 1);
    mbar_init(&ms.q_full, 1), mbar_init(&ms.q_empty, 1), mbar_init(&ms.drain, 1), mbar_init(&ms.claimed, 1);
    for (int g = 0; g < 2; ++g)
      mbar_init(&ms.s_full[g], 1), mbar_init(&ms.p_ready[g][0], 4), mbar_init(&ms.p_ready[g][1], 4), mbar_init(&ms.o_full[g], 1), mbar_init(&ms.o_free[g], 4);
    for (int i = 0; i < kTaskRing; ++i) mbar_init(&ms.tfull[i], 1), mbar_init(&ms.tempty[i], 8 + kLoaders);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) tmem_alloc(smem_addr(&ms.tmem_base), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp >= kSoftmaxWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    A::softmax(a, ms, (warp - kSoftmaxWarp) >> 2);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kMmaWarp) {
      A::mma_issuer(a, smem, ms);
    } else {
      A::loader(a, smem, ms, warp - kLoaderWarp);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(ms.tmem_base, kTmemCols);
  if (warp >= kSoftmaxWarp && (ms.clock.beat == kFailed || ms.lost)) A::give_up(a, ms);
}

template <typename T, int D, bool kCap>
cudaError_t launch(const AttendLaunch& a, cudaStream_t stream) {
  using L = Layout<D>;
  cudaError_t e = cudaFuncSetAttribute(attend_tc_kernel<T, D, kCap>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return e;
  const int step = 2 * (kRows / a.group);
  const int64_t tasks = (static_cast<int64_t>(a.tokens / step) + a.seqs) * a.splits * a.kv_heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tasks));   // CTAs that run take the tasks of those still waiting
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attend_tc_kernel<T, D, kCap>, a);
}

template <typename T>
cudaError_t launch_typed(const AttendLaunch& a, cudaStream_t stream) {
  if (a.head_dim == 64) return a.logit_cap > 0.f ? launch<T, 64, true>(a, stream) : launch<T, 64, false>(a, stream);
  return a.logit_cap > 0.f ? launch<T, 128, true>(a, stream) : launch<T, 128, false>(a, stream);
}

}  // namespace

cudaError_t launch_attend_tc(const AttendLaunch& a, cudaStream_t stream) {
  return a.dtype == SGLD_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(a, stream) : launch_typed<__half>(a, stream);
}

}  // namespace sgld
