// paged_attention for many rows per key/value head (chunks of prompts): 16-bit types, head_dim 64 .. 128,
// tensor cores with accumulators in tensor memory.
//
// An item (see kh_paged.cuh) is 256 rows of queries, two tiles of 128, against its keys in tiles of 128:
//   S_g = Q_g K^T   A = Q_g (shared memory, K-major), B = K tile (as it lies in the cache, K-major)
//   O_g += P_g V    A = P_g (tensor memory, 16-bit pairs), B = V tile (as it lies in the cache: its rows are
//                   keys, so it is the MN-major operand), accumulated in tensor memory over all tiles
// Tensor memory: S_0, S_1 (128 columns each; P_g is written over S_g once it is in registers) and O_0, O_1.
//
// One block per SM, 16 warps. Warpgroups 0 and 1, a thread per row, are the softmax of the two tiles; while one
// works, the tensor core does the other tile's P V and the next Q K^T, so the two keep it busy in turns. Warp 8
// issues the matrix instructions, warp 9 the copies, warp 10 works out the items, warps 12 to 15 bring in the queries of the next item while this
// one's last tile is worked on. The boxes of a tile of keys are looked up in the page table by one
// lane each and fetched by TMA straight out of the pages (a box is the largest power of two of slots that divides
// the page, so none crosses a page), keys and values through one ring. Pages therefore cost nothing but the
// look-up.
// Softmax with a lazy maximum: the reference a row's exponentials are taken against is only raised when the
// row's maximum has grown by more than 2^8, and only then is O_g rescaled (by the softmax threads themselves: the
// next scores being there means that the product before them is done). Until then P reaches at most 2^8, which costs
// no precision in floating point. P is rounded to the values' type (an operand of a 16-bit matrix
// instruction); the sum of the row is taken in fp32 before that rounding.
// Keys that no row of the item sees are masked by select, so K may hold anything there; of V such rows are
// zeroed in shared memory first (0 * NaN would reach every row), by the issuing warp, in the one or two tiles of an
// item that have any.
//
// Tensor-bound: 4 * 128 values * 256 rows * 128 keys = 16.8 Mflop per tile pair, 2048 clocks at the dense
// 16-bit rate; the 32768 exponentials of a pair take the special-function units the same 2048 clocks. Measured (a
// 2048-token chunk after 14336 tokens, 32 heads over 8, bf16): 441 us = 1.17 PFLOP/s, 2000 ns a pair; without the
// exponentials 400, without any softmax 365 (the products of a tile follow one another through four barriers).
// Measured and dropped: P handed over in two (447) or four (549) parts, an issuing warp per tile (445), 2 or 3 of 8
// exponentials by a polynomial on the multiply-add pipes (469, 490), two threads per row (556), the row maximum as a
// thread's first score (no change: 490 against 487 at the time), output rows stored by four lanes each (no change),
// half tiles of 64 keys with two buffers of scores, so that the next half's scores are there ahead (561: a product of 64 keys
// takes the tensor core as long as one of 128), one buffer of scores for both tiles, P in columns of its own and an issuing warp
// for each of the two products, so that scores are there ahead (431, but short items 5 to 10 % slower). The issuing warp is
// busy throughout: 52 clocks an instruction, 200 for a wait behind them, 3290 a pair. In a loop the device draws 990 W at
// 1.7 GHz.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kh_paged.cuh"
#include "kh_tcgen05.cuh"

namespace {

using khp::PagedParams;

constexpr int kTileRows = 128;
constexpr int kRows = 2 * kTileRows; // rows of an item
constexpr int kKeys = 128;           // keys of a tile
using Cut = khp::Grain<kRows, kKeys>;
constexpr int kThreads = 512;
constexpr int kMaxStages = 8;
constexpr int kIssueWarp = 8, kLoadWarp = 9, kPlanWarp = 10, kQueryWarp = 12, kQueryWarps = 4;
// registers after the warpgroups have traded them: two softmax groups, control, idle; 4 x 128 at launch
constexpr int kRegsSoftmax = 200, kRegsControl = 56;
constexpr float kLazy = 8.f;

template <int kDim> struct Config {
  static constexpr int kTileBytes = kKeys * kDim * 2; // K, V and Q tiles alike: kDim / 64 halves of 128 rows x 128 bytes; the host sizes 2 + kStages of them
  static constexpr int kStages = kDim == 128 ? 5 : 8;
};

template <int kRegs> __device__ __forceinline__ void registers_release() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs> __device__ __forceinline__ void registers_take() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const khd::TensorMap *map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
               "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
               "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t addr, const uint32_t (&r)[32]) {
  tmem_st_32x16(addr, *reinterpret_cast<const uint32_t(*)[16]>(&r[0]));
  tmem_st_32x16(addr + 16, *reinterpret_cast<const uint32_t(*)[16]>(&r[16]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The largest of three; NaN if any is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One arrival for the warp, after all its lanes (an arrival of every thread costs the barrier a turn each).
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) khd::mbar_arrive(bar);
}

// Operand descriptor of an MN-major tile in the 128-byte swizzle: rows (along K: keys) of 128 bytes hold 64
// values along MN; 8 rows are 1024 bytes, the next 64 values along MN lie `half_bytes` on. Fields as in
// khd::umma_desc_k128: leading offset = between blocks of 64 along MN, stride offset = between groups of 8 rows.
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t addr, uint32_t half_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(half_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

template <typename T> struct Types;
template <> struct Types<__half> {
  static constexpr uint32_t kFormat = 0;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct Types<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// A worker's part of an item.
struct alignas(16) Work {
  int q0, tokens, kv; // the sequence: first token, new tokens, keys
  int b, h, row0, rows; // rows: those of this item, up to 256
  int key_a, key_b;     // its keys in this stretch: [key_a, key_b), key_a on a tile
  int key_lo;           // the first key that any row sees
  int tiles;            // of keys; -1: nothing is left to do
  int part;             // the slot of a partial result, or -1 when the item is whole
};
// The worker's stretch of the line, item by item. Finding the next one is a few hundred dependent instructions, 4 us:
// one warp does it ahead of all others and hands it out through a short queue in shared memory.
struct Walker {
  int64_t at, until, from, start;
  int b, w;
  __device__ __forceinline__ void next(const PagedParams &P, Work &k) {
    khp::Item item;
    khp::Sequence s;
    for (;;) {
      if (at >= until) {
        k.tiles = -1;
        return;
      }
      s = khp::sequence<Cut>(P, b);
      while (at >= start + s.head_span * P.k_heads) {
        start += s.head_span * P.k_heads;
        s = khp::sequence<Cut>(P, ++b);
      }
      item = khp::item_at<Cut>(P, s, start, at);
      if (at - item.begin < item.keys.units) break;
      at = item.end; // what is left of the item is only what stands for its end
    }
    const int unit0 = static_cast<int>(at - item.begin);
    const int unit1 = static_cast<int>(min((until < item.end ? until : item.end) - item.begin, static_cast<int64_t>(item.keys.units)));
    k.q0 = s.q0;
    k.tokens = s.tokens;
    k.kv = s.kv;
    k.b = b;
    k.h = item.h;
    k.row0 = item.block * kRows;
    k.rows = min(kRows, s.rows - k.row0);
    k.key_lo = item.keys.lo;
    k.key_a = (item.keys.first_unit + unit0) * kKeys;
    k.key_b = static_cast<int>(min(static_cast<int64_t>(item.keys.first_unit + unit1) * kKeys, static_cast<int64_t>(item.keys.hi)));
    k.tiles = k.key_b > k.key_a ? (k.key_b - k.key_a + kKeys - 1) / kKeys : 0;
    k.part = unit0 == 0 && unit1 == item.keys.units ? -1 : (item.begin < from ? 2 * w : 2 * w + 1);
    at = until < item.end ? until : item.end;
  }
};
constexpr int kQueue = 4;
constexpr int kReaders = 8 + 1 + 1 + kQueryWarps; // warps that take every item

template <typename T, int kDim>
__device__ __forceinline__ void chunk_body(const PagedParams &P, const khd::TensorMap &tm_k, const khd::TensorMap &tm_v, int box_rows) {
  using Cfg = Config<kDim>;
  constexpr int kHalves = kDim / 64;
  constexpr uint32_t kHalfBytes = kKeys * 128; // 128 rows of 128 bytes
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[10 + 2 * kMaxStages + 2 * kQueue];
  __shared__ Work s_work[kQueue];
  __shared__ khp::LineScratch<kThreads> scratch;
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem_q = (khd::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t smem_ring = smem_q + 2 * Cfg::kTileBytes;
  const uint32_t bar_q = khd::smem_u32(&bars[0]), bar_s = khd::smem_u32(&bars[2]), bar_p = khd::smem_u32(&bars[4]),
                 bar_o = khd::smem_u32(&bars[6]), bar_q_free = khd::smem_u32(&bars[8]), bar_full = khd::smem_u32(&bars[10]),
                 bar_empty = khd::smem_u32(&bars[10 + kMaxStages]), bar_work = khd::smem_u32(&bars[10 + 2 * kMaxStages]),
                 bar_taken = khd::smem_u32(&bars[10 + 2 * kMaxStages + kQueue]);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int g = 0; g < 2; ++g) {
      khd::mbar_init(bar_q + 8 * g, kQueryWarps); // Q_g is in shared memory
      khd::mbar_init(bar_q_free + 8 * g, 1);           // the last S_g of an item is done: Q_g may go
      khd::mbar_init(bar_s + 8 * g, 1);                // S_g is done (and every product before it)
      khd::mbar_init(bar_p + 8 * g, 4);           // P_g is in tensor memory (an arrival per warp)
      khd::mbar_init(bar_o + 8 * g, 1);                // O_g is complete
    }
    for (int i = 0; i < kStages; ++i) {
      khd::mbar_init(bar_full + 8 * i, 1);
      khd::mbar_init(bar_empty + 8 * i, 1);
    }
    for (int i = 0; i < kQueue; ++i) {
      khd::mbar_init(bar_work + 8 * i, 1);
      khd::mbar_init(bar_taken + 8 * i, kReaders);
    }
    khd::mbar_fence_init();
    khd::tma_prefetch_descriptor(&tm_k);
    khd::tma_prefetch_descriptor(&tm_v);
  }
  if (warp == kIssueWarp) {
    khd::tmem_alloc(khd::smem_u32(&s_tmem_base), 512);
    khd::tmem_relinquish();
  }
  khd::tc_fence_before_sync();
  __syncthreads();
  khd::tc_fence_after_sync();
  const uint32_t tmem = s_tmem_base;
  khd::grid_dependency_wait();
  khd::grid_dependents_may_launch();

  const khp::Line line = khp::lay_line<kThreads, Cut>(P, blockIdx.x, scratch);
  // The next item of the queue, for a whole warp; false when there is none or a wait ran out.
  Work k;
  uint32_t work_count = 0;
  const auto take = [&] {
    const uint32_t i = work_count % kQueue;
    const bool ready = khd::mbar_wait(bar_work + 8 * i, (work_count / kQueue) & 1u, &s_abort, P.status, khd::kStatusEmptyWaitTimeout, 6900u);
    if (!__all_sync(0xffffffffu, ready)) return false;
    k = s_work[i];
    warp_arrive(bar_taken + 8 * i);
    ++work_count;
    return k.tiles >= 0;
  };

  if (warp >= 8) {
    registers_release<kRegsControl>();
    if (warp == kPlanWarp) {
      // ---- the worker's items, in turn, ahead of everybody ------------------------------------------------------
      Walker walker{};
      walker.w = blockIdx.x;
      if (walker.w < line.workers) {
        walker.from = walker.at = line.stretch(walker.w);
        walker.until = line.stretch(walker.w + 1);
        walker.b = scratch.b;
        walker.start = scratch.start;
      }
      for (uint32_t n = 0;; ++n) {
        const uint32_t i = n % kQueue;
        walker.next(P, k);
        const bool ready = khd::mbar_wait(bar_taken + 8 * i, ((n / kQueue) & 1u) ^ 1u, &s_abort, P.status, khd::kStatusEmptyWaitTimeout, 6950u);
        if (!__all_sync(0xffffffffu, ready)) break;
        if (lane == 0) {
          s_work[i] = k;
          khd::mbar_arrive(bar_work + 8 * i);
        }
        __syncwarp();
        if (k.tiles < 0) break;
      }
      if (lane == 0) {
        if (walker.w < line.workers) {
          const khp::Sequence s = khp::sequence<Cut>(P, scratch.b);
          khp::note_split<Cut>(P, line, walker.w, s, khp::item_at<Cut>(P, s, scratch.start, walker.from));
        } else {
          P.split_items[walker.w] = khp::SplitItem{};
        }
      }
    } else if (warp == kLoadWarp) {
      // ---- copies: K and V tiles of every item in turn through the ring. Lane i looks up and fetches box i. ----
      uint32_t slot = 0, phase = 0;
      bool ok = true;
      const int boxes = kKeys / box_rows;
      while (ok && take()) {
        const int32_t *table = P.table + k.b * P.table_stride;
        for (int j = 0; j < k.tiles && ok; ++j) {
          const int key = k.key_a + j * kKeys + lane * box_rows; // of this lane's box
          bool wanted = lane < boxes && key < k.key_b && key + box_rows > k.key_lo;
          int page = 0;
          if (wanted) {
            page = __ldg(table + key / P.page_size);
            if (page < 0 || page >= P.num_pages) {
              khd::report_status(P.status, khd::kStatusBadPage, static_cast<uint32_t>(k.b));
              wanted = false;
            }
          }
          const int place = key % P.page_size;
          const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, wanted))) * box_rows * 128u * kHalves;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = khd::mbar_wait(bar_empty + 8 * slot, phase ^ 1u, &s_abort, P.status, khd::kStatusEmptyWaitTimeout, 6000u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t bar = bar_full + 8 * slot, dst = smem_ring + slot * Cfg::kTileBytes + lane * box_rows * 128;
            if (lane == 0) khd::mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (wanted) {
#pragma unroll
              for (int x = 0; x < kHalves; ++x) tma_load_4d(dst + x * kHalfBytes, kv ? &tm_v : &tm_k, x * 64, place, k.h, page, bar);
            }
            if (++slot == kStages) {
              slot = 0;
              phase ^= 1u;
            }
          }
        }
      }
    } else if (warp == kIssueWarp) {
      // ---- matrix instructions, issued by one lane; the warp walks the loop together. Everything the instructions take
      //      is worked out warp-uniformly, outside the elected lane's branch: lengths come from lane 0 by shuffle,
      //      descriptors are a base plus constants (the address field counts 16 bytes). ----------------------------
      const bool leader = khd::elect_one();
      constexpr uint32_t kTypes = (Types<T>::kFormat << 7) | (Types<T>::kFormat << 10);
      constexpr uint32_t idesc_s = khd::umma_idesc_f16(kTileRows, kKeys) | kTypes;
      constexpr uint32_t idesc_o = khd::umma_idesc_f16(kTileRows, kDim) | kTypes | (1u << 16); // B is MN-major
      uint32_t slot = 0, phase = 0, p_phase[2] = {0, 0}, q_phase[2] = {0, 0};
      bool ok = true;
      const auto wait = [&](uint32_t bar, uint32_t parity, uint32_t code, uint32_t detail) {
        const bool ready = khd::mbar_wait(bar, parity, &s_abort, P.status, code, detail);
        return __all_sync(0xffffffffu, ready) != 0;
      };
      const auto advance = [&] {
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1u;
        }
      };
      const uint64_t desc_q = khd::umma_desc_k128(smem_q);
      const uint64_t desc_k = khd::umma_desc_k128(smem_ring), desc_v = umma_desc_mn128(smem_ring, kHalfBytes);
      constexpr uint32_t kStep = Cfg::kTileBytes >> 4;
      const auto issue_s = [&](int g, uint32_t k_slot, bool last, bool done) {
        const uint64_t a = desc_q + static_cast<uint32_t>(g) * kStep, b = desc_k + k_slot * kStep;
        if (leader) {
#pragma unroll
          for (int i = 0; i < kDim / 16; ++i) {
            const uint32_t off = (i >> 2) * (kHalfBytes >> 4) + (i & 3) * 2;
            khd::umma_f16_ss(tmem + g * 128, a + off, b + off, idesc_s, i != 0);
          }
          khd::umma_commit(bar_s + 8 * g);
          if (done) khd::umma_commit(bar_empty + 8 * k_slot);
          if (last) khd::umma_commit(bar_q_free + 8 * g);
        }
        __syncwarp();
      };
      while (ok && take()) {
        const int tiles = __shfl_sync(0xffffffffu, k.tiles, 0), groups = __shfl_sync(0xffffffffu, k.rows, 0) > kTileRows ? 2 : 1;
        const int key_a = __shfl_sync(0xffffffffu, k.key_a, 0), key_b = __shfl_sync(0xffffffffu, k.key_b, 0),
                  key_lo = __shfl_sync(0xffffffffu, k.key_lo, 0);
        if (tiles == 0) continue;
        for (int g = 0; g < groups && ok; ++g) {
          ok = wait(bar_q + 8 * g, q_phase[g], khd::kStatusEpilogueWaitTimeout, 6100u);
          q_phase[g] ^= 1u;
        }
        ok = ok && wait(bar_full + 8 * slot, phase, khd::kStatusTmaWaitTimeout, 6200u);
        if (!ok) break;
        khd::tc_fence_after_sync();
        for (int g = 0; g < groups; ++g) issue_s(g, slot, tiles == 1, g == groups - 1);
        advance();
        for (int j = 0; j < tiles && ok; ++j) {
          const uint32_t v_slot = slot;
          const uint64_t v = desc_v + v_slot * kStep;
          ok = wait(bar_full + 8 * slot, phase, khd::kStatusTmaWaitTimeout, 6300u);
          if (!ok) break;
          advance();
          // rows of V that no query sees: zeros
          const int key0 = key_a + j * kKeys, lo = max(0, key_lo - key0), hi = min(kKeys, key_b - key0);
          if (lo > 0 || hi < kKeys) {
            for (int i = lane; i < kHalves * kKeys * 8; i += 32) {
              const int row = (i >> 3) & (kKeys - 1);
              if (row < lo || row >= hi)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem_ring + v_slot * Cfg::kTileBytes + (i >> 10) * kHalfBytes +
                                                                                  (i & 1023) * 16),
                             "r"(0)
                             : "memory");
            }
            fence_async_shared();
            __syncwarp();
          }
          const bool more = j + 1 < tiles;
          if (more) {
            ok = wait(bar_full + 8 * slot, phase, khd::kStatusTmaWaitTimeout, 6500u);
            if (!ok) break;
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (g >= groups) break;
            ok = wait(bar_p + 8 * g, p_phase[g], khd::kStatusEpilogueWaitTimeout, 6400u);
            if (!ok) break;
            khd::tc_fence_after_sync();
            if (leader) {
#pragma unroll
              for (int i = 0; i < kKeys / 16; ++i) // 16 keys: 8 columns of P, two groups of 8 rows of V
                umma_ts(tmem + 256 + g * 128, tmem + g * 128 + i * 8, v + i * 128, idesc_o, j != 0 || i != 0);
              if (!more) khd::umma_commit(bar_o + 8 * g);
              if (g == groups - 1) khd::umma_commit(bar_empty + 8 * v_slot);
            }
            __syncwarp();
            p_phase[g] ^= 1u;
            if (more) issue_s(g, slot, j + 2 == tiles, g == groups - 1);
          }
          if (more) advance();
        }
      }
    }
    else if (warp >= kQueryWarp && warp < kQueryWarp + kQueryWarps) {
      // ---- queries: Q_g of the next item goes in as soon as the last S_g of this one is done. 16-byte chunk c of
      //      row x lies at chunk c ^ (x % 8) of its 128 bytes (the swizzle a TMA copy would have written). ----
      uint32_t phase[2] = {1, 1};
      bool ok = true;
      while (ok && take()) {
        if (k.tiles == 0) continue;
        for (int g = 0; g < 2 && g * kTileRows < k.rows && ok; ++g) {
          ok = khd::mbar_wait(bar_q_free + 8 * g, phase[g], &s_abort, P.status, khd::kStatusEmptyWaitTimeout, 6800u);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          phase[g] ^= 1u;
          constexpr int kChunks = kDim / 8;
#pragma unroll 4
          for (int i = 0; i < kTileRows * kChunks / (32 * kQueryWarps); ++i) {
            const int idx = (i * kQueryWarps + warp - kQueryWarp) * 32 + lane, x = idx / kChunks, c = idx % kChunks;
            const bool real = g * kTileRows + x < k.rows && c * 8 < P.head_dim;
            const int qr = k.row0 + (real ? g * kTileRows + x : 0), qt = qr / P.group;
            const T *src = reinterpret_cast<const T *>(P.q) + (k.q0 + qt) * P.q_token + (k.h * P.group + qr - qt * P.group) * P.q_head +
                           (real ? c * 8 : 0);
            const uint32_t dst = smem_q + g * Cfg::kTileBytes + (c >> 3) * kHalfBytes + x * 128 + (((c & 7) ^ (x & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_async_shared();
          warp_arrive(bar_q + 8 * g);
        }
      }
    }
  } else {
    registers_take<kRegsSoftmax>();
    // ---- softmax: a thread per row --------------------------------------------------------------------------
    const int g = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane; // in the tile
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + lanes + g * 128, t_o = tmem + lanes + 256 + g * 128;
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    while (ok && take()) {
      const int rows_here = k.rows - g * kTileRows; // of this tile
      if (rows_here <= 0) continue;
      const int r = k.row0 + g * kTileRows + row;
      const bool real = row < rows_here;
      const int t = real ? r / P.group : 0, head = k.h * P.group + (real ? r - t * P.group : 0);
      const int past = k.kv - k.tokens;
      const int see_hi = !real ? -1 : P.causal ? past + t : k.kv - 1;
      const int64_t first = P.window > 0 ? static_cast<int64_t>(past) + t - P.window + 1 : 0;
      const int see_lo = first > 0 ? static_cast<int>(min(first, static_cast<int64_t>(k.kv))) : 0;
      const bool idle = quad * 32 >= rows_here; // no row of this warp is real: its lanes of P may hold anything
      float m = -INFINITY, l = 0.f;             // reference and sum, in exp2 units
      for (int j = 0; j < k.tiles; ++j) {
        ok = khd::mbar_wait(bar_s + 8 * g, s_phase, &s_abort, P.status, khd::kStatusMmaWaitTimeout, 6600u);
        if (!ok) break;
        s_phase ^= 1u;
        khd::tc_fence_after_sync();
        if (!idle) {
          uint32_t s[kKeys];
#pragma unroll
          for (int i = 0; i < kKeys / 32; ++i) khd::tmem_ld_32x32(t_s + 32 * i, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * i]));
          khd::tmem_ld_wait();
          const int key0 = k.key_a + j * kKeys;
          const int lo = see_lo - key0, hi = see_hi - key0; // seen: lo <= i <= hi
          const bool masked = __any_sync(0xffffffffu, lo > 0 || hi < kKeys - 1);
          if (masked) {
#pragma unroll
            for (int i = 0; i < kKeys; ++i)
              if (i < lo || i > hi) s[i] = 0xff800000u; // -inf
          }
          float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kKeys; i += 8)
#pragma unroll
            for (int x = 0; x < 4; ++x) top4[x] = max3_nan(top4[x], __uint_as_float(s[i + 2 * x]), __uint_as_float(s[i + 2 * x + 1]));
          const float top = max3_nan(max3_nan(top4[0], top4[1], top4[2]), top4[3], -INFINITY) * P.scale_log2;
          const bool raise = !(top <= m + kLazy); // true of a NaN, which stays in m
          if (__any_sync(0xffffffffu, raise)) {   // (a row's own reference: its result does not depend on its neighbours)
            const float m_new = raise ? max3_nan(m, top, -INFINITY) : m, ref = m_new == -INFINITY ? 0.f : m_new;
            const float f = khd::exp2_approx(m - ref);
            m = m_new;
            l *= f;
            if (j > 0) { // O_g holds the tiles before: the product behind these scores' barrier is done
#pragma unroll
              for (int i = 0; i < kDim / 32; ++i) {
                uint32_t o[32];
                khd::tmem_ld_32x32(t_o + 32 * i, o);
                khd::tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                tmem_st_32x32(t_o + 32 * i, o);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.f : m;
          const float2 f2 = make_float2(P.scale_log2, P.scale_log2), off2 = make_float2(-ref, -ref);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int i = 0; i < kKeys / 32; ++i) {
            uint32_t p[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const float2 e = __ffma2_rn(make_float2(__uint_as_float(s[32 * i + 2 * x]), __uint_as_float(s[32 * i + 2 * x + 1])), f2, off2);
              const float2 v = make_float2(khd::exp2_approx(e.x), khd::exp2_approx(e.y));
              sum[x & 1] = __fadd2_rn(sum[x & 1], v);
              p[x] = Types<T>::pack(v.x, v.y);
            }
            tmem_st_32x16(t_s + 16 * i, p);
          }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          tmem_st_wait();
        }
        khd::tc_fence_before_sync();
        warp_arrive(bar_p + 8 * g);
      }
      if (!ok) break;
      // ---- the finished rows of this tile ------------------------------------------------------------------
      if (k.tiles > 0) {
        ok = khd::mbar_wait(bar_o + 8 * g, o_phase, &s_abort, P.status, khd::kStatusMmaWaitTimeout, 6700u);
        if (!ok) break;
        o_phase ^= 1u;
        khd::tc_fence_after_sync();
      }
      if (!idle) {
        const float inv = l != 0.f ? 1.f / l : 0.f; // a row that sees no key: zeros
        const int64_t at = static_cast<int64_t>(k.part) * kRows + g * kTileRows + row;
        T *dst = reinterpret_cast<T *>(P.o) + (k.q0 + t) * P.o_token + head * P.o_head;
#pragma unroll
        for (int i = 0; i < kDim / 32; ++i) {
          uint32_t o[32];
          if (k.tiles > 0) {
            khd::tmem_ld_32x32(t_o + 32 * i, o);
            khd::tmem_ld_wait();
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0u;
          }
          if (!real) continue;
          if (k.part >= 0) {
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<uint4 *>(P.partial_o + at * kDim + 32 * i + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          } else {
#pragma unroll
            for (int x = 0; x < 32; x += 8)
              if (32 * i + x < P.head_dim) {
                uint32_t v[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  v[y] = l != 0.f ? Types<T>::pack(__uint_as_float(o[x + 2 * y]) * inv, __uint_as_float(o[x + 2 * y + 1]) * inv) : 0u;
                *reinterpret_cast<uint4 *>(dst + 32 * i + x) = make_uint4(v[0], v[1], v[2], v[3]);
              }
          }
        }
        if (real) {
          if (k.part >= 0) P.partial_ml[at] = make_float2(m, l);
          else if (P.lse != nullptr)
            P.lse[static_cast<int64_t>(k.q0 + t) * (P.k_heads * P.group) + head] = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
        }
      }
    }
    khd::tc_fence_before_sync();
  }

  __syncthreads();
  if (s_abort) { // a wait ran out: let copies in flight land before the block's memory goes
    for (int i = 0; i < 64; ++i) __nanosleep(10000);
  }
  if (warp == kIssueWarp) {
    khd::tc_fence_after_sync();
    khd::tmem_dealloc(tmem, 512);
  }
}

} // namespace

#define KH_CHUNK(suffix, T, dim)                                                                                          \
  extern "C" __global__ void __launch_bounds__(kThreads, 1)                                                               \
  paged_attention_chunk_##suffix##_##dim(const __grid_constant__ PagedParams P, const __grid_constant__ khd::TensorMap tm_k, \
                                         const __grid_constant__ khd::TensorMap tm_v, int box_rows) {                      \
    chunk_body<T, dim>(P, tm_k, tm_v, box_rows);                                                                          \
  }                                                                                                                       \
  extern "C" __global__ void __launch_bounds__(256) paged_attention_chunk_combine_##suffix##_##dim(                       \
      const __grid_constant__ PagedParams P) {                                                                            \
    khp::combine_rows<kRows, dim>(P, [&](int token, int head, int c, float v) {                               \
      reinterpret_cast<T *>(P.o)[token * P.o_token + head * P.o_head + c] = Types<T>::from(v);                            \
    });                                                                                                                   \
  }

KH_CHUNK(bf16, __nv_bfloat16, 64)
KH_CHUNK(bf16, __nv_bfloat16, 128)
KH_CHUNK(f16, __half, 64)
KH_CHUNK(f16, __half, 128)
