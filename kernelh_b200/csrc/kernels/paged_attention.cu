// paged_attention: attention of new tokens over a paged cache, O = softmax(scale Q K^T + mask) V, for
// sequences of any lengths side by side: decoding (one new token), chunks of a prompt, or both in one call.
// fp32, bf16 or fp16; grouped key/value heads; causal and sliding-window masks; optional log-sum-exp.
//
// This file: the kernel for few rows per key/value head, and for types and head sizes that the tensor-memory
// kernel does not take. A block of warps works on one item (see kh_paged.cuh) at a time, 16 rows of queries,
// one m16 tile. Every warp streams its own 16 keys of each unit through a ring of its own (cp.async, no block
// barrier inside an item) and keeps its own running maximum, sum and 16 x head_dim output in registers; the
// warps are added up at the end of the item, through shared memory, in a fixed order.
//   S = Q K^T and O += P V run as mma.sync m16n8k16 (16-bit types) or as three m16n8k8 tf32 products of
//   hi/lo parts of 11 significant bits each (fp32; lo.lo is dropped: 2^-22 of a product).
// Few fp32 rows take plain multiply-adds (score_rows). Few items go to clusters, an item to each (kJoint).
// HBM-bound at decoding: 4 rows x 128 values of queries cost 0.5 flop per byte of cache per row, far below
// what any matrix unit needs; what counts is bytes in flight: two 16-key stages of keys and values per
// warp, 8 warps per SM, are 128 KiB. Scores, softmax and sums are fp32; P is rounded to the values' type for
// the second product (it is an operand of the 16-bit matrix instruction; 2^-9 of a probability in bf16), the
// row sum is taken before that rounding; fp32 keeps P in hi/lo parts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kh_paged.cuh"

namespace {

using khp::PagedParams;

constexpr int kRows = 16;    // rows of an item
constexpr int kKeys = 16;    // keys of a warp's step
constexpr int kStages = 3;   // ring of a warp
constexpr float kLazy = 8.f;

template <typename T, int kDim> struct Config {
  static constexpr int kRowBytes = kDim * static_cast<int>(sizeof(T));
  static constexpr int kWarps = kRowBytes <= 512 ? 4 : 2; // 3 stages of 16 keys and values per warp must fit
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kUnit = 64; // keys of a unit: the same for every type, so that the host can count
  using Cut = khp::Grain<kRows, kUnit>;
  static constexpr int kSteps = kUnit / (kKeys * kWarps);
  static constexpr int kPitch = kRowBytes + 16; // bytes between rows: ldmatrix and fp32 reads without bank conflicts
  static constexpr int kTile = kKeys * kPitch;
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kSmem = kWarps * kRing + (sizeof(T) == 4 ? kTile : 0); // fp32 queries lie behind the rings
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// nothing is read and zeros are written when !valid
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, both rounded to nearest at 11 significant bits (cut instead, the parts left over all have
// one sign and add up: 1.6e-6 of a decoding step's output in 2-norm against 8e-7). (An infinity gives NaN, inf - inf.)
__device__ __forceinline__ uint32_t round_tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t &hi, uint32_t &lo) {
  hi = round_tf32(__uint_as_float(x));
  lo = round_tf32(__uint_as_float(x) - __uint_as_float(hi));
}
template <int n> __device__ __forceinline__ void split_tf32(const uint32_t (&x)[n], uint32_t (&hi)[n], uint32_t (&lo)[n]) {
#pragma unroll
  for (int i = 0; i < n; ++i) split_tf32(x[i], hi[i], lo[i]);
}
__device__ __forceinline__ void mma8_fp32(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], uint32_t b0, uint32_t b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  mma8_tf32(d, al, h0, h1);
  mma8_tf32(d, ah, l0, l1);
  mma8_tf32(d, ah, h0, h1);
}

template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// The 16-row query tile as A fragments. 16-bit types keep them in registers: k-step s holds rows (g, g + 8) x columns
// 16 s + 2c (+1) and + 8 (g = lane / 4, c = lane % 4). fp32 rows are twice that: they lie in shared memory, padded like
// the keys, and a k-step's fragment (columns 8 s + c and + 4) is one ldmatrix. Zeros outside rows and head_dim.
template <typename T, int kDim> struct Queries {
  static constexpr int kStepsK = kDim / 16;
  uint32_t a[kStepsK][4];
  __device__ __forceinline__ void load(const PagedParams &P, const T *row0, const T *row1, uint32_t) {
    const int c = threadIdx.x & 3;
#pragma unroll
    for (int s = 0; s < kStepsK; ++s) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T *row = j & 1 ? row1 : row0;
        const int col = 16 * s + 2 * c + (j >> 1) * 8;
        a[s][j] = row != nullptr && col < P.head_dim ? *reinterpret_cast<const uint32_t *>(row + col) : 0u;
      }
    }
  }
};
template <int kDim> struct Queries<float, kDim> {
  static constexpr int kStepsK = kDim / 8;
  uint32_t at;
  // Every warp calls this; the block has passed a barrier since the last use, and passes one before the next.
  __device__ __forceinline__ void load(const PagedParams &P, const float *row0, const float *row1, uint32_t tile) {
    constexpr int kPitch = Config<float, kDim>::kPitch, kWarps = Config<float, kDim>::kWarps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int c = (warp * 4 + (lane & 3)) * 4; c < kDim; c += kWarps * 16) // this warp's share of the lane's two rows
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float *row = x ? row1 : row0;
        const float4 v = row != nullptr && c < P.head_dim ? *reinterpret_cast<const float4 *>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(tile + ((lane >> 2) + 8 * x) * kPitch + c * 4), "f"(v.x), "f"(v.y),
                     "f"(v.z), "f"(v.w)
                     : "memory");
      }
    at = tile + (lane & 15) * kPitch + (lane >> 4) * 16;
  }
};

// S (16 rows x 16 keys, two n8 tiles) of one tile of keys in shared memory
template <typename T, int kDim>
__device__ __forceinline__ void score_tile(const Queries<T, kDim> &q, uint32_t tile, float (&s)[2][4]) {
  using Cfg = Config<T, kDim>;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = 0.f;
  // matrices of one ldmatrix.x4: keys 0-7 and 8-15, each with the two 16-byte halves of the k-step
  const uint32_t at = tile + ((lane & 7) + ((lane >> 4) << 3)) * Cfg::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
  for (int k = 0; k < Queries<T, kDim>::kStepsK; ++k) {
    uint32_t b[4];
    ldsm4(b, at + k * 32);
    if constexpr (sizeof(T) == 2) {
      mma16<T>(s[0], q.a[k], b[0], b[1]);
      mma16<T>(s[1], q.a[k], b[2], b[3]);
    } else {
      uint32_t a[4], hi[4], lo[4];
      ldsm4(a, q.at + k * 32);
      split_tf32(a, hi, lo);
      mma8_fp32(s[0], hi, lo, b[0], b[1]);
      mma8_fp32(s[1], hi, lo, b[2], b[3]);
    }
  }
}

// O += P V for one tile: p holds the probabilities in the score layout
template <typename T, int kDim>
__device__ __forceinline__ void value_tile(const float (&p)[2][4], uint32_t tile, float (&o)[kDim / 8][4]) {
  using Cfg = Config<T, kDim>;
  const int lane = threadIdx.x & 31;
  if constexpr (sizeof(T) == 2) {
    const uint32_t a[4] = {pack<T>(p[0][0], p[0][1]), pack<T>(p[0][2], p[0][3]), pack<T>(p[1][0], p[1][1]), pack<T>(p[1][2], p[1][3])};
    const uint32_t at = tile + (lane & 15) * Cfg::kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < kDim / 16; ++n) {
      uint32_t b[4];
      ldsm4_trans(b, at + n * 32);
      mma16<T>(o[2 * n], a, b[0], b[1]);
      mma16<T>(o[2 * n + 1], a, b[2], b[3]);
    }
  } else {
    // k index c of the product stands for key 2c of its 8, c + 4 for key 2c + 1: the score layout as it is
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t a[4] = {__float_as_uint(p[t][0]), __float_as_uint(p[t][2]), __float_as_uint(p[t][1]), __float_as_uint(p[t][3])};
      uint32_t hi[4], lo[4];
      split_tf32(a, hi, lo);
      const uint32_t at = tile + (8 * t + 2 * (lane & 3)) * Cfg::kPitch + (lane >> 2) * 4;
#pragma unroll
      for (int n = 0; n < kDim / 8; ++n) {
        uint32_t b0, b1;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b0) : "r"(at + n * 32) : "memory");
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b1) : "r"(at + n * 32 + Cfg::kPitch) : "memory");
        mma8_fp32(o[n], hi, lo, b0, b1);
      }
    }
  }
}

// Few rows in fp32: most of the 16 rows of the products above would be padding, at seven instructions for every value that
// is split. Plain multiply-adds instead: scores with two lanes to a key, each half of its values, handed out in the
// layout above; P V with the lanes along head_dim, lane i's values 64 x + 2 i (+1) of row r in o[r * kDim / 64 + x][0 and 1].
// kFew rows are worked on: 1, 4, or 8 for longer rows than 64. (From a graph, against split products: 8 sequences of up to
// 1024 keys, 16 heads of 64, one row each, 16.5 us against 20.6. 16 x 8192 keys, 8 key/value heads: 4 rows of 64 values 122 against
// 149, of 128 214 against 430, 3 of 256 647 against 1669; 8 rows of 128 345 against 461, of 256 1399 against 1693, but 6 of
// 64 176 against 157.)
template <int kDim> constexpr int kFewRows = kDim == 64 ? 4 : 8;
template <int kDim, int kFew> __device__ __forceinline__ void score_rows(uint32_t q, uint32_t tile, float (&s)[2][4]) {
  constexpr int kPitch = Config<float, kDim>::kPitch;
  const int lane = threadIdx.x & 31;
  const uint32_t k = tile + (lane & 15) * kPitch + (lane >> 4) * (kDim * 2);
  q += (lane >> 4) * (kDim * 2);
  float2 sum[kFew][2];
#pragma unroll
  for (int r = 0; r < kFew; ++r) sum[r][0] = sum[r][1] = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kDim / 8; ++i) {
    float4 b;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w) : "r"(k + i * 16) : "memory");
#pragma unroll
    for (int r = 0; r < kFew; ++r) {
      float4 a;
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w) : "r"(q + r * kPitch + i * 16) : "memory");
      sum[r][0] = __ffma2_rn(make_float2(a.x, a.y), make_float2(b.x, b.y), sum[r][0]);
      sum[r][1] = __ffma2_rn(make_float2(a.z, a.w), make_float2(b.z, b.w), sum[r][1]);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[t][j] = 0.f;
#pragma unroll
  for (int r = 0; r < kFew; ++r) {
    float all = (sum[r][0].x + sum[r][0].y) + (sum[r][1].x + sum[r][1].y);
    all += __shfl_xor_sync(0xffffffffu, all, 16);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float v = __shfl_sync(0xffffffffu, all, 8 * t + 2 * (lane & 3) + j);
        if (lane >> 2 == r) s[t][j] = v;
      }
  }
}
template <int kDim, int kFew> __device__ __forceinline__ void value_rows(const float (&p)[2][4], uint32_t tile, float (&o)[kDim / 8][4]) {
  constexpr int kPitch = Config<float, kDim>::kPitch;
  const uint32_t at = tile + (threadIdx.x & 31) * 8;
#pragma unroll
  for (int k = 0; k < kKeys; ++k) {
    float w[kFew];
#pragma unroll
    for (int r = 0; r < kFew; ++r) w[r] = __shfl_sync(0xffffffffu, p[k >> 3][k & 1], 4 * r + ((k & 7) >> 1));
#pragma unroll
    for (int x = 0; x < kDim / 64; ++x) {
      float2 v;
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at + k * kPitch + x * 256) : "memory");
#pragma unroll
      for (int r = 0; r < kFew; ++r) {
        float(&to)[4] = o[r * (kDim / 64) + x];
        to[0] = fmaf(w[r], v.x, to[0]);
        to[1] = fmaf(w[r], v.y, to[1]);
      }
    }
  }
}

// Blocks of a cluster: barrier (every block makes the same number of arrivals, whatever it finds to do), and the
// shared memory of block `rank` at this block's address.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t address_in(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 load2_cluster(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 load4_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
constexpr int kMaxCluster = 8;

// kJoint: a cluster takes one item, each of its blocks a part of the keys, and adds the parts up through its shared
// memory. One launch and no workspace, for few items with keys enough for several blocks (see the host's rule).
template <typename T, int kDim, bool kJoint> __device__ __forceinline__ void attention_body(const PagedParams &P) {
  using Cfg = Config<T, kDim>;
  using Cut = typename Cfg::Cut;
  constexpr int kThreads = Cfg::kThreads, kWarps = Cfg::kWarps, kUnit = Cfg::kUnit;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ khp::LineScratch<kThreads> scratch;
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ float2 s_ml[kJoint ? kRows : 1]; // of the block
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t ring = smem_addr(smem) + warp * Cfg::kRing;
  if (P.head_dim < kDim) { // columns that no copy writes count as zeros
    for (int i = threadIdx.x * 16; i < kWarps * Cfg::kRing; i += kThreads * 16) *reinterpret_cast<uint4 *>(smem + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  khd::grid_dependency_wait();
  khd::grid_dependents_may_launch();
  const int ranks = kJoint ? static_cast<int>(cluster_size()) : 1, rank = kJoint ? static_cast<int>(cluster_rank()) : 0;
  const int w = static_cast<int>(blockIdx.x) / ranks;
  khp::Line line{};
  int64_t from = 0, until = 1;
  if constexpr (kJoint) {
    if (!khp::find_item<kThreads, Cut>(P, w, scratch)) {
      cluster_barrier();
      cluster_barrier();
      return;
    }
  } else {
    line = khp::lay_line<kThreads, Cut>(P, w, scratch);
    if (w >= line.workers) {
      if (threadIdx.x == 0 && !P.whole) P.split_items[w] = khp::SplitItem{};
      return;
    }
    from = line.stretch(w), until = line.stretch(w + 1);
  }
  int64_t at = from, start = scratch.start;
  int b = scratch.b;
  khp::Sequence s = khp::sequence<Cut>(P, b);
  if (!kJoint && P.whole) { // the first item that begins here
    const khp::Item item = khp::item_at<Cut>(P, s, start, at);
    if (item.begin < at) at = item.end;
  }

  const bool whole_steps = P.page_size % kKeys == 0; // a step's keys lie in one page
  const int chunks_per_row = P.head_dim * static_cast<int>(sizeof(T)) / 16; // 16-byte pieces that exist
  while (at < until) {
    khp::Item item;
    int unit0, unit1;
    if constexpr (kJoint) {
      item.h = static_cast<int>(w - start) / s.blocks;
      item.block = static_cast<int>(w - start) - item.h * s.blocks;
      item.keys = khp::keys_of<Cut>(P, s, item.block);
      item.begin = 0, item.end = 1;
      unit0 = static_cast<int>(static_cast<int64_t>(item.keys.units) * rank / ranks);
      unit1 = static_cast<int>(static_cast<int64_t>(item.keys.units) * (rank + 1) / ranks);
    } else {
      while (at >= start + s.head_span * P.k_heads) { // on to the next sequence that has rows
        start += s.head_span * P.k_heads;
        s = khp::sequence<Cut>(P, ++b);
      }
      item = khp::item_at<Cut>(P, s, start, at);
      if (at - item.begin >= item.keys.units) { // what is left of the item is only what stands for its end
        if (threadIdx.x == 0 && at == from && !P.whole) P.split_items[w] = khp::SplitItem{};
        at = item.end;
        continue;
      }
      unit0 = static_cast<int>(at - item.begin);
      unit1 = P.whole ? item.keys.units : static_cast<int>(min((until < item.end ? until : item.end) - item.begin, static_cast<int64_t>(item.keys.units)));
    }
    const int h = item.h;
    const int row0 = item.block * kRows, rows_here = min(kRows, s.rows - row0);
    const int t_first = row0 / P.group, t_last = (row0 + rows_here - 1) / P.group;
    const int past = s.kv - s.tokens; // position of token 0 (negative: its first tokens see nothing)
    // keys that rows of this block see, in this stretch
    const int lo_key = item.keys.lo;
    const int key_a = (item.keys.first_unit + unit0) * kUnit;
    const int key_b = static_cast<int>(min(static_cast<int64_t>(item.keys.first_unit + unit1) * kUnit, static_cast<int64_t>(item.keys.hi)));

    // this lane's two rows: their queries and the keys they see
    const int g = lane >> 2;
    const int few = sizeof(T) == 4 && rows_here <= kFewRows<kDim> ? rows_here : 0; // rows that score_rows takes
    int see_lo[2], see_hi[2];
    const T *q_row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + g + 8 * i;
      const bool real = r < s.rows;
      const int t = real ? r / P.group : 0, head = h * P.group + (real ? r - t * P.group : 0);
      q_row[i] = real ? reinterpret_cast<const T *>(P.q) + (s.q0 + t) * P.q_token + head * P.q_head : nullptr;
      see_hi[i] = !real ? -1 : P.causal ? past + t : s.kv - 1;
      const int64_t first = P.window > 0 ? static_cast<int64_t>(past) + t - P.window + 1 : 0;
      see_lo[i] = static_cast<int>(first > 0 ? first : 0);
    }
    // what all real rows of the warp's tile see: a step inside needs no mask (rows that are not real are not stored)
    const int all_hi = P.causal ? past + t_first : s.kv - 1;
    const int64_t last_lo = P.window > 0 ? static_cast<int64_t>(past) + t_last - P.window + 1 : 0;
    const int all_lo = static_cast<int>(min(max(last_lo, static_cast<int64_t>(0)), static_cast<int64_t>(s.kv)));
    Queries<T, kDim> q;
    q.load(P, q_row[0], q_row[1], smem_addr(smem) + kWarps * Cfg::kRing);
    if (sizeof(T) == 4) __syncthreads();

    float o[kDim / 8][4];
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const int32_t *table = P.table + b * P.table_stride;
    const char *k_base = P.k + static_cast<int64_t>(h) * P.k_head * sizeof(T), *v_base = P.v + static_cast<int64_t>(h) * P.v_head * sizeof(T);
    const int steps = key_b > key_a ? ((key_b - key_a + kUnit - 1) / kUnit) * Cfg::kSteps : 0;
    const auto key_of = [&](int i) { return key_a + (i / Cfg::kSteps) * kUnit + (i % Cfg::kSteps * kWarps + warp) * kKeys; };
    constexpr int kChunks = Cfg::kRowBytes / 16;
    // The page of the step after the one being fetched is looked up ahead of its use: one for the step where pages
    // are whole steps, else lane r < 16 looks up row r's.
    int page_next = 0;
    const auto look_up = [&](int i) {
      const int key = key_of(i) + (whole_steps ? 0 : lane & 15);
      page_next = i < steps && key < key_b ? __ldg(table + (P.page_shift >= 0 ? key >> P.page_shift : key / P.page_size)) : 0;
    };
    const auto issue = [&](int i) {
      const int key0 = key_of(i);
      if (i < steps && key0 < key_b) {
        const uint32_t k_tile = ring + (i % kStages) * 2 * Cfg::kTile;
        if (whole_steps && key0 >= lo_key && key0 + kKeys <= key_b && static_cast<unsigned>(page_next) < static_cast<unsigned>(P.num_pages)) {
          // sixteen rows of one page, all of them wanted: copy j takes the rows kStride further on
          constexpr int kStride = kChunks < 32 ? 32 / kChunks : 1;
          const int slot = (P.page_shift >= 0 ? key0 & (P.page_size - 1) : key0 % P.page_size) + lane / kChunks;
          const char *kp = k_base + (page_next * P.k_page + slot * P.k_slot) * static_cast<int64_t>(sizeof(T)) + lane % kChunks * 16;
          const char *vp = v_base + (page_next * P.v_page + slot * P.v_slot) * static_cast<int64_t>(sizeof(T)) + lane % kChunks * 16;
          const uint32_t dst = k_tile + lane / kChunks * Cfg::kPitch + lane % kChunks * 16;
          const int64_t k_step = kStride * P.k_slot * static_cast<int64_t>(sizeof(T)), v_step = kStride * P.v_slot * static_cast<int64_t>(sizeof(T));
          if (lane % kChunks < chunks_per_row) {
#pragma unroll
            for (int j = 0; j < kKeys / kStride; ++j) {
#pragma unroll
              for (int x = 0; x < (kChunks + 31) / 32; ++x) { // rows of more than 32 pieces take two copies
                if (x > 0 && lane + 32 * x >= chunks_per_row) break;
                copy16(dst + j * kStride * Cfg::kPitch + x * 512, kp + x * 512);
                copy16(dst + Cfg::kTile + j * kStride * Cfg::kPitch + x * 512, vp + x * 512);
              }
              kp += k_step;
              vp += v_step;
            }
          }
        } else {
          const int key = key0 + (lane & 15);
          bool good = key < key_b && key >= lo_key; // evicted keys before every row's window are not read
          const int page = page_next;
          if (good && (page < 0 || page >= P.num_pages)) {
            khd::report_status(P.status, khd::kStatusBadPage, static_cast<uint32_t>(b));
            good = false;
          }
          const int slot = key % P.page_size;
          const int64_t k_off = good ? (page * P.k_page + slot * P.k_slot) * static_cast<int64_t>(sizeof(T)) : -1;
          const int64_t v_off = good ? (page * P.v_page + slot * P.v_slot) * static_cast<int64_t>(sizeof(T)) : -1;
          const uint32_t v_tile = k_tile + Cfg::kTile;
#pragma unroll 4
          for (int j = 0; j < kKeys * kChunks / 32; ++j) {
            const int idx = j * 32 + lane, row = idx / kChunks, c = idx % kChunks;
            const int64_t ko = __shfl_sync(0xffffffffu, k_off, row), vo = __shfl_sync(0xffffffffu, v_off, row);
            if (c < chunks_per_row) {
              copy16_or_zero(k_tile + row * Cfg::kPitch + c * 16, ko >= 0 ? k_base + ko + c * 16 : k_base, ko >= 0);
              copy16_or_zero(v_tile + row * Cfg::kPitch + c * 16, vo >= 0 ? v_base + vo + c * 16 : v_base, vo >= 0);
            }
          }
        }
      }
      copy_commit();
      look_up(i + 1);
    };
    look_up(0);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
    if (!kJoint && threadIdx.x == 0 && at == from && !P.whole) khp::note_split<Cut>(P, line, w, s, item); // while the first copies fly
    for (int i = 0; i < steps; ++i) {
      __syncwarp(); // every lane is done with the slot that is refilled now
      issue(i + kStages - 1);
      copy_wait<kStages - 1>();
      __syncwarp();
      const int key0 = key_of(i);
      if (key0 >= key_b) continue;
      const uint32_t k_tile = ring + (i % kStages) * 2 * Cfg::kTile;
      float sc[2][4];
      if constexpr (sizeof(T) == 4) {
        if (few == 1) score_rows<kDim, 1>(smem_addr(smem) + kWarps * Cfg::kRing, k_tile, sc);
        else if (few > 0 && few <= 4) score_rows<kDim, 4>(smem_addr(smem) + kWarps * Cfg::kRing, k_tile, sc);
        else if (kFewRows<kDim> > 4 && few > 0) score_rows<kDim, kFewRows<kDim>>(smem_addr(smem) + kWarps * Cfg::kRing, k_tile, sc);
        else score_tile<T, kDim>(q, k_tile, sc);
      } else {
        score_tile<T, kDim>(q, k_tile, sc);
      }
      float top[2] = {-INFINITY, -INFINITY};
      if (key0 + kKeys - 1 <= all_hi && key0 >= all_lo) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[t][j] *= P.scale_log2;
            top[j >> 1] = fmaxf(top[j >> 1], sc[t][j]);
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + 8 * t + 2 * (lane & 3) + (j & 1), i2 = j >> 1;
            const bool seen = key <= see_hi[i2] && key >= see_lo[i2];
            sc[t][j] = seen ? sc[t][j] * P.scale_log2 : -INFINITY;
            top[i2] = fmaxf(top[i2], sc[t][j]);
          }
      }
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        top[i2] = fmaxf(top[i2], __shfl_xor_sync(0xffffffffu, top[i2], 1));
        top[i2] = fmaxf(top[i2], __shfl_xor_sync(0xffffffffu, top[i2], 2));
      }
      // The reference is raised when a maximum has outgrown it by 2^8 (the rows' first keys among that): until then
      // the exponentials reach at most 2^8, and the output need not be touched.
      if (__any_sync(0xffffffffu, top[0] > m[0] + kLazy || top[1] > m[1] + kLazy)) {
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const float m_new = top[i2] > m[i2] + kLazy ? top[i2] : m[i2]; // (a row's own: it does not depend on its neighbours)
          const float f = khd::exp2_approx(m[i2] - (m_new == -INFINITY ? 0.f : m_new));
          m[i2] = m_new;
          l[i2] *= f;
          if (few > 0) { // o is laid out along head_dim
            if (i2 == 0)
#pragma unroll
              for (int r = 0; r < kFewRows<kDim>; ++r) {
                const float f_row = __shfl_sync(0xffffffffu, f, 4 * r);
#pragma unroll
                for (int x = 0; x < kDim / 64; ++x) {
                  o[r * (kDim / 64) + x][0] *= f_row;
                  o[r * (kDim / 64) + x][1] *= f_row;
                }
              }
            continue;
          }
#pragma unroll
          for (int n = 0; n < kDim / 8; ++n) {
            o[n][2 * i2] *= f;
            o[n][2 * i2 + 1] *= f;
          }
        }
      }
      // a row that has seen no key yet keeps reference -inf; its exponentials are taken against 0 and are all 0
      const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sc[t][j] = khd::exp2_approx(sc[t][j] - ref[j >> 1]);
          l[j >> 1] += sc[t][j];
        }
      if constexpr (sizeof(T) == 4) {
        if (few == 1) value_rows<kDim, 1>(sc, k_tile + Cfg::kTile, o);
        else if (few > 0 && few <= 4) value_rows<kDim, 4>(sc, k_tile + Cfg::kTile, o);
        else if (kFewRows<kDim> > 4 && few > 0) value_rows<kDim, kFewRows<kDim>>(sc, k_tile + Cfg::kTile, o);
        else value_tile<T, kDim>(sc, k_tile + Cfg::kTile, o);
      } else {
        value_tile<T, kDim>(sc, k_tile + Cfg::kTile, o);
      }
    }

    // the warps' rows are added up: the rings are drained and serve as scratch
    copy_wait<0>();
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2) {
      l[i2] += __shfl_xor_sync(0xffffffffu, l[i2], 1);
      l[i2] += __shfl_xor_sync(0xffffffffu, l[i2], 2);
      if ((lane & 3) == 0) {
        s_m[warp][g + 8 * i2] = m[i2];
        s_l[warp][g + 8 * i2] = l[i2];
      }
    }
    __syncthreads();
    constexpr int kPitchF = kDim + 4;
    float *mine = reinterpret_cast<float *>(smem + warp * Cfg::kRing);
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2) {
      float top = s_m[0][g + 8 * i2];
#pragma unroll
      for (int x = 1; x < kWarps; ++x) top = fmaxf(top, s_m[x][g + 8 * i2]);
      const float f = exp2f(m[i2] - (top == -INFINITY ? 0.f : top));
      if (few > 0) {
        if (i2 == 0)
#pragma unroll
          for (int r = 0; r < kFewRows<kDim>; ++r) {
            const float f_row = __shfl_sync(0xffffffffu, f, 4 * r);
            if (r < few)
#pragma unroll
              for (int x = 0; x < kDim / 64; ++x) {
                const float(&from_row)[4] = o[r * (kDim / 64) + x];
                *reinterpret_cast<float2 *>(mine + r * kPitchF + 64 * x + 2 * lane) = make_float2(from_row[0] * f_row, from_row[1] * f_row);
              }
          }
        continue;
      }
#pragma unroll
      for (int n = 0; n < kDim / 8; ++n)
        *reinterpret_cast<float2 *>(mine + (g + 8 * i2) * kPitchF + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * i2] * f, o[n][2 * i2 + 1] * f);
    }
    __syncthreads();
    const bool whole = !kJoint && unit0 == 0 && unit1 == item.keys.units;
    const auto put = [&](int r, int c, float top, float sum, float (&v)[4]) { // the finished values c .. c + 3 of a row
      const int t = (row0 + r) / P.group, head = h * P.group + (row0 + r) - t * P.group;
      const float inv = 1.f / sum;
      if (c < P.head_dim) {
        T *dst = reinterpret_cast<T *>(P.o) + (s.q0 + t) * P.o_token + head * P.o_head + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = sum != 0.f ? v[j] * inv : 0.f; // a row that sees no key: zeros
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<uint2 *>(dst) = make_uint2(pack<T>(v[0], v[1]), pack<T>(v[2], v[3]));
      }
      if (c == 0 && P.lse != nullptr)
        P.lse[static_cast<int64_t>(s.q0 + t) * (P.k_heads * P.group) + head] = sum != 0.f ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
    };
    const int64_t part = item.begin < from ? 2 * static_cast<int64_t>(w) : 2 * static_cast<int64_t>(w) + 1;
    for (int i = threadIdx.x; i < rows_here * (kDim / 4); i += kThreads) {
      const int r = i / (kDim / 4), c = i % (kDim / 4) * 4;
      float top = s_m[0][r];
#pragma unroll
      for (int x = 1; x < kWarps; ++x) top = fmaxf(top, s_m[x][r]);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        sum += s_l[x][r] * exp2f(s_m[x][r] - ref);
        const float4 y = *reinterpret_cast<const float4 *>(smem + x * Cfg::kRing + (r * kPitchF + c) * 4);
        v[0] += y.x, v[1] += y.y, v[2] += y.z, v[3] += y.w;
      }
      if constexpr (kJoint) { // this thread alone has read these places
        *reinterpret_cast<float4 *>(smem + (r * kPitchF + c) * 4) = make_float4(v[0], v[1], v[2], v[3]);
        if (c == 0) s_ml[r] = make_float2(top, sum);
        continue;
      }
      if (!whole) {
        *reinterpret_cast<float4 *>(P.partial_o + (part * kRows + r) * kDim + c) = make_float4(v[0], v[1], v[2], v[3]);
        if (c == 0) P.partial_ml[part * kRows + r] = make_float2(top, sum);
        continue;
      }
      put(r, c, top, sum, v);
    }
    if constexpr (kJoint) {
      cluster_barrier();
      for (int i = rank * kThreads + threadIdx.x; i < rows_here * (kDim / 4); i += ranks * kThreads) {
        const int r = i / (kDim / 4), c = i % (kDim / 4) * 4;
        float2 ml[kMaxCluster];
        float4 y[kMaxCluster];
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < kMaxCluster; ++x)
          if (x < ranks) {
            ml[x] = load2_cluster(address_in(smem_addr(&s_ml[r]), x));
            y[x] = load4_cluster(address_in(smem_addr(smem) + (r * kPitchF + c) * 4, x));
            top = fmaxf(top, ml[x].x);
          }
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < kMaxCluster; ++x)
          if (x < ranks) {
            const float f = exp2f(ml[x].x - ref);
            sum = fmaf(ml[x].y, f, sum);
            v[0] = fmaf(y[x].x, f, v[0]), v[1] = fmaf(y[x].y, f, v[1]), v[2] = fmaf(y[x].z, f, v[2]), v[3] = fmaf(y[x].w, f, v[3]);
          }
        put(r, c, top, sum, v);
      }
      cluster_barrier(); // no block leaves while another reads from it
      return;
    }
    __syncthreads(); // the scratch becomes rings again
    if (P.head_dim < kDim) { // and their unwritten columns zeros
      for (int i = threadIdx.x * 16; i < kWarps * Cfg::kRing; i += kThreads * 16) *reinterpret_cast<uint4 *>(smem + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
    }
    at = until < item.end && !P.whole ? until : item.end;
  }
}

template <typename T, int kDim> __device__ __forceinline__ void combine(const PagedParams &P) {
  khp::combine_row<256, kRows, kDim>(P, [&](int token, int head, int c, float v) {
    reinterpret_cast<T *>(P.o)[token * P.o_token + head * P.o_head + c] = from_float<T>(v);
  });
}

} // namespace

#define KH_PAGED(suffix, T, dim)                                                                                              \
  extern "C" __global__ void __launch_bounds__(Config<T, dim>::kThreads)                                                      \
  paged_attention_##suffix##_##dim(const __grid_constant__ PagedParams P) { attention_body<T, dim, false>(P); }               \
  extern "C" __global__ void __launch_bounds__(Config<T, dim>::kThreads)                                                      \
  paged_attention_joint_##suffix##_##dim(const __grid_constant__ PagedParams P) { attention_body<T, dim, true>(P); }          \
  extern "C" __global__ void __launch_bounds__(256) paged_attention_combine_##suffix##_##dim(                                 \
      const __grid_constant__ PagedParams P) { combine<T, dim>(P); }

KH_PAGED(f32, float, 64)
KH_PAGED(f32, float, 128)
KH_PAGED(f32, float, 256)
KH_PAGED(bf16, __nv_bfloat16, 64)
KH_PAGED(bf16, __nv_bfloat16, 128)
KH_PAGED(bf16, __nv_bfloat16, 256)
KH_PAGED(f16, __half, 64)
KH_PAGED(f16, __half, 128)
KH_PAGED(f16, __half, 256)
