// qk_norm_rope: the per-head RMS norm of queries and keys with the rotation of positions, in one pass
// over both tensors; its backward pass; and the serving form, which also stores the finished keys and
// the values into a paged cache. fp32, bf16 or fp16 rows; all arithmetic in fp32.
//
// For a row x of one head (d values), weight w, R rotated values and position p:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,
//   (y_a, y_b) = (n_a cos - n_b sin, n_a sin + n_b cos)  with the angle p * inv_freq[j] of pair j < R/2,
// pair j being (j, j + R/2), or (2j, 2j + 1) when interleaved; values from R on are only normalised.
// Backward: g = the inverse rotation of dy, u = x r:  dw = sum over rows of g u,
//   dx = r (g w - u mean(g w u)).
//
// HBM-bound: 2 (forward) or 3 (backward) times the rows' bytes, nothing else of that order. A row belongs
// to a group of lanes of one warp, each holding the two 16-byte vectors that the rotation pairs up, so a
// rotation exchanges nothing between lanes and the norm is the only reduction (log2(lanes) shuffles). A
// row is read and written by the same lanes, read first: outputs may be the inputs themselves.
//
// A persistent grid whose blocks are dealt out to queries, keys (and values) by their share of the rows, so
// that a block has one weight and one set of weight-gradient sums. A block takes tiles of
// tokens; its groups walk the tile's rows, the next row's loads in flight while one is worked on.
// Angles: position * inv_freq in half turns, formed and reduced in 64 bits (a position of 10^6 times a
// frequency of 1 has 20 bits before the point, fp32 would keep 4 after it), the remainder in [-1, 1]
// rounded to fp32 for sincospif. They are worked out once per tile by the whole block into shared memory and
// shared by all its heads: 50 instructions each, which every row on its own would pay again. Arithmetic on
// pairs of values (fp32x2) and packed conversions: the kernels are bound by instructions before they are bound
// by HBM. Measured: 32768 tokens x 40 heads x 128 bf16 in 127 us, 5.3 TB/s (202 us with scalar arithmetic and every
// group computing addresses for three tensors, 370 instructions for four rows of a warp); 16384 x 40 x 128 fp32 in 112 us,
// 6.0 TB/s; backward of 16384 x 40 x 128 in 105 us (bf16, 4.8 TB/s) and 165 us (fp32, 6.1 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kh_device.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 1024; // pairs x tokens of a tile
// Blocks per SM (the host's grid counts on them). A lane of a 16-bit row holds twice the values: one block more spills
// (bf16 forward 127 -> 139 us, backward 105 -> 141 at the sizes above; fp32 118 -> 111 and 183 -> 165).
template <typename T> constexpr int kForwardBlocks = sizeof(T) == 4 ? 4 : 3;
template <typename T> constexpr int kBackwardBlocks = sizeof(T) == 4 ? 3 : 2;

// Rows of head_dim contiguous values: data + token * token_stride + head * head_stride (elements).
struct HeadRows {
  char *data;
  int64_t token_stride, head_stride;
};
struct PagedRows {
  char *data;
  int64_t page_stride, slot_stride, head_stride;
};

// Layout shared with the host (registry/qk_norm_rope_kernel.cpp).
struct NormRopeParams {
  HeadRows q, k;          // inputs
  HeadRows q_out, k_out;  // forward: outputs; backward: the gradients of q and k
  const float *q_weight, *k_weight; // nullptr: ones
  const float *inv_freq;
  const int64_t *positions;
  int64_t tokens;
  int32_t q_heads, k_heads, head_dim, rotary_dim;
  int32_t lanes;          // of a row
  float eps;
  int32_t blocks[3], tile[3]; // of queries, keys, values: blocks, and tokens of a tile
};
struct AppendParams {
  HeadRows v;
  PagedRows k_cache, v_cache;
  const int64_t *slots;
  int64_t num_slots;
  uint32_t *status;
  int32_t page_size;
};
struct BackwardParams {
  HeadRows dq_out, dk_out; // gradients that come in
  float *partials;         // [gridDim.x][head_dim]
};
struct WeightGradParams {
  const float *partials;
  float *dq_weight, *dk_weight; // either may be nullptr
  int32_t blocks[2], head_dim;
};

// Two values of 16 bits in a word.
__device__ __forceinline__ float2 unpack(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 unpack(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// The raw values of a lane's pairs: kSlots times two vectors of kVec values, of 16, 8, 4 or 2 bytes.
template <int kBytes> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <typename T, int kVec, int kSlots> struct RawPairs {
  using R = typename Raw<static_cast<int>(sizeof(T)) * kVec>::type;
  R a[kSlots], b[kSlots];
};

// A lane's pairs in fp32, two to a register pair.
template <int kPairs> struct Pairs {
  float2 a[kPairs / 2], b[kPairs / 2];
};

// How a kernel holds a row: kVec values per access; kSlots accesses per lane; kFull: every lane has all of them;
// kInterleaved: pair j is (2j, 2j + 1), and the two vectors of a lane lie side by side.
template <typename T_, int kVec_, int kSlots_, bool kFull_, bool kInterleaved_> struct Layout {
  using T = T_;
  static constexpr int kVec = kVec_, kSlots = kSlots_, kPairs = kVec * kSlots;
  static constexpr bool kFull = kFull_, kInterleaved = kInterleaved_;
  using RawT = RawPairs<T, kVec, kSlots>;
  using Values = Pairs<kPairs>;

  int first[kSlots], at_a[kSlots], at_b[kSlots]; // the slot's first pair, and where its vectors sit in a row
  bool on[kSlots];
  // Beyond the rotated part the remaining values are paired up the same way and pass through.
  __device__ __forceinline__ Layout(const NormRopeParams &P, int lane) {
    const int half = P.rotary_dim >> 1;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int p = lane + s * P.lanes;
      on[s] = kFull || 2 * p * kVec < P.head_dim;
      first[s] = on[s] ? p * kVec : 0;
      if (kInterleaved) {
        at_a[s] = 2 * first[s];
        at_b[s] = at_a[s] + kVec;
      } else if (first[s] < half) {
        at_a[s] = first[s];
        at_b[s] = half + first[s];
      } else {
        at_a[s] = P.rotary_dim + (first[s] - half);
        at_b[s] = at_a[s] + ((P.head_dim - P.rotary_dim) >> 1);
      }
    }
  }
  __device__ __forceinline__ void load(const T *row, RawT &v) const {
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (on[s]) {
        v.a[s] = __ldcs(reinterpret_cast<const typename RawT::R *>(row + at_a[s]));
        v.b[s] = __ldcs(reinterpret_cast<const typename RawT::R *>(row + at_b[s]));
      }
  }
  __device__ __forceinline__ void store(T *row, const RawT &v) const {
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (on[s]) {
        *reinterpret_cast<typename RawT::R *>(row + at_a[s]) = v.a[s];
        *reinterpret_cast<typename RawT::R *>(row + at_b[s]) = v.b[s];
      }
  }
  // Zeros for slots that are off.
  __device__ __forceinline__ void widen(const RawT &v, Values &x) const {
    float a[kPairs], b[kPairs];
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      float y[2 * kVec]; // the values of a, then of b
      if constexpr (sizeof(T) == 4) {
        const float *pa = reinterpret_cast<const float *>(&v.a[s]), *pb = reinterpret_cast<const float *>(&v.b[s]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[i] = pa[i], y[kVec + i] = pb[i];
      } else if constexpr (kVec == 1) {
        y[0] = unpack(v.a[s], T()).x;
        y[1] = unpack(v.b[s], T()).x;
      } else {
        const uint32_t *pa = reinterpret_cast<const uint32_t *>(&v.a[s]), *pb = reinterpret_cast<const uint32_t *>(&v.b[s]);
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
          const float2 p = unpack(pa[i], T()), q = unpack(pb[i], T());
          y[2 * i] = p.x, y[2 * i + 1] = p.y, y[kVec + 2 * i] = q.x, y[kVec + 2 * i + 1] = q.y;
        }
      }
      const bool keep = kFull || on[s];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        a[s * kVec + i] = keep ? y[kInterleaved ? 2 * i : i] : 0.f;
        b[s * kVec + i] = keep ? y[kInterleaved ? 2 * i + 1 : kVec + i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      x.a[i] = make_float2(a[2 * i], a[2 * i + 1]);
      x.b[i] = make_float2(b[2 * i], b[2 * i + 1]);
    }
  }
  // The one rounding to the tensors' type.
  __device__ __forceinline__ void narrow(const Values &x, RawT &v) const {
    float a[kPairs], b[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      a[2 * i] = x.a[i].x, a[2 * i + 1] = x.a[i].y;
      b[2 * i] = x.b[i].x, b[2 * i + 1] = x.b[i].y;
    }
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      float y[2 * kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        y[kInterleaved ? 2 * i : i] = a[s * kVec + i];
        y[kInterleaved ? 2 * i + 1 : kVec + i] = b[s * kVec + i];
      }
      if constexpr (sizeof(T) == 4) {
        float *pa = reinterpret_cast<float *>(&v.a[s]), *pb = reinterpret_cast<float *>(&v.b[s]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) pa[i] = y[i], pb[i] = y[kVec + i];
      } else if constexpr (kVec == 1) {
        v.a[s] = static_cast<uint16_t>(pack(y[0], 0.f, T()));
        v.b[s] = static_cast<uint16_t>(pack(y[1], 0.f, T()));
      } else {
        uint32_t *pa = reinterpret_cast<uint32_t *>(&v.a[s]), *pb = reinterpret_cast<uint32_t *>(&v.b[s]);
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) pa[i] = pack(y[2 * i], y[2 * i + 1], T()), pb[i] = pack(y[kVec + 2 * i], y[kVec + 2 * i + 1], T());
      }
    }
  }
  __device__ __forceinline__ int at(int s, int i, bool second) const {
    return kInterleaved ? at_a[s] + 2 * i + second : (second ? at_b[s] : at_a[s]) + i;
  }
  // This lane's values out of two tables by pair (cos and sin of a token; the weights of both values).
  __device__ __forceinline__ void look_up(const float *cs, const float *sn, float2 (&c)[kPairs / 2], float2 (&s)[kPairs / 2]) const {
    float fc[kPairs], fs[kPairs];
#pragma unroll
    for (int x = 0; x < kSlots; ++x) {
      if constexpr (kVec % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kVec; i += 4) {
          *reinterpret_cast<float4 *>(&fc[x * kVec + i]) = *reinterpret_cast<const float4 *>(cs + first[x] + i);
          *reinterpret_cast<float4 *>(&fs[x * kVec + i]) = *reinterpret_cast<const float4 *>(sn + first[x] + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          fc[x * kVec + i] = cs[first[x] + i];
          fs[x * kVec + i] = sn[first[x] + i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      c[i] = make_float2(fc[2 * i], fc[2 * i + 1]);
      s[i] = make_float2(fs[2 * i], fs[2 * i + 1]);
    }
  }
  // Turns the pairs by their angles (`sign` -1: back). Pairs from `half` on stay exactly as they are.
  template <int sign> __device__ __forceinline__ void rotate(Values &x, const float2 (&c)[kPairs / 2], const float2 (&s)[kPairs / 2], int half) const {
    if (kSlots == 1 && first[0] >= half) return;
    const bool all = kSlots == 1 && first[0] + kVec <= half;
    const Values old = x;
#pragma unroll
    for (int i = 0; i < kPairs / 2; ++i) {
      const float2 p = x.a[i], q = x.b[i];
      const float2 qs = __fmul2_rn(q, s[i]), ps = __fmul2_rn(p, s[i]);
      if (sign > 0) {
        x.a[i] = make_float2(fmaf(p.x, c[i].x, -qs.x), fmaf(p.y, c[i].y, -qs.y));
        x.b[i] = __ffma2_rn(q, c[i], ps);
      } else {
        x.a[i] = __ffma2_rn(p, c[i], qs);
        x.b[i] = make_float2(fmaf(q.x, c[i].x, -ps.x), fmaf(q.y, c[i].y, -ps.y));
      }
    }
    if (!all) { // a lane that holds pairs of both kinds
#pragma unroll
      for (int i = 0; i < kPairs / 2; ++i) {
        const bool x0 = first[2 * i / kVec] + 2 * i % kVec < half, x1 = first[(2 * i + 1) / kVec] + (2 * i + 1) % kVec < half;
        x.a[i] = make_float2(x0 ? x.a[i].x : old.a[i].x, x1 ? x.a[i].y : old.a[i].y);
        x.b[i] = make_float2(x0 ? x.b[i].x : old.b[i].x, x1 ? x.b[i].y : old.b[i].y);
      }
    }
  }
};

// The sum over the row's lanes (a power of two, aligned inside the warp), the same bits in every lane.
__device__ __forceinline__ float group_sum(float v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int kPairs> __device__ __forceinline__ float dot(const Pairs<kPairs> &x, const Pairs<kPairs> &y) {
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kPairs / 2; ++i) {
    s = __ffma2_rn(x.a[i], y.a[i], s);
    s = __ffma2_rn(x.b[i], y.b[i], s);
  }
  return s.x + s.y;
}

// cos and sin of every pair of the tile's tokens, (1, 0) past the rotated part.
// For 16-bit rows sin and cos come from the special-function units (error below 2^-21 of 1 in [-pi, pi], where the
// outputs keep 2^-12 at best); with few heads the angles are most of the work (32768 tokens x 9 heads 98 -> 51 us).
template <typename T>
__device__ __forceinline__ void fill_angles(const NormRopeParams &P, int64_t token0, int tokens, float *cs, float *sn) {
  const int pairs = P.head_dim >> 1, half = P.rotary_dim >> 1;
  for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const int t = i / pairs, j = i - t * pairs;
    float c = 1.f, s = 0.f;
    if (j < half) {
      const double turns = static_cast<double>(P.positions[token0 + t]) * static_cast<double>(P.inv_freq[j]) * 0.31830988618379067154;
      const float rest = static_cast<float>(turns - 2.0 * rint(0.5 * turns));
      if (sizeof(T) == 4) sincospif(rest, &s, &c);
      else __sincosf(rest * 3.14159265358979f, &s, &c);
    }
    cs[i] = c;
    sn[i] = s;
  }
}

// The block's weight into shared memory, by pair; a null one is all ones. The barrier is the caller's first.
template <bool kInterleaved> __device__ __forceinline__ void fetch_weight(const float *w, const NormRopeParams &P, float (*to)[128]) {
  const int half = P.rotary_dim >> 1;
  for (int j = threadIdx.x; j < P.head_dim >> 1; j += kThreads) {
    const int a = kInterleaved ? 2 * j : j < half ? j : P.rotary_dim + j - half;
    const int b = kInterleaved ? 2 * j + 1 : a + (j < half ? half : (P.head_dim - P.rotary_dim) >> 1);
    to[0][j] = w != nullptr ? w[a] : 1.f;
    to[1][j] = w != nullptr ? w[b] : 1.f;
  }
}

// A block's part of the work: which rows, and of them which tiles. Its groups of lanes walk the rows of a tile:
// group, group + groups, ...; a row is (token of the tile, head).
struct Share {
  int kind, heads, tile, block, blocks; // kind 0 queries, 1 keys, 2 values
  int groups, group, lane;
  int token_step, head_step, token_first, head_first;
  __device__ __forceinline__ Share(const NormRopeParams &P) {
    block = blockIdx.x;
    kind = 0;
    while (block >= P.blocks[kind]) block -= P.blocks[kind++];
    heads = kind == 0 ? P.q_heads : P.k_heads;
    tile = P.tile[kind];
    blocks = P.blocks[kind];
    groups = kThreads / P.lanes;
    group = threadIdx.x / P.lanes;
    lane = threadIdx.x % P.lanes;
    token_step = groups / heads;
    head_step = groups % heads;
    token_first = group / heads;
    head_first = group % heads;
  }
};
// A group's walk through the rows of a tile.
struct Place {
  int token, head;
  __device__ __forceinline__ Place(const Share &me) : token(me.token_first), head(me.head_first) {}
  __device__ __forceinline__ void next(const Share &me) {
    token += me.token_step;
    head += me.head_step;
    if (head >= me.heads) {
      head -= me.heads;
      ++token;
    }
  }
  template <typename T> __device__ __forceinline__ T *in(T *base, const HeadRows &rows) const { return base + token * rows.token_stride + head * rows.head_stride; }
};
template <typename T> __device__ __forceinline__ T *tile_of(const HeadRows &rows, int64_t token0) {
  return reinterpret_cast<T *>(rows.data) + token0 * rows.token_stride;
}

template <typename L, bool kAppend> __device__ __forceinline__ void forward_body(const NormRopeParams &P, const AppendParams &A) {
  using T = typename L::T;
  __shared__ __align__(16) float s_cos[2][kMaxAngles], s_sin[2][kMaxAngles];
  __shared__ __align__(16) float s_weight[2][128];
  __shared__ int64_t s_place[2][kAppend ? kMaxAngles : 1]; // where the token's rows go in the cache (INT64_MIN: nowhere)
  const Share me(P);
  const L lay(P, me.lane);
  const int half = P.rotary_dim >> 1, pairs = P.head_dim >> 1;
  const float scale = 1.f / static_cast<float>(P.head_dim);
  khd::grid_dependency_wait();
  khd::grid_dependents_may_launch();
  const HeadRows in = me.kind == 0 ? P.q : me.kind == 1 ? P.k : A.v;
  const HeadRows out = me.kind == 0 ? P.q_out : P.k_out;
  const PagedRows cache = me.kind == 1 ? A.k_cache : A.v_cache;
  fetch_weight<L::kInterleaved>(me.kind == 0 ? P.q_weight : P.k_weight, P, s_weight);
  const int64_t tiles = (P.tokens + me.tile - 1) / me.tile;
  int buffer = 0;
  for (int64_t tile = me.block; tile < tiles; tile += me.blocks, buffer ^= 1) {
    const int64_t token0 = tile * me.tile;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(me.tile), P.tokens - token0)), rows = tokens * me.heads;
    typename L::RawT raw[2]; // the next row and the one after it
    T *const in_tile = tile_of<T>(in, token0), *const out_tile = tile_of<T>(out, token0);
    Place at(me), ahead(me);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (me.group + i * me.groups < rows) lay.load(ahead.in(in_tile, in), raw[i]);
      ahead.next(me);
    }
    if (kAppend && me.kind > 0) {
      for (int i = threadIdx.x; i < tokens; i += kThreads) {
        const int64_t slot = A.slots[token0 + i];
        int64_t place = INT64_MIN;
        if (slot >= 0 && slot < A.num_slots) {
          const int64_t page = slot < (int64_t{1} << 31) ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(A.page_size) : slot / A.page_size;
          place = page * cache.page_stride + (slot - page * A.page_size) * cache.slot_stride;
        } else if (slot != -1) { // nothing is stored for this token, and the host is told
          khd::report_status(A.status, khd::kStatusBadSlot, static_cast<uint32_t>(token0 + i));
        }
        s_place[buffer][i] = place;
      }
    }
    if (me.kind < 2) fill_angles<T>(P, token0, tokens, s_cos[buffer], s_sin[buffer]);
    __syncthreads(); // the other buffers' readers passed the barrier before this one
    // every lane of a warp makes the same number of turns, so that the shuffles are always complete
    for (int r0 = 0; r0 < rows; r0 += me.groups) {
      const bool mine = r0 + me.group < rows;
      typename L::RawT cur = raw[0];
      raw[0] = raw[1];
      if (r0 + 2 * me.groups + me.group < rows) lay.load(ahead.in(in_tile, in), raw[1]);
      ahead.next(me);
      if (!kAppend || me.kind < 2) {
        typename L::Values x;
        lay.widen(cur, x); // (a group without a row works on what its registers hold, among its own lanes)
        const float r = rsqrtf(fmaf(group_sum(dot(x, x), P.lanes), scale, P.eps));
        if (mine) {
          float2 c[L::kPairs / 2], s[L::kPairs / 2];
          lay.look_up(s_cos[buffer] + at.token * pairs, s_sin[buffer] + at.token * pairs, c, s);
          typename L::Values w;
          lay.look_up(s_weight[0], s_weight[1], w.a, w.b);
          const float2 r2 = make_float2(r, r);
#pragma unroll
          for (int i = 0; i < L::kPairs / 2; ++i) {
            x.a[i] = __fmul2_rn(__fmul2_rn(x.a[i], r2), w.a[i]);
            x.b[i] = __fmul2_rn(__fmul2_rn(x.b[i], r2), w.b[i]);
          }
          lay.template rotate<1>(x, c, s, half);
          lay.narrow(x, cur);
        }
      }
      if (mine) {
        if (!kAppend || me.kind == 0) {
          lay.store(at.in(out_tile, out), cur);
        } else if (const int64_t place = s_place[buffer][at.token]; place != INT64_MIN) {
          lay.store(reinterpret_cast<T *>(cache.data) + place + at.head * cache.head_stride, cur);
        }
      }
      at.next(me);
    }
  }
}

// Backward. Every lane keeps the weight gradients of its own values in fp32 registers over all its rows. At the end
// the block adds its groups' sums in a fixed order into one row of `partials`, which qk_norm_weight_grad adds up
// over the blocks, again in a fixed order: no atomics, the same bits every time.
template <typename L> __device__ __forceinline__ void backward_body(const NormRopeParams &P, const BackwardParams &B) {
  using T = typename L::T;
  __shared__ __align__(16) float s_cos[2][kMaxAngles], s_sin[2][kMaxAngles];
  __shared__ __align__(16) float s_weight[2][128];
  __shared__ float s_sum[kThreads / 32][256];
  const Share me(P);
  const L lay(P, me.lane);
  const int half = P.rotary_dim >> 1, pairs = P.head_dim >> 1;
  const float scale = 1.f / static_cast<float>(P.head_dim);
  khd::grid_dependency_wait();
  khd::grid_dependents_may_launch();
  const HeadRows in = me.kind == 0 ? P.q : P.k, grad = me.kind == 0 ? B.dq_out : B.dk_out, out = me.kind == 0 ? P.q_out : P.k_out;
  fetch_weight<L::kInterleaved>(me.kind == 0 ? P.q_weight : P.k_weight, P, s_weight);
  typename L::Values sum;
#pragma unroll
  for (int i = 0; i < L::kPairs / 2; ++i) sum.a[i] = sum.b[i] = make_float2(0.f, 0.f);
  const int64_t tiles = (P.tokens + me.tile - 1) / me.tile;
  int buffer = 0;
  for (int64_t tile = me.block; tile < tiles; tile += me.blocks, buffer ^= 1) {
    const int64_t token0 = tile * me.tile;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(me.tile), P.tokens - token0)), rows = tokens * me.heads;
    typename L::RawT raw, draw;
    T *const in_tile = tile_of<T>(in, token0), *const grad_tile = tile_of<T>(grad, token0), *const out_tile = tile_of<T>(out, token0);
    Place at(me), ahead(me);
    if (me.group < rows) {
      lay.load(ahead.in(in_tile, in), raw);
      lay.load(ahead.in(grad_tile, grad), draw);
    }
    fill_angles<T>(P, token0, tokens, s_cos[buffer], s_sin[buffer]);
    __syncthreads(); // the other buffer's readers passed the barrier before this one
    for (int r0 = 0; r0 < rows; r0 += me.groups) {
      const bool mine = r0 + me.group < rows;
      typename L::Values u, g;
      lay.widen(raw, u); // (a group without a row works on what its registers hold, among its own lanes)
      lay.widen(draw, g);
      ahead.next(me);
      if (r0 + me.groups + me.group < rows) {
        lay.load(ahead.in(in_tile, in), raw);
        lay.load(ahead.in(grad_tile, grad), draw);
      }
      const float r = rsqrtf(fmaf(group_sum(dot(u, u), P.lanes), scale, P.eps));
      const float2 r2 = make_float2(r, r);
      float2 c[L::kPairs / 2], s[L::kPairs / 2];
      const int table = (mine ? at.token : 0) * pairs;
      lay.look_up(s_cos[buffer] + table, s_sin[buffer] + table, c, s);
      lay.template rotate<-1>(g, c, s, half);
      typename L::Values w;
      lay.look_up(s_weight[0], s_weight[1], w.a, w.b);
#pragma unroll
      for (int i = 0; i < L::kPairs / 2; ++i) {
        u.a[i] = __fmul2_rn(u.a[i], r2);
        u.b[i] = __fmul2_rn(u.b[i], r2);
        if (mine) {
          sum.a[i] = __ffma2_rn(g.a[i], u.a[i], sum.a[i]);
          sum.b[i] = __ffma2_rn(g.b[i], u.b[i], sum.b[i]);
        }
        g.a[i] = __fmul2_rn(g.a[i], w.a[i]);
        g.b[i] = __fmul2_rn(g.b[i], w.b[i]);
      }
      const float mean = group_sum(dot(g, u), P.lanes) * scale;
      if (mine) {
        const float2 m2 = make_float2(-mean, -mean);
#pragma unroll
        for (int i = 0; i < L::kPairs / 2; ++i) {
          g.a[i] = __fmul2_rn(__ffma2_rn(u.a[i], m2, g.a[i]), r2);
          g.b[i] = __fmul2_rn(__ffma2_rn(u.b[i], m2, g.b[i]), r2);
        }
        typename L::RawT res;
        lay.narrow(g, res);
        lay.store(at.in(out_tile, out), res);
      }
      at.next(me);
    }
  }
  // groups of a warp first (shuffles over the lanes that hold the same values), then the eight warps
#pragma unroll
  for (int i = 0; i < L::kPairs; ++i) {
    float a = i & 1 ? sum.a[i / 2].y : sum.a[i / 2].x, b = i & 1 ? sum.b[i / 2].y : sum.b[i / 2].x;
    for (int o = P.lanes; o < 32; o <<= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if ((threadIdx.x & 31) < P.lanes && lay.on[i / L::kVec]) {
      s_sum[threadIdx.x >> 5][lay.at(i / L::kVec, i % L::kVec, false)] = a;
      s_sum[threadIdx.x >> 5][lay.at(i / L::kVec, i % L::kVec, true)] = b;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < P.head_dim; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int x = 0; x < kThreads / 32; ++x) v += s_sum[x][i];
    B.partials[static_cast<int64_t>(blockIdx.x) * P.head_dim + i] = v;
  }
}

} // namespace

#define KH_NORM_ROPE_PAIRING(suffix, T, vec, slots, full, pairing)                                                      \
  extern "C" __global__ void __launch_bounds__(kThreads, kForwardBlocks<T>)                                                             \
  qk_norm_rope_##suffix(const __grid_constant__ NormRopeParams P) {                                                     \
    forward_body<Layout<T, vec, slots, full, pairing>, false>(P, AppendParams{});                                       \
  }                                                                                                                     \
  extern "C" __global__ void __launch_bounds__(kThreads, kForwardBlocks<T>)                                                             \
  qk_norm_rope_append_##suffix(const __grid_constant__ NormRopeParams P, const __grid_constant__ AppendParams A) {      \
    forward_body<Layout<T, vec, slots, full, pairing>, true>(P, A);                                                     \
  }                                                                                                                     \
  extern "C" __global__ void __launch_bounds__(kThreads, kBackwardBlocks<T>)                                                             \
  qk_norm_rope_backward_##suffix(const __grid_constant__ NormRopeParams P, const __grid_constant__ BackwardParams B) {  \
    backward_body<Layout<T, vec, slots, full, pairing>>(P, B);                                                          \
  }
#define KH_NORM_ROPE(suffix, T, vec, slots, full)                \
  KH_NORM_ROPE_PAIRING(suffix##_halves, T, vec, slots, full, false) \
  KH_NORM_ROPE_PAIRING(suffix##_inter, T, vec, slots, full, true)

// 16-byte vectors (full: and no idle lane); 8-byte ones for halves of a rotation, or addresses, that 16 bytes do not
// divide; single values (four pairs per lane) for everything else.
KH_NORM_ROPE(f32_v4_full, float, 4, 1, true)
KH_NORM_ROPE(f32_v4, float, 4, 1, false)
KH_NORM_ROPE(f32_v2, float, 2, 1, false)
KH_NORM_ROPE(f32_v1, float, 1, 4, false)
KH_NORM_ROPE(bf16_v8_full, __nv_bfloat16, 8, 1, true)
KH_NORM_ROPE(bf16_v8, __nv_bfloat16, 8, 1, false)
KH_NORM_ROPE(bf16_v4, __nv_bfloat16, 4, 1, false)
KH_NORM_ROPE(bf16_v1, __nv_bfloat16, 1, 4, false)
KH_NORM_ROPE(f16_v8_full, __half, 8, 1, true)
KH_NORM_ROPE(f16_v8, __half, 8, 1, false)
KH_NORM_ROPE(f16_v4, __half, 4, 1, false)
KH_NORM_ROPE(f16_v1, __half, 1, 4, false)

// dw[k][i] = the sum of partials[block][i] over the blocks of queries (k = 0) or keys: a warp per 32 columns and
// eighth of the blocks, the eighths added in order.
extern "C" __global__ void __launch_bounds__(256) qk_norm_weight_grad(const __grid_constant__ WeightGradParams P) {
  __shared__ float part[8][32];
  khd::grid_dependency_wait();
  const int k = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  const float *from = P.partials + static_cast<int64_t>(k == 0 ? 0 : P.blocks[0]) * P.head_dim;
  float v = 0.f;
  if (col < P.head_dim)
#pragma unroll 8
    for (int b = w; b < P.blocks[k]; b += 8) v += from[static_cast<int64_t>(b) * P.head_dim + col];
  part[w][threadIdx.x & 31] = v;
  __syncthreads();
  float *out = k == 0 ? P.dq_weight : P.dk_weight;
  if (w != 0 || col >= P.head_dim || out == nullptr) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += part[i][threadIdx.x];
  out[col] = sum;
}
