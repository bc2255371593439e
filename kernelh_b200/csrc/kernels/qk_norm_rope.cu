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
// Angles: position * inv_freq in half turns, formed and reduced in 64 bits (a position of 10^6 times a
// frequency of 1 has 20 bits before the point, fp32 would keep 4 after it), the remainder in [-1, 1]
// rounded to fp32 for sincospif. They are worked out once per token by the whole block into shared memory
// and shared by all its heads: 50 instructions each, which every head on its own would pay again.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kh_device.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;      // head_dim up to 256
constexpr int kMaxTokensPerTile = 4;

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
  int32_t interleaved, lanes, tile_tokens;
  float eps;
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
  float *partials;         // [gridDim.x][2][head_dim]
};
struct WeightGradParams {
  const float *partials;
  float *dq_weight, *dk_weight; // either may be nullptr
  int32_t blocks, head_dim;
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// kVec values of one access: 16, 8, 4 or 2 bytes.
template <int kBytes> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

template <typename T, int kVec> struct Vec {
  using R = typename Raw<sizeof(T) * kVec>::type;
  union {
    R raw;
    T v[kVec];
  };
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ void load(const T *p) { raw = __ldcs(reinterpret_cast<const R *>(p)); }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<R *>(p) = raw; }
};

// The sum over the row's lanes (a power of two, aligned inside the warp), the same bits in every lane.
__device__ __forceinline__ float group_sum(float v, int lanes) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Where the two vectors of pair-vector `p` (pairs p * kVec ..) sit in a row. Beyond the rotated part the
// remaining values are paired up the same way and pass through.
template <int kVec> __device__ __forceinline__ void pair_offsets(int p, const NormRopeParams &P, int &a, int &b) {
  if (P.interleaved) {
    a = 2 * p * kVec;
    b = a + kVec;
    return;
  }
  const int half = P.rotary_dim >> 1, first = p * kVec;
  if (first < half) {
    a = first;
    b = half + first;
  } else {
    a = P.rotary_dim + (first - half);
    b = a + ((P.head_dim - P.rotary_dim) >> 1);
  }
}

// cos and sin of every pair of the tile's tokens, (1, 0) past the rotated part. The sine's sign is the caller's.
__device__ __forceinline__ void fill_angles(const NormRopeParams &P, int64_t token0, float (*cs)[kMaxPairs], float (*sn)[kMaxPairs]) {
  const int pairs = P.head_dim >> 1, half = P.rotary_dim >> 1;
  for (int i = threadIdx.x; i < P.tile_tokens * pairs; i += kThreads) {
    const int t = i / pairs, j = i - t * pairs;
    float c = 1.f, s = 0.f;
    if (j < half && token0 + t < P.tokens) {
      const double turns = static_cast<double>(P.positions[token0 + t]) * static_cast<double>(P.inv_freq[j]) * 0.31830988618379067154;
      sincospif(static_cast<float>(turns - 2.0 * rint(0.5 * turns)), &s, &c);
    }
    cs[t][j] = c;
    sn[t][j] = s;
  }
}

// n = x r w for one row: `a` and `b` hold the raw pair vectors on entry, xa / xb their values x and the result is r.
template <typename T, int kVec, int kSlots>
__device__ __forceinline__ float row_rms(const Vec<T, kVec> (&a)[kSlots], const Vec<T, kVec> (&b)[kSlots], const bool (&on)[kSlots],
                                         const NormRopeParams &P, float (&xa)[kSlots][kVec], float (&xb)[kSlots][kVec]) {
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      xa[s][i] = on[s] ? to_float(a[s].v[i]) : 0.f;
      xb[s][i] = on[s] ? to_float(b[s].v[i]) : 0.f;
      sum = fmaf(xa[s][i], xa[s][i], sum);
      sum = fmaf(xb[s][i], xb[s][i], sum);
    }
  return rsqrtf(group_sum(sum, P.lanes) / static_cast<float>(P.head_dim) + P.eps);
}

// (a, b) turned by (c, s) pairwise, in place. Interleaved pairs lie in one vector: the i-th pair of the
// 2 kVec contiguous values is (value 2i, value 2i + 1). Pairs from `half` on stay as they are.
template <int kVec>
__device__ __forceinline__ void rotate(float (&a)[kVec], float (&b)[kVec], const float (&c)[kVec], const float (&s)[kVec], int first,
                                       int half, bool interleaved) {
  if (!interleaved) {
    if (first >= half) return;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = x * s[i] + y * c[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    float &ra = 2 * i < kVec ? a[(2 * i) % kVec] : b[(2 * i) % kVec];
    float &rb = 2 * i + 1 < kVec ? a[(2 * i + 1) % kVec] : b[(2 * i + 1) % kVec];
    if (first + i < half) {
      const float x = ra, y = rb;
      ra = x * c[i] - y * s[i];
      rb = x * s[i] + y * c[i];
    }
  }
}

template <typename T, int kVec, int kSlots>
__device__ __forceinline__ void load_row(Vec<T, kVec> (&a)[kSlots], Vec<T, kVec> (&b)[kSlots], const HeadRows &rows, int64_t token,
                                         int head, const int (&at_a)[kSlots], const int (&at_b)[kSlots], const bool (&on)[kSlots]) {
  const T *p = reinterpret_cast<const T *>(rows.data) + token * rows.token_stride + head * rows.head_stride;
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
    if (on[s]) {
      a[s].load(p + at_a[s]);
      b[s].load(p + at_b[s]);
    }
}

// The geometry of a lane: kSlots pair vectors `lane + s * lanes`, of which those inside the row are on.
template <int kVec, int kSlots> struct LaneMap {
  int first[kSlots], at_a[kSlots], at_b[kSlots];
  bool on[kSlots];
  __device__ __forceinline__ LaneMap(const NormRopeParams &P, int lane) {
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int p = lane + s * P.lanes;
      on[s] = 2 * p * kVec < P.head_dim;
      first[s] = on[s] ? p * kVec : 0;
      pair_offsets<kVec>(on[s] ? p : 0, P, at_a[s], at_b[s]);
    }
  }
};

// Weights of the lane's values: wa[s][i] belongs to offset at_a[s] + i. A null weight is all ones.
template <int kVec, int kSlots>
__device__ __forceinline__ void load_weights(const float *w, const LaneMap<kVec, kSlots> &m, float (&wa)[kSlots][kVec], float (&wb)[kSlots][kVec]) {
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      wa[s][i] = w != nullptr && m.on[s] ? __ldg(w + m.at_a[s] + i) : 1.f;
      wb[s][i] = w != nullptr && m.on[s] ? __ldg(w + m.at_b[s] + i) : 1.f;
    }
}

// Forward. A block takes tile_tokens tokens; its lane groups are dealt out to the tokens evenly and a group
// walks the heads of its token (queries, keys, and the values when they are appended) with its cosines in
// registers, the next row's loads in flight while it works on the current one.
template <typename T, int kVec, int kSlots, bool kAppend>
__device__ __forceinline__ void forward_body(const NormRopeParams &P, const AppendParams &A) {
  __shared__ float s_cos[kMaxTokensPerTile][kMaxPairs], s_sin[kMaxTokensPerTile][kMaxPairs];
  const int groups_per_token = kThreads / P.lanes / P.tile_tokens;
  const int group = threadIdx.x / P.lanes, lane = threadIdx.x % P.lanes;
  const int t = group / groups_per_token;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * P.tile_tokens;
  const int64_t token = token0 + t;
  const int heads = P.q_heads + P.k_heads + (kAppend ? P.k_heads : 0);
  const LaneMap<kVec, kSlots> m(P, lane);
  khd::grid_dependency_wait();
  khd::grid_dependents_may_launch();

  const bool live = token < P.tokens;
  Vec<T, kVec> a[kSlots], b[kSlots];
  const auto fetch = [&](int head) {
    if (head < P.q_heads) load_row<T, kVec, kSlots>(a, b, P.q, token, head, m.at_a, m.at_b, m.on);
    else if (head < P.q_heads + P.k_heads) load_row<T, kVec, kSlots>(a, b, P.k, token, head - P.q_heads, m.at_a, m.at_b, m.on);
    else if (kAppend) load_row<T, kVec, kSlots>(a, b, A.v, token, head - P.q_heads - P.k_heads, m.at_a, m.at_b, m.on);
  };
  int head = group % groups_per_token;
  if (live && head < heads) fetch(head);

  int64_t slot = -1, page = 0;
  int in_page = 0;
  if (kAppend && live) {
    slot = __ldg(A.slots + token);
    if (slot < -1 || slot >= A.num_slots) { // nothing is stored for this token, and the host is told
      if (lane == 0) khd::report_status(A.status, khd::kStatusBadSlot, static_cast<uint32_t>(token));
      slot = -1;
    }
    if (slot >= 0) {
      page = slot / A.page_size;
      in_page = static_cast<int>(slot - page * A.page_size);
    }
  }
  fill_angles(P, token0, s_cos, s_sin);
  __syncthreads();
  float c[kSlots][kVec], s[kSlots][kVec];
#pragma unroll
  for (int x = 0; x < kSlots; ++x)
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      c[x][i] = s_cos[t][m.first[x] + i];
      s[x][i] = s_sin[t][m.first[x] + i];
    }
  float wa[kSlots][kVec], wb[kSlots][kVec];
  int have = -1; // whose weights are in the registers: 0 queries, 1 keys
  const int half = P.rotary_dim >> 1;
  // every lane of a warp walks the same number of rows, so that the shuffles are always complete
  for (int h0 = 0; h0 < heads; h0 += groups_per_token, head += groups_per_token) {
    const bool mine = live && head < heads;
    const int kind = head < P.q_heads ? 0 : (head < P.q_heads + P.k_heads ? 1 : 2);
    Vec<T, kVec> oa[kSlots], ob[kSlots];
    float xa[kSlots][kVec], xb[kSlots][kVec];
    bool used[kSlots];
#pragma unroll
    for (int x = 0; x < kSlots; ++x) {
      used[x] = mine && m.on[x];
      oa[x] = a[x];
      ob[x] = b[x];
    }
    if (live && head + groups_per_token < heads) fetch(head + groups_per_token);
    const float r = row_rms<T, kVec, kSlots>(oa, ob, used, P, xa, xb);
    if (!mine) continue;
    if (kind < 2) {
      if (kind != have) {
        load_weights<kVec, kSlots>(kind == 0 ? P.q_weight : P.k_weight, m, wa, wb);
        have = kind;
      }
#pragma unroll
      for (int x = 0; x < kSlots; ++x) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          xa[x][i] = xa[x][i] * r * wa[x][i];
          xb[x][i] = xb[x][i] * r * wb[x][i];
        }
        rotate<kVec>(xa[x], xb[x], c[x], s[x], m.first[x], half, P.interleaved != 0);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          oa[x].v[i] = from_float<T>(xa[x][i]); // the one rounding to the tensors' type
          ob[x].v[i] = from_float<T>(xb[x][i]);
        }
      }
    }
    T *out;
    if (kind == 0) {
      out = reinterpret_cast<T *>(P.q_out.data) + token * P.q_out.token_stride + head * P.q_out.head_stride;
    } else if (!kAppend) {
      out = reinterpret_cast<T *>(P.k_out.data) + token * P.k_out.token_stride + (head - P.q_heads) * P.k_out.head_stride;
    } else {
      if (slot < 0) continue;
      const PagedRows &cache = kind == 1 ? A.k_cache : A.v_cache;
      const int at = head - P.q_heads - (kind == 2 ? P.k_heads : 0);
      out = reinterpret_cast<T *>(cache.data) + page * cache.page_stride + in_page * cache.slot_stride + at * cache.head_stride;
    }
#pragma unroll
    for (int x = 0; x < kSlots; ++x)
      if (m.on[x]) {
        oa[x].store(out + m.at_a[x]);
        ob[x].store(out + m.at_b[x]);
      }
  }
}

// Backward. A persistent grid: a block walks the tiles blockIdx.x, + gridDim.x, ... and every lane keeps the
// weight gradients of its own values, for queries and for keys, in fp32 registers over all its rows. At the
// end the block adds its groups' sums in a fixed order into one row of `partials`, which
// qk_norm_weight_grad adds up over the blocks, again in a fixed order: no atomics, the same bits every time.
template <typename T, int kVec, int kSlots> __device__ __forceinline__ void backward_body(const NormRopeParams &P, const BackwardParams &B) {
  __shared__ float s_cos[2][kMaxTokensPerTile][kMaxPairs], s_sin[2][kMaxTokensPerTile][kMaxPairs];
  __shared__ float s_sum[kThreads / 32][2][2 * kMaxPairs];
  const int groups_per_token = kThreads / P.lanes / P.tile_tokens;
  const int group = threadIdx.x / P.lanes, lane = threadIdx.x % P.lanes;
  const int t = group / groups_per_token;
  const int heads = P.q_heads + P.k_heads;
  const int half = P.rotary_dim >> 1;
  const LaneMap<kVec, kSlots> m(P, lane);
  float wsum[2][2][kSlots][kVec];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int x = 0; x < kSlots; ++x)
#pragma unroll
      for (int i = 0; i < kVec; ++i) wsum[k][0][x][i] = wsum[k][1][x][i] = 0.f;
  khd::grid_dependency_wait();
  khd::grid_dependents_may_launch();
  const int64_t tiles = (P.tokens + P.tile_tokens - 1) / P.tile_tokens;
  int buffer = 0;
  float wa[kSlots][kVec], wb[kSlots][kVec];
  int have = -1;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, buffer ^= 1) {
    const int64_t token0 = tile * P.tile_tokens, token = token0 + t;
    const bool live = token < P.tokens;
    Vec<T, kVec> a[kSlots], b[kSlots], da[kSlots], db[kSlots];
    const auto fetch = [&](int head) {
      const bool is_q = head < P.q_heads;
      const int at = is_q ? head : head - P.q_heads;
      load_row<T, kVec, kSlots>(a, b, is_q ? P.q : P.k, token, at, m.at_a, m.at_b, m.on);
      load_row<T, kVec, kSlots>(da, db, is_q ? B.dq_out : B.dk_out, token, at, m.at_a, m.at_b, m.on);
    };
    int head = group % groups_per_token;
    if (live && head < heads) fetch(head);
    fill_angles(P, token0, s_cos[buffer], s_sin[buffer]);
    __syncthreads(); // the other buffer's readers are past this barrier's predecessor before it is refilled
    float c[kSlots][kVec], s[kSlots][kVec];
#pragma unroll
    for (int x = 0; x < kSlots; ++x)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        c[x][i] = s_cos[buffer][t][m.first[x] + i];
        s[x][i] = -s_sin[buffer][t][m.first[x] + i]; // the inverse rotation
      }
    for (int h0 = 0; h0 < heads; h0 += groups_per_token, head += groups_per_token) {
      const bool mine = live && head < heads;
      const bool is_q = head < P.q_heads;
      float xa[kSlots][kVec], xb[kSlots][kVec], ga[kSlots][kVec], gb[kSlots][kVec];
      bool used[kSlots];
#pragma unroll
      for (int x = 0; x < kSlots; ++x) {
        used[x] = mine && m.on[x];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          ga[x][i] = used[x] ? to_float(da[x].v[i]) : 0.f;
          gb[x][i] = used[x] ? to_float(db[x].v[i]) : 0.f;
        }
      }
      const float r = row_rms<T, kVec, kSlots>(a, b, used, P, xa, xb);
      if (live && head + groups_per_token < heads) fetch(head + groups_per_token);
      if (mine && have != (is_q ? 0 : 1)) {
        have = is_q ? 0 : 1;
        load_weights<kVec, kSlots>(is_q ? P.q_weight : P.k_weight, m, wa, wb);
      }
      float dot = 0.f; // sum of g w u
#pragma unroll
      for (int x = 0; x < kSlots; ++x) {
        rotate<kVec>(ga[x], gb[x], c[x], s[x], m.first[x], half, P.interleaved != 0);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          xa[x][i] *= r; // u
          xb[x][i] *= r;
          const float va = ga[x][i] * xa[x][i], vb = gb[x][i] * xb[x][i];
          if (used[x]) {
            if (is_q) {
              wsum[0][0][x][i] += va;
              wsum[0][1][x][i] += vb;
            } else {
              wsum[1][0][x][i] += va;
              wsum[1][1][x][i] += vb;
            }
            dot = fmaf(va, wa[x][i], dot);
            dot = fmaf(vb, wb[x][i], dot);
          }
        }
      }
      const float mean = group_sum(dot, P.lanes) / static_cast<float>(P.head_dim);
      if (!mine) continue;
      const HeadRows &rows = is_q ? P.q_out : P.k_out;
      T *out = reinterpret_cast<T *>(rows.data) + token * rows.token_stride + (is_q ? head : head - P.q_heads) * rows.head_stride;
#pragma unroll
      for (int x = 0; x < kSlots; ++x)
        if (m.on[x]) {
          Vec<T, kVec> oa, ob;
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            oa.v[i] = from_float<T>(r * (ga[x][i] * wa[x][i] - xa[x][i] * mean));
            ob.v[i] = from_float<T>(r * (gb[x][i] * wb[x][i] - xb[x][i] * mean));
          }
          oa.store(out + m.at_a[x]);
          ob.store(out + m.at_b[x]);
        }
    }
  }
  // groups of a warp first (shuffles over the lanes that hold the same values), then the eight warps
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int x = 0; x < kSlots; ++x)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        float va = wsum[k][0][x][i], vb = wsum[k][1][x][i];
        for (int o = P.lanes; o < 32; o <<= 1) {
          va += __shfl_xor_sync(0xffffffffu, va, o);
          vb += __shfl_xor_sync(0xffffffffu, vb, o);
        }
        if ((threadIdx.x & 31) < P.lanes && m.on[x]) {
          s_sum[threadIdx.x >> 5][k][m.at_a[x] + i] = va;
          s_sum[threadIdx.x >> 5][k][m.at_b[x] + i] = vb;
        }
      }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * P.head_dim; i += kThreads) {
    const int k = i / P.head_dim, at = i - k * P.head_dim;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) v += s_sum[w][k][at];
    B.partials[(static_cast<int64_t>(blockIdx.x) * 2 + k) * P.head_dim + at] = v;
  }
}

} // namespace

#define KH_NORM_ROPE(suffix, T, vec, slots)                                                                              \
  extern "C" __global__ void __launch_bounds__(kThreads)                                                                \
  qk_norm_rope_##suffix(const __grid_constant__ NormRopeParams P) {                                                     \
    forward_body<T, vec, slots, false>(P, AppendParams{});                                                              \
  }                                                                                                                     \
  extern "C" __global__ void __launch_bounds__(kThreads)                                                                \
  qk_norm_rope_append_##suffix(const __grid_constant__ NormRopeParams P, const __grid_constant__ AppendParams A) {      \
    forward_body<T, vec, slots, true>(P, A);                                                                            \
  }                                                                                                                     \
  extern "C" __global__ void __launch_bounds__(kThreads)                                                                \
  qk_norm_rope_backward_##suffix(const __grid_constant__ NormRopeParams P, const __grid_constant__ BackwardParams B) {  \
    backward_body<T, vec, slots>(P, B);                                                                                 \
  }

// 16-byte vectors; 8-byte ones for halves of a rotation, or addresses, that 16 bytes do not divide; single
// values (four pairs per lane, 32 lanes) for everything else.
KH_NORM_ROPE(f32_v4, float, 4, 1)
KH_NORM_ROPE(f32_v2, float, 2, 1)
KH_NORM_ROPE(f32_v1, float, 1, 4)
KH_NORM_ROPE(bf16_v8, __nv_bfloat16, 8, 1)
KH_NORM_ROPE(bf16_v4, __nv_bfloat16, 4, 1)
KH_NORM_ROPE(bf16_v1, __nv_bfloat16, 1, 4)
KH_NORM_ROPE(f16_v8, __half, 8, 1)
KH_NORM_ROPE(f16_v4, __half, 4, 1)
KH_NORM_ROPE(f16_v1, __half, 1, 4)

// dw[k][i] = the sum over the blocks of partials[block][k][i]: a warp per 32 columns and eighth of the
// blocks, the eighths added in order.
extern "C" __global__ void __launch_bounds__(256) qk_norm_weight_grad(const __grid_constant__ WeightGradParams P) {
  __shared__ float part[8][32];
  khd::grid_dependency_wait();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float v = 0.f;
  if (col < 2 * P.head_dim)
    for (int b = w; b < P.blocks; b += 8) v += P.partials[static_cast<int64_t>(b) * 2 * P.head_dim + col];
  part[w][threadIdx.x & 31] = v;
  __syncthreads();
  if (w != 0 || col >= 2 * P.head_dim) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += part[i][threadIdx.x];
  const int k = col / P.head_dim, at = col - k * P.head_dim;
  float *out = k == 0 ? P.dq_weight : P.dk_weight;
  if (out != nullptr) out[at] = sum;
}
