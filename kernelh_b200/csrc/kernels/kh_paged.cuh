// What the kernels of attention over a paged cache share: the parameters, how a call's work is dealt out,
// and the buffers that partial results meet in.
//
// Rows. The queries of one sequence that share a key/value head (group = q_heads / k_heads of them per
// token) form rows: row r of head h is token r / group, query head h * group + r % group. A row block is
// kRows of them; a query head never needs a tile of its own, so a single token with 8 query heads per
// key/value head reads its keys and values once.
//
// Work. An item is (sequence, key/value head, row block) and takes n units of kUnit keys, n the same for all
// items of a sequence (its whole key range; the causal mask cuts the units at an item's end, which cost
// nothing). All units of all items form one line, and every worker (a block) takes an equal stretch of it,
// whatever the lengths are: a worker finishes the item it starts in, does whole ones, and leaves the last one
// to the next worker. Items that more than one worker touches leave (max, sum, unnormalised row) in the
// workspace: slot 2w + 1 for the worker that starts an item, 2w for those that continue it; a second launch
// adds them up in the order of the keys. The line is laid out from q_start and kv_len on the device, so a
// captured call follows lengths that change between replays.
#pragma once

#include "kh_device.cuh"

namespace khp {

// Layout shared with the host (registry/paged_attention_kernel.cpp). Strides in elements.
struct PagedParams {
  const char *q;
  int64_t q_token, q_head;
  char *o;
  int64_t o_token, o_head;
  const char *k;
  int64_t k_page, k_slot, k_head;
  const char *v;
  int64_t v_page, v_slot, v_head;
  const int32_t *table;
  int64_t table_stride;
  const int32_t *q_start, *kv_len;
  float *lse;       // [tokens, q_heads] or nullptr
  float *partial_o; // [2 * workers][rows of a block][padded head_dim]
  float2 *partial_ml;
  uint32_t *status;
  int32_t tokens, batch, q_heads, k_heads, group, head_dim, page_size, table_width, num_pages;
  int32_t causal, window;  // window 0: none
  int32_t workers, min_units;
  int32_t rows_above, rows_upto; // sequences with rows in (rows_above, rows_upto] are this launch's
  float scale_log2;              // scale * log2(e): scores are kept in exp2 units
};

struct Sequence {
  int q0, tokens, rows, kv; // first token, new tokens, tokens * group, keys
  int blocks, first_unit, units; // row blocks; the key units that any row sees
};

// The sequence's shape, with every offset forced into range (and reported when it was not).
template <int kRows, int kUnit> __device__ __forceinline__ Sequence sequence(const PagedParams &P, int b) {
  Sequence s;
  s.q0 = P.q_start[b];
  const int q1 = P.q_start[b + 1];
  s.kv = P.kv_len[b];
  const int64_t capacity = static_cast<int64_t>(P.table_width) * P.page_size;
  if (s.q0 < 0 || q1 < s.q0 || q1 > P.tokens || s.kv < 0 || s.kv > capacity) {
    khd::report_status(P.status, khd::kStatusBadPage, static_cast<uint32_t>(b));
    s.q0 = 0;
    s.tokens = 0;
    s.kv = 0;
  } else {
    s.tokens = q1 - s.q0;
  }
  const int64_t rows = static_cast<int64_t>(s.tokens) * P.group;
  s.rows = rows > P.rows_above && rows <= P.rows_upto ? static_cast<int>(rows) : 0;
  s.blocks = (s.rows + kRows - 1) / kRows;
  const int64_t first = P.window > 0 ? static_cast<int64_t>(s.kv) - s.tokens - P.window + 1 : 0;
  s.first_unit = first > 0 ? static_cast<int>(first / kUnit) : 0;
  s.units = max(1, (s.kv + kUnit - 1) / kUnit - s.first_unit); // an item without keys still has its zeros to write
  return s;
}
template <int kRows, int kUnit> __device__ __forceinline__ int64_t sequence_units(const PagedParams &P, int b) {
  const Sequence s = sequence<kRows, kUnit>(P, b);
  return static_cast<int64_t>(s.blocks) * s.units * P.k_heads;
}

// Row blocks are walked from both ends (0, last, 1, last - 1, ...): under the causal mask the work of two
// neighbours in that order adds up to the same.
__device__ __forceinline__ int block_of(int i, int blocks) { return i & 1 ? blocks - 1 - (i >> 1) : i >> 1; }

// The whole line and the place of one unit on it, worked out by the block together.
struct Line {
  int64_t total;
  int workers; // of which the first `workers` have any work
};
template <int kThreads> struct LineScratch {
  int64_t warp_sum[kThreads / 32];
  int64_t total, start;
  int b;
};

template <int kThreads> __device__ __forceinline__ int64_t block_scan(int64_t v, int64_t &inclusive, int64_t *warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  inclusive = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, inclusive, o);
    if (lane >= o) inclusive += x;
  }
  if (lane == 31) warp_sum[warp] = inclusive;
  __syncthreads();
  int64_t all = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = all;
    all += warp_sum[w];
  }
  inclusive += before;
  __syncthreads();
  return all;
}

template <int kThreads, int kRows, int kUnit>
__device__ __forceinline__ Line measure_line(const PagedParams &P, LineScratch<kThreads> &s) {
  int64_t mine = 0, inclusive;
  for (int b = threadIdx.x; b < P.batch; b += kThreads) mine += sequence_units<kRows, kUnit>(P, b);
  Line line;
  line.total = block_scan<kThreads>(mine, inclusive, s.warp_sum);
  const int64_t most = (line.total + P.min_units - 1) / P.min_units;
  line.workers = static_cast<int>(most < P.workers ? most : P.workers);
  return line;
}
// Where worker w's stretch begins (w = workers: the end of the line).
__device__ __forceinline__ int64_t stretch(const Line &line, int w) {
  return line.total / line.workers * w + line.total % line.workers * w / line.workers;
}
// The sequence that unit `at` (< total) belongs to, and where that sequence starts on the line.
template <int kThreads, int kRows, int kUnit>
__device__ __forceinline__ void locate(const PagedParams &P, int64_t at, LineScratch<kThreads> &s, int &b_out, int64_t &start) {
  int64_t before = 0;
  for (int base = 0; base < P.batch; base += kThreads) {
    const int b = base + static_cast<int>(threadIdx.x);
    const int64_t mine = b < P.batch ? sequence_units<kRows, kUnit>(P, b) : 0;
    int64_t inclusive;
    const int64_t all = block_scan<kThreads>(mine, inclusive, s.warp_sum);
    if (at < before + all) {
      if (mine > 0 && at >= before + inclusive - mine && at < before + inclusive) {
        s.b = b;
        s.start = before + inclusive - mine;
      }
      break;
    }
    before += all;
  }
  __syncthreads();
  b_out = s.b;
  start = s.start;
  __syncthreads();
}

// The item that worker w's stretch (w > 0) begins inside of, if no earlier stretch does, and its parts:
// part 0 in slot 2 (w - 1) + 1, part p in slot 2 (w - 1 + p).
struct Split {
  Sequence s;
  int h, row0, w, parts; // parts 0: nothing to add up here
  __device__ __forceinline__ int64_t slot(int p) const { return 2 * static_cast<int64_t>(w - 1 + p) + (p == 0 ? 1 : 0); }
};
template <int kThreads, int kRows, int kUnit> __device__ __forceinline__ Split find_split(const PagedParams &P, LineScratch<kThreads> &scratch) {
  Split x{};
  const Line line = measure_line<kThreads, kRows, kUnit>(P, scratch);
  x.w = blockIdx.x + 1;
  if (x.w >= line.workers) return x;
  const int64_t at = stretch(line, x.w);
  int b;
  int64_t start;
  locate<kThreads, kRows, kUnit>(P, at, scratch, b, start);
  x.s = sequence<kRows, kUnit>(P, b);
  const int64_t item = (at - start) / x.s.units; // head * blocks + place of the row block
  const int64_t begin = start + item * x.s.units, end = begin + x.s.units;
  if (begin == at || begin < stretch(line, x.w - 1)) return x; // nothing split here, or an earlier block's
  x.h = static_cast<int>(item / x.s.blocks);
  x.row0 = block_of(static_cast<int>(item - static_cast<int64_t>(x.h) * x.s.blocks), x.s.blocks) * kRows;
  int last = x.w; // the last worker with a part
  while (last + 1 < line.workers && stretch(line, last + 1) < end) ++last;
  x.parts = last - x.w + 2;
  return x;
}

// Adds up the parts of one row, for items with few rows and many parts: block (w - 1, y) takes row y of w's
// item. Its warps take every kThreads / 32-th part each with a running maximum and are added up in order.
template <typename T, int kThreads, int kRows, int kUnit, int kDim, typename Store>
__device__ __forceinline__ void combine_body(const PagedParams &P, Store store) {
  __shared__ LineScratch<kThreads> scratch;
  __shared__ float s_row[kThreads / 32][kDim];
  __shared__ float2 s_ml[kThreads / 32];
  khd::grid_dependency_wait();
  const Split x = find_split<kThreads, kRows, kUnit>(P, scratch);
  const Sequence &s = x.s;
  const int row = x.row0 + static_cast<int>(blockIdx.y), h = x.h, parts = x.parts;
  if (parts == 0 || static_cast<int>(blockIdx.y) >= kRows || row >= s.rows) return;
  constexpr int kWarps = kThreads / 32, kPer = kDim / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  for (int p = warp; p < parts; p += kWarps) {
    const int64_t slot = x.slot(p);
    const float2 ml = P.partial_ml[slot * kRows + blockIdx.y];
    const float *src = P.partial_o + (slot * kRows + blockIdx.y) * kDim + lane * kPer;
    float y[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] = src[i];
    const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
    const float f_old = exp2f(m - ref), f_new = exp2f(ml.x - ref);
    l = l * f_old + ml.y * f_new;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * f_old + y[i] * f_new;
    m = m_new;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_row[warp][lane * kPer + i] = acc[i];
  if (lane == 0) s_ml[warp] = make_float2(m, l);
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s_ml[i].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float f[kWarps], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    f[i] = exp2f(s_ml[i].x - ref);
    sum += s_ml[i].y * f[i];
  }
  const int token = s.q0 + row / P.group, head = h * P.group + row % P.group;
  for (int c = threadIdx.x; c < P.head_dim; c += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += s_row[i][c] * f[i];
    store(token, head, c, sum != 0.f ? v / sum : 0.f);
  }
  if (threadIdx.x == 0 && P.lse != nullptr)
    P.lse[static_cast<int64_t>(token) * P.q_heads + head] = sum != 0.f ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
}

// The same for items with many rows, which have few parts: block (w - 1, y) takes the rows y * 32 .. + 31 of w's
// item, a warp takes whole rows and goes through their parts in order.
template <int kThreads, int kRows, int kUnit, int kDim, typename Store>
__device__ __forceinline__ void combine_rows(const PagedParams &P, Store store) {
  __shared__ LineScratch<kThreads> scratch;
  khd::grid_dependency_wait();
  const Split x = find_split<kThreads, kRows, kUnit>(P, scratch);
  if (x.parts == 0) return;
  constexpr int kPer = kDim / 32, kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = warp; i < 32; i += kWarps) {
    const int in_block = static_cast<int>(blockIdx.y) * 32 + i, row = x.row0 + in_block;
    if (in_block >= kRows || row >= x.s.rows) return;
    float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] = 0.f;
    for (int p = 0; p < x.parts; ++p) {
      const int64_t at = x.slot(p) * kRows + in_block;
      const float2 ml = P.partial_ml[at];
      float y[kPer];
#pragma unroll
      for (int c = 0; c < kPer; ++c) y[c] = P.partial_o[at * kDim + c * 32 + lane];
      const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
      const float f_old = exp2f(m - ref), f_new = exp2f(ml.x - ref);
      l = l * f_old + ml.y * f_new;
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[c] = acc[c] * f_old + y[c] * f_new;
      m = m_new;
    }
    const int token = x.s.q0 + row / P.group, head = x.h * P.group + row % P.group;
#pragma unroll
    for (int c = 0; c < kPer; ++c)
      if (c * 32 + lane < P.head_dim) store(token, head, c * 32 + lane, l != 0.f ? acc[c] / l : 0.f);
    if (lane == 0 && P.lse != nullptr)
      P.lse[static_cast<int64_t>(token) * P.q_heads + head] = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
  }
}

} // namespace khp
