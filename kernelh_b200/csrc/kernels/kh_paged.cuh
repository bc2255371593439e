// What the kernels of attention over a paged cache share: the parameters, how a call's work is dealt out,
// and the buffers that partial results meet in.
//
// Rows. The queries of one sequence that share a key/value head (group = q_heads / k_heads of them per
// token) form rows: row r of head h is token r / group, query head h * group + r % group. A row block is
// kRows of them; a query head never needs a tile of its own, so a single token with 8 query heads per
// key/value head reads its keys and values once.
//
// Work. An item is (sequence, key/value head, row block) and takes n units of kUnit keys: from the first key that
// any of its rows sees to the last. With a few more that stand for its start and end, the units of all items form one
// line, and every worker (a block) takes an equal stretch of it, whatever the lengths are: a worker finishes the item
// it starts in, does whole ones, and leaves the last one to the next worker. Under the causal mask the blocks of a
// sequence differ in length; they lie on the line in pairs, shortest with longest, whose sum is nearly the same for
// all, so that a place on the line still leads to its item by one division. Items that more than one worker touches
// leave (max, sum, unnormalised row) in the workspace: slot 2w + 1 for the worker that starts an item, 2w for those
// that continue it. The first worker that begins inside an item also leaves a note of it, and a second launch adds the
// parts up in the order of the keys. The line is laid out from q_start and kv_len on the device, so a captured call
// follows lengths that change between replays.
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
  struct SplitItem *split_items; // [workers]
  uint32_t *status;
  int32_t tokens, batch, k_heads, group, head_dim, page_size, page_shift, table_width, num_pages; // page_size = 2^page_shift, or page_shift < 0
  int32_t causal, window;  // window 0: none
  int32_t workers, min_units;
  int32_t pad;   // units that stand for an item's start and end on the line
  int32_t whole; // 1: a worker takes the items that begin in its stretch, whole; nothing is split
  int32_t rows_above, rows_upto; // sequences with rows in (rows_above, rows_upto] are this launch's
  float scale_log2;              // scale * log2(e): scores are kept in exp2 units
};

// How a kernel cuts its work.
template <int kRows_, int kUnit_> struct Grain {
  static constexpr int kRows = kRows_, kUnit = kUnit_;
};
// 64-bit quotients cost a hundred instructions; nearly all of these fit 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int32_t b) {
  return a < (int64_t{1} << 31) ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

struct Sequence {
  int q0, tokens, rows, kv; // first token, new tokens, tokens * group, keys
  int blocks, pair_span, last_span; // row blocks; the length of two paired ones on the line, and of an odd last one
  int64_t head_span;                // of all blocks of one head
};

// The keys that row block `block` sees, [lo, hi), and the units they lie in.
struct Keys {
  int lo, hi, first_unit, units;
};
template <typename G> __device__ __forceinline__ Keys keys_of(const PagedParams &P, const Sequence &s, int block) {
  Keys k{0, s.kv, 0, 0};
  const int past = s.kv - s.tokens; // position of token 0 (negative: its first tokens see nothing)
  const int row0 = block * G::kRows;
  // (the last block ends with the sequence and the first begins with it: no quotient for a single one)
  if (P.causal && row0 + G::kRows < s.rows) k.hi = max(0, min(s.kv, past + (row0 + G::kRows - 1) / P.group + 1));
  if (P.window > 0) {
    const int64_t lo = static_cast<int64_t>(past) + (block > 0 ? row0 / P.group : 0) - P.window + 1;
    k.lo = lo > 0 ? static_cast<int>(min(lo, static_cast<int64_t>(s.kv))) : 0;
  }
  k.first_unit = k.lo / G::kUnit;
  k.units = max(1, (k.hi + G::kUnit - 1) / G::kUnit - k.first_unit); // an item without keys still has its zeros to write
  return k;
}

// The sequence's shape, with every offset forced into range (and reported when it was not).
template <typename G> __device__ __forceinline__ Sequence sequence(const PagedParams &P, int b) {
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
  s.blocks = (s.rows + G::kRows - 1) / G::kRows;
  s.pair_span = s.last_span = 0;
  if (s.blocks & 1) s.last_span = keys_of<G>(P, s, s.blocks - 1).units + P.pad;
  if (s.blocks > 1) {
    // No pair may be longer than pair_span. The last key a block sees grows linearly from block to block (cut off at 0,
    // which makes the sum of a pair largest at the ends), so does the first one under a window (cut off at 0, with the
    // opposite sign: largest in the middle). Either pair may be rounded up to units by two less than another is, by
    // four with a window, and the one at the ends may be short of a block's tokens, two units at most.
    const int last = (s.blocks & ~1) - 1;
    const int ends = keys_of<G>(P, s, 0).units + keys_of<G>(P, s, last).units;
    const int middle = keys_of<G>(P, s, last / 2).units + keys_of<G>(P, s, last / 2 + 1).units;
    s.pair_span = max(ends, middle) + (P.window > 0 ? 6 : 2) + 2 * P.pad;
  }
  s.head_span = static_cast<int64_t>(s.blocks >> 1) * s.pair_span + s.last_span;
  return s;
}
template <typename G> __device__ __forceinline__ int64_t sequence_span(const PagedParams &P, int b) { return sequence<G>(P, b).head_span * P.k_heads; }

// The item at a place on the line, of a sequence that begins at `start`: its stretch of the line [begin, end), of
// which the first keys.units are its units.
struct Item {
  int64_t begin, end;
  int h, block;
  Keys keys;
};
template <typename G> __device__ __forceinline__ Item item_at(const PagedParams &P, const Sequence &s, int64_t start, int64_t at) {
  Item x;
  const bool big = s.head_span >= (int64_t{1} << 31);
  x.h = static_cast<int>(big ? (at - start) / s.head_span : quotient(at - start, static_cast<int32_t>(s.head_span)));
  x.begin = start + x.h * s.head_span;
  const int64_t inside = at - x.begin, pairs = static_cast<int64_t>(s.blocks >> 1) * s.pair_span;
  if (inside >= pairs) {
    x.block = s.blocks - 1;
    x.keys = keys_of<G>(P, s, x.block);
    x.begin += pairs;
    x.end = x.begin + s.last_span;
    return x;
  }
  const int pair = static_cast<int>(quotient(inside, s.pair_span));
  x.begin += static_cast<int64_t>(pair) * s.pair_span;
  x.end = x.begin + s.pair_span;
  x.block = pair;
  x.keys = keys_of<G>(P, s, pair);
  const int64_t second = x.begin + x.keys.units + P.pad;
  if (at < second) {
    x.end = second;
  } else {
    x.begin = second;
    x.block = (s.blocks & ~1) - 1 - pair;
    x.keys = keys_of<G>(P, s, x.block);
  }
  return x;
}

// The whole line, dealt out evenly: worker w's stretch begins at stretch(w) (w = workers: the line's end).
struct Line {
  int64_t total, share;
  int workers, rest; // of which the first `workers` have any work
  __device__ __forceinline__ int64_t stretch(int w) const {
    return share * w + static_cast<int64_t>(static_cast<uint32_t>(rest) * static_cast<uint32_t>(w) / static_cast<uint32_t>(workers)); // both below 2^15
  }
};
template <int kThreads> struct LineScratch {
  int64_t warp_sum[kThreads / 32];
  int64_t start;
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

// The block works out the line together, and where worker w's stretch begins: in sequence scratch.b, which begins
// at scratch.start (both stay there). The order is that of the sequences; a thread takes one, of each kThreads.
template <int kThreads, typename G> __device__ __forceinline__ Line lay_line(const PagedParams &P, int w, LineScratch<kThreads> &scratch) {
  Line line;
  int64_t mine = 0, inclusive;
  for (int b = threadIdx.x; b < P.batch; b += kThreads) mine += sequence_span<G>(P, b);
  line.total = block_scan<kThreads>(mine, inclusive, scratch.warp_sum);
  const int64_t most = quotient(line.total + P.min_units - 1, P.min_units);
  line.workers = static_cast<int>(most < P.workers ? most : P.workers);
  if (w >= line.workers) return line;
  line.share = quotient(line.total, line.workers);
  line.rest = static_cast<int>(line.total - line.share * line.workers);
  const int64_t at = line.stretch(w);
  int64_t before = 0;
  for (int base = 0;; base += kThreads) { // with more sequences than threads, again group by group
    const int b = base + static_cast<int>(threadIdx.x);
    int64_t all = line.total;
    if (P.batch > kThreads) {
      mine = b < P.batch ? sequence_span<G>(P, b) : 0;
      all = block_scan<kThreads>(mine, inclusive, scratch.warp_sum);
    }
    if (at < before + all) {
      if (at >= before + inclusive - mine && at < before + inclusive) {
        scratch.b = b;
        scratch.start = before + inclusive - mine;
      }
      break;
    }
    before += all;
  }
  __syncthreads();
  return line;
}

// Item w of all, in the order of the sequences, their heads and their blocks, found by the block together: its
// sequence in scratch.b, whose first item is scratch.start. False when there are no more than w.
template <int kThreads, typename G> __device__ __forceinline__ bool find_item(const PagedParams &P, int w, LineScratch<kThreads> &scratch) {
  int64_t before = 0;
  for (int base = 0; base < P.batch; base += kThreads) {
    const int b = base + static_cast<int>(threadIdx.x);
    const int64_t mine = b < P.batch ? static_cast<int64_t>(sequence<G>(P, b).blocks) * P.k_heads : 0;
    int64_t inclusive;
    const int64_t all = block_scan<kThreads>(mine, inclusive, scratch.warp_sum);
    if (w < before + all) {
      if (w >= before + inclusive - mine && w < before + inclusive) {
        scratch.b = b;
        scratch.start = before + inclusive - mine;
      }
      __syncthreads();
      return true;
    }
    before += all;
  }
  return false;
}

// The item that worker w's stretch begins inside of, if no earlier stretch does (parts 0 otherwise). Its part 0
// lies in slot 2 (w - 1) + 1, part p in slot 2 (w - 1 + p).
struct alignas(32) SplitItem {
  int32_t q0, row0, rows, h, parts; // rows: of the item
};
__device__ __forceinline__ int64_t part_slot(int w, int p) { return 2 * static_cast<int64_t>(w - 1 + p) + (p == 0 ? 1 : 0); }
// One thread of worker w notes it down; `item` (of sequence s) is where its stretch begins.
template <typename G> __device__ __forceinline__ void note_split(const PagedParams &P, const Line &line, int w, const Sequence &s, const Item &item) {
  SplitItem x{};
  const int64_t at = line.stretch(w), end = item.begin + item.keys.units;
  if (item.begin < at && at < end && item.begin >= line.stretch(w - 1)) {
    x.q0 = s.q0;
    x.h = item.h;
    x.row0 = item.block * G::kRows;
    x.rows = min(G::kRows, s.rows - x.row0);
    // the last worker with a part: by proportion, then to the place
    int last = max(w, min(line.workers - 1, static_cast<int>((end - 1) * line.workers / line.total)));
    while (last + 1 < line.workers && line.stretch(last + 1) < end) ++last;
    while (last > w && line.stretch(last) >= end) --last;
    x.parts = last - w + 2;
  }
  P.split_items[w] = x;
}

// Adds up the parts of one row, for items with few rows and many parts: block (w - 1, y) takes row y of w's
// item. Its warps take every kThreads / 32-th part each with a running maximum and are added up in order.
template <int kThreads, int kRows, int kDim, typename Store> __device__ __forceinline__ void combine_row(const PagedParams &P, Store store) {
  __shared__ float s_row[kThreads / 32][kDim];
  __shared__ float2 s_ml[kThreads / 32];
  khd::grid_dependency_wait();
  const int w = blockIdx.x + 1;
  const SplitItem x = P.split_items[w];
  const int in_block = static_cast<int>(blockIdx.y), row = x.row0 + in_block;
  if (x.parts == 0 || in_block >= x.rows) return;
  constexpr int kWarps = kThreads / 32, kPer = kDim / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  constexpr int kAhead = 4; // parts on their way at once
  float2 mls[kAhead];
  float ys[kAhead][kPer];
  const auto fetch = [&](int p, float2 &ml, float (&y)[kPer]) {
    if (p >= x.parts) return;
    const int64_t at = part_slot(w, p) * kRows + in_block;
    ml = P.partial_ml[at];
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] = P.partial_o[at * kDim + i * 32 + lane];
  };
  for (int p0 = warp; p0 < x.parts; p0 += kAhead * kWarps) {
#pragma unroll
   for (int a = 0; a < kAhead; ++a) fetch(p0 + a * kWarps, mls[a], ys[a]);
#pragma unroll
   for (int a = 0; a < kAhead; ++a) {
    if (p0 + a * kWarps >= x.parts) break;
    const float2 ml = mls[a];
    const float (&y)[kPer] = ys[a];
    const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
    const float f_old = exp2f(m - ref), f_new = exp2f(ml.x - ref);
    l = l * f_old + ml.y * f_new;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * f_old + y[i] * f_new;
    m = m_new;
   }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_row[warp][i * 32 + lane] = acc[i];
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
  const int token = x.q0 + row / P.group, head = x.h * P.group + row % P.group;
  for (int c = threadIdx.x; c < P.head_dim; c += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += s_row[i][c] * f[i];
    store(token, head, c, sum != 0.f ? v / sum : 0.f);
  }
  if (threadIdx.x == 0 && P.lse != nullptr)
    P.lse[static_cast<int64_t>(token) * (P.k_heads * P.group) + head] = sum != 0.f ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
}

// The same for items with many rows, which have few parts: block (w - 1, y) takes the rows y * kBlockRows .. of w's
// item, a warp two of them at once, a row's parts in order.
constexpr int kBlockRows = 16;
template <int kRows, int kDim, typename Store> __device__ __forceinline__ void combine_rows(const PagedParams &P, Store store) {
  khd::grid_dependency_wait();
  const int w = blockIdx.x + 1;
  const SplitItem x = P.split_items[w];
  constexpr int kPer = kDim / 32, kAtOnce = kBlockRows / 8;
  const int lane = threadIdx.x & 31, first = static_cast<int>(blockIdx.y) * kBlockRows + static_cast<int>(threadIdx.x >> 5) * kAtOnce;
  if (x.parts == 0 || first >= x.rows) return;
  float m[kAtOnce], l[kAtOnce], acc[kAtOnce][kPer];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[i][c] = 0.f;
  }
  float2 ml[kAtOnce];
  float y[kAtOnce][kPer];
  const auto fetch = [&](int p) {
    const int64_t slot = part_slot(w, p) * kRows;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = slot + min(first + i, x.rows - 1);
      ml[i] = P.partial_ml[at];
#pragma unroll
      for (int c = 0; c < kPer; ++c) y[i][c] = P.partial_o[at * kDim + c * 32 + lane];
    }
  };
  fetch(0);
  for (int p = 0; p < x.parts; ++p) {
    float2 ml0[kAtOnce];
    float y0[kAtOnce][kPer];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      ml0[i] = ml[i];
#pragma unroll
      for (int c = 0; c < kPer; ++c) y0[i][c] = y[i][c];
    }
    if (p + 1 < x.parts) fetch(p + 1); // the next part is on its way while this one is added
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float m_new = fmaxf(m[i], ml0[i].x), ref = m_new == -INFINITY ? 0.f : m_new;
      const float f_old = exp2f(m[i] - ref), f_new = exp2f(ml0[i].x - ref);
      l[i] = l[i] * f_old + ml0[i].y * f_new;
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[i][c] = acc[i][c] * f_old + y0[i][c] * f_new;
      m[i] = m_new;
    }
  }
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    if (first + i >= x.rows) return;
    const int row = x.row0 + first + i, token = x.q0 + row / P.group, head = x.h * P.group + row % P.group;
#pragma unroll
    for (int c = 0; c < kPer; ++c)
      if (c * 32 + lane < P.head_dim) store(token, head, c * 32 + lane, l[i] != 0.f ? acc[i][c] / l[i] : 0.f);
    if (lane == 0 && P.lse != nullptr)
      P.lse[static_cast<int64_t>(token) * (P.k_heads * P.group) + head] = l[i] != 0.f ? (m[i] + log2f(l[i])) * 0.69314718055994531f : -INFINITY;
  }
}

} // namespace khp
