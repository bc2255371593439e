// Argument checks and launches of attention over a paged cache: kernels/paged_attention.cu for few rows per
// key/value head, kernels/paged_attention_chunk.cu for many. A typed entry point only: the registry's launch by
// name takes fp32 buffers of one layout.
#include "executor.hpp"

#include <bit>
#include <climits>
#include <cmath>
#include <string>

namespace kh {
namespace {

constexpr int kRows = 16, kUnit = 64;                  // kernels/paged_attention.cu
constexpr int kChunkRows = 256, kChunkKeys = 128;      // kernels/paged_attention_chunk.cu
constexpr int kMinUnits = 2;          // units per worker below which more workers cost more than they bring
constexpr int kWholeKeys = 512;       // see run_paged_attention
constexpr int kMaxCluster = 8;        // kernels/paged_attention.cu
constexpr long kMaxSms = 160;         // workspaces are sized for at most this many SMs

int element_size(int32_t dtype) { return dtype == KH_F32 ? 4 : 2; }
int padded_dim(int32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Layout shared with kernels/kh_paged.cuh.
struct PagedParams {
  const void *q;
  int64_t q_token, q_head;
  void *o;
  int64_t o_token, o_head;
  const void *k;
  int64_t k_page, k_slot, k_head;
  const void *v;
  int64_t v_page, v_slot, v_head;
  const int32_t *table;
  int64_t table_stride;
  const int32_t *q_start, *kv_len;
  float *lse, *partial_o;
  void *partial_ml, *split_items;
  uint32_t *status;
  int32_t tokens, batch, k_heads, group, head_dim, page_size, page_shift, table_width, num_pages;
  int32_t causal, window;
  int32_t workers, min_units, pad, whole;
  int32_t rows_above, rows_upto;
  float scale_log2;
};
static_assert(sizeof(PagedParams) <= LaunchArgs::kMaxStructBytes);

// Blocks of the kernel that an SM holds: by shared memory (a ring of 3 x 32 padded rows per warp) and registers.
struct Shape {
  int dim, warps, per_sm;
  size_t smem;
};
Shape kernel_shape(int32_t dtype, int32_t head_dim) {
  Shape s{};
  s.dim = padded_dim(head_dim);
  const int row_bytes = s.dim * element_size(dtype);
  s.warps = row_bytes <= 512 ? 4 : 2;
  s.per_sm = row_bytes <= 128 ? 3 : row_bytes <= 256 ? 2 : 1;
  s.smem = static_cast<size_t>(s.warps * 3 * 2 + (dtype == KH_F32 ? 1 : 0)) * 16 * (row_bytes + 16);
  return s;
}

// The tensor-memory kernel takes 16-bit types and head sizes of one or two 128-byte swizzle rows, and its copies
// want boxes of at least eight slots, strides a tensor map can hold, and a scale whose sign keeps maxima maxima.
bool chunk_kernel_fits(const kh_paged_attention_args &a) {
  if (a.dtype == KH_F32 || a.head_dim < 64 || a.head_dim > 128 || a.page_size % 8 != 0 || !(a.scale > 0.f)) return false;
  for (const kh_paged_rows &c : {a.k_cache, a.v_cache})
    for (const auto &[stride, count] : {std::pair<int64_t, int64_t>{c.page_stride, a.num_pages}, {c.slot_stride, a.page_size}, {c.head_stride, a.k_heads}})
      if (count > 1 && (stride <= 0 || stride >= (int64_t{1} << 38))) return false;
  return true;
}
// Whether some sequence may have more rows than one tile of the other kernel.
bool many_rows(const kh_paged_attention_args &a) { return static_cast<int64_t>(a.max_q_len) * (a.q_heads / a.k_heads) > kRows; }

// Grows with `sms` and with every length: the workspace, counted for kMaxSms, covers any device's launch.
int64_t item_count(const kh_paged_attention_args &a, int rows) { // at most
  return (a.tokens * (a.q_heads / a.k_heads) / rows + a.batch) * a.k_heads;
}
int64_t worker_count(const kh_paged_attention_args &a, int rows, int unit, int per_sm, long sms) {
  const int64_t items = item_count(a, rows);
  const int64_t units = (static_cast<int64_t>(std::max(a.max_kv_len, 1)) + unit - 1) / unit;
  const int64_t most = per_sm * std::min(sms, kMaxSms);
  return std::min<int64_t>(most, std::max<int64_t>(1, (items * units + kMinUnits - 1) / kMinUnits));
}
int64_t workspace_for(int64_t workers, int rows, int dim) { return workers * (2 * rows * (dim * 4 + 8) + 32); }

std::string check_stride(const char *name, const void *data, std::initializer_list<std::pair<int64_t, int64_t>> strides, int32_t head_dim,
                         int size, bool output) {
  if (data == nullptr) return std::string("buffer '") + name + "' is null";
  bool aligned = reinterpret_cast<uintptr_t>(data) % 16 == 0;
  for (const auto &[stride, count] : strides) {
    if (count <= 1) continue;
    aligned = aligned && stride * size % 16 == 0;
    if (output && std::abs(stride) < head_dim) return std::string("rows of output '") + name + "' overlap (a stride below head_dim)";
  }
  if (!aligned) return std::string("rows of '") + name + "' do not start on 16-byte boundaries (pass an aligned copy)";
  return "";
}

} // namespace

int64_t paged_attention_workspace(const kh_paged_attention_args &a) {
  if (a.q_heads < 1 || a.k_heads < 1 || a.head_dim < 1 || a.head_dim > 256 || a.tokens < 0 || a.batch < 0) return 0;
  const Shape s = kernel_shape(a.dtype, a.head_dim);
  int64_t bytes = workspace_for(worker_count(a, kRows, kUnit, s.per_sm, kMaxSms), kRows, s.dim);
  // the two kernels run one after the other and use the same memory
  if (a.dtype != KH_F32 && a.head_dim <= 128 && many_rows(a))
    bytes = std::max(bytes, workspace_for(worker_count(a, kChunkRows, kChunkKeys, 1, kMaxSms), kChunkRows, s.dim));
  return bytes;
}

Result<void> check_paged_attention(const kh_paged_attention_args &a) {
  const auto refuse = [&](const std::string &why) { return fail(2, "kh_paged_attention: " + why); };
  if (a.dtype != KH_F32 && a.dtype != KH_BF16 && a.dtype != KH_F16)
    return refuse("dtype must be KH_F32, KH_BF16 or KH_F16 (got " + std::to_string(a.dtype) + ")");
  if (a.q_heads < 1 || a.k_heads < 1 || a.q_heads > (1 << 20) || a.q_heads % a.k_heads != 0)
    return refuse("q_heads must be a positive multiple of k_heads, at most 2^20 (got " + std::to_string(a.q_heads) + " and " +
                  std::to_string(a.k_heads) + ")");
  if (a.head_dim < 8 || a.head_dim > 256 || a.head_dim % 8 != 0)
    return refuse("head_dim must be a multiple of 8 up to 256 (got " + std::to_string(a.head_dim) + ")");
  if (a.tokens < 0 || a.tokens > (INT_MAX - 1024) / (a.q_heads / a.k_heads))
    return refuse("tokens * q_heads / k_heads must lie in 0 .. 2^31 - 1025");
  if (a.batch < 0 || a.max_q_len < 0 || a.max_kv_len < 0) return refuse("batch, max_q_len and max_kv_len must not be negative");
  if (a.causal != 0 && a.causal != 1) return refuse("causal must be 0 or 1");
  if (a.window < 0) return refuse("window must not be negative (0: none)");
  if (!std::isfinite(a.scale)) return refuse("scale must be finite");
  if (a.num_pages < 1 || a.num_pages > INT_MAX || a.page_size < 1 || a.page_size > (1 << 24))
    return refuse("num_pages must lie in 1 .. 2^31 - 1 and page_size in 1 .. 2^24");
  if (a.table_width < 0 || static_cast<int64_t>(a.table_width) * a.page_size > INT_MAX - 1024)
    return refuse("a page table row must hold at most 2^31 - 1025 slots");
  if (a.batch > 1 && std::abs(a.table_stride) < a.table_width) return refuse("rows of the page table overlap");
  if (a.tokens == 0 || a.batch == 0) return {};
  const int size = element_size(a.dtype);
  std::string why = check_stride("q", a.q.data, {{a.q.token_stride, a.tokens}, {a.q.head_stride, a.q_heads}}, a.head_dim, size, false);
  if (why.empty()) why = check_stride("o", a.o.data, {{a.o.token_stride, a.tokens}, {a.o.head_stride, a.q_heads}}, a.head_dim, size, true);
  for (const auto &[name, c] : {std::pair<const char *, kh_paged_rows>{"k_cache", a.k_cache}, {"v_cache", a.v_cache}})
    if (why.empty())
      why = check_stride(name, c.data, {{c.page_stride, a.num_pages}, {c.slot_stride, a.page_size}, {c.head_stride, a.k_heads}}, a.head_dim,
                         size, false);
  for (const auto &[name, p] : {std::pair<const char *, const void *>{"page_table", a.page_table}, {"q_start", a.q_start}, {"kv_len", a.kv_len}, {"lse", a.lse}}) {
    if (!why.empty()) break;
    if (p == nullptr && name != std::string("lse") && !(name == std::string("page_table") && a.table_width == 0))
      why = std::string("buffer '") + name + "' is null";
    else if (reinterpret_cast<uintptr_t>(p) % 4 != 0) why = std::string("buffer '") + name + "' is not 4-byte aligned";
  }
  if (why.empty() && a.q.data == a.o.data) why = "o must not be q itself";
  if (!why.empty()) return refuse(why);
  const int64_t need = paged_attention_workspace(a);
  if (a.workspace == nullptr || a.workspace_bytes < need)
    return refuse("the workspace must have " + std::to_string(need) + " bytes (got " +
                  std::to_string(a.workspace == nullptr ? 0 : a.workspace_bytes) + ")");
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16 != 0) return refuse("the workspace is not 16-byte aligned");
  return {};
}

Result<void> run_paged_attention(Executor &ex, kh_paged_attention_args a, StreamHandle stream) {
  if (a.tokens == 0 || a.batch == 0) return {};
  long sms = query_cu_count(ex.limits());
  if (sms <= 0) sms = 148;
  const Shape s = kernel_shape(a.dtype, a.head_dim);
  PagedParams p{};
  const auto stride = [](int64_t v, int64_t count) { return count > 1 ? v : 0; };
  p.q = a.q.data, p.q_token = stride(a.q.token_stride, a.tokens), p.q_head = stride(a.q.head_stride, a.q_heads);
  p.o = a.o.data, p.o_token = stride(a.o.token_stride, a.tokens), p.o_head = stride(a.o.head_stride, a.q_heads);
  p.k = a.k_cache.data, p.k_page = stride(a.k_cache.page_stride, a.num_pages), p.k_slot = stride(a.k_cache.slot_stride, a.page_size);
  p.v = a.v_cache.data, p.v_page = stride(a.v_cache.page_stride, a.num_pages), p.v_slot = stride(a.v_cache.slot_stride, a.page_size);
  p.k_head = stride(a.k_cache.head_stride, a.k_heads), p.v_head = stride(a.v_cache.head_stride, a.k_heads);
  p.table = a.page_table, p.table_stride = a.batch > 1 ? a.table_stride : 0;
  p.q_start = a.q_start, p.kv_len = a.kv_len;
  p.lse = a.lse;
  p.partial_o = static_cast<float *>(a.workspace);
  p.status = ex.status_word();
  p.tokens = static_cast<int32_t>(a.tokens), p.batch = a.batch, p.k_heads = a.k_heads;
  p.group = a.q_heads / a.k_heads, p.head_dim = a.head_dim;
  p.page_size = a.page_size, p.page_shift = (a.page_size & (a.page_size - 1)) == 0 ? std::countr_zero(static_cast<unsigned>(a.page_size)) : -1;
  p.table_width = a.table_width, p.num_pages = static_cast<int32_t>(a.num_pages);
  p.causal = a.causal, p.window = a.window;
  p.min_units = kMinUnits;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  const std::string suffix = std::string(a.dtype == KH_F32 ? "f32_" : a.dtype == KH_BF16 ? "bf16_" : "f16_") + std::to_string(s.dim);
  const auto launch = [&](const char *image, const std::string &entry, LaunchDims grid, unsigned threads, size_t smem,
                          std::initializer_list<TensorMapBytes> maps, int box_rows, unsigned cluster = 1) -> Result<void> {
    LaunchStep step;
    step.entry = entry;
    step.grid = grid;
    step.block = {threads, 1, 1};
    step.dynamic_smem = smem;
    step.overlap_tail = true;
    step.cluster = cluster;
    LaunchArgs args;
    args.add_struct_bytes(&p, sizeof p);
    for (const TensorMapBytes &m : maps) args.add_tensor_map(m);
    if (box_rows > 0) args.add_scalar<int32_t>(box_rows);
    step.param_count = static_cast<int>(args.param_count());
    auto fn = ex.function(image, entry);
    if (!fn) return std::unexpected(fn.error());
    return ex.launch(*fn, step, args, stream);
  };
  const auto workers = [&](int rows, int unit, int per_sm) {
    const int64_t n = worker_count(a, rows, unit, per_sm, sms);
    p.workers = static_cast<int32_t>(n);
    // An item's start and end take about as long as four units of 128 keys and 256 rows, or three of 64 and 16. Where
    // items are fewer than workers, each is worked on by several, and units that stand for nothing would only leave
    // some of these without work. (64 ragged decoding sequences 200 us with 1, 172 with 3; 8 fp32 ones, 128 items,
    // 20.8 with 1, 24.2 with 3; 13 mixed ones 210 us in the chunk kernel with 0, 130 with 3 or 4.)
    p.pad = (rows == kChunkRows ? 2 : 1) + (item_count(a, rows) >= n ? 2 : 0);
    char *base = static_cast<char *>(a.workspace); // rows, notes of split items, (max, sum) pairs
    p.split_items = base + 2 * n * rows * s.dim * 4;
    p.partial_ml = base + 2 * n * rows * s.dim * 4 + n * 32;
    return static_cast<unsigned>(n);
  };
  const int64_t all_rows = a.tokens * p.group;
  p.rows_above = 0, p.rows_upto = INT_MAX;

  if (many_rows(a) && chunk_kernel_fits(a)) {
    // A sequence of at most 16 rows (a decoding one) goes to the other kernel, unless there can be none (when the
    // longest length times the batch is no more than the tokens, every sequence has that length), or so few that
    // they cost less among the chunks than two more launches: 13 sequences, 8 of them decoding, 155 us against 166 with
    // both kernels, but 32 of up to 8 tokens 170 against 150 (8 key/value heads).
    const bool alone = static_cast<int64_t>(a.batch) * a.max_q_len <= a.tokens || static_cast<int64_t>(a.batch) * a.k_heads <= sms;
    if (!alone) p.rows_above = kRows;
    int box_rows = kChunkKeys; // the largest power of two of slots that divides a page and a tile
    while (a.page_size % box_rows != 0) box_rows /= 2;
    TensorMapBytes maps[2];
    for (int i = 0; i < 2; ++i) {
      const kh_paged_rows &c = i == 0 ? a.k_cache : a.v_cache;
      TensorMapSpec t;
      t.global_address = c.data;
      t.rank = 4;
      t.elem_bytes = 2;
      const int64_t row = a.head_dim; // stands in for the stride of a dimension of size 1
      const int64_t counts[3] = {a.page_size, a.k_heads, a.num_pages}, strides[3] = {c.slot_stride, c.head_stride, c.page_stride};
      t.dims[0] = static_cast<uint64_t>(a.head_dim);
      for (int d = 0; d < 3; ++d) {
        t.dims[d + 1] = static_cast<uint64_t>(counts[d]);
        t.strides_bytes[d] = static_cast<uint64_t>(counts[d] > 1 ? strides[d] : row) * 2;
      }
      t.box[0] = 64;
      t.box[1] = static_cast<uint32_t>(box_rows);
      t.swizzle_bytes = 128;
      auto map = ex.backend().encode_tensor_map(t);
      if (!map) return std::unexpected(map.error());
      maps[i] = *map;
    }
    const unsigned n = workers(kChunkRows, kChunkKeys, 1);
    const int stages = s.dim == 128 ? 5 : 8;
    const size_t smem = static_cast<size_t>(2 + stages) * kChunkKeys * s.dim * 2 + 1024;
    if (auto r = launch("paged_attention_chunk", "paged_attention_chunk_" + suffix, {n, 1, 1}, 512, smem, {maps[0], maps[1]}, box_rows); !r) return r;
    if (n > 1) {
      // an item is split where a worker's stretch begins inside it: 16 rows of it per block
      const unsigned y = static_cast<unsigned>((std::min<int64_t>(kChunkRows, all_rows) + 15) / 16);
      if (auto r = launch("paged_attention_chunk", "paged_attention_chunk_combine_" + suffix, {n - 1, y, 1}, 256, 0, {}, 0); !r) return r;
    }
    if (alone) return {};
    p.rows_above = 0, p.rows_upto = kRows;
  }
  // Few items: each to a cluster of as many blocks as fit on the device at once and have keys to work on; one launch. Up to
  // the point where more blocks than a cluster has bring in the keys faster: 512 keys a block when the clusters fill more
  // than half the device, else 384, and 256 for several fp32 rows, whose arithmetic counts. (Replayed from a graph, against a
  // stretch of the line per block; 32 heads over 8 of 128 in bf16: one sequence of 400 keys 10.3 us against 12.4, 8 of 2000
  // 20.9 against 22.7, one of 4000 14.5 both, two of 4000 18.5 against 16.5; fp32, 16 heads of 64: 8 of 1000 18.6 against
  // 20.6, one of 4000 18.0 against 14.8; by split products, the slowest, 8 of 1000 24.7 against 20.7.)
  const int64_t few = item_count(a, kRows), units = (static_cast<int64_t>(a.max_kv_len) + kUnit - 1) / kUnit, blocks = s.per_sm * sms;
  int64_t ranks = kMaxCluster;
  while (ranks > 1 && (few * ranks > blocks || ranks > units)) ranks /= 2;
  const bool several = static_cast<int64_t>(a.max_q_len) * p.group > 1;
  const int64_t keys = a.dtype == KH_F32 && several ? 256 : 2 * few * ranks > blocks ? 512 : 384; // a block's
  if (ranks > 1 && a.max_kv_len <= ranks * keys)
    return launch("paged_attention", "paged_attention_joint_" + suffix, {static_cast<unsigned>(few * ranks), 1, 1}, 32u * s.warps, s.smem, {}, 0,
                  static_cast<unsigned>(ranks));
  // Short key ranges are not split: an item takes less than the second launch that would add its parts up. (Replayed
  // from a graph, 32 heads over 8 of 128 in bf16: 8 sequences of 200 keys 10.4 us against 13.4, 64 of 400 keys 27.1
  // against 34.7, one of 800 keys 16.6 against 12.4, 64 of 800 keys 45.6 against 51.8.)
  unsigned n = workers(kRows, kUnit, s.per_sm);
  if (a.max_kv_len <= kWholeKeys || (a.max_kv_len <= 2 * kWholeKeys && item_count(a, kRows) >= s.per_sm * sms)) {
    p.whole = 1;
    p.min_units = 1;
    n = static_cast<unsigned>(std::min<int64_t>(item_count(a, kRows), s.per_sm * sms)); // writes nothing to the workspace
    p.workers = static_cast<int32_t>(n);
  }
  if (auto r = launch("paged_attention", "paged_attention_" + suffix, {n, 1, 1}, 32u * s.warps, s.smem, {}, 0); !r) return r;
  if (n == 1 || p.whole) return {};
  const unsigned y = static_cast<unsigned>(std::min<int64_t>(kRows, all_rows)); // a row per block
  return launch("paged_attention", "paged_attention_combine_" + suffix, {n - 1, y, 1}, 256, 0, {}, 0);
}

} // namespace kh
