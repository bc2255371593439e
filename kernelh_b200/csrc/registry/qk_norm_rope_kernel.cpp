// Argument checks and launches of the query/key norm with rotation (kernels/qk_norm_rope.cu): forward,
// backward and the form that appends to a paged cache. Typed entry points only: the registry's launch by
// name takes fp32 buffers of one layout, these take rows of three types with strides.
#include "executor.hpp"

#include <bit>
#include <cmath>
#include <string>

namespace kh {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 256;
// Blocks per SM (as the kernels are bounded: a wide row's lane holds half the values), and at most in the backward
// pass, where each leaves a row of weight-gradient sums.
constexpr int forward_blocks(int32_t dtype) { return dtype == KH_F32 ? 4 : 3; }
constexpr int backward_blocks(int32_t dtype) { return dtype == KH_F32 ? 3 : 2; }
constexpr int kBackwardMaxBlocks = 3 * 160;
constexpr int kMaxAngles = 1024; // pairs x tokens of a tile (kernels/qk_norm_rope.cu)

int element_size(int32_t dtype) { return dtype == KH_F32 ? 4 : 2; }

// Layouts shared with kernels/qk_norm_rope.cu.
struct NormRopeParams {
  kh_head_rows q, k, q_out, k_out;
  const float *q_weight, *k_weight, *inv_freq;
  const int64_t *positions;
  int64_t tokens;
  int32_t q_heads, k_heads, head_dim, rotary_dim;
  int32_t lanes;
  float eps;
  int32_t blocks[3], tile[3];
};
static_assert(sizeof(NormRopeParams) <= LaunchArgs::kMaxStructBytes);
struct AppendParams {
  kh_head_rows v;
  kh_paged_rows k_cache, v_cache;
  const int64_t *slots;
  int64_t num_slots;
  uint32_t *status;
  int32_t page_size;
};
struct BackwardParams {
  kh_head_rows dq_out, dk_out;
  float *partials;
};
struct WeightGradParams {
  const float *partials;
  float *dq_weight, *dk_weight;
  int32_t blocks[2], head_dim;
};

// The stride of a dimension of size 1 says nothing.
kh_head_rows normalised(kh_head_rows r, int64_t tokens, int32_t heads) {
  if (tokens <= 1) r.token_stride = 0;
  if (heads <= 1) r.head_stride = 0;
  return r;
}

std::string check_rows(const char *name, const kh_head_rows &r, int64_t tokens, int32_t heads, int32_t head_dim,
                       int size, bool output) {
  if (r.data == nullptr) return std::string("buffer '") + name + "' is null";
  if (reinterpret_cast<uintptr_t>(r.data) % static_cast<uintptr_t>(size) != 0)
    return std::string("buffer '") + name + "' is not aligned to its elements";
  if (!output) return "";
  const auto overlaps = [&](int64_t stride, int64_t count) { return count > 1 && std::abs(stride) < head_dim; };
  if (overlaps(r.token_stride, tokens) || overlaps(r.head_stride, heads))
    return std::string("rows of output '") + name + "' overlap (a stride below head_dim)";
  return "";
}

std::string check_cache(const char *name, const kh_paged_rows &c, int64_t pages, int32_t page_size, int32_t heads,
                        int32_t head_dim, int size) {
  const kh_head_rows rows{c.data, page_size > 1 ? c.slot_stride : c.page_stride, c.head_stride};
  std::string why = check_rows(name, rows, page_size > 1 ? page_size : pages, heads, head_dim, size, true);
  if (why.empty() && pages > 1 && std::abs(c.page_stride) < head_dim)
    why = std::string("rows of output '") + name + "' overlap (a stride below head_dim)";
  return why;
}

// Whether every row of `r` starts on a multiple of `bytes`.
bool rows_aligned(const kh_head_rows &r, int size, int bytes) {
  return reinterpret_cast<uintptr_t>(r.data) % static_cast<uintptr_t>(bytes) == 0 && r.token_stride * size % bytes == 0 &&
         r.head_stride * size % bytes == 0;
}
bool rows_aligned(const kh_paged_rows &c, int size, int bytes) {
  return rows_aligned(kh_head_rows{c.data, c.slot_stride, c.head_stride}, size, bytes) && c.page_stride * size % bytes == 0;
}

// Values per access: the largest vector that divides the address and strides of every buffer, the halves
// of the rotation (a pair vector must not straddle one) and the row. Single values otherwise.
int vector_width(const NormRopeCall &c) {
  const kh_qk_norm_rope_args &a = c.args;
  const int size = element_size(a.dtype);
  for (int bytes : {16, 8}) {
    const int vec = bytes / size;
    if (a.head_dim % (2 * vec) != 0 || a.head_dim / (2 * vec) > 32) continue;
    if (!a.interleaved && (a.rotary_dim / 2 % vec != 0 || (a.head_dim - a.rotary_dim) / 2 % vec != 0)) continue;
    bool ok = rows_aligned(a.q, size, bytes) && rows_aligned(a.k, size, bytes) && rows_aligned(c.q_out, size, bytes);
    if (c.kind != NormRopeCall::Append) ok = ok && rows_aligned(c.k_out, size, bytes);
    if (c.kind == NormRopeCall::Backward) ok = ok && rows_aligned(c.dq_out, size, bytes) && rows_aligned(c.dk_out, size, bytes);
    if (c.kind == NormRopeCall::Append)
      ok = ok && rows_aligned(c.v, size, bytes) && rows_aligned(c.k_cache, size, bytes) && rows_aligned(c.v_cache, size, bytes);
    if (ok) return vec;
  }
  return 1;
}

} // namespace

int64_t qk_norm_rope_backward_workspace(int32_t head_dim) {
  return static_cast<int64_t>(kBackwardMaxBlocks) * std::max(head_dim, 0) * 4;
}

Result<void> check_qk_norm_rope(const char *entry, const NormRopeCall &c) {
  const kh_qk_norm_rope_args &a = c.args;
  const auto refuse = [&](const std::string &why) { return fail(2, std::string(entry) + ": " + why); };
  if (a.dtype != KH_F32 && a.dtype != KH_BF16 && a.dtype != KH_F16)
    return refuse("dtype must be KH_F32, KH_BF16 or KH_F16 (got " + std::to_string(a.dtype) + ")");
  if (a.tokens < 0 || a.tokens > (int64_t{1} << 31) - 16) return refuse("tokens must lie in 0 .. 2^31 - 16");
  if (a.q_heads < 1 || a.k_heads < 1 || a.q_heads > (1 << 20) || a.k_heads > (1 << 20))
    return refuse("q_heads and k_heads must lie in 1 .. 2^20");
  if (a.head_dim < 2 || a.head_dim > kMaxHeadDim || a.head_dim % 2 != 0)
    return refuse("head_dim must be even and at most 256 (got " + std::to_string(a.head_dim) + ")");
  if (a.rotary_dim < 0 || a.rotary_dim > a.head_dim || a.rotary_dim % 2 != 0)
    return refuse("rotary_dim must be even and lie in 0 .. head_dim (got " + std::to_string(a.rotary_dim) + ")");
  if (a.interleaved != 0 && a.interleaved != 1) return refuse("interleaved must be 0 or 1");
  if (!(a.eps >= 0.f) || !std::isfinite(a.eps)) return refuse("eps must be finite and not negative");
  if (c.kind == NormRopeCall::Backward && a.tokens > 0) {
    if (c.workspace == nullptr || c.workspace_bytes < qk_norm_rope_backward_workspace(a.head_dim))
      return refuse("the workspace must have " + std::to_string(qk_norm_rope_backward_workspace(a.head_dim)) + " bytes (got " +
                    std::to_string(c.workspace == nullptr ? 0 : c.workspace_bytes) + ")");
    if (reinterpret_cast<uintptr_t>(c.workspace) % 4 != 0) return refuse("the workspace is not 4-byte aligned");
  }
  if (c.kind == NormRopeCall::Append) {
    if (c.page_size < 1 || c.num_pages < 1 || c.num_pages > (int64_t{1} << 31))
      return refuse("page_size and num_pages must be positive, num_pages at most 2^31");
  }
  for (const float *w : {a.q_weight, a.k_weight, a.inv_freq, static_cast<const float *>(c.dq_weight), static_cast<const float *>(c.dk_weight)})
    if (reinterpret_cast<uintptr_t>(w) % 4 != 0) return refuse("a weight, its gradient or inv_freq is not 4-byte aligned");
  for (const int64_t *w : {a.positions, c.slots})
    if (reinterpret_cast<uintptr_t>(w) % 8 != 0) return refuse("positions or slots are not 8-byte aligned");
  if (a.tokens == 0) return {};
  const int size = element_size(a.dtype);
  std::string why = check_rows("q", a.q, a.tokens, a.q_heads, a.head_dim, size, false);
  const auto next = [&](const char *name, const kh_head_rows &r, int32_t heads, bool output) {
    if (why.empty()) why = check_rows(name, r, a.tokens, heads, a.head_dim, size, output);
  };
  next("k", a.k, a.k_heads, false);
  const bool backward = c.kind == NormRopeCall::Backward;
  next(backward ? "dq" : "q_out", c.q_out, a.q_heads, true);
  if (c.kind != NormRopeCall::Append) next(backward ? "dk" : "k_out", c.k_out, a.k_heads, true);
  if (backward) {
    next("dq_out", c.dq_out, a.q_heads, false);
    next("dk_out", c.dk_out, a.k_heads, false);
  }
  if (c.kind == NormRopeCall::Append) {
    next("v", c.v, a.k_heads, false);
    if (why.empty()) why = check_cache("k_cache", c.k_cache, c.num_pages, c.page_size, a.k_heads, a.head_dim, size);
    if (why.empty()) why = check_cache("v_cache", c.v_cache, c.num_pages, c.page_size, a.k_heads, a.head_dim, size);
    if (why.empty() && c.slots == nullptr) why = "buffer 'slots' is null";
  }
  if (why.empty() && a.positions == nullptr) why = "buffer 'positions' is null";
  if (why.empty() && a.inv_freq == nullptr && a.rotary_dim > 0) why = "buffer 'inv_freq' is null";
  if (!why.empty()) return refuse(why);
  return {};
}

Result<void> run_qk_norm_rope(Executor &ex, NormRopeCall c, StreamHandle stream) {
  kh_qk_norm_rope_args &a = c.args;
  const bool backward = c.kind == NormRopeCall::Backward, append = c.kind == NormRopeCall::Append;
  for (kh_head_rows *r : {&a.q, &c.q_out, &c.dq_out}) *r = normalised(*r, a.tokens, a.q_heads);
  for (kh_head_rows *r : {&a.k, &c.k_out, &c.dk_out, &c.v}) *r = normalised(*r, a.tokens, a.k_heads);
  for (kh_paged_rows *p : {&c.k_cache, &c.v_cache}) {
    if (c.num_pages <= 1) p->page_stride = 0;
    if (c.page_size <= 1) p->slot_stride = 0;
    if (a.k_heads <= 1) p->head_stride = 0;
  }
  long sms = query_cu_count(ex.limits());
  if (sms <= 0) sms = 148;
  NormRopeParams p{};
  if (a.tokens > 0) {
    const int vec = vector_width(c), slots = vec == 1 ? 4 : 1;
    const int pair_vectors = (a.head_dim / 2 + vec - 1) / vec;
    p.q = a.q, p.k = a.k, p.q_out = c.q_out, p.k_out = c.k_out;
    p.q_weight = a.q_weight, p.k_weight = a.k_weight, p.inv_freq = a.inv_freq, p.positions = a.positions;
    p.tokens = a.tokens;
    p.q_heads = a.q_heads, p.k_heads = a.k_heads, p.head_dim = a.head_dim, p.rotary_dim = a.rotary_dim;
    p.eps = a.eps;
    p.lanes = static_cast<int>(std::bit_ceil(static_cast<unsigned>((pair_vectors + slots - 1) / slots)));
    // Blocks go to queries, keys and values by their rows, a token's angles counting as four of them: at least one
    // each and none without a tile. A tile has at most about eight rows for every group of lanes, and every block the
    // same number of tiles or one less.
    const int kinds = append ? 3 : 2, groups = kThreads / p.lanes;
    const int64_t most = backward ? std::min<int64_t>(backward_blocks(a.dtype) * sms, kBackwardMaxBlocks) : forward_blocks(a.dtype) * sms;
    const int64_t heads[3] = {a.q_heads, a.k_heads, a.k_heads}, cost[3] = {a.q_heads + 4, a.k_heads + 4, append ? a.k_heads : 0};
    const auto pieces = [](int64_t n, int64_t size) { return (n + size - 1) / size; };
    int64_t blocks = 0;
    for (int i = 0; i < kinds; ++i) {
      const int64_t share = std::max<int64_t>(1, most * cost[i] / (cost[0] + cost[1] + cost[2]));
      const int64_t largest = std::max<int64_t>(1, std::min<int64_t>(8 * groups / heads[i], kMaxAngles / (a.head_dim / 2)));
      p.tile[i] = static_cast<int32_t>(pieces(a.tokens, share * pieces(a.tokens, share * largest)));
      p.blocks[i] = static_cast<int32_t>(std::min(share, pieces(a.tokens, p.tile[i])));
      blocks += p.blocks[i];
    }
    LaunchStep step;
    step.entry = std::string(append ? "qk_norm_rope_append_" : backward ? "qk_norm_rope_backward_" : "qk_norm_rope_") +
                 (a.dtype == KH_F32 ? "f32_v" : a.dtype == KH_BF16 ? "bf16_v" : "f16_v") + std::to_string(vec) +
                 (vec * element_size(a.dtype) == 16 && pair_vectors == p.lanes ? "_full" : "") + (a.interleaved ? "_inter" : "_halves");
    step.block = {kThreads, 1, 1};
    step.overlap_tail = true;
    step.grid = {static_cast<unsigned>(blocks), 1, 1};
    LaunchArgs args;
    args.add_struct_bytes(&p, sizeof p);
    if (append) {
      const AppendParams q{c.v, c.k_cache, c.v_cache, c.slots, c.num_pages * c.page_size, ex.status_word(), c.page_size};
      args.add_struct_bytes(&q, sizeof q);
    }
    if (backward) {
      const BackwardParams q{c.dq_out, c.dk_out, static_cast<float *>(c.workspace)};
      args.add_struct_bytes(&q, sizeof q);
    }
    step.param_count = static_cast<int>(args.param_count());
    auto fn = ex.function("qk_norm_rope", step.entry);
    if (!fn) return std::unexpected(fn.error());
    if (auto r = ex.launch(*fn, step, args, stream); !r) return r;
  }
  if (!backward || (c.dq_weight == nullptr && c.dk_weight == nullptr)) return {};
  LaunchStep step;
  step.entry = "qk_norm_weight_grad";
  step.block = {256, 1, 1};
  step.grid = {static_cast<unsigned>((a.head_dim + 31) / 32), 2, 1};
  step.overlap_tail = true;
  step.param_count = 1;
  const WeightGradParams q{static_cast<const float *>(c.workspace), c.dq_weight, c.dk_weight, {p.blocks[0], p.blocks[1]}, a.head_dim};
  LaunchArgs args;
  args.add_struct_bytes(&q, sizeof q);
  auto fn = ex.function("qk_norm_rope", step.entry);
  if (!fn) return std::unexpected(fn.error());
  return ex.launch(*fn, step, args, stream);
}

} // namespace kh
