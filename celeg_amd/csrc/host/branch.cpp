#include "branch.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "kernels.hpp"

namespace celeg {

namespace {
// A launch has fewer than 2^32 threads: more rows, pairs or requests than this are launched in turns.
constexpr long long MOST_A_LAUNCH = 1 << 20;

void need(bool ok, const char* message) {
    if (!ok) throw ArgumentError(message);
}
// addresses of values of `size` bytes each
void aligned(std::initializer_list<const void*> addresses, size_t size, const char* message) {
    for (const void* p : addresses) need(reinterpret_cast<uintptr_t>(p) % size == 0, message);
}
void floats(DType dtype, const char* message) { need(dtype == DType::F32 || dtype == DType::BF16, message); }

// the pages and the table of a group, as the kernels address them
void check_cache(const KVView& kv) {
    floats(kv.dtype, "cache: the pages are float32 or bfloat16");
    need(kv.k && kv.table, "cache: the pages or the table are missing");
    aligned({kv.k, kv.v}, dtype_size(kv.dtype), "cache: the pages must lie on a boundary of their type");
    aligned({kv.table}, 4, "cache: the table must lie on a boundary of 4 bytes");
    need(kv.n_pages > 0 && kv.n_layers > 0 && kv.kv_heads > 0 && kv.page_tokens > 0 && kv.head_dim > 0 && kv.v_head_dim >= 0 &&
             kv.table_rows > 0 && kv.table_stride > 0, "cache: sizes must be positive");
    need((kv.v_head_dim > 0) == (kv.v != nullptr), "cache: values and their width come together (keys only: neither)");
    need(static_cast<long long>(kv.table_stride) * kv.page_tokens < (1LL << 31) - 4096, "cache: a request's places must fit 31 bits");
    need(static_cast<long long>(kv.n_layers) * kv.kv_heads <= 65535, "cache: more than 65,535 layers times heads");
}
void check_workspace(const void* workspace, size_t bytes, size_t needed) {
    if (!needed) return;
    need(workspace && bytes >= needed, "the workspace is missing or smaller than the size asked for it");
    need(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must lie on a boundary of 16 bytes");
}
}  // namespace

// ---------------------------------------------------------------------------- log probabilities
static void check_sizes(const TokenLogprobs& a) {
    floats(a.dtype, "token_logprobs: logits must be float32 or bfloat16");
    need(a.rows >= 0 && a.rows < (1LL << 31), "token_logprobs: the number of rows must be in [0, 2^31)");
    need(a.vocab > 0 && a.vocab <= (1LL << 24), "token_logprobs: the vocabulary must be in [1, 2^24]");
    need(a.rows * (a.vocab / 8192 + 2) < (1LL << 31), "token_logprobs: too many logits for one call");
    need(a.per_row >= 0 && a.per_row <= TokenLogprobs::MAX_PER_ROW, "token_logprobs: up to 8 tokens a row");
    need(a.top >= 0 && a.top <= TokenLogprobs::MAX_TOP && a.top <= a.vocab, "token_logprobs: top must be in [0, 128] and not above the vocabulary");
    need(a.row_stride >= 0 && (a.rows <= 1 || a.row_stride == 0 || a.row_stride >= a.vocab),
         "token_logprobs: rows must not overlap in part (a row stride of 0 or at least the vocabulary)");
}

static void check(const TokenLogprobs& a) {
    check_sizes(a);
    if (a.rows == 0) return;
    need(a.logits != nullptr, "token_logprobs: the logits are missing");
    need(a.per_row == 0 || (a.tokens && a.logprobs && a.ranks), "token_logprobs: tokens, logprobs and ranks come together");
    need(a.top == 0 || (a.top_ids && a.top_logprobs), "token_logprobs: top_ids and top_logprobs are missing");
    aligned({a.logits}, dtype_size(a.dtype), "token_logprobs: logits must lie on a boundary of their type");
    aligned({a.tokens, a.logprobs, a.ranks, a.entropy, a.top_ids, a.top_logprobs}, 4, "token_logprobs: lists and results must lie on boundaries of 4 bytes");
}

// rows of a launch: a workgroup or more for each
static long long rows_at_once(const TokenLogprobs& a) { return std::min(a.rows, std::max(1LL, 8 * MOST_A_LAUNCH / (a.vocab / 1024 + 2))); }

size_t token_logprobs_workspace(const TokenLogprobs& a) {
    check_sizes(a);
    if (a.rows == 0) return 0;
    // (the last launch's rows may be few, which are cut into more parts)
    const long long most = rows_at_once(a), last = a.rows % most;
    const auto bytes = [&](long long rows) {
        return rows ? celeg_logprobs_workspace(static_cast<int>(a.dtype), rows, static_cast<int>(a.vocab), a.per_row, a.top) : 0;
    };
    return std::max(bytes(most), bytes(last));
}

void token_logprobs(const TokenLogprobs& a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    check(a);
    if (a.rows == 0) return;
    check_workspace(workspace, workspace_bytes, token_logprobs_workspace(a));
    const long long most = rows_at_once(a);
    const auto at = [](auto* list, long long offset) { return list ? list + offset : nullptr; };
    for (long long first = 0; first < a.rows; first += most) {
        const char* logits = static_cast<const char*>(a.logits) + first * a.row_stride * static_cast<long long>(dtype_size(a.dtype));
        kernel_check(celeg_logprobs_rows(logits, static_cast<int>(a.dtype), std::min(most, a.rows - first), static_cast<int>(a.vocab), a.row_stride,
                                         at(a.tokens, first * a.per_row), a.per_row, a.top, at(a.logprobs, first * a.per_row),
                                         at(a.ranks, first * a.per_row), at(a.entropy, first), at(a.top_ids, first * a.top),
                                         at(a.top_logprobs, first * a.top), workspace, stream), "token_logprobs");
    }
}

// ---------------------------------------------------------------------------- attention of trees
static void check_sizes(const TreeAttention& a, const KVView& kv) {
    check_cache(kv);
    need(kv.v_head_dim == kv.head_dim, "tree_attention: values of the keys' width only");
    need(kv.layer >= 0 && kv.layer < kv.n_layers, "tree_attention: layer outside the cache");
    need(kv.head_dim <= TreeAttention::MAX_HEAD_DIM, "tree_attention: heads of up to 256");
    need(a.rows >= 0 && a.requests >= 0, "tree_attention: negative counts");
    need(a.heads > 0 && a.heads <= 65535 && a.heads % kv.kv_heads == 0, "tree_attention: heads must be a multiple of the cache's key/value heads");
    need(a.max_nodes > 0 && a.max_nodes <= TreeAttention::MAX_NODES, "tree_attention: max_nodes must be in [1, 256]");
    need(static_cast<long long>(a.requests) * a.max_nodes <= TreeAttention::MAX_REQUEST_NODES, "tree_attention: more than 65,535 requests times max_nodes");
    need(a.window >= 0 && a.max_context >= 0, "tree_attention: window and max_context must not be negative");
    need(std::isfinite(a.scale), "tree_attention: the scale must be finite");
    const long long width = static_cast<long long>(a.heads) * kv.head_dim;
    need(a.rows <= 1 || a.q_stride >= width, "tree_attention: the rows of q overlap");
    need(a.q_stride >= 0 && a.q_stride < (1LL << 31), "tree_attention: the row stride of q must be in [0, 2^31)");
}

static void check(const TreeAttention& a, const KVView& kv) {
    check_sizes(a, kv);
    if (a.rows == 0 || a.requests == 0) return;
    need(a.q && a.out && a.slots && a.starts && a.offsets && a.parents, "tree_attention: an argument is missing");
    aligned({a.q, a.out}, dtype_size(kv.dtype), "tree_attention: q and out must lie on a boundary of their type");
    aligned({a.slots, a.starts, a.offsets, a.parents}, 4, "tree_attention: lists must lie on boundaries of 4 bytes");
}

// Parts that the contexts are cut into, 0: the kernel for any sizes, which reads single values.
static int tree_parts(const TreeAttention& a, const KVView& kv) {
    const uintptr_t low = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(kv.k) |
                          reinterpret_cast<uintptr_t>(kv.v) | (a.rows > 1 ? static_cast<uintptr_t>(a.q_stride) * dtype_size(kv.dtype) : 0);
    const long long page_bytes = static_cast<long long>(kv.n_layers) * kv.kv_heads * kv.page_tokens * kv.head_dim * static_cast<long long>(dtype_size(kv.dtype));
    if (low % 16 || page_bytes >= (1LL << 31) || !celeg_tree_attention_fast_ok(kv.head_dim, kv.page_tokens)) return 0;
    const long long room = static_cast<long long>(kv.table_stride) * kv.page_tokens;
    int context = static_cast<int>(a.max_context > 0 ? std::min<long long>(a.max_context, room) : room);
    if (a.window > 0) context = std::min(context, a.window);        // (nothing before it is read)
    return celeg_tree_attention_parts(static_cast<int>(kv.dtype), kv.head_dim, a.requests, kv.kv_heads, a.heads / kv.kv_heads, a.max_nodes, context);
}

size_t tree_attention_workspace(const TreeAttention& a, const KVView& kv) {
    check_sizes(a, kv);
    if (a.rows == 0 || a.requests == 0) return 0;
    const int parts = tree_parts(a, kv);
    return parts > 1 ? static_cast<size_t>(a.rows) * a.heads * parts * (kv.head_dim + 2) * sizeof(float) : 0;
}

void tree_attention(const TreeAttention& a, const KVView& kv, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    check(a, kv);
    if (a.rows == 0 || a.requests == 0) return;
    check_workspace(workspace, workspace_bytes, tree_attention_workspace(a, kv));
    const int parts = tree_parts(a, kv);
    if (parts > 0) {
        kernel_check(celeg_tree_attention_fast(a.q, static_cast<int>(a.q_stride), static_cast<int>(kv.dtype), kv.k, kv.v, kv.n_pages,
                                               kv.n_layers, kv.layer, a.heads, kv.kv_heads, kv.head_dim, kv.page_tokens, kv.table,
                                               kv.table_rows, kv.table_stride, a.slots, a.starts, a.offsets, a.parents, a.requests, a.rows,
                                               a.max_nodes, parts, a.scale, a.window, a.out, workspace, stream),
                     "tree_attention (matrix cores)");
        return;
    }
    kernel_check(celeg_tree_attention_general(a.q, static_cast<int>(a.q_stride), static_cast<int>(kv.dtype), kv.k, kv.v, kv.n_pages,
                                              kv.n_layers, kv.layer, a.heads, kv.kv_heads, kv.head_dim, kv.page_tokens, kv.table,
                                              kv.table_rows, kv.table_stride, a.slots, a.starts, a.offsets, a.parents, a.requests, a.rows,
                                              a.max_nodes, a.scale, a.window, a.out, stream), "tree_attention");
}

// ---------------------------------------------------------------------------- tokens and pages
void move_tokens(const MoveTokens& a, const KVView& kv, hipStream_t stream) {
    check_cache(kv);
    need(a.requests >= 0 && a.n_places >= 0, "move_tokens: negative counts");
    if (a.requests == 0 || a.n_places == 0) return;
    need(a.src_slots && a.dst_slots && a.offsets && a.places && a.dst_starts, "move_tokens: an argument is missing");
    aligned({a.src_slots, a.dst_slots, a.offsets, a.places, a.dst_starts}, 4, "move_tokens: lists must lie on boundaries of 4 bytes");
    for (long long first = 0; first < a.requests; first += MOST_A_LAUNCH)
        kernel_check(celeg_move_token_list(kv.k, kv.v, static_cast<int>(kv.dtype), kv.n_pages, kv.n_layers, kv.kv_heads, kv.page_tokens,
                                           kv.head_dim, kv.v_head_dim, kv.table, kv.table_rows, kv.table_stride, a.src_slots + first,
                                           a.dst_slots + first, a.offsets + first, a.places, a.dst_starts + first,
                                           static_cast<int>(std::min(MOST_A_LAUNCH, a.requests - first)), a.n_places, stream), "move_tokens");
}

void copy_pages(const KVView& kv, const int* src, const int* dst, int n, hipStream_t stream) {
    check_cache(kv);
    need(n >= 0, "copy_pages: a negative count");
    if (n == 0) return;
    need(src && dst, "copy_pages: the lists of pages are missing");
    aligned({src, dst}, 4, "copy_pages: lists must lie on boundaries of 4 bytes");
    const size_t per_dim = static_cast<size_t>(kv.n_layers) * kv.kv_heads * kv.page_tokens * dtype_size(kv.dtype);
    for (long long first = 0; first < n; first += MOST_A_LAUNCH)
        kernel_check(celeg_copy_page_list(kv.k, kv.v, per_dim * kv.head_dim, per_dim * kv.v_head_dim, kv.n_pages, src + first, dst + first,
                                          static_cast<int>(std::min(MOST_A_LAUNCH, n - first)), stream), "copy_pages");
}

}  // namespace celeg
