// The C interface of the operators in branch.hpp (include/celeg_amd.h).
#include "../include/celeg_amd.h"

#include "branch.hpp"

using namespace celeg;

extern "C" void celeg_set_last_error_(const char* message);

namespace {
template <typename F>
celeg_status guarded(F&& body) {
    try {
        body();
        return CELEG_OK;
    } catch (const ArgumentError& e) {
        celeg_set_last_error_(e.what());
        return CELEG_INVALID_ARGUMENT;
    } catch (const std::exception& e) {
        celeg_set_last_error_(e.what());
        return CELEG_ERROR;
    } catch (...) {
        celeg_set_last_error_("unknown failure");
        return CELEG_ERROR;
    }
}

DType dtype_of(int32_t dtype) {
    if (dtype != 0 && dtype != 1) throw ArgumentError("dtype must be 0 (float32) or 1 (bfloat16)");
    return static_cast<DType>(dtype);
}

template <typename T>
const T& given(const T* args) {
    if (!args) throw ArgumentError("the arguments are missing");
    if (args->struct_size < sizeof(T)) throw ArgumentError("struct_size is smaller than this library's struct");
    return *args;
}

KVView view_of(const celeg_paged_cache* cache, int32_t layer = 0) {
    const celeg_paged_cache& c = given(cache);
    KVView kv;
    kv.k = c.k;
    kv.v = c.v;
    kv.dtype = dtype_of(c.dtype);
    kv.layer = layer;
    kv.n_pages = c.n_pages;
    kv.n_layers = c.n_layers;
    kv.kv_heads = c.kv_heads;
    kv.page_tokens = c.page_tokens;
    kv.head_dim = c.head_dim;
    kv.v_head_dim = c.v_head_dim;
    // (the kernels write keys and values, never the table)
    kv.table = const_cast<int*>(c.table);
    kv.table_rows = c.table_rows;
    kv.table_stride = c.table_stride;
    return kv;
}

TokenLogprobs logprobs_of(const celeg_token_logprobs_args* args) {
    const celeg_token_logprobs_args& g = given(args);
    TokenLogprobs a;
    a.logits = g.logits;
    a.dtype = dtype_of(g.dtype);
    a.rows = g.rows;
    a.vocab = g.vocab;
    a.row_stride = g.row_stride;
    a.tokens = g.tokens;
    a.per_row = g.per_row;
    a.top = g.top;
    a.logprobs = g.logprobs;
    a.ranks = g.ranks;
    a.entropy = g.entropy;
    a.top_ids = g.top_ids;
    a.top_logprobs = g.top_logprobs;
    return a;
}

TreeAttention tree_of(const celeg_tree_attention_args* args) {
    const celeg_tree_attention_args& g = given(args);
    TreeAttention a;
    a.q = g.q;
    a.q_stride = g.q_stride;
    a.out = g.out;
    a.rows = g.rows;
    a.heads = g.heads;
    a.requests = g.requests;
    a.slots = g.slots;
    a.starts = g.starts;
    a.offsets = g.offsets;
    a.parents = g.parents;
    a.scale = g.scale;
    a.window = g.window;
    a.max_nodes = g.max_nodes;
    a.max_context = g.max_context;
    return a;
}
}  // namespace

extern "C" {

celeg_status celeg_token_logprobs_workspace(const celeg_token_logprobs_args* args, size_t* bytes) {
    return guarded([&] {
        if (!bytes) throw ArgumentError("bytes is missing");
        *bytes = token_logprobs_workspace(logprobs_of(args));
    });
}

celeg_status celeg_token_logprobs(const celeg_token_logprobs_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] { token_logprobs(logprobs_of(args), workspace, workspace_bytes, static_cast<hipStream_t>(stream)); });
}

celeg_status celeg_tree_attention_workspace(const celeg_tree_attention_args* args, const celeg_paged_cache* cache, size_t* bytes) {
    return guarded([&] {
        if (!bytes) throw ArgumentError("bytes is missing");
        *bytes = tree_attention_workspace(tree_of(args), view_of(cache, given(args).layer));
    });
}

celeg_status celeg_tree_attention(const celeg_tree_attention_args* args, const celeg_paged_cache* cache, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    return guarded([&] {
        tree_attention(tree_of(args), view_of(cache, given(args).layer), workspace, workspace_bytes, static_cast<hipStream_t>(stream));
    });
}

celeg_status celeg_move_tokens(const celeg_paged_cache* cache, int32_t requests, const int32_t* src_slots, const int32_t* dst_slots,
                               const int32_t* offsets, const int32_t* places, int32_t n_places, const int32_t* dst_starts, void* stream) {
    return guarded([&] {
        MoveTokens a;
        a.requests = requests;
        a.n_places = n_places;
        a.src_slots = src_slots;
        a.dst_slots = dst_slots;
        a.offsets = offsets;
        a.places = places;
        a.dst_starts = dst_starts;
        move_tokens(a, view_of(cache), static_cast<hipStream_t>(stream));
    });
}

celeg_status celeg_copy_pages(const celeg_paged_cache* cache, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    return guarded([&] { copy_pages(view_of(cache), src, dst, n, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
