// Operators for requests that go on in several ways: what logits say about given tokens, attention of a tree of drafted
// tokens, cached tokens brought together, pages copied.
//
// They keep nothing between calls: the caller brings the stream and, where a kernel leaves parts for a second one, the
// workspace (its size from the *_workspace function of the same arguments), so that calls on several streams or in several
// recorded graphs share nothing that their caller does not share.  Arguments are checked here, before anything is launched:
// ArgumentError says what is wrong.  What only the device knows (slots, places, parents) is bounded by the kernels.
#pragma once
#include <hip/hip_runtime_api.h>

#include "cache.hpp"

namespace celeg {

struct ArgumentError : KernelError { using KernelError::KernelError; };

struct TokenLogprobs {
    const void* logits = nullptr;          // [rows, vocab], rows row_stride elements apart
    DType dtype = DType::F32;
    long long rows = 0, vocab = 0, row_stride = 0;
    const int* tokens = nullptr;           // [rows, per_row]
    int per_row = 0, top = 0;
    float* logprobs = nullptr;             // [rows, per_row]
    int* ranks = nullptr;                  // [rows, per_row]
    float* entropy = nullptr;              // [rows], or null
    int* top_ids = nullptr;                // [rows, top]
    float* top_logprobs = nullptr;         // [rows, top]
    static constexpr int MAX_PER_ROW = 8, MAX_TOP = 128;
};
size_t token_logprobs_workspace(const TokenLogprobs& a);
void token_logprobs(const TokenLogprobs& a, void* workspace, size_t workspace_bytes, hipStream_t stream);

struct TreeAttention {
    const void* q = nullptr;               // [rows, heads * head_dim], rows q_stride elements apart
    long long q_stride = 0;
    void* out = nullptr;                   // [rows, heads * head_dim]
    int rows = 0, heads = 0, requests = 0;
    const int *slots = nullptr, *starts = nullptr;       // [requests]: row of the table, tokens of the context
    const int* offsets = nullptr;          // [requests + 1]: each request's first row
    const int* parents = nullptr;          // [rows]
    float scale = 1.f;
    int window = 0;                        // 0: none
    int max_nodes = 0;                     // most nodes of a request; what lies behind them is left alone
    int max_context = 0;                   // about the longest context (0: what the table holds); decides how the work is cut, nothing else
    static constexpr int MAX_NODES = 256, MAX_HEAD_DIM = 256;
    static constexpr int MAX_REQUEST_NODES = 65535;      // requests times max_nodes of a call
};
size_t tree_attention_workspace(const TreeAttention& a, const KVView& kv);
void tree_attention(const TreeAttention& a, const KVView& kv, void* workspace, size_t workspace_bytes, hipStream_t stream);

struct MoveTokens {
    int requests = 0, n_places = 0;
    const int *src_slots = nullptr, *dst_slots = nullptr;      // [requests]
    const int* offsets = nullptr;          // [requests + 1]: each request's first entry of places
    const int* places = nullptr;           // [n_places]
    const int* dst_starts = nullptr;       // [requests]
};
void move_tokens(const MoveTokens& a, const KVView& kv, hipStream_t stream);

// pages src[i] -> dst[i] of the group, all layers
void copy_pages(const KVView& kv, const int* src, const int* dst, int n, hipStream_t stream);

}  // namespace celeg
