// Pages and tokens of a group's cache copied, all layers at once.
//   K [pages, layers, kv_heads, page_tokens, head_dim]      a token's key: head_dim values in a row
//   V [pages, layers, kv_heads, v_head_dim, page_tokens]    a token's value: a column of its page
// Nothing is computed: the bytes are read once and written once.  What a list names outside the pool, the table or a
// request's pages is left out (nothing is read or written for it).
#include "common.h"

// ---------------------------------------------------------------------------- whole pages
// A page of a group is one block of memory for all layers and heads.  A workgroup copies a share of one page of K or V.
template <typename W>
__global__ __launch_bounds__(256) void copy_pages_kernel(W* __restrict__ k, W* __restrict__ v, size_t k_words, size_t v_words,
                                                         int n_pages, const int* __restrict__ src, const int* __restrict__ dst) {
    const int from = src[blockIdx.x], to = dst[blockIdx.x];
    if (from < 0 || from >= n_pages || to < 0 || to >= n_pages || from == to) return;
    W* pool = blockIdx.z ? v : k;
    const size_t words = blockIdx.z ? v_words : k_words;
    for (size_t i = blockIdx.y * 256 + threadIdx.x; i < words; i += static_cast<size_t>(gridDim.y) * 256)
        pool[to * words + i] = pool[from * words + i];
}

extern "C" int celeg_copy_page_list(void* k, void* v, size_t k_bytes, size_t v_bytes, int n_pages, const int* src, const int* dst,
                                    int n, hipStream_t stream) {
    const size_t most = k_bytes > v_bytes ? k_bytes : v_bytes;
    const uintptr_t low = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | k_bytes | v_bytes;
    auto run = [&](auto* word) {
        using W = std::remove_pointer_t<decltype(word)>;
        const size_t words = most / sizeof(W);
        const unsigned shares = static_cast<unsigned>(words < 4096 ? 1 : words / 4096 < 64 ? words / 4096 : 64);
        copy_pages_kernel<W><<<dim3(n, shares, v_bytes ? 2 : 1), dim3(256), 0, stream>>>(
            static_cast<W*>(k), static_cast<W*>(v), k_bytes / sizeof(W), v_bytes / sizeof(W), n_pages, src, dst);
    };
    if (low % 16 == 0) run(static_cast<uint4*>(nullptr));
    else run(static_cast<uint16_t*>(nullptr));
    return CELEG_LAUNCH_RESULT();
}

// ---------------------------------------------------------------------------- tokens
// Token i of request r goes from place places[offsets[r] + i] of slot src_slots[r] to place dst_starts[r] + i of slot
// dst_slots[r].  Within one slot the places rise and no token moves up (place >= dst_starts[r] + i): what a token is
// written over is then never read for a later one, so a workgroup that has read a token before it writes it may take the
// tokens in order.  A workgroup owns one layer and head of K or V.
template <typename T>
__global__ __launch_bounds__(256) void move_tokens_kernel(T* __restrict__ k, T* __restrict__ v, int n_pages, int n_layers, int kv_heads,
                                                          int page_tokens, int head_dim, int v_head_dim, const int* __restrict__ table,
                                                          int table_rows, int table_stride, const int* __restrict__ src_slots,
                                                          const int* __restrict__ dst_slots, const int* __restrict__ offsets,
                                                          const int* __restrict__ places, const int* __restrict__ dst_starts, int n_places) {
    const int r = blockIdx.x, lh = blockIdx.y;
    const int a = src_slots[r], b = dst_slots[r];
    if (a < 0 || a >= table_rows || b < 0 || b >= table_rows) return;
    const int first = max(offsets[r], 0), last = min(offsets[r + 1], n_places), start = dst_starts[r];
    if (start < 0) return;
    const int width = blockIdx.z ? v_head_dim : head_dim;
    const long long room = static_cast<long long>(table_stride) * page_tokens;
    T* pool = blockIdx.z ? v : k;
    const size_t page_size = static_cast<size_t>(n_layers) * kv_heads * page_tokens * width;
    auto where = [&](int slot, long long place) -> T* {
        if (place < 0 || place >= room) return nullptr;
        const int page = table[static_cast<size_t>(slot) * table_stride + place / page_tokens];
        if (page < 0 || page >= n_pages) return nullptr;
        const int at = static_cast<int>(place % page_tokens);
        return pool + page * page_size + static_cast<size_t>(lh) * page_tokens * width + (blockIdx.z ? at : at * width);
    };
    const int step = blockIdx.z ? page_tokens : 1;
    for (int i = first; i < last; ++i) {
        const T* from = where(a, places[i]);
        T* to = where(b, static_cast<long long>(start) + (i - first));
        if (!from || !to || from == to) continue;
        for (int d = threadIdx.x; d < width; d += 256) to[static_cast<size_t>(d) * step] = from[static_cast<size_t>(d) * step];
    }
}

extern "C" int celeg_move_token_list(void* k, void* v, int dtype, int n_pages, int n_layers, int kv_heads, int page_tokens, int head_dim,
                                     int v_head_dim, const int* table, int table_rows, int table_stride, const int* src_slots,
                                     const int* dst_slots, const int* offsets, const int* places, const int* dst_starts, int n,
                                     int n_places, hipStream_t stream) {
    auto run = [&](auto* word) {
        using W = std::remove_pointer_t<decltype(word)>;
        move_tokens_kernel<W><<<dim3(n, n_layers * kv_heads, v_head_dim ? 2 : 1), dim3(256), 0, stream>>>(
            static_cast<W*>(k), static_cast<W*>(v), n_pages, n_layers, kv_heads, page_tokens, head_dim, v_head_dim, table, table_rows,
            table_stride, src_slots, dst_slots, offsets, places, dst_starts, n_places);
    };
    if (dtype == CELEG_BF16) run(static_cast<uint16_t*>(nullptr));
    else run(static_cast<uint32_t*>(nullptr));
    return CELEG_LAUNCH_RESULT();
}
