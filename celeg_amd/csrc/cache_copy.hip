// Pages and tokens of a group's cache copied, all layers at once.
//   K [pages, layers, kv_heads, page_tokens, head_dim]      a token's key: head_dim values in a row
//   V [pages, layers, kv_heads, v_head_dim, page_tokens]    a token's value: a column of its page
// Nothing is computed: the bytes are read once and written once.  What a list names outside the pool, the table or a
// request's pages is left out (nothing is read or written for it).
#include "common.h"
#include <algorithm>

// ---------------------------------------------------------------------------- whole pages
// A page of a group is one block of memory for all layers and heads.  A workgroup copies 1,024 words (16 KB) of a page of K or V, a
// thread four of them, asked for together.  Bound by the bytes.
#define COPY_EACH 4

template <typename W>
__global__ __launch_bounds__(256) void copy_pages_kernel(W* __restrict__ k, W* __restrict__ v, size_t k_words, size_t v_words,
                                                         int n_pages, const int* __restrict__ src, const int* __restrict__ dst) {
    const int from = src[blockIdx.x], to = dst[blockIdx.x];
    if (from < 0 || from >= n_pages || to < 0 || to >= n_pages || from == to) return;
    const size_t words = blockIdx.z ? v_words : k_words;
    const W* in = (blockIdx.z ? v : k) + from * words;
    W* out = (blockIdx.z ? v : k) + to * words;
    for (size_t base = blockIdx.y * static_cast<size_t>(256 * COPY_EACH) + threadIdx.x; base < words; base += gridDim.y * static_cast<size_t>(256 * COPY_EACH)) {
        W held[COPY_EACH];
#pragma unroll
        for (int e = 0; e < COPY_EACH; ++e)
            if (base + 256 * e < words) held[e] = in[base + 256 * e];
#pragma unroll
        for (int e = 0; e < COPY_EACH; ++e)
            if (base + 256 * e < words) out[base + 256 * e] = held[e];
    }
}

extern "C" int celeg_copy_page_list(void* k, void* v, size_t k_bytes, size_t v_bytes, int n_pages, const int* src, const int* dst,
                                    int n, hipStream_t stream) {
    const size_t most = k_bytes > v_bytes ? k_bytes : v_bytes;
    const uintptr_t low = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | k_bytes | v_bytes;
    auto run = [&](auto* word) {
        using W = std::remove_pointer_t<decltype(word)>;
        const size_t shares = (most / sizeof(W) + 256 * COPY_EACH - 1) / (256 * COPY_EACH);
        copy_pages_kernel<W><<<dim3(n, static_cast<unsigned>(std::min<size_t>(shares, 65535)), v_bytes ? 2 : 1), dim3(256), 0, stream>>>(
            static_cast<W*>(k), static_cast<W*>(v), k_bytes / sizeof(W), v_bytes / sizeof(W), n_pages, src, dst);
    };
    typedef unsigned int piece __attribute__((ext_vector_type(4)));
    if (low % 16 == 0) run(static_cast<piece*>(nullptr));
    else run(static_cast<uint16_t*>(nullptr));
    return CELEG_LAUNCH_RESULT();
}

// ---------------------------------------------------------------------------- tokens
// Token i of request r goes from place places[offsets[r] + i] of slot src_slots[r] to place dst_starts[r] + i of slot
// dst_slots[r].  Within one slot the places rise and no token moves up (place >= dst_starts[r] + i): what a token is
// written over is then never read for a later one, so tokens are taken in runs that are read as a whole before they are
// written, the runs in order.
struct MoveArgs {
    void *k, *v;
    const int* table;
    const int *src_slots, *dst_slots, *offsets, *places, *dst_starts;
    int n_pages, n_layers, kv_heads, page_tokens, head_dim, v_head_dim, table_rows, table_stride, n_places;
    int blocks_each;             // layers and heads (one after the other) of a workgroup
    int shares;                  // workgroups that share a request's runs, where it moves between two slots
};

// A request of a call.
struct MoveRequest {
    int from_slot, to_slot, first, count, start;
    bool ok;
    __device__ __forceinline__ MoveRequest(const MoveArgs& a, int r) {
        from_slot = a.src_slots[r];
        to_slot = a.dst_slots[r];
        first = max(a.offsets[r], 0);
        const int to = min(a.offsets[r + 1], a.n_places);
        count = to > first ? to - first : 0;
        start = a.dst_starts[r];
        ok = from_slot >= 0 && from_slot < a.table_rows && to_slot >= 0 && to_slot < a.table_rows && start >= 0 && count > 0;
    }
};

// The page of a place, or -1 if it is on none.
__device__ __forceinline__ int page_of_place(const MoveArgs& a, int slot, long long place) {
    if (place < 0 || place >= static_cast<long long>(a.table_stride) * a.page_tokens) return -1;
    const int page = a.table[static_cast<size_t>(slot) * a.table_stride + static_cast<int>(place) / a.page_tokens];
    return page >= 0 && page < a.n_pages ? page : -1;
}

// Any sizes: a workgroup owns one layer and head of K or V; a thread owns some of its dimensions and takes the tokens in order.
template <typename T>
__global__ __launch_bounds__(256) void move_tokens_general_kernel(const MoveArgs a) {
    const MoveRequest q(a, blockIdx.x);
    if (!q.ok) return;
    const int lh = blockIdx.y, width = blockIdx.z ? a.v_head_dim : a.head_dim;
    T* pool = static_cast<T*>(blockIdx.z ? a.v : a.k);
    const size_t per_block = static_cast<size_t>(a.page_tokens) * width, page_size = per_block * a.n_layers * a.kv_heads;
    auto where = [&](int slot, long long place) -> T* {
        const int page = page_of_place(a, slot, place);
        if (page < 0) return nullptr;
        const int at = static_cast<int>(place) % a.page_tokens;
        return pool + page * page_size + lh * per_block + (blockIdx.z ? at : static_cast<size_t>(at) * width);
    };
    const int step = blockIdx.z ? a.page_tokens : 1;
    for (int i = 0; i < q.count; ++i) {
        const T* from = where(q.from_slot, a.places[q.first + i]);
        T* to = where(q.to_slot, static_cast<long long>(q.start) + i);
        if (!from || !to || from == to) continue;
        for (int d = threadIdx.x; d < width; d += 256) to[static_cast<size_t>(d) * step] = from[static_cast<size_t>(d) * step];
    }
}

// x / d for x and d whose product is below 2^32 (d > 1), by a multiplication
__device__ __forceinline__ unsigned reciprocal(unsigned d) { return 0xffffffffu / d + 1u; }
__device__ __forceinline__ unsigned quotient(unsigned x, unsigned by, unsigned d) { return d == 1 ? x : __umulhi(x, by); }

// Keys in pieces of 16 bytes, values (columns of their pages) in groups of as many tokens as 16 bytes hold, gathered one by one and
// written as a whole, the groups of 16 tokens, which are a line, by neighbouring lanes.  A workgroup has K or V of `blocks_each` layers and heads of a request: one where the runs are long, more
// where a request moves a few tokens, so that the way to them (slots, places, table) is gone once.  A run has as many tokens as its
// workgroup's threads hold, MOVE_EACH pieces (groups) a thread.
// Bound by the bytes: 8 requests that keep 4,001 to 3,500 of 8,192 tokens, 6 layers of 8 heads of 64 in bfloat16 (737 MB, and the values
// that lie between those kept, 184 MB): 212 us, 4.3 TB/s; the keys alone 82 us, 4.5 TB/s.  Sixteen tokens' groups side by side in
// neighbouring lanes, so that a store writes whole lines: 277 -> 226 us.
#define MOVE_EACH 4
#define MOVE_RUN 256             // most tokens of a run

template <typename T>
__global__ __launch_bounds__(256) void move_tokens_kernel(const MoveArgs a) {
    constexpr int GROUP = 16 / sizeof(T), SIDE = 16 / GROUP, CAPACITY = 256 * MOVE_EACH;
    typedef unsigned int piece __attribute__((ext_vector_type(4)));
    typedef T group_t __attribute__((ext_vector_type(GROUP)));
    __shared__ long long from_of[MOVE_RUN], to_of[MOVE_RUN];           // elements from the pool's start, -1: the token is left out
    const MoveRequest q(a, blockIdx.x);
    const bool values = blockIdx.z & 1;
    int share = blockIdx.z >> 1, shares = a.shares;
    if (!q.ok || (values && !a.v)) return;
    if (q.from_slot == q.to_slot) {        // in place: the runs in order
        if (share > 0) return;
        shares = 1;
    }
    const int tid = threadIdx.x, width = values ? a.v_head_dim : a.head_dim;
    const int lh0 = blockIdx.y * a.blocks_each, blocks = min(a.blocks_each, a.n_layers * a.kv_heads - lh0);
    T* pool = static_cast<T*>(values ? a.v : a.k);
    const size_t per_block = static_cast<size_t>(a.page_tokens) * width, page_size = per_block * a.n_layers * a.kv_heads;
    pool += lh0 * per_block;
    // tokens of a run; a run of values begins on a boundary of a group, but for the request's first
    const unsigned pieces = width / GROUP;
    const int lead = values ? q.start % 16 : 0;
    const int run = values ? max(min(CAPACITY / (width * blocks * SIDE), MOVE_RUN / 16), 1) * 16 : min(CAPACITY / (static_cast<int>(pieces) * blocks), MOVE_RUN);
    const unsigned by_inner = reciprocal(values ? width : pieces);
    for (int base = share * run - lead; base < q.count; base += shares * run) {
        const int i0 = max(base, 0), n = min(base + run, q.count) - i0;
        for (int i = tid; i < n; i += 256) {
            const int place = a.places[q.first + i0 + i];
            const long long target = static_cast<long long>(q.start) + i0 + i;
            const int from_page = page_of_place(a, q.from_slot, place), to_page = page_of_place(a, q.to_slot, target);
            const bool there = from_page >= 0 && to_page >= 0;
            const size_t unit = values ? 1 : width;
            // (a token that is left out is read from the pool's first page, and not written)
            from_of[i] = there ? from_page * page_size + (place % a.page_tokens) * unit : 0;
            to_of[i] = there ? static_cast<long long>(to_page * page_size + (static_cast<int>(target) % a.page_tokens) * unit) : -1;
        }
        __syncthreads();
        if (!values) {
            const unsigned items = n * pieces * blocks, by_n = reciprocal(n);
            piece held[MOVE_EACH];
            // item x: piece x % pieces of token (x / pieces) % n of block x / pieces / n
            auto item = [&](int e, unsigned& i) {
                const unsigned x = min(tid + 256u * e, items - 1), y = quotient(x, by_inner, pieces), block = quotient(y, by_n, n);
                i = y - block * n;
                return block * per_block + (x - y * pieces) * GROUP;
            };
#pragma unroll
            for (int e = 0; e < MOVE_EACH; ++e) {
                if (256u * e >= items) break;
                unsigned i;
                const size_t at = item(e, i);
                held[e] = *reinterpret_cast<const piece*>(pool + from_of[i] + at);
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < MOVE_EACH; ++e) {
                if (256u * e >= items) break;
                unsigned i;
                const size_t at = item(e, i);
                if (tid + 256u * e < items && to_of[i] >= 0) *reinterpret_cast<piece*>(pool + to_of[i] + at) = held[e];
            }
        } else {
            // Sixteen tokens' groups lie side by side, so that neighbouring lanes write what follows one another: line n of the run
            // holds its tokens 16 n - skip .. + 15
            const int skip = i0 - base;
            const unsigned lines = (skip + n + 15) / 16, items = lines * width * blocks * SIDE, by_lines = reciprocal(lines);
            group_t held[MOVE_EACH];
            // item x: group x % SIDE of dimension (x / SIDE) % width of line (x / SIDE / width) % lines of block x / SIDE / width / lines
            auto item = [&](int e, int& first) {
                const unsigned x = min(tid + 256u * e, items - 1), u = x / SIDE, y = quotient(u, by_inner, width), block = quotient(y, by_lines, lines);
                first = static_cast<int>((y - block * lines) * 16 + x % SIDE * GROUP) - skip;
                return block * per_block + static_cast<size_t>(u - y * width) * a.page_tokens;
            };
#pragma unroll
            for (int e = 0; e < MOVE_EACH; ++e) {
                if (256u * e >= items) break;
                int i;
                const T* from = pool + item(e, i);
#pragma unroll
                for (int t = 0; t < GROUP; ++t) held[e][t] = from[from_of[min(max(i + t, 0), n - 1)]];
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < MOVE_EACH; ++e) {
                if (256u * e >= items) break;
                if (tid + 256u * e >= items) continue;
                int i;
                T* to = pool + item(e, i);
                bool whole = i >= 0 && i + GROUP <= n;
#pragma unroll
                for (int t = 0; t < GROUP; ++t) whole = whole && to_of[min(max(i + t, 0), n - 1)] >= 0;
                if (whole) {
                    *reinterpret_cast<group_t*>(to + to_of[i]) = held[e];
                } else {
#pragma unroll
                    for (int t = 0; t < GROUP; ++t)
                        if (i + t >= 0 && i + t < n && to_of[i + t] >= 0) to[to_of[i + t]] = held[e][t];
                }
            }
        }
        __syncthreads();         // (the lists are made anew)
    }
}

extern "C" int celeg_move_token_list(void* k, void* v, int dtype, int n_pages, int n_layers, int kv_heads, int page_tokens, int head_dim,
                                     int v_head_dim, const int* table, int table_rows, int table_stride, const int* src_slots,
                                     const int* dst_slots, const int* offsets, const int* places, const int* dst_starts, int n,
                                     int n_places, hipStream_t stream) {
    const MoveArgs base{k, v, table, src_slots, dst_slots, offsets, places, dst_starts, n_pages, n_layers, kv_heads, page_tokens, head_dim,
                        v_head_dim, table_rows, table_stride, n_places, 1, 1};
    const int lh = n_layers * kv_heads, sides = v_head_dim ? 2 : 1;
    auto run = [&](auto* word) {
        using T = std::remove_pointer_t<decltype(word)>;
        constexpr int GROUP = 16 / sizeof(T);
        MoveArgs a = base;
        const bool aligned = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0;
        if (!aligned || page_tokens % GROUP || head_dim % GROUP || head_dim > 256 || v_head_dim > 256) {
            move_tokens_general_kernel<T><<<dim3(n, lh, sides), dim3(256), 0, stream>>>(a);
            return;
        }
        // Few tokens a request: several layers and heads a workgroup, as many as its threads hold of a line of values, while there
        // are 768 workgroups (32 requests of up to 5 tokens, 6 layers of 8 heads of 64: 9.3 us, with 192 of them 15.6).
        const long long blocks = static_cast<long long>(n) * lh * sides;
        const int tokens = n_places / n + 1, most = std::max(1, 256 * MOVE_EACH / (2 * 16 / GROUP * std::max(head_dim, v_head_dim)));
        a.blocks_each = std::min({std::max(1, MOVE_RUN / 4 / tokens), most, std::max(1, static_cast<int>(blocks / 768))});
        const int groups = (lh + a.blocks_each - 1) / a.blocks_each;
        // Long runs: as many workgroups share them as the chip holds a few times over (2,048 to 65,536 in all: 238, 226, 219, 217 us for
        // the requests above).
        const int run = std::max(256 * MOVE_EACH / (std::max(head_dim, v_head_dim) * a.blocks_each * 16 / GROUP), 1) * 16;
        a.shares = std::max(1, std::min(tokens / run, static_cast<int>(8192 / (static_cast<long long>(n) * groups * sides) + 1)));
        move_tokens_kernel<T><<<dim3(n, groups, 2 * a.shares), dim3(256), 0, stream>>>(a);
    };
    if (dtype == CELEG_BF16) run(static_cast<uint16_t*>(nullptr));
    else run(static_cast<uint32_t*>(nullptr));
    return CELEG_LAUNCH_RESULT();
}
