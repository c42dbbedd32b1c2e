// Attention of a tree of drafted tokens over the paged cache.
//
// A request's context lies at the places 0 .. start - 1 of its pages, the keys and values of its tree's nodes behind it, node i
// at place start + i.  Node i stands at position start + depth(i); it sees the context, its ancestors and itself, of them (with a
// window w) the keys at positions above its own less w.  out = softmax(scale q . k) v over what it sees.
// parents[row]: the index inside its request's tree of a node's parent; what is not an index below the node's own makes it a root.
//   K [pages, layers, kv_heads, page_tokens, head_dim], V [pages, layers, kv_heads, head_dim, page_tokens]
#include "common.h"

#define TREE_MAX_NODES 256

// What a key outside the tree or an ancestor is to a node: all arguments in places, positions and depths.
__device__ __forceinline__ int tree_depth(const int* parents, int node) {
    int depth = 0;
    for (int at = node;;) {
        const int up = parents[at];
        if (up < 0 || up >= at) return depth;      // (indices fall, so the way ends)
        at = up;
        ++depth;
    }
}

// ---------------------------------------------------------------------------- any sizes
// A wavefront a node and query head.  Keys are taken 64 at a time, a lane a key for the scores (running maximum and sum of the
// softmax), a lane a dimension (and the one 64, 128, 192 further on) for the output.
template <typename T>
__global__ __launch_bounds__(64) void tree_attention_general_kernel(
    const T* __restrict__ q, int ldq, const T* __restrict__ k_pool, const T* __restrict__ v_pool, int n_pages, int n_layers, int layer,
    int heads, int kv_heads, int head_dim, int page_tokens, const int* __restrict__ table, int table_rows, int table_stride,
    const int* __restrict__ slots, const int* __restrict__ starts, const int* __restrict__ offsets, const int* __restrict__ parents,
    int n_rows, int max_nodes, float scale, int window, T* __restrict__ out) {
    const int r = blockIdx.y / max_nodes, node = blockIdx.y % max_nodes, h = blockIdx.x, lane = threadIdx.x;
    const int first = offsets[r], count = min(offsets[r + 1] - first, max_nodes);
    const int slot = slots[r], start = max(starts[r], 0);
    if (node >= count || first < 0 || first + node >= n_rows || slot < 0 || slot >= table_rows) return;
    const int* up = parents + first;
    const int depth = tree_depth(up, node), low = window > 0 ? max(0, start + depth - window + 1) : 0;
    __shared__ float qs[256];
    __shared__ float weights[64];
    __shared__ int blocks[64];
    __shared__ unsigned long long seen[TREE_MAX_NODES / 64];
    const T* qrow = q + static_cast<size_t>(first + node) * ldq + static_cast<size_t>(h) * head_dim;
    for (int d = lane; d < head_dim; d += 64) qs[d] = to_float(qrow[d]);
    if (lane < TREE_MAX_NODES / 64) seen[lane] = 0ull;
    __syncthreads();
    if (lane == 0) {
        int at = node;
        for (int steps = 0; steps <= depth && (window <= 0 || steps < window); ++steps) {
            seen[at >> 6] |= 1ull << (at & 63);
            at = up[at];
        }
    }
    __syncthreads();
    const int end = start + count;
    const size_t per_head = static_cast<size_t>(page_tokens) * head_dim;
    const size_t head_block = (static_cast<size_t>(layer) * kv_heads + h / (heads / kv_heads)) * per_head;
    const size_t page_size = static_cast<size_t>(n_layers) * kv_heads * per_head;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int base = low & ~63; base < end; base += 64) {
        const int key = base + lane, i = key - start;
        const int entry = key / page_tokens;
        bool visible = key >= low && key < end && entry < table_stride;
        if (visible && i >= 0) visible = (seen[i >> 6] >> (i & 63)) & 1ull;
        int page = visible ? table[static_cast<size_t>(slot) * table_stride + entry] : 0;
        visible = visible && page >= 0 && page < n_pages;
        float s = -INFINITY;
        if (visible) {
            const T* kr = k_pool + page * page_size + head_block + static_cast<size_t>(key % page_tokens) * head_dim;
            float dot = 0.f;
            for (int d = 0; d < head_dim; ++d) dot = fmaf(qs[d], to_float(kr[d]), dot);
            s = dot * scale;
        }
        const float high = fmaxf(m, wave_max(s));
        const float shift = high == -INFINITY ? 0.f : high;
        const float p = visible ? expf(s - shift) : 0.f, keep = expf(m - shift);
        l = l * keep + wave_sum(p);
        m = high;
        __syncthreads();
        weights[lane] = p;
        blocks[lane] = visible ? page : -1;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= keep;
        for (int j = 0; j < 64; ++j) {
            const int from = blocks[j];
            if (from < 0) continue;                  // (a key that is not seen is not read: it may hold anything)
            const T* vr = v_pool + from * page_size + head_block + (base + j) % page_tokens;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (lane + 64 * e < head_dim) o[e] = fmaf(weights[j], to_float(vr[static_cast<size_t>(lane + 64 * e) * page_tokens]), o[e]);
        }
    }
    T* orow = out + static_cast<size_t>(first + node) * heads * head_dim + static_cast<size_t>(h) * head_dim;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < head_dim) orow[lane + 64 * e] = from_float<T>(o[e] / l);
}

extern "C" int celeg_tree_attention_general(const void* q, int ldq, int dtype, const void* k_pool, const void* v_pool, int n_pages,
                                            int n_layers, int layer, int heads, int kv_heads, int head_dim, int page_tokens,
                                            const int* table, int table_rows, int table_stride, const int* slots, const int* starts,
                                            const int* offsets, const int* parents, int n_requests, int n_rows, int max_nodes, float scale,
                                            int window, void* out, hipStream_t stream) {
    auto run = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        tree_attention_general_kernel<T><<<dim3(heads, n_requests * max_nodes), dim3(64), 0, stream>>>(
            static_cast<const T*>(q), ldq, static_cast<const T*>(k_pool), static_cast<const T*>(v_pool), n_pages, n_layers, layer, heads,
            kv_heads, head_dim, page_tokens, table, table_rows, table_stride, slots, starts, offsets, parents, n_rows, max_nodes, scale,
            window, static_cast<T*>(out));
    };
    if (dtype == CELEG_BF16) run(static_cast<bf16*>(nullptr));
    else run(static_cast<float*>(nullptr));
    return CELEG_LAUNCH_RESULT();
}
