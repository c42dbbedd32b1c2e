// Attention of a tree of drafted tokens over the paged cache.
//
// A request's context lies at the places 0 .. start - 1 of its pages, the keys and values of its tree's nodes behind it, node i
// at place start + i.  Node i stands at position start + depth(i); it sees the context, its ancestors and itself, of them (with a
// window w) the keys at positions above its own less w.  out = softmax(scale q . k) v over what it sees, zeros if that is nothing.
// parents[row]: the index inside its request's tree of a node's parent; what is not an index below the node's own makes it a root.
//   K [pages, layers, kv_heads, page_tokens, head_dim], V [pages, layers, kv_heads, head_dim, page_tokens]
//
// The query heads that share a key/value head, for all nodes of a tree, are the rows of matrix instructions, so that a key is asked
// for once for many rows.  Up to 32 rows: a workgroup's four wavefronts take rounds of keys in turn, each with a running maximum,
// sum and output of its own, and meet in LDS.  More, in bfloat16: 64, 128 or 256 rows a workgroup share rounds of 64 keys that are
// staged in LDS.  Long contexts are cut into parts for as many workgroups, which a second kernel joins.
// Bound by: few rows, the bytes of keys and values (16 trees of 1 node behind 12,001 to 16,384 tokens, 32 heads of 128 on 8: 175
// us, 5.3 TB/s, of 16 nodes 183) or, in short contexts, a chain of reads; many rows, vector and matrix instructions (of 64 nodes: 319 to 335
// us, by the clock, 710 to 745 TFLOP/s, 2.8 to 2.9 TB/s; 14 us of it join two parts).
//
// Scores, maxima, sums and outputs are 32-bit.  In bfloat16 the weights enter the product with the values rounded to bfloat16 (half a step each,
// 2^-8; the sum is of the exact ones); the kernel for any sizes, which has no matrix instructions, keeps them in 32 bits.  Against 64 bits
// results are off by 0.0022 of their size here, of which their own rounding is 0.0017.
#include "common.h"
#include <algorithm>
#include <climits>

#define TREE_MAX_NODES 256

typedef __bf16 tree_bf16x8 __attribute__((ext_vector_type(8)));
typedef float tree_f4 __attribute__((ext_vector_type(4)));
typedef unsigned int tree_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int tree_depth(const int* parents, int node) {
    int depth = 0;
    for (int at = node;;) {
        const int up = parents[at];
        if (up < 0 || up >= at) return depth;      // (indices fall, so the way ends)
        at = up;
        ++depth;
    }
}

// Rows of request r from `first` on that the arrays hold (lists may name anything).
__device__ __forceinline__ int tree_count(const int* offsets, int r, int n_rows, int max_nodes) {
    const int first = offsets[r], to = min(offsets[r + 1], n_rows);
    return first >= 0 && to > first ? min(to - first, max_nodes) : 0;
}

// The context's tokens, so far below the largest number that nothing added to it passes that.
__device__ __forceinline__ int tree_start(const int* starts, int r) { return min(max(starts[r], 0), INT_MAX - 4096); }

// ---------------------------------------------------------------------------- on the matrix cores
struct TreeArgs {
    const void* q;
    const void* k_pool;
    const void* v_pool;
    const int* table;
    const int *slots, *starts, *offsets, *parents;
    void* out;
    float* ws_o;                 // [rows, heads, parts, head_dim]: outputs of parts, not divided
    float* ws_ml;                // [rows, heads, parts, 2]: their maximum (in powers of two) and sum
    int ldq, n_pages, n_layers, layer, heads, kv_heads, group, page_tokens, page_shift, table_rows, table_stride, requests, n_rows, max_nodes;
    int parts, row_blocks, units;      // units: requests * kv_heads * parts
    float scale;                 // its size times log2(e); `turned`: it is negative, and q enters with the other sign
    bool turned;
    int window;
};

// How keys and values lie in the operands.  A round holds KEYS keys; `a` of a key tile is 16 keys by the head's values, a
// lane's (c, qd) = (lane % 16, lane / 16) share of it key(tile, c); a score tile leaves a lane the scores of row c with four keys that
// follow one another, which are in turn the keys that the lane's weights have to stand for in the product with the values.
template <typename T, int HD> struct TreeOps;

template <int HD> struct TreeOps<bf16, HD> {
    static constexpr int KEYS = HD <= 64 ? 64 : 32, TILES = KEYS / 16, KS = HD / 32, DT = HD / 16, VG = KEYS / 32, VKEYS = 8;
    typedef tree_bf16x8 Frag;
    static __device__ __forceinline__ int key(int tile, int c) { return 32 * (tile >> 1) + 8 * (c >> 2) + 4 * (tile & 1) + (c & 3); }
    // whether a row that sees the keys of `seen` sees those of its scores: bits of the word that shown() gives
    static __device__ __forceinline__ unsigned shown(unsigned long long seen, int tile, int qd) {
        return static_cast<unsigned>(tile >> 1 ? seen >> 32 : seen) >> (8 * qd);
    }
    static __device__ __forceinline__ constexpr int bit(int tile, int i) { return 4 * (tile & 1) + i; }
    static __device__ __forceinline__ int vkey(int g, int qd) { return 32 * g + 8 * qd; }
    static __device__ __forceinline__ int dim(int s, int qd) { return 32 * s + 8 * qd; }
    static __device__ __forceinline__ tree_f4 scores(const Frag (&k)[KS], const Frag (&q)[KS]) {
        tree_f4 acc = tree_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[s], q[s], acc, 0, 0, 0);
        return acc;
    }
    // o += V^T p; the weights enter rounded to bfloat16 (half a step, 2^-8 of each; the sum l is taken of the exact ones)
    static __device__ __forceinline__ void values(const Frag (&v)[DT][VG], const tree_f4 (&p)[TILES], tree_f4 (&o)[DT]) {
#pragma unroll
        for (int g = 0; g < VG; ++g) {
            Frag b;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b[i] = static_cast<__bf16>(p[2 * g][i]);
                b[4 + i] = static_cast<__bf16>(p[2 * g + 1][i]);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[dt][g], b, o[dt], 0, 0, 0);
        }
    }
    static __device__ __forceinline__ void turn(Frag& f) { f = __builtin_bit_cast(Frag, __builtin_bit_cast(tree_u4, f) ^ 0x80008000u); }
    // a bit for every half word whose exponent is all ones (infinities and NaN), and the same with them made 0
    static __device__ __forceinline__ unsigned not_finite(const Frag& f) {
        const tree_u4 u = __builtin_bit_cast(tree_u4, f);
        unsigned bad = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= ((u[e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        return bad;
    }
    static __device__ __forceinline__ void make_finite(Frag& f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = static_cast<float>(f[e]);
            if (!(fabsf(x) < INFINITY)) f[e] = static_cast<__bf16>(0.f);
        }
    }
};

template <int HD> struct TreeOps<float, HD> {
    static constexpr int KEYS = 32, TILES = KEYS / 16, KS = HD / 16, DT = HD / 16, VG = TILES, VKEYS = 4;
    typedef tree_f4 Frag;
    static __device__ __forceinline__ int key(int tile, int c) { return 16 * tile + c; }
    static __device__ __forceinline__ unsigned shown(unsigned long long seen, int, int qd) { return static_cast<unsigned>(seen) >> (4 * qd); }
    static __device__ __forceinline__ constexpr int bit(int tile, int i) { return 16 * tile + i; }
    static __device__ __forceinline__ int vkey(int g, int qd) { return 16 * g + 4 * qd; }
    // (a product sums over the head's values in any order: a lane holds a quarter of them that lie side by side)
    static __device__ __forceinline__ int dim(int s, int qd) { return (HD / 4) * qd + 4 * s; }
    static __device__ __forceinline__ tree_f4 scores(const Frag (&k)[KS], const Frag (&q)[KS]) {
        tree_f4 acc = tree_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][e], q[s][e], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ void values(const Frag (&v)[DT][VG], const tree_f4 (&p)[TILES], tree_f4 (&o)[DT]) {
#pragma unroll
        for (int g = 0; g < VG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[dt][g][i], p[g][i], o[dt], 0, 0, 0);
    }
    static __device__ __forceinline__ void turn(Frag& f) { f = -f; }
    static __device__ __forceinline__ unsigned not_finite(const Frag& f) {
        unsigned bad = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= !(fabsf(f[e]) < INFINITY);
        return bad;
    }
    static __device__ __forceinline__ void make_finite(Frag& f) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(fabsf(f[e]) < INFINITY)) f[e] = 0.f;
    }
};

// The keys of a round of 64 from place `base` on that a node sees, a bit each: of the context those from `low` on, of the tree those
// that the node's words name.
__device__ __forceinline__ unsigned long long tree_visible(int base, int start, int low, const unsigned long long (&words)[TREE_MAX_NODES / 64]) {
    const int off = base - start;
    unsigned long long seen = 0ull;
    if (off < 0) {
        const int context = min(-off, 64);
        seen = context == 64 ? ~0ull : (1ull << context) - 1ull;
        const int before = low - base;
        if (before > 0) seen = before >= 64 ? 0ull : seen & (~0ull << before);
        if (context < 64) seen |= words[0] << context;
    } else {
#pragma unroll
        for (int w = 0; w < TREE_MAX_NODES / 64; ++w) {
            if ((off >> 6) == w) seen |= words[w] >> (off & 63);
            if ((off >> 6) + 1 == w && (off & 63)) seen |= words[w] << (64 - (off & 63));
        }
    }
    return seen;
}

// The request of a workgroup: which rows and keys it has.  ok: there is something to do.
struct TreeRequest {
    int first, count, slot, start, rows, end;
    bool ok;
    const int* pages;
    __device__ __forceinline__ TreeRequest(const TreeArgs& a, int r) {
        // (the same for all lanes: said so that they take no vector registers)
        first = __builtin_amdgcn_readfirstlane(a.offsets[r]);
        count = __builtin_amdgcn_readfirstlane(tree_count(a.offsets, r, a.n_rows, a.max_nodes));
        slot = __builtin_amdgcn_readfirstlane(a.slots[r]);
        start = __builtin_amdgcn_readfirstlane(tree_start(a.starts, r));
        rows = count * a.group;
        // (places behind what the table holds are seen by nobody)
        const int room = a.table_stride << a.page_shift;
        end = start < room ? min(start + count, room) : room;
        ok = count > 0 && slot >= 0 && slot < a.table_rows;
        pages = a.table + static_cast<size_t>(ok ? slot : 0) * a.table_stride;
    }
};

// The ways up the tree of the nodes n0 .. n1 (at most as many as threads), and from where on each sees the context; all
// threads call it, and meet a barrier afterwards.
template <int THREADS>
__device__ __forceinline__ void tree_ways(const TreeArgs& a, const TreeRequest& q, int n0, int n1, int* up,
                                          unsigned long long (*words_of)[TREE_MAX_NODES / 64], int* low_of) {
    constexpr int WORDS = TREE_MAX_NODES / 64;
    const int tid = threadIdx.x;
    for (int i = tid; i < q.count; i += THREADS) up[i] = a.parents[q.first + i];
    __syncthreads();
    if (tid <= n1 - n0) {
        unsigned long long words[WORDS] = {};
        int depth = 0;
        for (int at = n0 + tid;;) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
                if ((at >> 6) == w && (a.window <= 0 || depth < a.window)) words[w] |= 1ull << (at & 63);
            const int next = up[at];
            if (next < 0 || next >= at) break;         // (indices fall, so the way ends)
            at = next;
            ++depth;
        }
#pragma unroll
        for (int w = 0; w < WORDS; ++w) words_of[tid][w] = words[w];
        low_of[tid] = a.window > 0 ? max(0, q.start + depth - a.window + 1) : 0;
    }
    __syncthreads();
}

// The rounds of a part, r_begin .. r_end.  In those that begin at `plain` or later and end before the tree every row sees every
// key, as long as all pages are there.
struct TreeRounds {
    int r_begin, r_end, plain;
    __device__ __forceinline__ TreeRounds(const TreeArgs& a, const TreeRequest& q, int part, int keys) {
        const int first = a.window > 0 ? max(0, q.start - a.window + 1) / keys : 0, last = q.end > 0 ? (q.end - 1) / keys : -1;
        const int total = max(last - first + 1, 0), per = (total + a.parts - 1) / a.parts;
        // (the same for all lanes, as TreeRequest's)
        r_begin = __builtin_amdgcn_readfirstlane(first + part * per);
        r_end = __builtin_amdgcn_readfirstlane(min(last, r_begin + per - 1));
        plain = __builtin_amdgcn_readfirstlane(a.window > 0 ? max(0, q.start + q.count - a.window) : 0);
    }
};

// The scores of a round, of RT row tiles, into weights; the rows' running maximum m (in powers of two), sum l (a lane's own keys;
// the four lanes of a row meet at the end) and output o brought up to date.  MASKED: the scores are scaled and hidden ones -inf
// already.  The maximum follows the scores only when some row's grows by more than 8 (a factor 2^8): until then the weights are taken
// against the older one, and numerator and denominator carry the same factor.  Whether one grows so far needs no exchange between the
// lanes of a row: one of them sees it.
template <bool MASKED, int RT, int TILES, int DT>
__device__ __forceinline__ void tree_softmax(tree_f4 (&s)[RT][TILES], float (&m)[RT], float (&l)[RT], tree_f4 (&o)[RT][DT], float scale) {
    float high[RT];
    bool grows = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        high[t] = s[t][0][0];
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
            for (int i = 0; i < 4; ++i) high[t] = fmaxf(high[t], s[t][tile][i]);
        if (!MASKED) high[t] *= scale;
        grows |= high[t] > m[t] + 8.f;
    }
    if (__ballot(grows) != 0ull) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float now = fmaxf(m[t], max_half32(max_row16(high[t])));
            const float keep = m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[t] - now);
            m[t] = now;
            l[t] *= keep;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[t][dt] *= keep;
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float shift = m[t] == -INFINITY ? 0.f : m[t];
        tree_f4 sum = tree_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[t][tile][i] = __builtin_amdgcn_exp2f(MASKED ? s[t][tile][i] - shift : fmaf(s[t][tile][i], scale, -shift));
            sum += s[t][tile];
        }
        l[t] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
}

// The same for a round in which every row sees every key, without looking for the maximum: the scores become weights against the
// running one as it stands, which is left where it is as long as no lane's weights add up to more than 2^12 (false: s is of
// no use, the round has to be taken by tree_softmax; so the first one is).
template <int RT, int TILES>
__device__ __forceinline__ bool tree_weights(tree_f4 (&s)[RT][TILES], const float (&m)[RT], float (&l)[RT], float scale) {
    float sums[RT];
    bool in_range = true;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        tree_f4 sum = tree_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][tile][i] = __builtin_amdgcn_exp2f(fmaf(s[t][tile][i], scale, -m[t]));
            sum += s[t][tile];
        }
        sums[t] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        in_range = in_range && sums[t] <= 4096.f;
    }
    if (__ballot(!in_range) != 0ull) return false;
#pragma unroll
    for (int t = 0; t < RT; ++t) l[t] += sums[t];
    return true;
}

// The keys of the round from `base` on that a row sees, a bit each (page: the lane's page of the round, `gone` if it is none).
template <int KEYS>
__device__ __forceinline__ unsigned long long tree_seen(const TreeArgs& a, const TreeRequest& q, int base, bool all_there, bool gone, int last_page,
                                                        int low, const unsigned long long* words_of) {
    unsigned long long words[TREE_MAX_NODES / 64];
#pragma unroll
    for (int w = 0; w < TREE_MAX_NODES / 64; ++w) words[w] = words_of[w];
    unsigned long long seen = tree_visible(base, q.start, low, words);
    if (base + 64 > q.end) seen &= (1ull << (q.end - base)) - 1ull;
    if (!all_there) {
        const int n = min(a.page_tokens, KEYS), first_page = base >> a.page_shift;
        for (int i = 0; i < KEYS; i += n)
            if (__shfl(static_cast<int>(gone), min((base + i) >> a.page_shift, last_page) - first_page, 64))
                seen &= ~((n == 64 ? ~0ull : (1ull << n) - 1ull) << i);
    }
    return seen;
}

// What the matrix instructions left out of a round: infinities and NaN among the values, for the rows that see them.
template <typename T, int KEYS, int DT>
__device__ __noinline__ void tree_odd_values_of(tree_f4 (&o)[DT], const T* from_head, size_t page_size, int page_shift, int base, int last_page, int page,
                                             unsigned long long seen) {
    const int qd = (threadIdx.x & 63) >> 4;
    for (int i = 0; i < KEYS; ++i) {
        if (!__ballot((seen >> i) & 1ull)) continue;
        const int key = base + i;
        const T* from = from_head + __shfl(page, min(key >> page_shift, last_page) - (base >> page_shift), 64) * page_size +
                        (key & ((1 << page_shift) - 1));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = to_float(from[static_cast<size_t>(16 * dt + 4 * qd + e) << page_shift]);
                if (((seen >> i) & 1ull) && !(fabsf(x) < INFINITY)) o[dt][e] += x;
            }
    }
}

// (a copy goes to the function, so that the outputs themselves stay in registers)
template <typename T, int KEYS, int DT>
__device__ __forceinline__ void tree_odd_values(tree_f4 (&o)[DT], const T* from_head, size_t page_size, int page_shift, int base, int last_page,
                                                int page, unsigned long long seen) {
    tree_f4 copy[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) copy[dt] = o[dt];
    tree_odd_values_of<T, KEYS, DT>(copy, from_head, page_size, page_shift, base, last_page, page, seen);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = copy[dt];
}

// A row's result: to `out`, or, where the context is cut, its part's maximum, sum and output to the workspace.
template <typename T, int HD>
__device__ __forceinline__ void tree_store(const TreeArgs& a, size_t row, int head, int part, int qd, float m, float l, const tree_f4 (&o)[HD / 16]) {
    if (a.parts == 1) {
        T* to = static_cast<T*>(a.out) + (row * a.heads + head) * HD + 4 * qd;
        const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) {
            const float x[4] = {o[dt][0] * inverse, o[dt][1] * inverse, o[dt][2] * inverse, o[dt][3] * inverse};
            Vec4<T>::store(to + 16 * dt, x);
        }
    } else {
        const size_t at = (row * a.heads + head) * a.parts + part;
        if (qd == 0) {
            a.ws_ml[2 * at] = m;
            a.ws_ml[2 * at + 1] = l;
        }
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) *reinterpret_cast<tree_f4*>(a.ws_o + at * HD + 16 * dt + 4 * qd) = o[dt];
    }
}

template <typename T, int HD, int RT>
__device__ __forceinline__ void tree_queries(const TreeArgs& a, const TreeRequest& w, int kvh, int j0, typename TreeOps<T, HD>::Frag (&q)[RT][TreeOps<T, HD>::KS],
                                             int (&node_of)[RT]) {
    using O = TreeOps<T, HD>;
    const int lane = threadIdx.x & 63, c = lane & 15, qd = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int j = min(j0 + 16 * t + c, w.rows - 1), node = j / a.group;
        node_of[t] = node;
        const T* from = static_cast<const T*>(a.q) + static_cast<size_t>(w.first + node) * a.ldq +
                        static_cast<size_t>(kvh * a.group + j % a.group) * HD;
#pragma unroll
        for (int s = 0; s < O::KS; ++s) {
            q[t][s] = *reinterpret_cast<const typename O::Frag*>(from + O::dim(s, qd));
            if (a.turned) O::turn(q[t][s]);
        }
    }
}

// ---- few rows: operands straight from memory, the wavefronts take the rounds in turn
template <typename T, int HD, int RT>
__global__ __launch_bounds__(256, 2) void tree_few_kernel(const TreeArgs a) {
    using O = TreeOps<T, HD>;
    using Frag = typename O::Frag;
    constexpr int KEYS = O::KEYS, TILES = O::TILES, KS = O::KS, DT = O::DT, VG = O::VG, ROWS = 16 * RT;
    __shared__ int up[TREE_MAX_NODES];
    __shared__ unsigned long long words_of[ROWS][TREE_MAX_NODES / 64];
    __shared__ int low_of[ROWS];
    __shared__ __align__(16) float join_o[2][ROWS][HD];
    __shared__ float join_ml[2][ROWS][2];
    // row blocks of the same keys lie a multiple of 8 workgroups apart: on one die, whose cache then holds the keys for all of them
    const int spread = (a.units + 7) & ~7, block = blockIdx.x / spread, unit = blockIdx.x % spread;
    if (unit >= a.units) return;
    const int kvh = unit % a.kv_heads, part = unit / a.kv_heads % a.parts, r = unit / (a.kv_heads * a.parts);
    const TreeRequest w(a, r);
    const int j0 = block * ROWS;
    if (!w.ok || j0 >= w.rows) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, qd = lane >> 4;
    const size_t per_head = static_cast<size_t>(HD) << a.page_shift, page_size = per_head * a.kv_heads * a.n_layers;
    const size_t head_block = per_head * (static_cast<size_t>(a.layer) * a.kv_heads + kvh);
    const T* __restrict__ k_pool = static_cast<const T*>(a.k_pool) + head_block;
    const T* __restrict__ v_pool = static_cast<const T*>(a.v_pool) + head_block;
    const int page_mask = a.page_tokens - 1;
    Frag q[RT][KS];
    int node_of[RT];
    tree_queries<T, HD, RT>(a, w, kvh, j0, q, node_of);
    const int n0 = j0 / a.group, n1 = min(j0 + ROWS - 1, w.rows - 1) / a.group;      // the block's nodes
    const TreeRounds rounds(a, w, part, KEYS);
    // the pages of a round, a lane each; asked for a round ahead (the first one's before the ways up the tree are gone)
    auto pages_of = [&](int round) {
        const int base = round * KEYS, last = (min(base + KEYS, w.end) - 1) >> a.page_shift;
        return round <= rounds.r_end ? w.pages[min((base >> a.page_shift) + lane, last)] : 0;
    };
    int next_page = pages_of(rounds.r_begin + wave);
    tree_ways<256>(a, w, n0, n1, up, words_of, low_of);
    float m[RT], l[RT];
    tree_f4 o[RT][DT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] = tree_f4{0.f, 0.f, 0.f, 0.f};
    }
    for (int round = rounds.r_begin + (tid >> 6); round <= rounds.r_end; round += 4) {
        const int base = round * KEYS, top = min(base + KEYS, w.end) - 1;
        const int first_page = base >> a.page_shift, last_page = top >> a.page_shift;
        int page = next_page;
        const bool there = page >= 0 && page < a.n_pages;
        const bool all_there = __ballot(!there) == 0ull;
        page = there ? page : 0;
        Frag k[TILES][KS], v[DT][VG];
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile) {
            const int key = min(base + O::key(tile, c), top);
            const T* from = k_pool + __shfl(page, (key >> a.page_shift) - first_page, 64) * page_size + static_cast<size_t>(key & page_mask) * HD;
#pragma unroll
            for (int s = 0; s < KS; ++s) k[tile][s] = *reinterpret_cast<const Frag*>(from + O::dim(s, qd));
        }
#pragma unroll
        for (int g = 0; g < VG; ++g) {
            const int key = min(base + O::vkey(g, qd), top & ~(O::VKEYS - 1));
            const T* from = v_pool + __shfl(page, (key >> a.page_shift) - first_page, 64) * page_size + (key & page_mask);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                v[dt][g] = *reinterpret_cast<const Frag*>(from + (static_cast<size_t>(16 * dt + c) << a.page_shift));
        }
        next_page = pages_of(round + 4);
        if (base >= rounds.plain && base + KEYS <= w.start && all_there) {
            tree_f4 s[RT][TILES];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int tile = 0; tile < TILES; ++tile) s[t][tile] = O::scores(k[tile], q[t]);
            tree_softmax<false>(s, m, l, o, a.scale);
#pragma unroll
            for (int t = 0; t < RT; ++t) O::values(v, s[t], o[t]);
            continue;
        }
        // A weight of 0 times an infinity or a NaN is no 0: such values are taken out, and added for the rows that see them
        unsigned bad = 0;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < VG; ++g) bad |= O::not_finite(v[dt][g]);
        const bool odd_values = __ballot(bad != 0) != 0ull;
        if (odd_values) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < VG; ++g) O::make_finite(v[dt][g]);
        }
        tree_f4 s[RT][TILES];
        unsigned long long seen_of[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int tile = 0; tile < TILES; ++tile) s[t][tile] = O::scores(k[tile], q[t]);
            const unsigned long long seen = tree_seen<KEYS>(a, w, base, all_there, !there, last_page, low_of[node_of[t] - n0], words_of[node_of[t] - n0]);
#pragma unroll
            for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[t][tile][i] = (O::shown(seen, tile, qd) >> O::bit(tile, i)) & 1u ? s[t][tile][i] * a.scale : -INFINITY;
            seen_of[t] = seen;
        }
        tree_softmax<true>(s, m, l, o, 1.f);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            O::values(v, s[t], o[t]);
            if (odd_values) tree_odd_values<T, KEYS>(o[t], v_pool, page_size, a.page_shift, base, last_page, page, seen_of[t]);
        }
    }
    // the four wavefronts' results: the upper two to the lower two, then those
#pragma unroll
    for (int t = 0; t < RT; ++t) l[t] = sum_half32(sum_row16(l[t]));
    for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                if (qd == 0) {
                    join_ml[wave - half][16 * t + c][0] = m[t];
                    join_ml[wave - half][16 * t + c][1] = l[t];
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<tree_f4*>(&join_o[wave - half][16 * t + c][16 * dt + 4 * qd]) = o[t][dt];
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const float other = join_ml[wave][16 * t + c][0], now = fmaxf(m[t], other), shift = now == -INFINITY ? 0.f : now;
                const float mine = __builtin_amdgcn_exp2f(m[t] - shift), theirs = __builtin_amdgcn_exp2f(other - shift);
                l[t] = l[t] * mine + join_ml[wave][16 * t + c][1] * theirs;
                m[t] = now;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    o[t][dt] = o[t][dt] * mine + *reinterpret_cast<const tree_f4*>(&join_o[wave][16 * t + c][16 * dt + 4 * qd]) * theirs;
            }
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int j = j0 + 16 * t + c;
        if (j < w.rows) tree_store<T, HD>(a, w.first + node_of[t], kvh * a.group + j % a.group, part, qd, m[t], l[t], o[t]);
    }
}

// ---- many rows, bfloat16: the keys and values of a round are staged in LDS for the NW wavefronts, each of which has 16 RT rows of
// its own.  Rounds travel straight from memory to one of NB buffers, NB - 1 ahead of the one that is worked on.
// Keys lie in LDS in the order of the score tiles; the 16-byte pieces of a row change places by the row's number, so that the lanes
// that are served together, which read the same piece of as many rows, read from all banks.
#define TREE_GLOBAL(p) reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(p))
#define TREE_LDS(p) reinterpret_cast<__attribute__((address_space(3))) void*>(reinterpret_cast<uintptr_t>(p))
#define TREE_PAGES 1024          // entries of a request's table row that are in LDS at a time

template <int N>
__device__ __forceinline__ void tree_wait_loads() {        // at most N of the wavefront's loads are still on their way
    static_assert(N < 64, "what the counter holds");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

template <int HD, int RT, int NW, int NB>
__global__ __launch_bounds__(64 * NW, 2) void tree_rows_kernel(const TreeArgs a) {
    // (rounds of 64 keys for any head size: staged keys cost no registers)
    using O = TreeOps<bf16, HD>;
    using O64 = TreeOps<bf16, 64>;
    using Frag = tree_bf16x8;
    constexpr int KEYS = 64, TILES = 4, KS = O::KS, DT = O::DT, ROWS = 16 * RT * NW, CH = HD / 8, THREADS = 64 * NW;
    constexpr int LOADS = HD / 8, PER = (LOADS + NW - 1) / NW;      // of keys, and of values, a round: 1 KB each
    struct Buffer {
        __bf16 k[KEYS * HD];
        __bf16 v[HD * KEYS];
    };
    extern __shared__ __align__(1024) char tree_lds[];
    Buffer* const buffers = reinterpret_cast<Buffer*>(tree_lds);       // [NB]
    __shared__ int up[TREE_MAX_NODES];
    __shared__ unsigned long long words_of[ROWS < TREE_MAX_NODES ? ROWS : TREE_MAX_NODES][TREE_MAX_NODES / 64];
    __shared__ int low_of[ROWS < TREE_MAX_NODES ? ROWS : TREE_MAX_NODES];
    __shared__ int page_list[TREE_PAGES + 1];
    __shared__ int any_gone;
    const int spread = (a.units + 7) & ~7, block = blockIdx.x / spread, unit = blockIdx.x % spread;
    if (unit >= a.units) return;
    const int kvh = unit % a.kv_heads, part = unit / a.kv_heads % a.parts, r = unit / (a.kv_heads * a.parts);
    const TreeRequest w(a, r);
    const int b0 = block * ROWS;
    if (!w.ok || b0 >= w.rows) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, qd = lane >> 4;
    const int j0 = b0 + wave * 16 * RT;
    const bool active = j0 < w.rows;       // (the others only help to stage)
    const size_t per_head = static_cast<size_t>(HD) << a.page_shift, page_size = per_head * a.kv_heads * a.n_layers;
    const size_t head_block = per_head * (static_cast<size_t>(a.layer) * a.kv_heads + kvh);
    const __bf16* __restrict__ k_pool = static_cast<const __bf16*>(a.k_pool) + head_block;
    const __bf16* __restrict__ v_pool = static_cast<const __bf16*>(a.v_pool) + head_block;
    const char* __restrict__ k_bytes = reinterpret_cast<const char*>(k_pool);
    const char* __restrict__ v_bytes = reinterpret_cast<const char*>(v_pool);
    const unsigned page_bytes = static_cast<unsigned>(2 * page_size);      // (below 2^31: checked by the host)
    const int page_mask = a.page_tokens - 1;
    Frag q[RT][KS];
    int node_of[RT];
    tree_queries<bf16, HD, RT>(a, w, kvh, j0, q, node_of);
    const int n0 = b0 / a.group, n1 = min(b0 + ROWS - 1, w.rows - 1) / a.group;
    if (tid == 0) any_gone = 0;
    tree_ways<THREADS>(a, w, n0, n1, up, words_of, low_of);
    const TreeRounds rounds(a, w, part, KEYS);

    // ---- the part's pages: whether all are there, and the first of them in LDS
    const int last_page = rounds.r_end >= rounds.r_begin ? (min(rounds.r_end * KEYS + KEYS, w.end) - 1) >> a.page_shift : 0;
    const int span = max(TREE_PAGES * a.page_tokens / KEYS, 1);        // rounds that the list serves
    int list_round = rounds.r_begin, list_page = 0;
    auto fill_list = [&](int round) {
        list_round = round;
        list_page = round * KEYS >> a.page_shift;
        for (int i = tid; i <= TREE_PAGES; i += THREADS) {
            const int page = w.pages[min(list_page + i, last_page)];
            page_list[i] = page >= 0 && page < a.n_pages ? page : 0;
        }
    };
    if (rounds.r_begin <= rounds.r_end) {
        fill_list(rounds.r_begin);
        bool gone = false;
        for (int i = (rounds.r_begin * KEYS >> a.page_shift) + tid; i <= last_page; i += THREADS) gone |= w.pages[i] < 0 || w.pages[i] >= a.n_pages;
        if (gone) any_gone = 1;
    }
    __syncthreads();
    const bool all_there = __builtin_amdgcn_readfirstlane(any_gone) == 0;

    // The load number wave + NW i of the keys (values) fills 64 pieces of 16 bytes from piece 64 (wave + NW i) on: the lane's row of
    // keys is CH pieces long, and of values 8.  What hangs on the lane is the same for every i, but for heads of 96.
    const int v_dim = 8 * wave + (lane >> 3), v_key = 8 * ((lane & 7) ^ ((lane >> 3) & 7));      // dimension v_dim + 8 NW i
    const int k_row = (64 * wave + lane) / CH;                                                     // row k_row + 64 NW / CH i
    const int k_piece = HD == 32 ? (lane & 3) ^ ((k_row >> 1) & 3) : HD == 128 ? (lane % CH) ^ (2 * (k_row & 7)) : (lane % CH) ^ (k_row & 7);
    auto key_of_row = [](int row) { return 32 * (row >> 5) + 8 * ((row >> 2) & 3) + 4 * ((row >> 4) & 1) + (row & 3); };
    auto fetch = [&](int round, Buffer& to) {
        const int base = round * KEYS, top = min(base + KEYS, w.end) - 1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (LOADS % NW && wave + NW * i >= LOADS) break;
            int row_key, piece;
            if (HD != 96) {
                row_key = key_of_row(k_row) + key_of_row(64 * NW / CH * i);
                piece = k_piece;
            } else {
                const int x = (wave + NW * i) * 64 + lane, row = x / CH;
                row_key = key_of_row(row);
                piece = (x % CH) ^ (row & 3);
            }
            const int key = min(base + row_key, top);
            const char* from = k_bytes + static_cast<uint64_t>(static_cast<unsigned>(page_list[(key >> a.page_shift) - list_page])) * page_bytes +
                               static_cast<unsigned>((key & page_mask) * (2 * HD) + piece * 16);
            __builtin_amdgcn_global_load_lds(TREE_GLOBAL(from), TREE_LDS(to.k + (wave + NW * i) * 512), 16, 0, 0);
        }
        const int key = min(base + v_key, top & ~7);
        const char* from = v_bytes + static_cast<uint64_t>(static_cast<unsigned>(page_list[(key >> a.page_shift) - list_page])) * page_bytes +
                           static_cast<unsigned>(2 * ((v_dim << a.page_shift) + (key & page_mask)));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (LOADS % NW && wave + NW * i >= LOADS) break;
            __builtin_amdgcn_global_load_lds(TREE_GLOBAL(from + (static_cast<unsigned>(16 * NW * i) << a.page_shift)),
                                             TREE_LDS(to.v + (wave + NW * i) * 512), 16, 0, 0);
        }
    };
    // where the lane's pieces of a row lie in LDS
    const int v_piece0 = qd ^ (c & 7), v_piece1 = (4 + qd) ^ (c & 7);
    auto k_piece_of = [&](int x) {
        return HD == 128 ? (4 * x + qd) ^ (2 * (c & 7)) : HD == 64 ? (x ? v_piece1 : v_piece0) : HD == 96 ? 4 * x + (qd ^ (c & 3)) : qd ^ ((c >> 1) & 3);
    };
    float m[RT], l[RT];
    tree_f4 o[RT][DT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] = tree_f4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < NB - 1; ++i)
        if (rounds.r_begin + i <= rounds.r_end) fetch(rounds.r_begin + i, buffers[i]);
    int cur = 0;
    for (int round = rounds.r_begin; round <= rounds.r_end; ++round, cur = cur + 1 == NB ? 0 : cur + 1) {
        // the round has arrived, for all wavefronts, and nobody reads the buffer of the one before any more
        if (NB > 2 && LOADS % NW == 0 && round + NB - 2 <= rounds.r_end) tree_wait_loads<(NB - 2) * 2 * PER>();
        else tree_wait_loads<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int ahead = round + NB - 1;
        if (ahead <= rounds.r_end) {
            if (ahead >= list_round + span) {       // (everybody has read what it needs of the list: the barrier)
                fill_list(ahead);
                __syncthreads();
            }
            fetch(ahead, buffers[cur == 0 ? NB - 1 : cur - 1]);
        }
        const Buffer& from = buffers[cur];
        auto keys_of = [&](int tile, int x) {
            return *reinterpret_cast<const Frag*>(from.k + (16 * tile + c) * HD + k_piece_of(x) * 8);
        };
        auto values_of = [&](int dt, int g) {
            return *reinterpret_cast<const Frag*>(from.v + (16 * dt + c) * KEYS + (g ? v_piece1 : v_piece0) * 8);
        };
        auto weights_of = [&](const tree_f4 (&s)[TILES], int g) {
            Frag p;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = static_cast<__bf16>(s[2 * g][i]);
                p[4 + i] = static_cast<__bf16>(s[2 * g + 1][i]);
            }
            return p;
        };
        const int base = round * KEYS;
        tree_f4 s[RT][TILES];
        auto scores = [&]() {
#pragma unroll
            for (int tile = 0; tile < TILES; ++tile) {
                Frag k[KS];
#pragma unroll
                for (int x = 0; x < KS; ++x) k[x] = keys_of(tile, x);
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t][tile] = O::scores(k, q[t]);
            }
        };
        if (active && base >= rounds.plain && base + KEYS <= w.start && all_there) {
            scores();
            if (!tree_weights(s, m, l, a.scale)) {
                scores();
                tree_softmax<false>(s, m, l, o, a.scale);
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                Frag p[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) p[t] = weights_of(s[t], g);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const Frag v = values_of(dt, g);
#pragma unroll
                    for (int t = 0; t < RT; ++t) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[t], o[t][dt], 0, 0, 0);
                }
            }
        } else if (active) {
            // A weight of 0 times an infinity or a NaN is no 0: such values are taken out, and added for the rows that see them
            const int first_page = base >> a.page_shift, end_page = (min(base + KEYS, w.end) - 1) >> a.page_shift;
            int page = w.pages[min(first_page + lane, end_page)];
            const bool gone = page < 0 || page >= a.n_pages;
            page = gone ? 0 : page;
            const bool round_there = __ballot(gone) == 0ull;
            unsigned long long seen[RT];
            scores();
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                seen[t] = tree_seen<KEYS>(a, w, base, round_there, gone, end_page, low_of[node_of[t] - n0], words_of[node_of[t] - n0]);
#pragma unroll
                for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[t][tile][i] = (O64::shown(seen[t], tile, qd) >> O64::bit(tile, i)) & 1u ? s[t][tile][i] * a.scale : -INFINITY;
            }
            tree_softmax<true>(s, m, l, o, 1.f);
            unsigned bad = 0;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                Frag p[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) p[t] = weights_of(s[t], g);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    Frag v = values_of(dt, g);
                    const unsigned b = O::not_finite(v);
                    if (b) O::make_finite(v);
                    bad |= b;
#pragma unroll
                    for (int t = 0; t < RT; ++t) o[t][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[t], o[t][dt], 0, 0, 0);
                }
            }
            if (__ballot(bad != 0)) {
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    tree_odd_values<bf16, KEYS>(o[t], reinterpret_cast<const bf16*>(v_pool), page_size, a.page_shift, base, end_page, page, seen[t]);
            }
        }
    }
    if (!active) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] = sum_half32(sum_row16(l[t]));
        const int j = j0 + 16 * t + c;
        if (j < w.rows) tree_store<bf16, HD>(a, w.first + node_of[t], kvh * a.group + j % a.group, part, qd, m[t], l[t], o[t]);
    }
}

template <int HD, int RT, int NW, int NB>
static void launch_tree_rows(const TreeArgs& a, dim3 grid, hipStream_t stream) {
    constexpr int bytes = NB * 2 * 64 * HD * 2;
    // (more than 64 KB a workgroup has to be asked for; the same call every time, which costs nothing next to the launch)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(tree_rows_kernel<HD, RT, NW, NB>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    tree_rows_kernel<HD, RT, NW, NB><<<grid, dim3(64 * NW), bytes, stream>>>(a);
}

// The parts of a node and query head: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  A wavefront each; four to a workgroup.
template <typename T, int HD>
__global__ __launch_bounds__(256) void tree_join_kernel(const TreeArgs a) {
    const int lane = threadIdx.x & 63;
    const long long id = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int head = static_cast<int>(id % a.heads), node = static_cast<int>(id / a.heads % a.max_nodes);
    const long long r = id / (static_cast<long long>(a.heads) * a.max_nodes);
    if (r >= a.requests) return;
    const int first = a.offsets[r], slot = a.slots[r];
    if (node >= tree_count(a.offsets, r, a.n_rows, a.max_nodes) || slot < 0 || slot >= a.table_rows) return;
    const size_t at = (static_cast<size_t>(first + node) * a.heads + head) * a.parts;
    // A part (of up to 64) a lane: its weight, which the others take from there.  Up to eight parts' outputs are asked for together (8
    // parts of 208 nodes, 32 heads of 64: 4.5 us, one after the other 6.3).
    const bool has = lane < a.parts;
    const float m = has ? a.ws_ml[2 * (at + lane)] : -INFINITY, l = has ? a.ws_ml[2 * (at + lane) + 1] : 0.f;
    const float high = wave_max(m), weight = __builtin_amdgcn_exp2f(m - (high == -INFINITY ? 0.f : high));
    const float sum = wave_sum(weight * l);
    constexpr int PER = (HD + 63) / 64;
    float o[PER] = {};
    auto add = [&](auto together, int p0) {
        constexpr int N = decltype(together)::value;
        float from[N][PER];
#pragma unroll
        for (int p = 0; p < N; ++p)
#pragma unroll
            for (int e = 0; e < PER; ++e) from[p][e] = a.ws_o[(at + min(p0 + p, a.parts - 1)) * HD + min(lane + 64 * e, HD - 1)];
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), p0 + p));
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] = p0 + p < a.parts ? fmaf(w, from[p][e], o[e]) : o[e];
        }
    };
    for (int p0 = 0; p0 < a.parts;) {
        if (a.parts - p0 <= 2) {
            add(std::integral_constant<int, 2>{}, p0);
            p0 += 2;
        } else {
            add(std::integral_constant<int, 8>{}, p0);
            p0 += 8;
        }
    }
    T* to = static_cast<T*>(a.out) + (static_cast<size_t>(first + node) * a.heads + head) * HD;
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (lane + 64 * e < HD) to[lane + 64 * e] = from_float<T>(sum == 0.f ? 0.f : o[e] / sum);
}

// The form of a launch: whether keys are staged, row tiles of a wavefront, rows of a workgroup, keys of a round, and workgroups
// that a compute unit holds.
//   Up to 32 rows nothing is gained by staging: four wavefronts read 16 or 32 rows' keys themselves.  Above, staged: 64 rows by four
// wavefronts, 128 by four with two row tiles each, and more by eight, which read every key once for 256 rows, from four buffers (16
// trees of 64 nodes behind 16,384 tokens, 32 heads of 128 on 8: 368 us, in workgroups of 128 rows 419; behind 14,192, heads of 64: 205 and
// 221; 8 trees of 64 behind 8,192 tokens, heads of 64: 69 and 72, of 128 112 and 119).
struct TreeForm {
    bool staged;
    int tiles, rows, keys, resident;
};
static TreeForm tree_form(int dtype, int head_dim, int rows) {
    if (dtype == CELEG_BF16 && rows > 32) {
        if (rows <= 64) return {true, 1, 64, 64, 2};
        if (rows <= 128) return {true, 2, 128, 64, 2};
        return {true, 2, 256, 64, 1};
    }
    const int tiles = rows <= 16 || (dtype != CELEG_BF16 && head_dim > 64) ? 1 : 2;
    return {false, tiles, 16 * tiles, dtype == CELEG_BF16 && head_dim <= 64 ? 64 : 32, 2};
}

// Whether the matrix cores take these sizes.
extern "C" int celeg_tree_attention_fast_ok(int head_dim, int page_tokens) {
    return (head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128) && page_tokens >= 16 && (page_tokens & (page_tokens - 1)) == 0;
}

// Parts that the contexts are cut into (0: more workgroups than a launch has).
//   Few rounds are one workgroup's: up to 12 (4 where keys are staged) a second kernel costs more than the wait (1 request of 8 nodes,
// 16 heads of 64 on 8, behind 500, 700, 760, 900, 1,100 and 1,500: 8.4, 9.3, 9.6, 10.5, 11.6 and 13.6 us, in the best number of parts 9.8,
// 10.6, 10.8, 10.3, 10.4 and 10.4, and a launch less for the host; of 4 requests behind 760 and 1,100 11.8 and 13.8, 12.6 and 11.9).  In 32 bits, whose
// rounds take longer, the two meet earlier (3 of 13 behind 200, 300 and 500: 12.9, 15.6 and 20.3, 13.2, 13.4 and 14.0), but a launch more
// is the host's.
//   More: 256 workgroups, one a compute unit, each wavefront (each workgroup that stages: two) with a round at least: a second one beside it
// gains less than its part costs to join (4 trees of 8 behind 6,000, 32 heads of 64 on 8: 20.0 us, of 512 workgroups 22.9; heads
// of 128 29.7 and 34.9).  Staged rounds in long parts gain more from it; the limits, 16 rounds a part and 40 of wider heads, lie where no case loses.
// Heads of 64, 8 trees of 26 behind 2,500, 4,000, 6,000 and 16,000 (10, 16, 24 and 63 rounds a part of 256 workgroups): 25.6, 30.2, 39.2 and 84
// us, of 512 25.3, 27.3, 34.5 and 70; 4 trees (5, 8, 12 and 31) 18.5, 21.1, 26.2 and 46, 19.2, 21.7, 25.1 and 40.  Heads of 128, 8 trees behind 6,000, 8,000
// and 16,000 (24, 31 and 63) 60, 77 and 134, 61, 73 and 121; 4 trees behind 8,000, 11,000 and 16,000 (16, 22 and 31) 40, 54 and 74, 47, 57 and 72.
extern "C" int celeg_tree_attention_parts(int dtype, int head_dim, int requests, int kv_heads, int group, int max_nodes, int max_context) {
    const int rows = max_nodes * group;
    const TreeForm form = tree_form(dtype, head_dim, rows);
    const long long groups = static_cast<long long>(requests) * kv_heads * ((rows + form.rows - 1) / form.rows);
    const long long rounds = (static_cast<long long>(max_context) + max_nodes + form.keys - 1) / form.keys;
    // (a launch has fewer than 2^32 threads, here of up to 512 a workgroup)
    const auto fits = [&](long long parts) {
        return (groups * parts + 8LL * ((rows + form.rows - 1) / form.rows)) * 512 < 1LL << 32 &&
               (parts == 1 || static_cast<long long>(requests) * max_nodes * kv_heads * group / 4 + 1 < 1LL << 24);
    };
    if (rounds <= (form.staged ? 4 : 12)) return fits(1) ? 1 : 0;
    long long parts = (256 + groups - 1) / groups;
    if (form.staged && form.resident > 1 && rounds > (head_dim > 64 ? 40 : 16) * parts) parts = (256 * form.resident + groups - 1) / groups;
    parts = std::max(1LL, std::min({parts, form.staged ? (rounds + 1) / 2 : (rounds + 3) / 4, 64LL}));
    return fits(parts) ? static_cast<int>(parts) : 0;
}

extern "C" int celeg_tree_attention_fast(const void* q, int ldq, int dtype, const void* k_pool, const void* v_pool, int n_pages, int n_layers,
                                         int layer, int heads, int kv_heads, int head_dim, int page_tokens, const int* table, int table_rows,
                                         int table_stride, const int* slots, const int* starts, const int* offsets, const int* parents,
                                         int n_requests, int n_rows, int max_nodes, int parts, float scale, int window, void* out,
                                         void* workspace, hipStream_t stream) {
    TreeArgs a;
    a.q = q;
    a.k_pool = k_pool;
    a.v_pool = v_pool;
    a.table = table;
    a.slots = slots;
    a.starts = starts;
    a.offsets = offsets;
    a.parents = parents;
    a.out = out;
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = parts > 1 ? a.ws_o + static_cast<size_t>(n_rows) * heads * parts * head_dim : nullptr;
    a.ldq = ldq;
    a.n_pages = n_pages;
    a.n_layers = n_layers;
    a.layer = layer;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.group = heads / kv_heads;
    a.page_tokens = page_tokens;
    a.page_shift = __builtin_ctz(page_tokens);
    a.table_rows = table_rows;
    a.table_stride = table_stride;
    a.requests = n_requests;
    a.n_rows = n_rows;
    a.max_nodes = max_nodes;
    a.parts = parts;
    a.units = n_requests * kv_heads * parts;
    a.scale = fabsf(scale) * 1.44269504088896340736f;
    a.turned = scale < 0.f;
    a.window = window;
    const int rows = max_nodes * a.group;
    const TreeForm form = tree_form(dtype, head_dim, rows);
    a.row_blocks = (rows + form.rows - 1) / form.rows;
    const dim3 grid(static_cast<unsigned>((a.units + 7) / 8 * 8) * a.row_blocks);
    const dim3 join(static_cast<unsigned>((static_cast<long long>(n_requests) * max_nodes * heads + 3) / 4));
    auto run = [&](auto* type, auto dim) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int HD = decltype(dim)::value;
        constexpr bool B = std::is_same<T, bf16>::value;
        if (form.staged) {
            if constexpr (B) {
                if (form.rows == 256) launch_tree_rows<HD, 2, 8, 4>(a, grid, stream);
                else if (form.tiles == 2) launch_tree_rows<HD, 2, 4, 2>(a, grid, stream);
                else launch_tree_rows<HD, 1, 4, 2>(a, grid, stream);
            }
        } else if (form.tiles == 2) {
            if constexpr (B || HD <= 64) tree_few_kernel<T, HD, 2><<<grid, dim3(256), 0, stream>>>(a);
        } else {
            tree_few_kernel<T, HD, 1><<<grid, dim3(256), 0, stream>>>(a);
        }
        if (parts > 1) tree_join_kernel<T, HD><<<join, dim3(256), 0, stream>>>(a);
    };
    auto by_dim = [&](auto* type) {
        if (head_dim == 32) run(type, std::integral_constant<int, 32>{});
        else if (head_dim == 64) run(type, std::integral_constant<int, 64>{});
        else if (head_dim == 96) run(type, std::integral_constant<int, 96>{});
        else run(type, std::integral_constant<int, 128>{});
    };
    if (dtype == CELEG_BF16) by_dim(static_cast<bf16*>(nullptr));
    else by_dim(static_cast<float*>(nullptr));
    return CELEG_LAUNCH_RESULT();
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
    const int first = offsets[r], count = tree_count(offsets, r, n_rows, max_nodes);
    const int slot = slots[r], start = tree_start(starts, r);
    if (node >= count || slot < 0 || slot >= table_rows) return;
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
    const int room = table_stride * page_tokens;       // (below 2^31: checked by the host; places behind it are seen by nobody)
    const int end = start < room ? min(start + count, room) : room;
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
        if (lane + 64 * e < head_dim) orow[lane + 64 * e] = from_float<T>(l == 0.f ? 0.f : o[e] / l);
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
