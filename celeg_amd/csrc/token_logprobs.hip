// What rows of logits say about tokens: log probability and rank of given tokens, the entropy, the best alternatives.
//   m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):  logprob(t) = x_t - m - ln S,  entropy = ln S - T / S;
//   rank(t) = how many logits stand ahead of t's: larger ones, and equal ones of lower index.
// The exponentials and T are kept in powers of two, d = (x - m) log2(e), so that an exponential is one instruction.
// A logit of -inf has probability 0.  A row without a distribution (a NaN, a +inf, nothing but -inf) gets NaN for
// log probabilities and entropy; one that holds a NaN has no order either: ranks and alternatives are -1 then.
// A token outside the vocabulary gets NaN and -1; nothing is read for it.
//
// What bounds it is the one read of the logits.  A workgroup of 256 threads takes a part of a row into its registers (up to
// 64 logits a thread), and finds there in turn the maximum, the sums, the tokens' ranks and the part's best: four such
// workgroups share a compute unit, so that one's arithmetic runs while another's loads are on their way.  Few rows are cut into
// more parts, so that all compute units take part; a second kernel, a workgroup a row, joins the parts.
//
// The best of a part: the top-th largest of the maxima of 64 (256) groups of threads is not above the top-th largest logit,
// so that the logits not below it hold all that is sought and little more; they are collected and counted against one another.
// Where too many are (thousands of equal logits), the bound is raised by halving first the logits, then the indices.
#include "common.h"

#define LP_THREADS 256
#define LP_WAVES 4
#define LP_LIST 512           // logits that a part's best are chosen from
#define LP_GROUPS 256         // groups of 16 bytes that hold one of them
#define LP_JOIN 2048          // candidates of a row looked at together
#define LP_MAX_TOKENS 8
#define LP_MAX_TOP 128

typedef float lp_f4 __attribute__((ext_vector_type(4)));
typedef unsigned int lp_u4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// 16 bytes of logits as they lie in memory
template <typename T> struct LogitGroup;
template <> struct LogitGroup<float> {
    static constexpr int N = 4;
    lp_f4 v;
    __device__ __forceinline__ void none() { v = lp_f4{NAN, NAN, NAN, NAN}; }
    __device__ __forceinline__ float get(int e) const { return v[e]; }
};
template <> struct LogitGroup<bf16> {
    static constexpr int N = 8;
    lp_u4 v;
    __device__ __forceinline__ void none() { v = lp_u4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}; }
    __device__ __forceinline__ float get(int e) const { return __uint_as_float((e & 1) ? (v[e >> 1] & 0xffff0000u) : (v[e >> 1] << 16)); }
};

// the next float below a finite one or +inf (of -0 and +0: the smallest negative one)
__device__ __forceinline__ float next_below(float x) {
    const unsigned u = __float_as_uint(x);
    return x == 0.f ? __uint_as_float(0x80000001u) : __uint_as_float((u & 0x80000000u) ? u + 1u : u - 1u);
}

struct LogprobOut {
    float* logprobs;
    int* ranks;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
};

// What a part of a row leaves for the join.  stats: m, S, T, and how its order stands (1: a NaN).
struct LogprobParts {
    float4* stats;                   // [rows, parts]
    int* ranks;                      // [rows, parts, per_row]
    unsigned long long* best;        // [rows, parts, top], falling, 0 where the part has no more
};

__device__ __forceinline__ float best_logit(unsigned long long packed) {
    const uint32_t key = static_cast<uint32_t>(packed >> 32);
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ float logprob_of(float x, float m, float log2_sum) { return (x - m) - log2_sum * LN2; }

// Of n packed logits in `list` (all different), the `top` largest in falling order: put(place, packed).  All threads call it.
template <typename F>
__device__ __forceinline__ void sorted_best(const unsigned long long* list, int n, int top, F put) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const unsigned long long mine = list[i];
        int ahead = 0;
        for (int j = 0; j < n; ++j) ahead += list[j] > mine;
        if (ahead < top) put(ahead, mine);
    }
}

// ---------------------------------------------------------------------------- a part of a row
// Too many logits lie at or above the bound for the list (thousands of equal ones, or a bound of -inf where a vocabulary is
// masked down to a few tokens): exactly the `top` best of columns c0 .. c1 - 1 go to the list.  The logits are read again for
// every halving; all threads call it.  (No NaN among them.)
template <typename T>
__device__ __noinline__ int best_by_halving(const T* __restrict__ x, int c0, int c1, int top, float bound, float high,
                                            unsigned long long* list, int* counts, int* count) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int turn = 0;
    auto count_of = [&](auto take) {
        int n = 0;
        for (int c = c0 + tid; c < c1; c += LP_THREADS) n += take(order_key(to_float(x[c]) + 0.0f), c);
        const float of_wave = wave_sum(static_cast<float>(n));
        turn ^= 1;                       // (the other half of counts may still be read)
        if (lane == 0) counts[turn * LP_WAVES + wave] = static_cast<int>(of_wave);
        __syncthreads();
        const int* of = counts + turn * LP_WAVES;
        return of[0] + of[1] + of[2] + of[3];
    };
    // the largest key that `wanted` logits are not below
    const int wanted = min(top, c1 - c0);
    uint32_t key = order_key(bound + 0.0f), most = order_key(high + 0.0f);
    while (key < most) {
        const uint32_t middle = key + (most - key) / 2 + 1;
        if (count_of([&](uint32_t k, int) { return k >= middle; }) >= wanted) key = middle;
        else most = middle - 1;
    }
    // of those that have it, the lowest index up to which there are enough
    const int above = count_of([&](uint32_t k, int) { return k > key; });
    int last = c0, end = c1 - 1;
    while (last < end) {
        const int middle = last + (end - last) / 2;
        if (above + count_of([&](uint32_t k, int c) { return k == key && c <= middle; }) >= wanted) end = middle;
        else last = middle + 1;
    }
    __syncthreads();
    if (tid == 0) *count = 0;
    __syncthreads();
    for (int c = c0 + tid; c < c1; c += LP_THREADS) {
        const float v = to_float(x[c]);
        const uint32_t k = order_key(v + 0.0f);
        if (k > key || (k == key && c <= last)) {
            const int place = atomicAdd(count, 1);
            if (place < LP_LIST) list[place] = packed_logit(v, c);
        }
    }
    __syncthreads();
    return min(*count, LP_LIST);
}

// A thread holds GROUPS groups of 16 bytes, and one logit more where the part begins or ends off a boundary of 16 bytes.  What
// it holds beyond the part is a NaN: no comparison and no sum takes it.
template <typename T, int GROUPS>
__global__ __launch_bounds__(LP_THREADS, 4) void logprobs_part_kernel(
    const T* __restrict__ logits, long long row_stride, const int* __restrict__ tokens, int vocab, int per_row, int top, int parts,
    int part_size, const LogprobParts left, const LogprobOut out) {
    using Group = LogitGroup<T>;
    constexpr int N = Group::N;
    __shared__ float wave_of[LP_WAVES][2 + LP_MAX_TOKENS];
    __shared__ float wave_high[LP_WAVES];
    __shared__ int wave_bad[LP_WAVES];
    __shared__ __align__(16) float maxima[LP_THREADS];
    __shared__ float bounds[LP_WAVES];
    __shared__ int n_groups, count, counts[2 * LP_WAVES];
    __shared__ Group hit[LP_GROUPS];
    __shared__ int hit_at[LP_GROUPS];
    __shared__ unsigned long long list[LP_LIST];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int part = blockIdx.x % parts;
    const size_t row = blockIdx.x / parts;
    const T* __restrict__ x = logits + row * static_cast<size_t>(row_stride);
    const int c0 = part * part_size, c1 = min(vocab, c0 + part_size);
    // whole groups: `whole` of them from column a0 on
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x + c0) / sizeof(T)) % N);
    const int a0 = min(c0 + (N - off) % N, c1), whole = (c1 - a0) / N;
    Group g[GROUPS];
    if (whole > 0) {
        const decltype(g[0].v)* from = reinterpret_cast<const decltype(g[0].v)*>(x + a0);
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) g[j].v = from[min(tid + j * LP_THREADS, whole - 1)];
    } else {
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) g[j].none();
    }
    // the logits before a0 (threads 0 .. N - 1) and behind the last whole group (threads N .. 2N - 1)
    const int edge = tid < N ? c0 + tid : a0 + whole * N + (tid - N);
    const bool has_edge = tid < N ? edge < a0 : tid < 2 * N && edge < c1;
    const float extra = has_edge ? to_float(x[edge]) : NAN;
    // (token i of the row and its logit in lane i)
    int token = -1;
    float at = INFINITY;
    if (lane < per_row) {
        token = tokens[row * per_row + lane];
        if (token >= 0 && token < vocab) at = to_float(x[token]);
    }
    if (tid == 0) {
        n_groups = 0;
        count = 0;
    }
    if (whole < GROUPS * LP_THREADS) {
#pragma unroll
        for (int j = 0; j < GROUPS; ++j)
            if (tid + j * LP_THREADS >= whole) g[j].none();
    }
    // ---- the maximum
    float high = fmaxf(-INFINITY, extra);
    bool bad = has_edge && extra != extra;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
        bool of_group = false;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float v = g[j].get(e);
            high = fmaxf(high, v);
            of_group |= v != v;
        }
        bad |= of_group && tid + j * LP_THREADS < whole;
    }
    const bool any_bad = __ballot(bad) != 0ull;
    const float wave_max_value = wave_max(high);
    // (the maxima of 4 lanes each where 64 are well more than are sought)
    const bool few = top <= 40;
    if (few) {
        float of_four = fmaxf(high, lane_move<LANES_XOR_1>(high));
        of_four = fmaxf(of_four, lane_move<LANES_XOR_2>(of_four));
        if ((lane & 3) == 0) maxima[tid >> 2] = of_four;
    } else {
        maxima[tid] = high;
    }
    if (lane == 0) {
        wave_high[wave] = wave_max_value;
        wave_bad[wave] = any_bad;
    }
    __syncthreads();
    high = fmaxf(fmaxf(wave_high[0], wave_high[1]), fmaxf(wave_high[2], wave_high[3]));
    bad = (wave_bad[0] | wave_bad[1] | wave_bad[2] | wave_bad[3]) != 0;
    // ---- the bound for the best: the least of the maxima that fewer than `top` others lie above
    if (top > 0 && tid < (few ? 64 : LP_THREADS)) {
        const int n = few ? 64 : LP_THREADS;
        const float mine = maxima[tid];
        int above = 0;
        for (int j = 0; j < n; j += 4) {
            const lp_f4 o = *reinterpret_cast<const lp_f4*>(maxima + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) above += o[e] > mine;
        }
        const float least = -wave_max(above < top ? -mine : -INFINITY);
        if (lane == 0) bounds[wave] = least;
    }
    // ---- the sums.  (The maximum is taken off first: a mask of the type's lowest value times log2(e) would be no number.)
    // Below -2000 the exponential is 0 in any case, and 0 times -2000 is no NaN.
    const float m = high == -INFINITY ? 0.f : high;
    float sum = 0.f, moment = 0.f;
    auto add = [&](float v) {
        const float d = fmaxf((v - m) * LOG2E, -2000.f);
        const float p = __builtin_amdgcn_exp2f(d);
        sum += p;
        moment = fmaf(p, d, moment);
    };
#pragma unroll
    for (int j = 0; j < GROUPS; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) add(g[j].get(e));
    add(extra);
    sum = wave_sum(sum);
    moment = wave_sum(moment);
    if (lane == 0) {
        wave_of[wave][0] = sum;
        wave_of[wave][1] = moment;
    }
    // ---- the tokens' ranks: logits above the token's, and, before it, equal ones
    for (int i = 0; i < per_row; ++i) {
        const int t = __builtin_amdgcn_readlane(token, i);
        const float v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, at), i));
        int ahead = 0;
        if (v == -INFINITY) {                   // (nothing is below it: counted from memory)
            for (int c = c0 + tid; c < c1; c += LP_THREADS) ahead += to_float(x[c]) > v || c < t;
        } else {
            const float below = next_below(v);
            // before the token, "not below it" is "above the next number below it"
            const int before = t >= a0 ? (t - a0) / N : 0;
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
                const float over = tid + j * LP_THREADS < before ? below : v;
#pragma unroll
                for (int e = 0; e < N; ++e) ahead += g[j].get(e) > over;
            }
            ahead += extra > v || (extra == v && edge < t);
            // the group that the token lies in
            if (before < whole && tid == before % LP_THREADS)
                for (int c = a0 + before * N; c < t; ++c) ahead += to_float(x[c]) == v;
        }
        const float total = wave_sum(static_cast<float>(ahead));       // (at most 16,384: exact)
        if (lane == 0) wave_of[wave][2 + i] = total;
    }
    __syncthreads();
    // ---- the best: groups with a logit not below the bound, then those logits
    int have = 0;
    if (top > 0 && !bad) {
        const float bound = few ? bounds[0] : fminf(fminf(bounds[0], bounds[1]), fminf(bounds[2], bounds[3]));
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
            float of_group = g[j].get(0);
#pragma unroll
            for (int e = 1; e < N; ++e) of_group = fmaxf(of_group, g[j].get(e));
            if (of_group >= bound) {
                const int place = atomicAdd(&n_groups, 1);
                if (place < LP_GROUPS) {
                    hit[place] = g[j];
                    hit_at[place] = a0 + (tid + j * LP_THREADS) * N;
                }
            }
        }
        if (extra >= bound) list[atomicAdd(&count, 1)] = packed_logit(extra, edge);        // (up to 2N of them)
        __syncthreads();
        const int hits = min(n_groups, LP_GROUPS);
        for (int i = tid; i < hits * N; i += LP_THREADS) {
            const float v = hit[i / N].get(i % N);
            if (v >= bound) {
                const int place = atomicAdd(&count, 1);
                if (place < LP_LIST) list[place] = packed_logit(v, hit_at[i / N] + i % N);
            }
        }
        __syncthreads();
        have = count;
        if (n_groups > LP_GROUPS || have > LP_LIST) have = best_by_halving(x, c0, c1, top, bound, high, list, counts, &count);
    }
    sum = wave_of[0][0] + wave_of[1][0] + wave_of[2][0] + wave_of[3][0];
    moment = wave_of[0][1] + wave_of[1][1] + wave_of[2][1] + wave_of[3][1];
    if (parts > 1) {
        const size_t at_part = row * parts + part;
        if (tid == 0) left.stats[at_part] = make_float4(high, sum, moment, bad ? 1.f : 0.f);
        if (tid < per_row)
            left.ranks[at_part * per_row + tid] =
                static_cast<int>(wave_of[0][2 + tid] + wave_of[1][2 + tid] + wave_of[2][2 + tid] + wave_of[3][2 + tid]);
        unsigned long long* best = left.best + at_part * top;
        for (int k = have + tid; k < top; k += LP_THREADS) best[k] = 0ull;
        sorted_best(list, have, top, [&](int place, unsigned long long packed) { best[place] = packed; });
        return;
    }
    const bool none = bad || high == INFINITY || high == -INFINITY;
    const float log2_sum = none ? NAN : __builtin_amdgcn_logf(sum);
    if (tid == 0 && out.entropy) out.entropy[row] = (log2_sum - moment / sum) * LN2;
    if (tid < per_row) {
        const int t = tokens[row * per_row + tid];
        const bool valid = t >= 0 && t < vocab;
        const float total = wave_of[0][2 + tid] + wave_of[1][2 + tid] + wave_of[2][2 + tid] + wave_of[3][2 + tid];
        out.logprobs[row * per_row + tid] = valid ? logprob_of(to_float(x[t]), m, log2_sum) : NAN;
        out.ranks[row * per_row + tid] = valid && !bad ? static_cast<int>(total) : -1;
    }
    if (bad) {
        for (int k = tid; k < top; k += LP_THREADS) {
            out.top_ids[row * top + k] = -1;
            out.top_logprobs[row * top + k] = NAN;
        }
        return;
    }
    sorted_best(list, have, top, [&](int place, unsigned long long packed) {
        out.top_ids[row * top + place] = packed_logit_index(packed);
        out.top_logprobs[row * top + place] = logprob_of(best_logit(packed), m, log2_sum);
    });
}

// ---------------------------------------------------------------------------- the parts of a row joined
// The best of several falling lists: with `depth` taken of each of n lists, the ceil(top / depth)-th largest of their depth-th
// entries has `top` entries not below it; what is not below it is sorted.  More lists than fit are taken in turn, the best so far
// among them.
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_join_kernel(
    const T* __restrict__ logits, long long row_stride, const int* __restrict__ tokens, int vocab, int per_row, int top, int parts,
    const LogprobParts left, const LogprobOut out) {
    __shared__ unsigned long long all[LP_JOIN], list[LP_JOIN], so_far[LP_MAX_TOP];
    __shared__ unsigned long long bound_shared;
    __shared__ float wave_of[3][LP_WAVES];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    const T* __restrict__ x = logits + row * static_cast<size_t>(row_stride);
    const float4* stats = left.stats + row * parts;
    float high = -INFINITY, bad = 0.f;
    for (int p = tid; p < parts; p += LP_THREADS) {
        high = fmaxf(high, stats[p].x);
        bad += stats[p].w;
    }
    high = wave_max(high);
    bad = wave_sum(bad);
    if (lane == 0) {
        wave_of[0][wave] = high;
        wave_of[1][wave] = bad;
    }
    __syncthreads();
    high = fmaxf(fmaxf(wave_of[0][0], wave_of[0][1]), fmaxf(wave_of[0][2], wave_of[0][3]));
    bad = wave_of[1][0] + wave_of[1][1] + wave_of[1][2] + wave_of[1][3];
    const float m = high == -INFINITY ? 0.f : high;
    float sum = 0.f, moment = 0.f;
    for (int p = tid; p < parts; p += LP_THREADS) {
        const float4 s = stats[p];
        const float d = fmaxf((s.x - m) * LOG2E, -2000.f), w = __builtin_amdgcn_exp2f(d);
        sum = fmaf(w, s.y, sum);
        moment = fmaf(w, fmaf(d, s.y, s.z), moment);
    }
    sum = wave_sum(sum);
    moment = wave_sum(moment);
    __syncthreads();
    if (lane == 0) {
        wave_of[0][wave] = sum;
        wave_of[2][wave] = moment;
    }
    __syncthreads();
    sum = wave_of[0][0] + wave_of[0][1] + wave_of[0][2] + wave_of[0][3];
    moment = wave_of[2][0] + wave_of[2][1] + wave_of[2][2] + wave_of[2][3];
    const bool none = bad > 0.f || high == INFINITY || high == -INFINITY;
    const float log2_sum = none ? NAN : __builtin_amdgcn_logf(sum);
    if (tid == 0 && out.entropy) out.entropy[row] = (log2_sum - moment / sum) * LN2;
    // a wavefront a token: the parts' counts
    for (int i = wave; i < per_row; i += LP_WAVES) {
        int total = 0;
        for (int p = lane; p < parts; p += 64) total += left.ranks[(row * parts + p) * per_row + i];
        total = static_cast<int>(wave_sum(static_cast<float>(total)));       // (at most 2^24: exact)
        if (lane == 0) {
            const int t = tokens[row * per_row + i];
            const bool valid = t >= 0 && t < vocab;
            out.logprobs[row * per_row + i] = valid ? logprob_of(to_float(x[t]), m, log2_sum) : NAN;
            out.ranks[row * per_row + i] = valid && bad == 0.f ? total : -1;
        }
    }
    if (top == 0) return;
    if (bad > 0.f) {
        for (int k = tid; k < top; k += LP_THREADS) {
            out.top_ids[row * top + k] = -1;
            out.top_logprobs[row * top + k] = NAN;
        }
        return;
    }
    const int room = LP_JOIN / top;
    for (int done = 0; done < parts;) {
        const int kept = done > 0 ? 1 : 0, fresh = min(parts - done, room - kept), lists = kept + fresh;
        __syncthreads();
        for (int i = tid; i < kept * top; i += LP_THREADS) all[i] = so_far[i];
        for (int i = tid; i < fresh * top; i += LP_THREADS) all[kept * top + i] = left.best[(row * parts + done) * top + i];
        if (tid == 0) {
            count = 0;
            bound_shared = 1ull;
        }
        __syncthreads();
        const int depth = (top + lists - 1) / lists, nth = (top + depth - 1) / depth;
        for (int i = tid; i < lists; i += LP_THREADS) {
            const unsigned long long mine = all[i * top + depth - 1];
            int ahead = 0;
            for (int j = 0; j < lists; ++j) {
                const unsigned long long other = all[j * top + depth - 1];
                ahead += other > mine || (other == mine && j < i);
            }
            if (ahead == nth - 1 && mine > 0ull) bound_shared = mine;       // (0: a list has no such entry; then everything counts)
        }
        __syncthreads();
        const unsigned long long bound = bound_shared;
        for (int i = tid; i < lists * top; i += LP_THREADS)
            if (all[i] >= bound) list[atomicAdd(&count, 1)] = all[i];
        __syncthreads();
        done += fresh;
        const int have = count;
        if (done < parts) {
            for (int k = tid; k < top; k += LP_THREADS)
                if (k >= have) so_far[k] = 0ull;
            sorted_best(list, have, top, [&](int place, unsigned long long packed) { so_far[place] = packed; });
        } else {
            sorted_best(list, have, top, [&](int place, unsigned long long packed) {
                out.top_ids[row * top + place] = packed_logit_index(packed);
                out.top_logprobs[row * top + place] = logprob_of(best_logit(packed), m, log2_sum);
            });
        }
    }
}

// ---------------------------------------------------------------------------- how a call is cut
// Parts of a row, and logits of a part.  A part holds at most `most` logits; with few rows it is smaller, down to 1,024.
static void logprobs_cut(long long rows, int vocab, int dtype, bool aligned, int& parts, int& part_size, int& groups) {
    const int n = dtype == CELEG_BF16 ? 8 : 4;
    const int sizes[3] = {1, dtype == CELEG_BF16 ? 2 : 4, dtype == CELEG_BF16 ? 8 : 16};
    for (int i = 0; i < 3; ++i) {
        groups = sizes[i];
        // (rows that begin off a boundary need a group more)
        const int most = LP_THREADS * groups * n - (aligned ? 0 : n);
        parts = (vocab + most - 1) / most;
        part_size = ((vocab + parts - 1) / parts + n - 1) / n * n;
        if (part_size > most) part_size = most;
        parts = (vocab + part_size - 1) / part_size;
        if (rows * parts <= 1024 && parts <= 64) return;
    }
}

static bool logprobs_aligned(const void* logits, int dtype, long long row_stride, long long rows) {
    const long long n = dtype == CELEG_BF16 ? 8 : 4;
    return reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (rows <= 1 || row_stride % n == 0);
}

// Bytes of workspace of a call (for any alignment of the logits).
extern "C" size_t celeg_logprobs_workspace(int dtype, long long rows, int vocab, int per_row, int top) {
    size_t bytes = 0;
    for (int aligned = 0; aligned < 2; ++aligned) {
        int parts, part_size, groups;
        logprobs_cut(rows, vocab, dtype, aligned != 0, parts, part_size, groups);
        const size_t all = static_cast<size_t>(rows) * parts;
        const size_t b = parts > 1 ? all * 16 + all * top * 8 + all * per_row * 4 : 0;
        bytes = b > bytes ? b : bytes;
    }
    return (bytes + 15) / 16 * 16;
}

extern "C" int celeg_logprobs_rows(const void* logits, int dtype, long long rows, int vocab, long long row_stride, const int* tokens,
                                   int per_row, int top, float* logprobs, int* ranks, float* entropy, int* top_ids,
                                   float* top_logprobs, void* workspace, hipStream_t stream) {
    int parts, part_size, groups;
    logprobs_cut(rows, vocab, dtype, logprobs_aligned(logits, dtype, row_stride, rows), parts, part_size, groups);
    const size_t all = static_cast<size_t>(rows) * parts;
    char* ws = static_cast<char*>(workspace);
    LogprobParts left{};
    if (parts > 1) {
        left.stats = reinterpret_cast<float4*>(ws);
        left.best = reinterpret_cast<unsigned long long*>(ws + all * 16);
        left.ranks = reinterpret_cast<int*>(ws + all * 16 + all * top * 8);
    }
    const LogprobOut out{logprobs, ranks, entropy, top_ids, top_logprobs};
    auto run = [&](auto* x) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
        constexpr bool B = std::is_same<T, bf16>::value;
        const dim3 grid(static_cast<unsigned>(all)), block(LP_THREADS);
        auto part = [&](auto count) {
            logprobs_part_kernel<T, decltype(count)::value><<<grid, block, 0, stream>>>(x, row_stride, tokens, vocab, per_row, top, parts,
                                                                                      part_size, left, out);
        };
        if (groups == 1) part(std::integral_constant<int, 1>{});
        else if (groups == (B ? 2 : 4)) part(std::integral_constant<int, B ? 2 : 4>{});
        else part(std::integral_constant<int, B ? 8 : 16>{});
        if (parts > 1)
            logprobs_join_kernel<T><<<dim3(static_cast<unsigned>(rows)), block, 0, stream>>>(x, row_stride, tokens, vocab, per_row, top, parts,
                                                                                           left, out);
    };
    if (dtype == CELEG_BF16) run(static_cast<const bf16*>(logits));
    else run(static_cast<const float*>(logits));
    return CELEG_LAUNCH_RESULT();
}
