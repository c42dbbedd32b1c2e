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
// workgroups share a compute unit, so that one's arithmetic runs while another's loads are on their way; a second kernel, a
// workgroup a row, joins the parts.  2,048 rows of 65,536 32-bit logits, 5 best: 106 us (5.1 TB/s, as a large copy); of bfloat16 80 us,
// bound by the vector instructions (an exponential is four of the about 20 a logit).  Up to 256 rows, one a compute unit, have
// nothing to overlap with: there a workgroup of 1,024 threads takes a whole row of up to 65,536 logits, and nothing is joined (one row 10.6
// us where parts and their join take 12.0, and a launch and a workspace less for the host; 64 rows, 20 best 12.5 and 14.7; 128 best
// of one row 25 and 140).
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
constexpr float LP_FITS = 16777216.f;     // below it m log2(e) is rounded by at most 1

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

// What a part of a row leaves for the join.  stats: m, S and T (against m log2(e) as rounded), and how its order stands (1: a NaN).
struct LogprobParts {
    float4* stats;                   // [rows, parts]
    int* ranks;                      // [rows, parts, per_row]
    unsigned long long* best;        // [rows, parts, top], falling, 0 where the part has no more
};

__device__ __forceinline__ float best_logit(unsigned long long packed) {
    const uint32_t key = static_cast<uint32_t>(packed >> 32);
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// What the rounding of m log2(e), from which the sums take their distances, left out of it: the same for every logit, so that 2^-this
// brings a sum against the rounded product to one against m itself.  Below LP_FITS it is no more than 1; from there on m is taken off
// first, and nothing is left out (a row of 1,000 logits of 1e10 is off by 440 powers of two otherwise).
__device__ __forceinline__ float left_out(float m) { return fabsf(m) < LP_FITS ? fmaf(m, LOG2E, -(m * LOG2E)) : 0.f; }

// (log2_sum: of the exponentials against m itself)
__device__ __forceinline__ float logprob_of(float x, float m, float log2_sum) { return (x - m) - log2_sum * LN2; }

// Of n packed logits in `list` (all different), the `top` largest in falling order: put(place, packed).  All threads call it, behind a
// barrier; there is one more in it.  They are counted against one another eight at a time, whose reads are under way together (the list
// has room for eight more, which are made 0): one at a time 128 best took twice as long as all the rest.
template <int THREADS, typename F>
__device__ __forceinline__ void sorted_best(unsigned long long* list, int n, int top, F put) {
    typedef unsigned long long two __attribute__((ext_vector_type(2)));
    if (threadIdx.x < 8) list[n + threadIdx.x] = 0ull;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long mine = list[i];
        int ahead = 0;
        for (int j = 0; j < n; j += 8) {
            two of[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) of[e] = *reinterpret_cast<const two*>(list + j + 2 * e);
#pragma unroll
            for (int e = 0; e < 4; ++e) ahead += (of[e][0] > mine) + (of[e][1] > mine);
        }
        if (ahead < top) put(ahead, mine);
    }
}

// ---------------------------------------------------------------------------- a part of a row
// Too many logits lie at or above the bound for the list (thousands of equal ones, or a bound of -inf where a vocabulary is
// masked down to a few tokens): exactly the `top` best of columns c0 .. c1 - 1 go to the list.  The logits are read again for
// every halving; all threads call it.  (No NaN among them.)
template <typename T, int THREADS>
__device__ __noinline__ int best_by_halving(const T* __restrict__ x, int c0, int c1, int top, float bound, float high,
                                            unsigned long long* list, int* counts, int* count) {
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int turn = 0;
    auto count_of = [&](auto take) {
        int n = 0;
        for (int c = c0 + tid; c < c1; c += THREADS) n += take(order_key(to_float(x[c]) + 0.0f), c);
        const float of_wave = wave_sum(static_cast<float>(n));
        turn ^= 1;                       // (the other half of counts may still be read)
        if (lane == 0) counts[turn * WAVES + wave] = static_cast<int>(of_wave);
        __syncthreads();
        const int* of = counts + turn * WAVES;
        int all = 0;
        for (int i = 0; i < WAVES; ++i) all += of[i];
        return all;
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
    for (int c = c0 + tid; c < c1; c += THREADS) {
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
template <typename T, int GROUPS, int THREADS>
__global__ __launch_bounds__(THREADS, 1024 / THREADS) void logprobs_part_kernel(
    const T* __restrict__ logits, long long row_stride, const int* __restrict__ tokens, int vocab, int per_row, int top, int parts,
    int part_size, const LogprobParts left, const LogprobOut out) {
    using Group = LogitGroup<T>;
    constexpr int N = Group::N, WAVES = THREADS / 64;
    __shared__ float wave_of[WAVES][2 + LP_MAX_TOKENS];
    __shared__ float wave_high[WAVES];
    __shared__ int wave_bad[WAVES];
    __shared__ __align__(16) float maxima[256];
    __shared__ float bounds[4];
    __shared__ int n_groups, count, counts[2 * WAVES];
    __shared__ Group hit[LP_GROUPS];
    __shared__ int hit_at[LP_GROUPS];
    __shared__ __align__(16) unsigned long long list[LP_LIST + 8];
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
        for (int j = 0; j < GROUPS; ++j) g[j].v = from[min(tid + j * THREADS, whole - 1)];
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
    if (whole < GROUPS * THREADS) {
#pragma unroll
        for (int j = 0; j < GROUPS; ++j)
            if (tid + j * THREADS >= whole) g[j].none();
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
        bad |= of_group && tid + j * THREADS < whole;
    }
    const bool any_bad = __ballot(bad) != 0ull;
    const float wave_max_value = wave_max(high);
    // 256 maxima, or 64 (of four times as many threads) where those are well more than are sought
    const bool few = top <= 40;
    float of_some = high;
    if (THREADS > 256) {
        of_some = fmaxf(of_some, lane_move<LANES_XOR_1>(of_some));
        of_some = fmaxf(of_some, lane_move<LANES_XOR_2>(of_some));
    }
    if (few) {
        if (THREADS > 256) {
            of_some = fmaxf(of_some, lane_move<LANES_ROTATE_8>(of_some));
            of_some = fmaxf(of_some, lane_move<LANES_ROTATE_4>(of_some));
            if ((lane & 15) == 0) maxima[tid >> 4] = of_some;
        } else {
            of_some = fmaxf(of_some, lane_move<LANES_XOR_1>(of_some));
            of_some = fmaxf(of_some, lane_move<LANES_XOR_2>(of_some));
            if ((lane & 3) == 0) maxima[tid >> 2] = of_some;
        }
    } else if (THREADS == 256 || (lane & 3) == 0) {
        maxima[THREADS == 256 ? tid : tid >> 2] = of_some;
    }
    if (lane == 0) {
        wave_high[wave] = wave_max_value;
        wave_bad[wave] = any_bad;
    }
    __syncthreads();
    high = wave_high[0];
    int any = wave_bad[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        high = fmaxf(high, wave_high[i]);
        any |= wave_bad[i];
    }
    bad = any != 0;
    // ---- the bound for the best: the least of the maxima that fewer than `top` others lie above
    if (top > 0 && tid < (few ? 64 : 256)) {
        const int n = few ? 64 : 256;
        const float mine = maxima[tid];
        int above = 0;
        for (int j = 0; j < n; j += 32) {
            lp_f4 o[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] = *reinterpret_cast<const lp_f4*>(maxima + j + 4 * x);
#pragma unroll
            for (int x = 0; x < 8; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) above += o[x][e] > mine;
        }
        const float least = -wave_max(above < top ? -mine : -INFINITY);
        if (lane == 0) bounds[wave] = least;
    }
    // ---- the sums, of d = x log2(e) - m log2(e).  Below -2000 the exponential is 0 in any case, and 0 times -2000 is no NaN.
    // Where m log2(e) is rounded by more than 1 (a row masked throughout by -1e10), the maximum is taken off first.
    const float m = high == -INFINITY ? 0.f : high;
    float sum = 0.f, moment = 0.f;
    auto add = [&](float d) {
        d = fmaxf(d, -2000.f);
        const float p = __builtin_amdgcn_exp2f(d);
        sum += p;
        moment = fmaf(p, d, moment);
    };
    if (fabsf(m) < LP_FITS) {
        const float m2 = m * LOG2E;
#pragma unroll
        for (int j = 0; j < GROUPS; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) add(fmaf(g[j].get(e), LOG2E, -m2));
        add(fmaf(extra, LOG2E, -m2));
    } else {
        // (from memory: such rows are rare, and a second loop over the registers would take more of them)
        for (int c = c0 + tid; c < c1; c += THREADS) add((to_float(x[c]) - m) * LOG2E);
    }
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
            for (int c = c0 + tid; c < c1; c += THREADS) ahead += to_float(x[c]) > v || c < t;
        } else {
            const float below = next_below(v);
            // before the token, "not below it" is "above the next number below it"
            const int before = t >= a0 ? (t - a0) / N : 0;
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
                const float over = tid + j * THREADS < before ? below : v;
#pragma unroll
                for (int e = 0; e < N; ++e) ahead += g[j].get(e) > over;
            }
            ahead += extra > v || (extra == v && edge < t);
            // the group that the token lies in
            if (before < whole && tid == before % THREADS)
                for (int c = a0 + before * N; c < t; ++c) ahead += to_float(x[c]) == v;
        }
        const float total = wave_sum(static_cast<float>(ahead));       // (at most 2^17: exact)
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
                    hit_at[place] = a0 + (tid + j * THREADS) * N;
                }
            }
        }
        if (extra >= bound) list[atomicAdd(&count, 1)] = packed_logit(extra, edge);        // (up to 2N of them)
        __syncthreads();
        const int hits = min(n_groups, LP_GROUPS);
        for (int i = tid; i < hits * N; i += THREADS) {
            const float v = hit[i / N].get(i % N);
            if (v >= bound) {
                const int place = atomicAdd(&count, 1);
                if (place < LP_LIST) list[place] = packed_logit(v, hit_at[i / N] + i % N);
            }
        }
        __syncthreads();
        have = count;
        if (n_groups > LP_GROUPS || have > LP_LIST) have = best_by_halving<T, THREADS>(x, c0, c1, top, bound, high, list, counts, &count);
    }
    auto of_all = [&](int i) {
        float all = (wave_of[0][i] + wave_of[1][i]) + (wave_of[2][i] + wave_of[3][i]);
#pragma unroll
        for (int w = 4; w < WAVES; w += 4) all += (wave_of[w][i] + wave_of[w + 1][i]) + (wave_of[w + 2][i] + wave_of[w + 3][i]);
        return all;
    };
    sum = of_all(0);
    moment = of_all(1);
    if (parts > 1) {
        const size_t at_part = row * parts + part;
        if (tid == 0) left.stats[at_part] = make_float4(high, sum, moment, bad ? 1.f : 0.f);
        if (tid < per_row)
            left.ranks[at_part * per_row + tid] = static_cast<int>(of_all(2 + tid));       // (at most 2^17: exact)
        unsigned long long* best = left.best + at_part * top;
        for (int k = have + tid; k < top; k += THREADS) best[k] = 0ull;
        sorted_best<THREADS>(list, have, top, [&](int place, unsigned long long packed) { best[place] = packed; });
        return;
    }
    const bool none = bad || high == INFINITY || high == -INFINITY;
    if (tid == 0 && out.entropy) out.entropy[row] = none ? NAN : (__builtin_amdgcn_logf(sum) - moment / sum) * LN2;
    const float log2_sum = none ? NAN : __builtin_amdgcn_logf(sum) - left_out(m);
    if (tid < per_row) {
        const int t = tokens[row * per_row + tid];
        const bool valid = t >= 0 && t < vocab;
        const float total = of_all(2 + tid);
        out.logprobs[row * per_row + tid] = valid ? logprob_of(to_float(x[t]), m, log2_sum) : NAN;
        out.ranks[row * per_row + tid] = valid && !bad ? static_cast<int>(total) : -1;
    }
    if (bad) {
        for (int k = tid; k < top; k += THREADS) {
            out.top_ids[row * top + k] = -1;
            out.top_logprobs[row * top + k] = NAN;
        }
        return;
    }
    sorted_best<THREADS>(list, have, top, [&](int place, unsigned long long packed) {
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
    __shared__ __align__(16) unsigned long long all[LP_JOIN], list[LP_JOIN + 8], so_far[LP_MAX_TOP];
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
        // (the part's sums are against its own largest as the part has it)
        const float d = fmaxf((s.x - m) * LOG2E - left_out(s.x), -2000.f), w = __builtin_amdgcn_exp2f(d);
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
            for (int j = 0; j < lists; j += 8) {
                unsigned long long other[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) other[e] = all[min(j + e, lists - 1) * top + depth - 1];
#pragma unroll
                for (int e = 0; e < 8; ++e) ahead += j + e < lists && (other[e] > mine || (other[e] == mine && j + e < i));
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
            sorted_best<LP_THREADS>(list, have, top, [&](int place, unsigned long long packed) { so_far[place] = packed; });
        } else {
            sorted_best<LP_THREADS>(list, have, top, [&](int place, unsigned long long packed) {
                out.top_ids[row * top + place] = packed_logit_index(packed);
                out.top_logprobs[row * top + place] = logprob_of(best_logit(packed), m, log2_sum);
            });
        }
    }
}

// ---------------------------------------------------------------------------- how a call is cut
// Parts of a row, logits of a part, and the threads of a workgroup with the groups that each holds.
struct LogprobCut {
    int parts, part_size, groups, threads;
    LogprobCut(long long rows, int vocab, int dtype, bool aligned, int top) {
        const bool bf = dtype == CELEG_BF16;
        const int n = bf ? 8 : 4;
        // (rows that begin off a boundary need a group more)
        const int lost = aligned ? 0 : n;
        auto cut_into = [&](int most) {
            parts = (vocab + most - 1) / most;
            part_size = ((vocab + parts - 1) / parts + n - 1) / n * n;
            if (part_size > most) part_size = most;
            parts = (vocab + part_size - 1) / part_size;
        };
        // Up to 256 rows, one a compute unit: a row is a workgroup's, and nothing is joined.
        if (rows <= 256) {
            threads = LP_THREADS;
            groups = bf ? 2 : 4;
            cut_into(threads * groups * n - lost);
            if (parts == 1) return;
            threads = 1024;
            // (where a row has fewer maxima than twice what is sought, the bound that they give is too low)
            if (vocab >= 2 * top * n * 4)
                for (int g : {bf ? 2 : 4, bf ? 4 : 8, bf ? 8 : 16}) {
                    groups = g;
                    cut_into(threads * groups * n - lost);
                    // (long lists from few large parts are joined sooner than from many small ones)
                    if (parts == 1 || (g * n == 64 && top > 32)) return;
                }
        }
        // a part holds at most `most` logits; with few rows it is smaller, down to 1,024
        threads = LP_THREADS;
        for (int g : {1, bf ? 2 : 4, bf ? 8 : 16}) {
            groups = g;
            cut_into(threads * groups * n - lost);
            if (rows * parts <= 1024 && parts <= 64) return;
        }
    }
};

static bool logprobs_aligned(const void* logits, int dtype, long long row_stride, long long rows) {
    const long long n = dtype == CELEG_BF16 ? 8 : 4;
    return reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (rows <= 1 || row_stride % n == 0);
}

// Bytes of workspace of a call (for any alignment of the logits).
extern "C" size_t celeg_logprobs_workspace(int dtype, long long rows, int vocab, int per_row, int top) {
    size_t bytes = 0;
    for (int aligned = 0; aligned < 2; ++aligned) {
        const LogprobCut cut(rows, vocab, dtype, aligned != 0, top);
        const size_t all = static_cast<size_t>(rows) * cut.parts;
        const size_t b = cut.parts > 1 ? all * 16 + all * top * 8 + all * per_row * 4 : 0;
        bytes = b > bytes ? b : bytes;
    }
    return (bytes + 15) / 16 * 16;
}

extern "C" int celeg_logprobs_rows(const void* logits, int dtype, long long rows, int vocab, long long row_stride, const int* tokens,
                                   int per_row, int top, float* logprobs, int* ranks, float* entropy, int* top_ids,
                                   float* top_logprobs, void* workspace, hipStream_t stream) {
    const LogprobCut cut(rows, vocab, dtype, logprobs_aligned(logits, dtype, row_stride, rows), top);
    const size_t all = static_cast<size_t>(rows) * cut.parts;
    char* ws = static_cast<char*>(workspace);
    LogprobParts left{};
    if (cut.parts > 1) {
        left.stats = reinterpret_cast<float4*>(ws);
        left.best = reinterpret_cast<unsigned long long*>(ws + all * 16);
        left.ranks = reinterpret_cast<int*>(ws + all * 16 + all * top * 8);
    }
    const LogprobOut out{logprobs, ranks, entropy, top_ids, top_logprobs};
    auto run = [&](auto* x) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
        constexpr bool B = std::is_same<T, bf16>::value;
        auto part = [&](auto groups, auto threads) {
            constexpr int THREADS = decltype(threads)::value;
            logprobs_part_kernel<T, decltype(groups)::value, THREADS><<<dim3(static_cast<unsigned>(all)), dim3(THREADS), 0, stream>>>(
                x, row_stride, tokens, vocab, per_row, top, cut.parts, cut.part_size, left, out);
        };
        auto of = [](auto value) { return value; };
        if (cut.threads == 1024) {
            const auto threads = of(std::integral_constant<int, 1024>{});
            if (cut.groups == (B ? 2 : 4)) part(std::integral_constant<int, B ? 2 : 4>{}, threads);
            else if (cut.groups == (B ? 4 : 8)) part(std::integral_constant<int, B ? 4 : 8>{}, threads);
            else part(std::integral_constant<int, B ? 8 : 16>{}, threads);
        } else {
            const auto threads = of(std::integral_constant<int, LP_THREADS>{});
            if (cut.groups == 1) part(std::integral_constant<int, 1>{}, threads);
            else if (cut.groups == (B ? 2 : 4)) part(std::integral_constant<int, B ? 2 : 4>{}, threads);
            else part(std::integral_constant<int, B ? 8 : 16>{}, threads);
        }
        if (cut.parts > 1)
            logprobs_join_kernel<T><<<dim3(static_cast<unsigned>(rows)), dim3(LP_THREADS), 0, stream>>>(x, row_stride, tokens, vocab, per_row, top,
                                                                                                        cut.parts, left, out);
    };
    if (dtype == CELEG_BF16) run(static_cast<const bf16*>(logits));
    else run(static_cast<const float*>(logits));
    return CELEG_LAUNCH_RESULT();
}
