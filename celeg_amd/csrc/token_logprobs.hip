// What rows of logits say about tokens: log probability and rank of given tokens, the entropy, the best alternatives.
//   m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):  logprob(t) = x_t - m - ln S,  entropy = ln S - T / S;
//   rank(t) = how many logits stand ahead of t's: larger ones, and equal ones of lower index.
// A logit of -inf has probability 0.  A row without a distribution (a NaN, a +inf, nothing but -inf) gets NaN for
// log probabilities and entropy; one that holds a NaN has no order either: ranks and alternatives are -1 then.
// A token outside the vocabulary gets NaN and -1; nothing is read for it.
#include "common.h"

#define LP_THREADS 1024

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void token_logprobs_kernel(
    const T* __restrict__ logits, long long row_stride, int vocab, const int* __restrict__ tokens, int per_row, int top,
    float* __restrict__ logprobs, int* __restrict__ ranks, float* __restrict__ entropy, int* __restrict__ top_ids,
    float* __restrict__ top_logprobs) {
    __shared__ float scratch[16];
    __shared__ unsigned long long best[16];
    const int tid = threadIdx.x;
    const size_t row = blockIdx.x;
    const T* __restrict__ x = logits + row * static_cast<size_t>(row_stride);
    float high = -INFINITY, bad = 0.f;
    for (int i = tid; i < vocab; i += LP_THREADS) {
        const float v = to_float(x[i]);
        high = fmaxf(high, v);
        if (v != v) bad = 1.f;
    }
    const int lane = tid & 63, wave = tid >> 6;
    high = wave_max(high);
    if (lane == 0) scratch[wave] = high;
    __syncthreads();
    high = scratch[0];
    for (int w = 1; w < LP_THREADS / 64; ++w) high = fmaxf(high, scratch[w]);
    const bool no_order = block_sum(bad, scratch) > 0.f;
    float sum = 0.f, moment = 0.f;
    for (int i = tid; i < vocab; i += LP_THREADS) {
        const float d = fmaxf(to_float(x[i]) - high, -200.f);      // (e^-200 is 0 in 32 bits: -inf adds nothing to either sum)
        const float e = expf(d);
        sum += e;
        moment = fmaf(e, d, moment);
    }
    sum = block_sum(sum, scratch);
    moment = block_sum(moment, scratch);
    const bool none = no_order || high == INFINITY || high == -INFINITY;
    const float log_sum = none ? NAN : logf(sum);
    if (tid == 0 && entropy) entropy[row] = none ? NAN : log_sum - moment / sum;
    for (int j = 0; j < per_row; ++j) {
        const int t = tokens[row * per_row + j];
        const bool valid = t >= 0 && t < vocab;
        const float at = valid ? to_float(x[t]) : 0.f;
        float ahead = 0.f;                                          // (counts below 2^24: exact)
        for (int i = tid; i < vocab; i += LP_THREADS) {
            const float v = to_float(x[i]);
            if (v > at || (v == at && i < t)) ahead += 1.f;
        }
        ahead = block_sum(ahead, scratch);
        if (tid == 0) {
            logprobs[row * per_row + j] = valid ? (at - high) - log_sum : NAN;
            ranks[row * per_row + j] = valid && !no_order ? static_cast<int>(ahead) : -1;
        }
    }
    unsigned long long before = ~0ull;
    for (int k = 0; k < top; ++k) {
        unsigned long long mine = 0ull;
        for (int i = tid; i < vocab; i += LP_THREADS) {
            const unsigned long long p = packed_logit(to_float(x[i]), i);
            if (p < before && p > mine) mine = p;
        }
        mine = wave_max_u64(mine);
        __syncthreads();
        if (lane == 0) best[wave] = mine;
        __syncthreads();
        mine = best[0];
        for (int w = 1; w < LP_THREADS / 64; ++w) mine = max(mine, best[w]);
        before = mine;
        if (tid == 0) {
            const int id = packed_logit_index(mine);
            top_ids[row * top + k] = no_order ? -1 : id;
            top_logprobs[row * top + k] = no_order ? NAN : (to_float(x[id]) - high) - log_sum;
        }
    }
}

extern "C" int celeg_logprobs_rows(const void* logits, int dtype, long long rows, int vocab, long long row_stride, const int* tokens,
                                   int per_row, int top, float* logprobs, int* ranks, float* entropy, int* top_ids,
                                   float* top_logprobs, hipStream_t stream) {
    auto run = [&](auto* x) {
        token_logprobs_kernel<<<dim3(static_cast<unsigned>(rows)), dim3(LP_THREADS), 0, stream>>>(
            x, row_stride, vocab, tokens, per_row, top, logprobs, ranks, entropy, top_ids, top_logprobs);
    };
    if (dtype == CELEG_BF16) run(static_cast<const bf16*>(logits));
    else run(static_cast<const float*>(logits));
    return CELEG_LAUNCH_RESULT();
}
