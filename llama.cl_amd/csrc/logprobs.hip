// Log probabilities of given tokens, the entropy of the distributions they come from, and the likeliest tokens beside them.
//
// For a row z of V logits, top M = max z:  S = sum exp(z - M),  log p_i = z_i - M - log S,
//   entropy = - sum p_i log p_i = log S - (sum exp(z - M) (z - M)) / S,
//   the likeliest `top` tokens in the order of their logits, equal ones in the order of their numbers.
//
//   1. logprob_runs_kernel   a run of a row (up to 8192 logits) to a workgroup, whose logits stay in registers: maximum, both sums, its likeliest tokens
//   2. logprob_rows_kernel or logprob_sums_kernel   joins a row's runs, if it has several
//
// The likeliest of a run: the `top`-th largest of the 64 lanes' own maxima is found in each wave bit by bit (a comparison and a count of lanes for each
// bit, most of it on the scalar unit), and no logit below the largest of the four waves' can be among them; that leaves some 3 * top logits, of which each
// counts how many others are before it.  Where that bound is minus infinity (few tokens are allowed) they are all logits above it, and the run's first ones
// that are not.  Rows of equal logits leave more; where that is more than there is room for, the same search goes over all logits and then over the
// numbers of those that are equal to the last.
// fp32 sums over a thread's logits and a workgroup's threads; runs are joined, and logarithms taken, in 64 bits.
#include <limits.h>

#include "common.h"
#include "extents.h"
#include "gemv_device.h"

namespace llmops {

constexpr int kMostTop = 64, kHeld = 1024;  // (logits that there is room for)

struct LogprobArgs {
    const float* logits;
    const int64_t* tokens;
    int64_t lsb, lsl, tsb, tsl;  // strides, elements
    int L, V, runs, top;
    float4* stat;       // [rows][runs]: M, S, sum exp(z - M) (z - M)
    struct Held* best;  // [rows][runs][top]
    float *logprobs, *entropy, *top_logprobs;
    int64_t* top_tokens;
};

// Logits as whole numbers in their order; NaN and minus infinity are one and the same (nothing), and so are zeros of either sign
__device__ __forceinline__ float something(float z) { return fmaxf(z, -INFINITY); }
__device__ __forceinline__ uint32_t rank_key(float z) {
    const uint32_t u = __float_as_uint(something(z) + 0.0f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// a logit and its token, of which (key, -token) counts
struct Held {
    uint32_t key;
    int32_t at;
};
__device__ __forceinline__ int is_ahead(Held a, Held b) { return a.key > b.key || (a.key == b.key && a.at < b.at) ? 1 : 0; }
// how many of `held` (n, and up to three that are nothing behind them) are before one of them; four neighbouring lanes count a quarter each
__device__ __forceinline__ int how_many_ahead(const Held* held, int n, Held one) {
    int before = 0;
#pragma unroll 2
    for (int t = 4 * (threadIdx.x & 3); t < n; t += 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(held + t), y = *reinterpret_cast<const uint4*>(held + t + 2);
        before += is_ahead({x.x, (int)x.y}, one) + is_ahead({x.z, (int)x.w}, one) + is_ahead({y.x, (int)y.y}, one) + is_ahead({y.z, (int)y.w}, one);
    }
    before += __shfl_xor(before, 1, 64);
    return before + __shfl_xor(before, 2, 64);
}
__device__ __forceinline__ Held nothing_held() { return {0u, INT_MAX}; }

// the workgroup's count of what its threads' E values hold true
template <int E, typename F>
__device__ __forceinline__ int count_all(int* sums, F is) {
    int mine = 0;
#pragma unroll
    for (int e = 0; e < E; e++) mine += (int)__builtin_popcountll(__ballot(is(e)));
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = mine;
    __syncthreads();
    const int all = sums[0] + sums[1] + sums[2] + sums[3];
    __syncthreads();
    return all;
}

// A row's top, the logarithm of its sum, its entropy
struct RowSums {
    float M;
    double log_s, entropy;
};
__device__ __forceinline__ RowSums row_sums_of(float M, double S, double T) {
    const double log_s = M == -INFINITY ? NAN : log(S);
    return {M, log_s, log_s - T / S};
}
__device__ __forceinline__ float logprob_of(const RowSums& s, float v) { return (float)((v == s.M ? 0.0 : (double)v - (double)s.M) - s.log_s); }
// .. its token
struct RowToken {
    bool real = false;
    float its = 0.0f;
    __device__ __forceinline__ RowToken() {}
    __device__ __forceinline__ RowToken(const LogprobArgs& a, int row) {
        const int b = row / a.L, l = row - b * a.L;
        const int64_t token = a.tokens[b * a.tsb + l * a.tsl];
        real = token >= 0 && token < a.V;
        its = real ? something(a.logits[b * a.lsb + l * a.lsl + token]) : 0.0f;
    }
    __device__ __forceinline__ void answer(const LogprobArgs& a, int row, const RowSums& s) const {
        a.logprobs[row] = real ? logprob_of(s, its) : 0.0f, a.entropy[row] = (float)s.entropy;
    }
};

// 32 logits to a thread: with fewer the reductions and the search weigh more, with more the registers of six workgroups to a compute unit do not suffice.
// 2100 rows of 32003: 269 MB in 45 us, 6.0 TB/s.  With tokens to be found and all workgroups at work at once loads come first and arithmetic behind: 160 rows of
// 55296, 35 MB, 15 us, of which memory takes 7 and the vector ALU, with 20 instructions a logit, 5.
template <int E, bool WHOLE>
__global__ __launch_bounds__(256) void logprob_runs_kernel(LogprobArgs a) {
    __shared__ float red[3][4];
    __shared__ int sums[4], count;
    __shared__ uint32_t bounds[4];
    __shared__ RowSums row_of;
    __shared__ __align__(16) Held held[kHeld + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = WHOLE ? blockIdx.x : blockIdx.x / a.runs, run = WHOLE ? 0 : blockIdx.x - row * a.runs, b = row / a.L, l = row - b * a.L;
    const float* z = a.logits + b * a.lsb + l * a.lsl;
    const buffer_rsrc r = make_rsrc(z, (uint32_t)a.V * 4u);
    const int base = run * 256 * E + 4 * threadIdx.x;
    float x[E];
    RowToken token;
    if (WHOLE && threadIdx.x == 192) token = RowToken(a, row);
#pragma unroll
    for (int u = 0; u < E / 4; u++) {
        const float4 y = buf_ldf4(r, (uint32_t)(base + 1024 * u) * 4u, 0);
        x[4 * u] = y.x, x[4 * u + 1] = y.y, x[4 * u + 2] = y.z, x[4 * u + 3] = y.w;
    }
    if ((run + 1) * 256 * E > a.V) {
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = base + 1024 * (e >> 2) + (e & 3) < a.V ? x[e] : -INFINITY;
    }
    float own = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; e++) own = fmaxf(own, x[e]);
    const float wave_top = wave_max(own);
    if (lane == 0) red[0][wave] = wave_top;
    if (a.top > 0) {
        const uint32_t key = rank_key(own);
        uint32_t bound = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 12; bit--) {  // (a bound need not be the nearest: the lower bits leave a few more and take as long as the others)
            const uint32_t more = bound | 1u << bit;
            if ((int)__builtin_popcountll(__ballot(key >= more)) >= a.top) bound = more;
        }
        if (lane == 0) bounds[wave] = bound;
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float S = 0.0f, T = 0.0f;
    if (M == INFINITY) {  // plus infinities share the row
#pragma unroll
        for (int e = 0; e < E; e++) S += x[e] == INFINITY ? 1.0f : 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float t = fmaxf(x[e] - M, -200.0f), w = __builtin_amdgcn_exp2f(t * 1.44269504f);  // (nothing: exp(-200) is 0 in fp32)
            S += w;
            T = fmaf(w, t, T);
        }
    }
    S = wave_sum(S), T = wave_sum(T);
    if (lane == 0) red[1][wave] = S, red[2][wave] = T;
    auto at = [&](int e) { return base + 1024 * (e >> 2) + (e & 3); };
    if (a.top > 0) {
        const uint32_t bound = max(max(bounds[0], bounds[1]), max(bounds[2], bounds[3]));
        // (one arrival for a wave, its lanes in order)
        const float least = of_key(max(bound, 0x00800000u));  // (something: at least the lowest finite logit)
        int its = 0;
#pragma unroll
        for (int e = 0; e < E; e++) its += (int)__builtin_popcountll(__ballot(x[e] >= least));
        int to = 0;
        if (lane == 0 && its > 0) to = atomicAdd(&count, its);
        to = __builtin_amdgcn_readfirstlane(to);
        float again = least;  // (the comparisons made again: 32 of their results kept take more scalar registers than there are)
        asm volatile("" : "+v"(again));
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool taken = x[e] >= again;
            const uint64_t all = __ballot(taken);
            if (all != 0) {
                const int slot = to + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
                if (taken && slot < kHeld) held[slot] = {rank_key(x[e]), at(e)};
                to += (int)__builtin_popcountll(all);
            }
        }
        // Few tokens allowed: fewer than `top` in each wave, so that there may be fewer than `top` of them, and tokens that are nothing follow, which are
        // equal.  Their first ones are among the run's first 2 * top tokens, of which fewer than `top` are something if they are needed.
        if (bound < 0x00800000u && 4 * (int)threadIdx.x < 2 * a.top) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (!(x[e] >= least)) {  // (behind the row's end too: what a run leaves are `top` tokens, and those are behind all that are there)
                    const int slot = atomicAdd(&count, 1);
                    if (slot < kHeld) held[slot] = {rank_key(x[e]), at(e)};
                }
        }
    }
    __syncthreads();
    const bool sums_thread = threadIdx.x == (WHOLE ? 192 : 0);  // (of a whole row: beside the other waves' comparisons)
    if (sums_thread) {
        const float all = red[1][0] + red[1][1] + red[1][2] + red[1][3], weighed = red[2][0] + red[2][1] + red[2][2] + red[2][3];
        if constexpr (WHOLE) {
            row_of = row_sums_of(M, all, weighed);
            token.answer(a, row, row_of);
        } else {
            a.stat[(int64_t)row * a.runs + run] = make_float4(M, all, weighed, 0.0f);
        }
    }
    if (a.top == 0) return;
    if (count > kHeld) {  // (the same in all threads)
        uint32_t last = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t more = last | 1u << bit;
            if (count_all<E>(sums, [&](int e) { return rank_key(x[e]) >= more; }) >= a.top) last = more;
        }
        const int equals = a.top - count_all<E>(sums, [&](int e) { return rank_key(x[e]) > last; });
        int upto = 0;  // the largest number below which there are too few of them
#pragma unroll 1
        for (int bit = 27; bit >= 0; bit--) {
            const int more = upto | 1 << bit;
            if (count_all<E>(sums, [&](int e) { return rank_key(x[e]) == last && at(e) < more; }) < equals) upto = more;
        }
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t key = rank_key(x[e]);
            if (key > last || (key == last && at(e) <= upto)) held[atomicAdd(&count, 1)] = {key, at(e)};
        }
        __syncthreads();
    }
    const int n = count;
    if (threadIdx.x < 4) held[n + threadIdx.x] = nothing_held();
    __syncthreads();
    const int64_t to = (WHOLE ? (int64_t)row : (int64_t)row * a.runs + run) * a.top;
    for (int c = (int)threadIdx.x >> 2; c < n; c += 64) {
        const int before = how_many_ahead(held, n, held[c]);
        if (before >= a.top || (threadIdx.x & 3) != 0) continue;
        if constexpr (WHOLE) a.top_tokens[to + before] = held[c].at, a.top_logprobs[to + before] = logprob_of(row_of, of_key(held[c].key));
        else a.best[to + before] = held[c];
    }
}

// A row's runs, in one wave
__device__ __forceinline__ RowSums row_sums(const LogprobArgs& a, int row, int lane) {
    const float4* stat = a.stat + (int64_t)row * a.runs;
    float4 s = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    if (lane < a.runs) s = stat[lane];
    float M = s.x;
    for (int r = lane + 64; r < a.runs; r += 64) M = fmaxf(M, stat[r].x);
    M = wave_max(M);
    double S = 0.0, T = 0.0;
    for (int r = lane; r < a.runs; r += 64) {
        if (r >= 64) s = stat[r];
        if (s.x == -INFINITY) continue;
        const double lower = s.x == M ? 0.0 : (double)s.x - (double)M, w = s.x == M ? 1.0 : exp(lower);  // (a run below one with plus infinity: 0 * -inf)
        S += w * s.y;
        if (w > 0.0) T += w * ((double)s.z + lower * s.y);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) S += __shfl_xor(S, o, 64), T += __shfl_xor(T, o, 64);
    return row_sums_of(M, S, T);
}
__device__ __forceinline__ void row_answers(const LogprobArgs& a, int row, int lane, RowSums& s) {
    const RowToken token(a, row);
    s = row_sums(a, row, lane);
    if (lane == 0) token.answer(a, row, s);
}

// without likeliest tokens: a wave to a row
__global__ __launch_bounds__(256) void logprob_sums_kernel(LogprobArgs a, int rows) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    RowSums s;
    if (row < rows) row_answers(a, row, threadIdx.x & 63, s);
}

// a workgroup to a row: one wave its sums, all its likeliest tokens, those of 512 / top runs after the other
__global__ __launch_bounds__(1024) void logprob_rows_kernel(LogprobArgs a) {
    __shared__ __align__(16) Held held[512 + kMostTop + 4], best[kMostTop];
    __shared__ RowSums sums;
    const int row = blockIdx.x, threads = blockDim.x;
    const int64_t n = (int64_t)a.runs * a.top;
    const Held* from = a.best + (int64_t)row * n;
    int kept = 0;
    const bool sums_wave = threadIdx.x >= threads - 64;
    for (int64_t c0 = 0; c0 < n; c0 += 512) {
        const int more = (int)min((int64_t)512, n - c0), m = more + kept;
        for (int c = threadIdx.x; c < more + 4; c += threads) held[kept + c] = c < more ? from[c0 + c] : nothing_held();
        if ((int)threadIdx.x < kept) held[threadIdx.x] = best[threadIdx.x];
        __syncthreads();
        if (!sums_wave) {
            for (int c = (int)threadIdx.x >> 2; c < m; c += (threads - 64) / 4) {
                const int before = how_many_ahead(held, m, held[c]);
                if (before < a.top && (threadIdx.x & 3) == 0) best[before] = held[c];
            }
        } else if (c0 == 0) {  // (beside the others' comparisons)
            RowSums s;
            row_answers(a, row, threadIdx.x & 63, s);
            if (threadIdx.x == threads - 64) sums = s;
        }
        kept = min(m, a.top);
        __syncthreads();
    }
    if ((int)threadIdx.x < a.top) {
        a.top_tokens[(int64_t)row * a.top + threadIdx.x] = best[threadIdx.x].at;
        a.top_logprobs[(int64_t)row * a.top + threadIdx.x] = logprob_of(sums, of_key(best[threadIdx.x].key));
    }
}

// logits to a thread: eight where that is the whole row
static int logprob_each(int64_t V) { return V <= 2048 ? 8 : 32; }

struct LogprobLayout {
    size_t stat, best, total;
    int64_t runs;
};
static LogprobLayout layout_logprobs(int64_t rows, int64_t V, int64_t top) {
    LogprobLayout w{};
    const int64_t run = 256 * logprob_each(V);
    w.runs = (V + run - 1) / run;
    w.stat = 0;
    w.best = w.stat + (size_t)(rows * w.runs) * 16;
    w.total = w.best + (size_t)(rows * w.runs * top) * 8;
    return w;
}

}  // namespace llmops

using namespace llmops;

static bool logprob_sizes_fit(int64_t B, int64_t L, int64_t V, int64_t top) {
    return B > 0 && L > 0 && V > 0 && B < ((int64_t)1 << 24) && L < ((int64_t)1 << 24) && B * L < ((int64_t)1 << 24) && V <= ((int64_t)1 << 27) && top >= 0 &&
           top <= kMostTop && top <= V;
}

extern "C" size_t llmops_token_logprobs_workspace_bytes(int64_t B, int64_t L, int64_t V, int64_t top) {
    if (!logprob_sizes_fit(B, L, V, top)) return 0;
    return layout_logprobs(B * L, V, top).total;
}

extern "C" int llmops_token_logprobs(const float* logits, int64_t stride_b, int64_t stride_l, int64_t B, int64_t L, int64_t V, const int64_t* tokens,
                                     int64_t token_stride_b, int64_t token_stride_l, int64_t top, float* logprobs, float* entropy, int64_t* top_tokens,
                                     float* top_logprobs, void* workspace, size_t workspace_bytes, llmops_stream_t stream) {
    LLMOPS_REQUIRE(logits != nullptr && tokens != nullptr && logprobs != nullptr && entropy != nullptr);
    LLMOPS_REQUIRE(logprob_sizes_fit(B, L, V, top));
    LLMOPS_REQUIRE(top == 0 || (top_tokens != nullptr && top_logprobs != nullptr));
    LLMOPS_REQUIRE(aligned(logits, 4) && aligned(tokens, 8) && aligned(logprobs, 4) && aligned(entropy, 4) && aligned(top_tokens, 8) && aligned(top_logprobs, 4));
    const LogprobLayout w = layout_logprobs(B * L, V, top);
    LLMOPS_REQUIRE(B * L * w.runs < ((int64_t)1 << 24));  // (a launch has fewer than 2^32 threads)
    if (workspace == nullptr || workspace_bytes < w.total)
        return fail(LLMOPS_EWORKSPACE, "token_logprobs needs %zu workspace bytes, got %zu", w.total, workspace == nullptr ? (size_t)0 : workspace_bytes);
    LLMOPS_REQUIRE(aligned(workspace, 16));
    const Extent out[4] = {Extent(logprobs, (Wide)B * L * 4), Extent(entropy, (Wide)B * L * 4), Extent(top_tokens, (Wide)B * L * top * 8),
                           Extent(top_logprobs, (Wide)B * L * top * 4)},
                 logits_at(logits, B, (Wide)stride_b * 4, L, (Wide)stride_l * 4, (Wide)V * 4), tokens_at(tokens, B, (Wide)token_stride_b * 8, L, (Wide)token_stride_l * 8, 8);
    for (int i = 0; i < 4; i++) {
        LLMOPS_REQUIRE(apart(out[i], logits_at));
        LLMOPS_REQUIRE(apart(out[i], tokens_at));
        for (int k = 0; k < i; k++) LLMOPS_REQUIRE(apart(out[i], out[k]));
    }
    char* ws = reinterpret_cast<char*>(workspace);
    LogprobArgs a{logits, tokens, stride_b, stride_l, token_stride_b, token_stride_l, (int)L, (int)V, (int)w.runs, (int)top};
    a.stat = reinterpret_cast<float4*>(ws + w.stat), a.best = reinterpret_cast<Held*>(ws + w.best);
    a.logprobs = logprobs, a.entropy = entropy, a.top_tokens = top_tokens, a.top_logprobs = top_logprobs;
    hipStream_t st = as_stream(stream);
    // One launch where a run is a whole row (us with two launches and with one, 5 likeliest: a row of 1500 7.6 and 5.1, 32 of 6000 10.1 and 6.8, 2100 of 6000 23.5 and 17.8;
    // longer rows, of 9000 to 32768, to a workgroup of 1024 threads gain with 240 rows and 5 likeliest, 10.9 to 13.8 and 9.7 to 10.7, and lose with 20, 13.5 and 14.2, and with
    // 960 rows, 28 and 40: they stay with two)
    if (w.runs == 1) {
        if (V <= 2048) logprob_runs_kernel<8, true><<<(unsigned)(B * L), 256, 0, st>>>(a);
        else logprob_runs_kernel<32, true><<<(unsigned)(B * L), 256, 0, st>>>(a);
        LLMOPS_LAUNCH_CHECK();
        return LLMOPS_OK;
    }
    logprob_runs_kernel<32, false><<<(unsigned)(B * L * w.runs), 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    // (us in workgroups of 256, 512 and 1024: 2100 rows with 20 tokens of runs to compare 51 and 58, 160 rows with 140 19.5, 18.5 and 18.2, 32 rows with 320 28.2, 19.5 and 17.3)
    if (top > 0) logprob_rows_kernel<<<(unsigned)(B * L), w.runs * top <= 96 ? 256 : 1024, 0, st>>>(a);
    else logprob_sums_kernel<<<(unsigned)((B * L + 3) / 4), 256, 0, st>>>(a, (int)(B * L));
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}
