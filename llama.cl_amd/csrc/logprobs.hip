// Log probabilities of given tokens, the entropy of the distributions they come from, and the likeliest tokens beside them.
//
// For a row z of V logits, top M = max z:  S = sum exp(z - M),  log p_i = z_i - M - log S,
//   entropy = - sum p_i log p_i = log S - (sum exp(z - M) (z - M)) / S,
//   the likeliest `top` tokens in the order of their logits, equal ones in the order of their numbers.
//
//   1. logprob_runs_kernel   a run of a row to a workgroup, whose logits stay in registers: maximum, both sums, its likeliest tokens
//   2. logprob_rows_kernel   joins a row's runs
//
// The likeliest of a run: the `top` largest of the threads' own maxima bound what can be among them, which leaves little more than `top`
// logits (and top * E at most, all from those threads); each of these counts how many others are before it.
// fp32 sums over a thread's logits and a workgroup's threads; runs are joined, and logarithms taken, in 64 bits.
#include "common.h"
#include "extents.h"
#include "gemv_device.h"

namespace llmops {

constexpr int kMostTop = 64;

struct LogprobArgs {
    const float* logits;
    const int64_t* tokens;
    int64_t lsb, lsl, tsb, tsl;  // strides, elements
    int L, V, runs, top;
    float4* stat;      // [rows][runs]: M, S, sum exp(z - M) (z - M)
    float* best;       // [rows][runs][top]
    int32_t* best_at;  // [rows][runs][top]
    float *logprobs, *entropy, *top_logprobs;
    int64_t* top_tokens;
};

// NaN and minus infinity are one and the same: nothing
__device__ __forceinline__ float something(float z) { return fmaxf(z, -INFINITY); }
__device__ __forceinline__ bool ahead(float v, int at, float w, int wat) { return v > w || (v == w && at < wat); }

template <int E>
__global__ __launch_bounds__(256) void logprob_runs_kernel(LogprobArgs a) {
    __shared__ float red[3][4], most[256];
    __shared__ int most_at[256];
    __shared__ float held[E * kMostTop];
    __shared__ int held_at[E * kMostTop], count, bound_at;
    __shared__ float bound;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x / a.runs, run = blockIdx.x - row * a.runs, b = row / a.L, l = row - b * a.L;
    const float* z = a.logits + b * a.lsb + l * a.lsl;
    const buffer_rsrc r = make_rsrc(z, (uint32_t)a.V * 4u);
    const int base = run * 256 * E + 4 * threadIdx.x;
    float x[E];
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
    if (a.top > 0) {
        int at = 0;
#pragma unroll
        for (int e = E - 1; e >= 0; e--) at = something(x[e]) == own ? e : at;
        most[threadIdx.x] = own, most_at[threadIdx.x] = base + 1024 * (at >> 2) + (at & 3);
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    if (threadIdx.x == 0) a.stat[(int64_t)row * a.runs + run] = make_float4(M, red[1][0] + red[1][1] + red[1][2] + red[1][3], red[2][0] + red[2][1] + red[2][2] + red[2][3], 0.0f);
    if (a.top == 0) return;
    {
        int before = 0;
        const int mine = most_at[threadIdx.x];
        for (int t = 0; t < 256; t++) before += ahead(most[t], most_at[t], own, mine) ? 1 : 0;
        if (before == a.top - 1) bound = own, bound_at = mine;
    }
    __syncthreads();
    const float least = bound;
    const int least_at = bound_at;
    if (!ahead(least, least_at, own, most_at[threadIdx.x])) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int at = base + 1024 * (e >> 2) + (e & 3);
            const float v = something(x[e]);
            if (!ahead(least, least_at, v, at)) {
                const int slot = atomicAdd(&count, 1);
                held[slot] = v, held_at[slot] = at;
            }
        }
    }
    __syncthreads();
    const int n = count;
    const int64_t to = ((int64_t)row * a.runs + run) * a.top;
    for (int c = threadIdx.x; c < n; c += 256) {
        const float v = held[c];
        const int at = held_at[c];
        int before = 0;
        for (int t = 0; t < n; t++) before += ahead(held[t], held_at[t], v, at) ? 1 : 0;
        if (before < a.top) a.best[to + before] = v, a.best_at[to + before] = at;
    }
}

// a workgroup to a row
__global__ __launch_bounds__(256) void logprob_rows_kernel(LogprobArgs a) {
    __shared__ double red[3][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x, b = row / a.L, l = row - b * a.L;
    const float* z = a.logits + b * a.lsb + l * a.lsl;
    const int64_t token = a.tokens[b * a.tsb + l * a.tsl];
    const bool real = token >= 0 && token < a.V;
    const float its = real ? something(z[token]) : 0.0f;
    const float4* stat = a.stat + (int64_t)row * a.runs;
    float top = -INFINITY;
    for (int r = threadIdx.x; r < a.runs; r += 256) top = fmaxf(top, stat[r].x);
    top = wave_max(top);
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
    const float M = (float)fmax(fmax(red[0][0], red[0][1]), fmax(red[0][2], red[0][3]));
    double S = 0.0, T = 0.0;
    for (int r = threadIdx.x; r < a.runs; r += 256) {
        const float4 s = stat[r];
        if (s.x == -INFINITY) continue;
        const double lower = s.x == M ? 0.0 : (double)s.x - (double)M, w = exp(lower);  // (a run below one with plus infinity: 0 * -inf)
        S += w * s.y;
        if (w > 0.0) T += w * ((double)s.z + lower * s.y);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) S += __shfl_xor(S, o, 64), T += __shfl_xor(T, o, 64);
    if (lane == 0) red[1][wave] = S, red[2][wave] = T;
    __syncthreads();
    S = red[1][0] + red[1][1] + red[1][2] + red[1][3], T = red[2][0] + red[2][1] + red[2][2] + red[2][3];
    const double log_s = M == -INFINITY ? NAN : log(S);
    auto logprob = [&](float v) { return (float)((v == M ? 0.0 : (double)v - (double)M) - log_s); };
    if (threadIdx.x == 0) {
        a.logprobs[row] = real ? logprob(its) : 0.0f;
        a.entropy[row] = (float)(log_s - T / S);
    }
    const int n = a.runs * a.top;
    const float* best = a.best + (int64_t)row * n;
    const int32_t* best_at = a.best_at + (int64_t)row * n;
    for (int c = threadIdx.x; c < n; c += 256) {
        const float v = best[c];
        const int at = best_at[c];
        int before = 0;
        for (int t = 0; t < n; t++) before += ahead(best[t], best_at[t], v, at) ? 1 : 0;
        if (before < a.top) a.top_tokens[(int64_t)row * a.top + before] = at, a.top_logprobs[(int64_t)row * a.top + before] = logprob(v);
    }
}

// logits to a thread: eight where that leaves workgroups for the whole chip
static int logprob_each(int64_t rows, int64_t V) { return rows * ((V + 2047) / 2048) <= 1024 ? 8 : 32; }

struct LogprobLayout {
    size_t stat, best, best_at, total;
    int64_t runs;
};
static LogprobLayout layout_logprobs(int64_t rows, int64_t V, int64_t top) {
    LogprobLayout w{};
    const int64_t run = 256 * logprob_each(rows, V);
    w.runs = (V + run - 1) / run;
    w.stat = 0;
    w.best = w.stat + (size_t)(rows * w.runs) * 16;
    w.best_at = w.best + (size_t)(rows * w.runs * top) * 4;
    w.total = w.best_at + (size_t)(rows * w.runs * top) * 4;
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
    a.stat = reinterpret_cast<float4*>(ws + w.stat), a.best = reinterpret_cast<float*>(ws + w.best), a.best_at = reinterpret_cast<int32_t*>(ws + w.best_at);
    a.logprobs = logprobs, a.entropy = entropy, a.top_tokens = top_tokens, a.top_logprobs = top_logprobs;
    hipStream_t st = as_stream(stream);
    const unsigned grid = (unsigned)(B * L * w.runs);
    if (logprob_each(B * L, V) == 8) logprob_runs_kernel<8><<<grid, 256, 0, st>>>(a);
    else logprob_runs_kernel<32><<<grid, 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    logprob_rows_kernel<<<(unsigned)(B * L), 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}
