// Drafted tokens against the target's logits, from given random numbers.  (The reference decodes token by token and has no
// counterpart.)
//
// Row i of a sequence: w_j = exp((z_j - max z) / T), p_j = w_j / sum w.  Draft x_i is accepted while u_i * q_i(x_i) < p_i(x_i), q_i the
// distribution that it was drawn from (1 for a draft without one).  Behind the accepted drafts comes one more token: where a draft was
// refused, drawn from max(p_i - q_i, 0) (without q: from p_i but x_i), else from the row behind the last draft; the smallest j whose
// running sum is above u * total.  T not above 0: the likeliest token, the lowest of equals, and drafts that equal it.
//
//   1. verify_rows_kernel   per row and run of the vocabulary: maximum, its place, sum of exponentials
//   2. verify_rest_kernel   how many drafts are accepted; per run, the sum of the distribution that the next token is drawn from
//   3. verify_pick_kernel   the run, then the token, where the running sum passes
//
// Answers are whole numbers that a rounding can change: a running sum over V tokens passes a border wrongly once in about
// 1 / (V * error) draws, so that exponentials and sums are in 64 bits.  A row is read once by 1; 2 and 3 read the one row per sequence
// that the next token comes from.  Logits that are NaN, and minus infinity, weigh nothing; plus infinities share the row.
#include <math.h>

#include "common.h"

namespace llmops {

constexpr int kRun = 4096;  // logits to a workgroup: 16 to a thread, in registers between maximum and sum

struct VerifyArgs {
    const float *logits, *probs, *uniforms, *temperature;
    const int64_t* drafts;
    const int32_t* draft_lens;
    float one_temperature;
    int B, K, V, runs;
    int64_t *tokens;
    int32_t* accepted;
    double *sum, *rest;  // [B*(K+1)][runs], [B][runs]
    float* top;          // [B*(K+1)][runs]
    int32_t* place;      // [B*(K+1)][runs]
};

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) { return a.draft_lens != nullptr ? max(0, min(a.draft_lens[b], a.K)) : a.K; }
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int b) { return a.temperature != nullptr ? a.temperature[b] : a.one_temperature; }
// exp((z - top) / T); a row without a value above minus infinity has no weight anywhere
__device__ __forceinline__ double weight(float z, float top, double inv_t) {
    if (!(z > -INFINITY)) return 0.0;
    return z == top ? 1.0 : top == INFINITY ? 0.0 : exp(((double)z - (double)top) * inv_t);
}
// what a run's sum counts for beside the row's maximum
__device__ __forceinline__ double share(float run_top, float top, double inv_t) {
    return run_top == top ? 1.0 : run_top == -INFINITY || top == INFINITY ? 0.0 : exp(((double)run_top - (double)top) * inv_t);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyArgs a) {
    __shared__ float tops[4];
    __shared__ int places[4];
    __shared__ double sums[4];
    const int row = blockIdx.x, run = blockIdx.y, b = row / (a.K + 1), i = row - b * (a.K + 1);
    if (i > drafts_of(a, b)) return;  // (a row behind the last draft's is not looked at)
    const float t = temperature_of(a, b);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j0 = run * kRun;
    const float* z = a.logits + (int64_t)row * a.V + j0;
    const int n = min(kRun, a.V - j0);
    float x[16];
    float top = -INFINITY;
    int place = 0x7fffffff;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const int j = threadIdx.x + 256 * e;
        x[e] = j < n ? z[j] : -INFINITY;
        if (x[e] > top) top = x[e], place = j0 + j;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float y = __shfl_xor(top, o, 64);
        const int p = __shfl_xor(place, o, 64);
        if (y > top || (y == top && p < place)) top = y, place = p;
    }
    if (lane == 0) tops[wave] = top, places[wave] = place;
    __syncthreads();
    top = tops[0], place = places[0];
#pragma unroll
    for (int w = 1; w < 4; w++)
        if (tops[w] > top || (tops[w] == top && places[w] < place)) top = tops[w], place = places[w];
    double sum = 0.0;
    if (t > 0.0f) {
        const double inv_t = 1.0 / (double)t;
#pragma unroll
        for (int e = 0; e < 16; e++) sum += weight(x[e], top, inv_t);
        sum = wave_sum64(sum);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    if (threadIdx.x == 0) {
        const int64_t at = (int64_t)row * a.runs + run;
        a.top[at] = top;
        a.place[at] = place;
        a.sum[at] = sum;
    }
}

// a row's maximum, its place, its sum, by one thread
struct Row {
    float top;
    int place;
    double sum;
};
__device__ __forceinline__ Row row_of(const VerifyArgs& a, int row, double inv_t) {
    Row r{-INFINITY, -1, 0.0};
    const int64_t at = (int64_t)row * a.runs;
    for (int c = 0; c < a.runs; c++)
        if (a.top[at + c] > r.top) r.top = a.top[at + c], r.place = a.place[at + c];
    for (int c = 0; c < a.runs; c++) r.sum += a.sum[at + c] * share(a.top[at + c], r.top, inv_t);
    return r;
}
__device__ __forceinline__ bool draft_fits(const VerifyArgs& a, int b, int i, float t, double inv_t) {
    const int64_t x = a.drafts[(int64_t)b * a.K + i];
    if (x < 0 || x >= a.V) return false;
    const int row = b * (a.K + 1) + i;
    const Row r = row_of(a, row, inv_t);
    if (!(t > 0.0f)) return x == r.place;
    const double q = a.probs != nullptr ? (double)a.probs[((int64_t)b * a.K + i) * a.V + x] : 1.0;
    return (double)a.uniforms[(int64_t)b * (a.K + 1) + i] * q * r.sum < weight(a.logits[(int64_t)row * a.V + x], r.top, inv_t);
}
// how many drafts are accepted, by the whole workgroup
__device__ __forceinline__ int accepted_of(const VerifyArgs& a, int b, int n, float t, double inv_t, int* shared) {
    if (threadIdx.x == 0) *shared = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x)
        if (!draft_fits(a, b, i, t, inv_t)) atomicMin(shared, i);
    __syncthreads();
    return *shared;
}

// what token j of a row weighs for the next token; q: the draft's distribution (or null), x: a draft without one (or -1)
__device__ __forceinline__ double rest_weight(const Row& r, float z, double inv_t, const float* q, int64_t x, int j) {
    const double p = weight(z, r.top, inv_t) / r.sum;
    if (q != nullptr) {
        const double d = p - (double)q[j];
        return d > 0.0 ? d : 0.0;
    }
    return j == x ? 0.0 : p;
}

__device__ __forceinline__ double block_sum64(double v, double* red) {
    v = wave_sum64(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const double s = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return s;
}

// threads take 16 neighbours each, so that sums run in the tokens' order
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyArgs a) {
    __shared__ int shared;
    __shared__ Row shared_row;
    __shared__ double red[4];
    const int b = blockIdx.x, run = blockIdx.y, n = drafts_of(a, b);
    const float t = temperature_of(a, b);
    const double inv_t = 1.0 / (double)t;
    const int done = accepted_of(a, b, n, t, inv_t, &shared);
    if (run == 0 && threadIdx.x == 0) a.accepted[b] = done;
    if (!(t > 0.0f)) return;
    const int row = b * (a.K + 1) + done;
    if (threadIdx.x == 0) shared_row = row_of(a, row, inv_t);
    __syncthreads();
    const Row r = shared_row;
    const bool refused = done < n;
    const float* q = refused && a.probs != nullptr ? a.probs + ((int64_t)b * a.K + done) * a.V : nullptr;
    const int64_t x = refused && a.probs == nullptr ? a.drafts[(int64_t)b * a.K + done] : -1;
    const int j0 = run * kRun + 16 * threadIdx.x, j1 = min(a.V, j0 + 16);
    double sum = 0.0;
    for (int j = j0; j < j1; j++) sum += rest_weight(r, a.logits[(int64_t)row * a.V + j], inv_t, q, x, j);
    sum = block_sum64(sum, red);
    if (threadIdx.x == 0) a.rest[(int64_t)b * a.runs + run] = sum;
}

__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
    __shared__ Row shared_row;
    __shared__ double sums[256];
    __shared__ int found, last;
    const int b = blockIdx.x, n = drafts_of(a, b), done = a.accepted[b], row = b * (a.K + 1) + done;
    const float t = temperature_of(a, b);
    const double inv_t = 1.0 / (double)t;
    if (threadIdx.x == 0) shared_row = row_of(a, row, inv_t), found = 0x7fffffff, last = -1;
    __syncthreads();
    const Row r = shared_row;
    int64_t* tokens = a.tokens + (int64_t)b * (a.K + 1);
    for (int i = threadIdx.x; i <= a.K; i += 256)
        if (i != done) tokens[i] = i < done ? a.drafts[(int64_t)b * a.K + i] : -1;
    if (!(t > 0.0f) || r.top == -INFINITY) {  // the likeliest; nothing to take: none
        if (threadIdx.x == 0) tokens[done] = r.place;
        return;
    }
    const bool refused = done < n;
    const float* q = refused && a.probs != nullptr ? a.probs + ((int64_t)b * a.K + done) * a.V : nullptr;
    int64_t x = refused && a.probs == nullptr ? a.drafts[(int64_t)b * a.K + done] : -1;
    const double* rest = a.rest + (int64_t)b * a.runs;
    double total = 0.0;
    for (int c = 0; c < a.runs; c++) total += rest[c];
    const bool none = !(total > 0.0);  // nothing above the draft's distribution: the target's own
    if (none) q = nullptr, x = -1;
    const int64_t at = (int64_t)row * a.runs;
    auto run_sum = [&](int c) { return none ? a.sum[at + c] * share(a.top[at + c], r.top, inv_t) / r.sum : rest[c]; };
    if (none) {
        total = 0.0;
        for (int c = 0; c < a.runs; c++) total += run_sum(c);
    }
    const double goal = (double)a.uniforms[(int64_t)b * (a.K + 1) + a.K] * total;
    double before = 0.0;
    int run = 0, heavy = 0;
    double heavy_before = 0.0;
    for (; run < a.runs; run++) {
        const double s = run_sum(run);
        if (s > 0.0) heavy = run, heavy_before = before;
        if (before + s > goal) break;
        before += s;
    }
    if (run == a.runs) run = heavy, before = heavy_before;  // (rounding, or a random number of 1: the last token with a weight)
    const int j0 = run * kRun + 16 * threadIdx.x, j1 = min(a.V, j0 + 16);
    double sum = 0.0;
    for (int j = j0; j < j1; j++) sum += rest_weight(r, a.logits[(int64_t)row * a.V + j], inv_t, q, x, j);
    sums[threadIdx.x] = sum;
    __syncthreads();
    for (unsigned u = 0; u < threadIdx.x; u++) before += sums[u];
    for (int j = j0; j < j1; j++) {
        const double w = rest_weight(r, a.logits[(int64_t)row * a.V + j], inv_t, q, x, j);
        before += w;
        if (w > 0.0) {
            atomicMax(&last, j);
            if (before > goal) {
                atomicMin(&found, j);
                break;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) tokens[done] = found != 0x7fffffff ? found : last;
}

struct VerifyLayout {
    size_t sum, rest, top, place, total;
};
static VerifyLayout layout_verify(int64_t B, int64_t K, int64_t runs) {
    VerifyLayout w{};
    const size_t rows = (size_t)(B * (K + 1) * runs);
    w.sum = 0;
    w.rest = w.sum + rows * 8;
    w.top = w.rest + (size_t)(B * runs) * 8;
    w.place = w.top + rows * 4;
    w.total = w.place + rows * 4;
    return w;
}

}  // namespace llmops

using namespace llmops;

static bool verify_sizes_fit(int64_t B, int64_t K, int64_t V) {
    return B > 0 && K >= 0 && V > 0 && V <= ((int64_t)1 << 27) && K < ((int64_t)1 << 20) && B < ((int64_t)1 << 24) && B * (K + 1) < ((int64_t)1 << 24);
}

extern "C" size_t llmops_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V) {
    if (!verify_sizes_fit(B, K, V)) return 0;
    return layout_verify(B, K, (V + kRun - 1) / kRun).total;
}

extern "C" int llmops_verify_drafts(const float* logits, int64_t B, int64_t K, int64_t V, const int64_t* drafts, const float* draft_probs,
                                    const float* uniforms, const float* temperature, float one_temperature, const int32_t* draft_lens, int64_t* tokens,
                                    int32_t* accepted, void* workspace, size_t workspace_bytes, llmops_stream_t stream) {
    LLMOPS_REQUIRE(logits != nullptr && uniforms != nullptr && tokens != nullptr && accepted != nullptr);
    LLMOPS_REQUIRE(verify_sizes_fit(B, K, V));
    LLMOPS_REQUIRE(drafts != nullptr || K == 0);
    LLMOPS_REQUIRE(aligned(logits, 4) && aligned(draft_probs, 4) && aligned(uniforms, 4) && aligned(drafts, 8) && aligned(tokens, 8));
    VerifyArgs a{};
    a.runs = (int)((V + kRun - 1) / kRun);
    const VerifyLayout w = layout_verify(B, K, a.runs);
    if (workspace == nullptr || workspace_bytes < w.total)
        return fail(LLMOPS_EWORKSPACE, "verify_drafts needs %zu workspace bytes, got %zu", w.total, workspace == nullptr ? (size_t)0 : workspace_bytes);
    LLMOPS_REQUIRE(aligned(workspace, 8));
    char* ws = reinterpret_cast<char*>(workspace);
    a.logits = logits, a.probs = draft_probs, a.uniforms = uniforms, a.temperature = temperature, a.drafts = drafts, a.draft_lens = draft_lens;
    a.one_temperature = one_temperature;
    a.B = (int)B, a.K = (int)K, a.V = (int)V, a.tokens = tokens, a.accepted = accepted;
    a.sum = reinterpret_cast<double*>(ws + w.sum), a.rest = reinterpret_cast<double*>(ws + w.rest), a.top = reinterpret_cast<float*>(ws + w.top);
    a.place = reinterpret_cast<int32_t*>(ws + w.place);
    hipStream_t st = as_stream(stream);
    verify_rows_kernel<<<dim3((unsigned)(B * (K + 1)), (unsigned)a.runs), 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    verify_rest_kernel<<<dim3((unsigned)B, (unsigned)a.runs), 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    verify_pick_kernel<<<(unsigned)B, 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}
