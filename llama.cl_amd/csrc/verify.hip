// Drafted tokens against the target's logits, from given random numbers.  (The reference decodes token by token and has no
// counterpart.)
//
// Row i of a sequence: w_j = exp((z_j - max z) / T), p_j = w_j / sum w.  Draft x_i is accepted while u_i * q_i(x_i) < p_i(x_i), q_i the
// distribution that it was drawn from (1 for a draft without one).  Behind the accepted drafts comes one more token: where a draft was
// refused, drawn from max(p_i - q_i, 0) (without q: from p_i but x_i), else from the row behind the last draft; the smallest j whose
// running sum is above u * total.  T not above 0: the likeliest token, the lowest of equals, and drafts that equal it.
//
//   1. verify_rows_kernel   per row and run of the vocabulary: maximum, its place, sum of exponentials
//   2. verify_next_kernel   how many drafts are accepted; per run, the sum of what the next token is drawn from; the workgroup of a
//                           sequence that is done last takes the run, then the token, where the running sum passes
//
// Answers are whole numbers that a rounding can change: a running sum over V tokens passes a border wrongly once in about
// 1 / (V * error) draws, so that exponentials (to 2e-14) and sums are in 64 bits.  A row is read once by 1; 2 reads the one row per
// sequence that the next token comes from.  Logits that are NaN, and minus infinity, weigh nothing; plus infinities share the row.
#include <math.h>

#include "common.h"
#include "extents.h"

namespace llmops {

constexpr double kLog2e = 1.4426950408889634;
constexpr int kRun = 4096;  // logits to a workgroup: 16 to a thread, in registers between maximum and sum

// a draft and what it is judged by, beside its row's sums, so that the second launch finds it without following the draft
struct Draft {
    float z, q, u;  // its logit (-inf: not a token), its probability where it was drawn, its random number
    int x;
};

struct VerifyArgs {
    const float *logits, *probs, *uniforms, *temperature;
    const int64_t* drafts;
    const int32_t* draft_lens;
    float one_temperature;
    int B, K, V, runs;
    int64_t *tokens;
    int32_t* accepted;
    double *sum, *rest;  // [B*(K+1)][runs], [B][runs]
    int32_t* arrived;    // [B]
    Draft* draft;        // [B*(K+1)]
    float* top;          // [B*(K+1)][runs]
    int32_t* place;      // [B*(K+1)][runs]
};

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) { return a.draft_lens != nullptr ? max(0, min(a.draft_lens[b], a.K)) : a.K; }
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int b) { return a.temperature != nullptr ? a.temperature[b] : a.one_temperature; }

// 2^y for y <= 0: a whole power and a polynomial over [-1/2, 1/2] (degree 9, interpolated at Chebyshev's points: off by 1.9e-14 at
// most, half the instructions of exp(), which is as exact as the type).  What is not above -1100, NaN too, gives 0
__device__ __forceinline__ double power_of_two(double y) {
    y = fmax(y, -1100.0);
    const double whole = rint(y), f = y - whole;
    double p = 0x1.b6571de2f2351p-24;
    p = fma(p, f, 0x1.63ef969a64d3cp-20);
    p = fma(p, f, 0x1.ffcb76789860fp-17);
    p = fma(p, f, 0x1.43088e257f341p-13);
    p = fma(p, f, 0x1.5d87fe908f88ap-10);
    p = fma(p, f, 0x1.3b2ab72b175eep-7);
    p = fma(p, f, 0x1.c6b08d7044119p-5);
    p = fma(p, f, 0x1.ebfbdff8149f2p-3);
    p = fma(p, f, 0x1.62e42fefa39f7p-1);
    p = fma(p, f, 0x1.000000000003dp+0);
    return ldexp(p, (int)whole);
}
// exp((z - top) / T), per_t = log2(e) / T: 1 at the maximum, infinite or not; 0 for minus infinity and NaN, and everywhere in a row without
// a value above minus infinity.  (Twenty instructions an element, two thirds of what the first launch issues.  The
// rounding of `shift` is the same in all of a row's weights.)
struct Weigher {
    float one;  // the logit that weighs 1; NaN: none
    double per_t, shift;
    __device__ __forceinline__ Weigher(float top, double per) : one(top > -INFINITY ? top : NAN), per_t(per), shift(-(double)top * per) {}
    __device__ __forceinline__ double operator()(float z) const {
        const double p = power_of_two(fma((double)z, per_t, shift));
        return z == one ? 1.0 : p;
    }
};
// what a run's sum counts for beside the row's maximum
__device__ __forceinline__ double share(float run_top, float top, double per_t) { return Weigher(top, per_t)(run_top); }

// Reductions over a wave whose steps stay in the vector ALU (a step through LDS waits some 100 cycles, and there are eight reductions one
// behind the other in a call): neighbours at 1, 2, 4, 8 lanes below within rows of 16, then the rows' ends.  `other`: what lanes without
// a neighbour take, the operation's zero.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t below(uint32_t x, uint32_t other) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)other, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float below(float x, float other) {
    return __uint_as_float(below<CTRL, ROWS>(__float_as_uint(x), __float_as_uint(other)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double below(double x, double) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)below<CTRL, ROWS>((uint32_t)(u >> 32), 0u) << 32 | below<CTRL, ROWS>((uint32_t)u, 0u));
}
// every lane: the lanes up to it and itself
template <typename V, typename F>
__device__ __forceinline__ V wave_scan(V v, V zero, F f) {
    v = f(v, below<0x111, 0xf>(v, zero));
    v = f(v, below<0x112, 0xf>(v, zero));
    v = f(v, below<0x114, 0xf>(v, zero));
    v = f(v, below<0x118, 0xf>(v, zero));
    v = f(v, below<0x142, 0xa>(v, zero));  // lane 15 to row 1, lane 47 to row 3
    return f(v, below<0x143, 0xc>(v, zero));  // lane 31 to rows 2 and 3
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ float lane_of(float v, int lane) { return __uint_as_float(lane_of(__float_as_uint(v), lane)); }
__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)lane_of((uint32_t)(u >> 32), lane) << 32 | lane_of((uint32_t)u, lane));
}
__device__ __forceinline__ double scan64(double v) { return wave_scan(v, 0.0, [](double x, double y) { return x + y; }); }
__device__ __forceinline__ double wave_sum64(double v) { return lane_of(scan64(v), 63); }
__device__ __forceinline__ float wave_top(float v) {
    return lane_of(wave_scan(v, -INFINITY, [](float x, float y) { return fmaxf(x, y); }), 63);
}
__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    return lane_of(wave_scan(v, 0xffffffffu, [](uint32_t x, uint32_t y) { return x < y ? x : y; }), 63);
}
constexpr uint32_t kNowhere = 0x7fffffff;

// A workgroup: 4096 logits of a row.  Bound by loads and then the vector ALU in 64 bits, one behind the other, since all workgroups start at
// once (128 rows of 55296, a quarter at temperature 0: 28 MB in 11.3 us, 2.5 TB/s; 31 instructions a logit, most of them at half rate), by latency
// with few rows (4 of 55296: 3.8 us).
__global__ __launch_bounds__(256) void verify_rows_kernel(VerifyArgs a) {
    __shared__ float tops[4];
    __shared__ uint32_t places[4];
    __shared__ double sums[4];
    const int row = blockIdx.x, run = blockIdx.y, b = row / (a.K + 1), i = row - b * (a.K + 1);
    if (i > drafts_of(a, b)) return;  // (a row behind the last draft's is not looked at)
    if (i == 0 && run == 0 && threadIdx.x == 0) a.arrived[b] = 0;  // (for the launch behind this one)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j0 = run * kRun;
    const float* z = a.logits + (int64_t)row * a.V + j0;
    const int n = min(kRun, a.V - j0);
    float x[16];  // (unconditional loads: behind a branch each, they would be waited for one by one)
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = z[min((int)threadIdx.x + 256 * e, n - 1)];
    const float t = temperature_of(a, b);
    if (run == 0 && threadIdx.x == 255 && i < a.K) {
        const int64_t x = a.drafts[(int64_t)b * a.K + i];
        const bool inside = x >= 0 && x < a.V;
        Draft d;
        d.z = inside ? a.logits[(int64_t)row * a.V + x] : -INFINITY;
        d.q = inside && a.probs != nullptr ? a.probs[((int64_t)b * a.K + i) * a.V + x] : 1.0f;
        d.u = a.uniforms[row];
        d.x = inside ? (int)x : -1;
        a.draft[row] = d;
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        if ((int)threadIdx.x + 256 * e >= n) x[e] = -INFINITY;
        top = fmaxf(top, x[e]);
    }
    top = wave_top(top);
    if (t > 0.0f) {  // sums beside a wave's own maximum: the waves meet once
        const double per_t = kLog2e / (double)t;
        double sum = 0.0;
        const Weigher weigh(top, per_t);
#pragma unroll
        for (int e = 0; e < 16; e++) sum += weigh(x[e]);
        sum = wave_sum64(sum);
        if (lane == 0) tops[wave] = top, sums[wave] = sum;
        __syncthreads();
        if (wave != 0) return;
        const float mine = tops[lane & 3], all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        sum = wave_sum64(lane < 4 ? sums[lane] * share(mine, all, per_t) : 0.0);
        if (lane == 0) a.top[(int64_t)row * a.runs + run] = all, a.sum[(int64_t)row * a.runs + run] = sum;
    } else {
        uint32_t place = kNowhere;
#pragma unroll
        for (int e = 15; e >= 0; e--)
            if (x[e] == top && top > -INFINITY) place = j0 + threadIdx.x + 256 * e;
        place = wave_least(place);
        if (lane == 0) tops[wave] = top, places[wave] = place;
        __syncthreads();
        if (wave != 0) return;
        const float mine = tops[lane & 3], all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        place = wave_least(mine == all ? places[lane & 3] : kNowhere);
        if (lane == 0) a.top[(int64_t)row * a.runs + run] = all, a.place[(int64_t)row * a.runs + run] = (int)place;
    }
}

// a row's maximum; the maximum's place (-1: there is none) or, where tokens are drawn, the sum and its inverse: by one wave, a run to a lane
struct Row {
    float top;
    int place;
    double sum, inv;
};
__device__ __forceinline__ Row row_of(const VerifyArgs& a, int row, bool draws, double per_t, int lane) {
    Row r{-INFINITY, -1, 0.0, 0.0};
    const int64_t at = (int64_t)row * a.runs;
    for (int c0 = 0; c0 < a.runs; c0 += 64) {
        const bool has = c0 + lane < a.runs;
        const float mine = has ? a.top[at + c0 + lane] : -INFINITY;
        if (draws) {
            const double sum = has ? a.sum[at + c0 + lane] : 0.0;
            const float up = fmaxf(r.top, wave_top(mine));
            r.sum = r.sum * share(r.top, up, per_t) + wave_sum64(sum * share(mine, up, per_t));
            r.top = up;
        } else {
            const uint32_t place = has ? (uint32_t)a.place[at + c0 + lane] : kNowhere;
            const float top = wave_top(mine);
            const uint32_t least = wave_least(mine == top ? place : kNowhere);
            if (top > r.top) r.top = top, r.place = (int)least;
        }
    }
    r.inv = 1.0 / r.sum;
    return r;
}

// what token j of a row weighs for the next token; q: its weight in the draft's distribution (behind a refused draft that has one)
__device__ __forceinline__ double rest_weight(const Weigher& weigh, double inv, float z, bool less, float q, bool out) {
    const double p = weigh(z) * inv;
    const double d = less ? fmax(p - (double)q, 0.0) : p;
    return out ? 0.0 : d;
}

// A workgroup: a run of the row that the next token of a sequence comes from (all but the first end at once where the first launch's sums do).  Bound by
// latency, a chain of dependent steps: rows' sums, the accepted drafts, the run's sum, the arrival, the run, the token (12.0 us for 32
// sequences, 55296; with four waves 12.6, with sixteen 16).
constexpr int kNextWaves = 8, kNext = 64 * kNextWaves, kEach = kRun / kNext;
__global__ __launch_bounds__(kNext) void verify_next_kernel(VerifyArgs a) {
    __shared__ int first, arrivals, found, last;
    __shared__ Row shared_row;
    __shared__ Draft shared_draft[kNextWaves];
    __shared__ int refused_token;
    __shared__ double red[kNextWaves];
    __shared__ float neighbours[2][kRun + kNext];  // (a thread's in a row and a gap: on banks of their own)
    const int b = blockIdx.x / (unsigned)a.runs, run = blockIdx.x - b * a.runs, n = drafts_of(a, b), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float t = temperature_of(a, b);
    const bool draws = t > 0.0f;
    const double per_t = draws ? kLog2e / (double)t : 0.0;
    if (!draws && run > 0) return;  // (the likeliest token needs no sums)
    if (threadIdx.x == 0) first = n;
    __syncthreads();
    // drafts, a wave to each, until one is refused
    const int row0 = b * (a.K + 1);
    const float* probs = a.probs != nullptr ? a.probs + (int64_t)b * a.K * a.V : nullptr;
    for (int i0 = 0; i0 <= n; i0 += kNextWaves) {
        const int i = i0 + wave;
        Row r{};
        if (i <= n) {
            const Draft d = a.draft[row0 + i];  // (behind the last draft: whatever is there, and not looked at)
            r = row_of(a, row0 + i, draws, per_t, lane);
            const bool fits = d.x >= 0 && (draws ? (double)d.u * (double)d.q * r.sum < Weigher(r.top, per_t)(d.z) : d.x == r.place);
            if (lane == 0) shared_draft[wave] = d;
            if (lane == 0 && i < n && !fits) atomicMin(&first, i);
        }
        __syncthreads();
        const int done = first;
        if (done == i && lane == 0) shared_row = r, refused_token = shared_draft[wave].x;
        __syncthreads();
        if (done < i0 + kNextWaves) break;
    }
    const int done = first, row = row0 + done;
    const Row r = shared_row;
    const Weigher weigh(r.top, per_t);
    const bool refused = done < n;
    const float *zrow = a.logits + (int64_t)row * a.V, *qrow = refused && probs != nullptr ? probs + (int64_t)done * a.V : nullptr;
    bool less = qrow != nullptr;
    int x = refused && qrow == nullptr ? refused_token : -1;
    int64_t* tokens = a.tokens + row0;
    if (run == 0) {
        if (threadIdx.x == 0) a.accepted[b] = done;
        for (int i = threadIdx.x; i <= a.K; i += kNext)
            if (i != done) tokens[i] = i < done ? a.drafts[(int64_t)b * a.K + i] : -1;
    }
    if (!draws || r.top == -INFINITY) {  // the likeliest; nothing to take: none
        if (run == 0 && threadIdx.x == 0) tokens[done] = r.place;
        return;
    }
    // Where a draft with a distribution was refused, every run has a sum to form; else the sums are those of the first launch, but for the
    // run of a refused draft without one
    const bool spread = less;
    if (!spread && run > 0) return;
    double* rest = a.rest + (int64_t)b * a.runs;
    // a thread's part of a run, kNext apart; what lies behind the row weighs nothing
    auto load = [&](int at_run, float (&z)[kEach], float (&q)[kEach]) {
        const int j0 = at_run * kRun + threadIdx.x;
#pragma unroll
        for (int e = 0; e < kEach; e++) z[e] = zrow[min(j0 + kNext * e, a.V - 1)];
        if (qrow != nullptr) {
#pragma unroll
            for (int e = 0; e < kEach; e++) q[e] = qrow[min(j0 + kNext * e, a.V - 1)];
        } else {
#pragma unroll
            for (int e = 0; e < kEach; e++) q[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < kEach; e++)
            if (j0 + kNext * e >= a.V) z[e] = -INFINITY;
    };
    const int sum_run = spread ? run : x >= 0 ? x / kRun : -1;
    double sum = 0.0;
    if (sum_run >= 0) {
        float z[kEach], q[kEach];
        load(sum_run, z, q);
#pragma unroll
        for (int e = 0; e < kEach; e++) sum += rest_weight(weigh, r.inv, z[e], less, q[e], sum_run * kRun + (int)threadIdx.x + kNext * e == x);
        sum = wave_sum64(sum);
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int u = 0; u < kNextWaves; u++) sum += red[u];
    }
    if (threadIdx.x == 0) found = (int)kNowhere, last = -1;
    if (spread) {
        if (threadIdx.x == 0) {
            // the exchange has come back before the arrival is counted: whoever counts the last one finds every sum.  (Nothing else is
            // handed over; a release and an acquire of the device's scope would write back and empty the L2 in every workgroup.)
            double before = __hip_atomic_exchange(&rest[run], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("" : "+v"(before) : : "memory");
            arrivals = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (arrivals != a.runs - 1) return;
    }

    // the last one (or the only one): every wave finds the run, a run to a lane
    const double sum_left = sum;
    const int64_t at = (int64_t)row * a.runs;
    auto run_sum = [&](int c, bool own) {
        if (c >= a.runs) return 0.0;
        if (own && x >= 0 && c == sum_run) return sum_left;
        return own ? a.sum[at + c] * share(a.top[at + c], r.top, per_t) * r.inv : __hip_atomic_load(&rest[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    double held = run_sum(lane, !spread);  // (of the first 64 runs, mostly all there are: asked for once)
    auto sum_of = [&](bool own) {
        double t = wave_sum64(held);
        for (int c0 = 64; c0 < a.runs; c0 += 64) t += wave_sum64(run_sum(c0 + lane, own));
        return t;
    };
    double total = sum_of(!spread);
    const bool none = !(total > 0.0);  // nothing above the draft's distribution: the target's own
    if (none) {
        less = false, x = -1;
        held = run_sum(lane, true);
        total = sum_of(true);
    }
    const double goal = (double)a.uniforms[row0 + a.K] * total;
    double before = 0.0, heavy_before = 0.0;  // sums of the runs before the one, and before the last with a weight
    int at_run = -1, heavy = 0;
    for (int c0 = 0; c0 < a.runs && at_run < 0; c0 += 64) {
        const double mine = c0 == 0 ? held : run_sum(c0 + lane, none || !spread);
        const double to = before + scan64(mine);  // up to and with this lane's run
        const uint64_t past = __ballot(to > goal && mine > 0.0), some = __ballot(mine > 0.0);
        if (some != 0) {
            const int h = 63 - __builtin_clzll(some);
            heavy = c0 + h;
            heavy_before = h > 0 ? lane_of(to, h - 1) : before;
        }
        if (past != 0) {
            const int f = __builtin_ctzll(past);
            at_run = c0 + f;
            before = f > 0 ? lane_of(to, f - 1) : before;
        } else {
            before = lane_of(to, 63);
        }
    }
    if (at_run < 0) at_run = heavy, before = heavy_before;  // (rounding, or a random number of 1: the last token with a weight)
    // its tokens in their order, kEach to a thread
    {
        float z[kEach], q[kEach];
        load(at_run, z, q);
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const int p = threadIdx.x + kNext * e, at = p + p / kEach;
            neighbours[0][at] = z[e];
            neighbours[1][at] = q[e];
        }
    }
    __syncthreads();
    const int j0 = at_run * kRun + kEach * threadIdx.x;
    double w[kEach];
    sum = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        w[e] = rest_weight(weigh, r.inv, neighbours[0][(kEach + 1) * threadIdx.x + e], less, neighbours[1][(kEach + 1) * threadIdx.x + e], j0 + e == x);
        sum += w[e];
    }
    const double to = scan64(sum);
    if (lane == 63) red[wave] = to;
    __syncthreads();
    for (int u = 0; u < wave; u++) before += red[u];
    before += to - sum;
    int mine = (int)kNowhere, some = -1;
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        before += w[e];
        if (w[e] > 0.0) {
            some = j0 + e;
            if (before > goal) mine = min(mine, j0 + e);
        }
    }
    mine = (int)wave_least((uint32_t)mine);
    const uint64_t with = __ballot(some >= 0);
    some = with != 0 ? (int)lane_of((uint32_t)some, 63 - __builtin_clzll(with)) : -1;  // (the highest lane has the highest tokens)
    if (lane == 0) atomicMin(&found, mine), atomicMax(&last, some);
    __syncthreads();
    if (threadIdx.x == 0) tokens[done] = found != (int)kNowhere ? found : last;
}

struct VerifyLayout {
    size_t draft, sum, rest, top, place, arrived, total;
};
static VerifyLayout layout_verify(int64_t B, int64_t K, int64_t runs) {
    VerifyLayout w{};
    const size_t rows = (size_t)(B * (K + 1) * runs);
    w.draft = 0;
    w.sum = w.draft + (size_t)(B * (K + 1)) * sizeof(Draft);
    w.rest = w.sum + rows * 8;
    w.top = w.rest + (size_t)(B * runs) * 8;
    w.place = w.top + rows * 4;
    w.arrived = w.place + rows * 4;
    w.total = w.arrived + (size_t)B * 4;
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
    LLMOPS_REQUIRE(B * a.runs < ((int64_t)1 << 32) / kNext);  // (a launch has fewer than 2^32 threads)
    const VerifyLayout w = layout_verify(B, K, a.runs);
    if (workspace == nullptr || workspace_bytes < w.total)
        return fail(LLMOPS_EWORKSPACE, "verify_drafts needs %zu workspace bytes, got %zu", w.total, workspace == nullptr ? (size_t)0 : workspace_bytes);
    LLMOPS_REQUIRE(aligned(workspace, 16));
    // (a workgroup reads a sequence's drafts and lengths while another may have written its answer)
    const Wide rows = (Wide)B * (K + 1);
    const Extent first(tokens, rows * 8), second(accepted, B * 4), drafts_at(drafts, (Wide)B * K * 8), logits_at(logits, rows * V * 4),
        random_at(uniforms, rows * 4), probs_at(draft_probs, draft_probs != nullptr ? (Wide)B * K * V * 4 : 0),
        temperatures_at(temperature, temperature != nullptr ? B * 4 : 0), lens_at(draft_lens, draft_lens != nullptr ? B * 4 : 0);
    LLMOPS_REQUIRE(apart(first, second));
    for (const Extent& out : {first, second}) {
        LLMOPS_REQUIRE(apart(out, drafts_at));
        LLMOPS_REQUIRE(apart(out, logits_at));
        LLMOPS_REQUIRE(apart(out, random_at));
        LLMOPS_REQUIRE(apart(out, probs_at));
        LLMOPS_REQUIRE(apart(out, temperatures_at));
        LLMOPS_REQUIRE(apart(out, lens_at));
    }
    char* ws = reinterpret_cast<char*>(workspace);
    a.logits = logits, a.probs = draft_probs, a.uniforms = uniforms, a.temperature = temperature, a.drafts = drafts, a.draft_lens = draft_lens;
    a.one_temperature = one_temperature;
    a.B = (int)B, a.K = (int)K, a.V = (int)V, a.tokens = tokens, a.accepted = accepted;
    a.draft = reinterpret_cast<Draft*>(ws + w.draft), a.sum = reinterpret_cast<double*>(ws + w.sum), a.rest = reinterpret_cast<double*>(ws + w.rest), a.top = reinterpret_cast<float*>(ws + w.top);
    a.place = reinterpret_cast<int32_t*>(ws + w.place), a.arrived = reinterpret_cast<int32_t*>(ws + w.arrived);
    hipStream_t st = as_stream(stream);
    verify_rows_kernel<<<dim3((unsigned)(B * (K + 1)), (unsigned)a.runs), 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    verify_next_kernel<<<(unsigned)(B * a.runs), kNext, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}
