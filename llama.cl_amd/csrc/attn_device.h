// What the attention kernels of several requests have in common (attn_prefix.hip, attn_q4.hip): extents of a batch's sequences, queries as
// operands of the fp16 matrix cores, and a softmax's running maximum and sum.
#pragma once

#include <float.h>

#include "common.h"
#include "gemv_device.h"

namespace llmops {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kS = 128;
constexpr float kLift = 14.0f, kLifted = 16384.0f;  // weights are exp2(.. + kLift)

// rows that sequence b has and new tokens that it brings; what does not fit the cache counts as padding
__device__ __forceinline__ void own_extent(const int32_t* __restrict__ lengths, const int32_t* __restrict__ q_lens, int b, int qL, int64_t maxlen,
                                           int& len, int& n) {
    len = (int)max((int64_t)0, min((int64_t)lengths[b], maxlen));
    const int want = q_lens != nullptr ? min(q_lens[b], qL) : qL;
    n = (int)max((int64_t)0, min((int64_t)want, maxlen - len));
}

// eight values of a rotated query as halves, in their order, and its factor.  top: the largest magnitude of all of the query's; bad: it holds an infinity or NaN
__device__ __forceinline__ float halves_of(const float (&x)[8], float top, bool bad, bool live, v8h& hi, v8h& lo) {
    const bool use = live && !bad && top > 0.0f;
    // (2^123 at most: the factor stays a normal number.  It would lose its bits below 2^-126, and at 0 make NaN of a masked score's -inf)
    const int e2 = use ? min(123, 13 - ilogbf(top)) : 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y = use ? ldexpf(x[e], e2) : 0.0f;
        const _Float16 h = (_Float16)y;
        hi[e] = h;
        lo[e] = (_Float16)(y - (float)h);
    }
    // (a query that holds an infinity or NaN has no score that is a number)
    return live && bad ? NAN : ldexpf(1.44269504f * 0.08838834764831845f, -e2);
}
struct QueryRow {
    uint4 hi, lo;
    float c;
};
__device__ __forceinline__ QueryRow query_row(const float (&x)[8], bool live) {
    float top = 0.0f;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e])), fine &= fabsf(x[e]) <= FLT_MAX;
    float bad = fine ? 0.0f : 1.0f;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64)), bad = fmaxf(bad, __shfl_xor(bad, o, 64));
    v8h h, l;
    const float c = halves_of(x, top, bad != 0.0f, live, h, l);
    return {__builtin_bit_cast(uint4, h), __builtin_bit_cast(uint4, l), c};
}

__device__ __forceinline__ v8h as_v8h(uint4 u) { return *reinterpret_cast<const v8h*>(&u); }
__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// queries 16*rt + lane % 16 of a wave: factor, running maximum (log2), this lane's part of the sum, O^T
template <int RT>
struct Queries {
    float c[RT], m[RT], l[RT];
    int see[RT];  // rows below this one are seen
    v4f o[RT][8];
    // cq: the factor of query m0
    __device__ __forceinline__ void start(const float* cq, int m0, int m_end, int i) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            c[rt] = cq[min(16 * rt + i, m_end - 1 - m0)];
            m[rt] = -INFINITY;
            l[rt] = 0.0f;
#pragma unroll
            for (int c8 = 0; c8 < 8; c8++) o[rt][c8] = v4f{0.f, 0.f, 0.f, 0.f};
        }
    }
};
// the larger of this lane's value and those of the lanes 16, 32 and 48 away
__device__ __forceinline__ float over_groups(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t w = __float_as_uint(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
    const auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// scores (before the factor, which is positive) to weights: the running maximum, the sum, and what the sums so far shrink by.
// sc[tt]: rows t + 16*tt + 4*g + v.  With the lift in exp2's argument that is rounded between 8 and 16 for all weights that count, and they are off by
// 2^-22 of themselves in the mean.  NEAR: lifted by a product of their own (an instruction for each), right to exp2's own unit beside the largest;
// also scores so far from 0 that their products with the factor may not be left unrounded beside the rounded maximum (from 2^31 on the weight of
// the maximum itself would be infinite)
template <bool NEAR = false, int RT, int N>
__device__ __forceinline__ void weigh(Queries<RT>& s, int rt, v4f (&sc)[N], int t, int g, bool masked) {
    if (masked) {
#pragma unroll
        for (int tt = 0; tt < N; tt++)
#pragma unroll
            for (int v = 0; v < 4; v++) sc[tt][v] = t + 16 * tt + 4 * g + v < s.see[rt] ? sc[tt][v] : -INFINITY;
    }
    float top = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3]));
#pragma unroll
    for (int tt = 1; tt < N; tt++) top = fmaxf(top, fmaxf(fmaxf(sc[tt][0], sc[tt][1]), fmaxf(sc[tt][2], sc[tt][3])));
    top = over_groups(top) * s.c[rt];
    if (__any(top > s.m[rt])) {
        const float m = fmaxf(s.m[rt], top), shrink = s.m[rt] == m ? 1.0f : __builtin_amdgcn_exp2f(s.m[rt] - m);
        s.m[rt] = m;
        s.l[rt] *= shrink;
#pragma unroll
        for (int c = 0; c < 8; c++) s.o[rt][c] *= shrink;
    }
    if (NEAR && __any(fabsf(s.m[rt]) > 0x1p20f && s.m[rt] != -INFINITY)) {
#pragma unroll
        for (int tt = 0; tt < N; tt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const float x = sc[tt][v] * s.c[rt];
                sc[tt][v] = __builtin_amdgcn_exp2f(s.m[rt] == -INFINITY ? x : x - s.m[rt]) * kLifted;
                s.l[rt] += sc[tt][v];
            }
        return;
    }
    const float base = s.m[rt] == -INFINITY ? 0.0f : NEAR ? -s.m[rt] : kLift - s.m[rt];  // (nothing seen yet: every weight is exp2(-inf) = 0)
#pragma unroll
    for (int tt = 0; tt < N; tt++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float w = __builtin_amdgcn_exp2f(fmaf(sc[tt][v], s.c[rt], base));
            sc[tt][v] = NEAR ? w * kLifted : w;
            s.l[rt] += sc[tt][v];
        }
}

// the weights of 32 rows as operands: hi, lo, hi / 2048
struct Weights {
    v8h hi, lo, low;
};
template <typename T>
__device__ __forceinline__ Weights weights_of(const v4f (&sc)[2]) {
    Weights w;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float x = sc[j >> 2][j & 3], y = sc[j >> 2][(j & 3) + 1];
        const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
        const v2h hv = __builtin_bit_cast(v2h, h);
        w.hi[j] = hv[0], w.hi[j + 1] = hv[1];
        w.lo[j] = (_Float16)fmaf((float)hv[0], -1.0f, x), w.lo[j + 1] = (_Float16)fmaf((float)hv[1], -1.0f, y);
    }
    if constexpr (sizeof(T) == 4) w.low = w.hi * (_Float16)(1.0f / 2048.0f);
    return w;
}

// `lane_at` is hidden from the compiler here so that it adds `at` where it loads, up to 4095 in the instruction, and does not keep
// sixteen sums in registers
__device__ __forceinline__ uint32_t unseen(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ uint4 ask16(buffer_rsrc r, uint32_t lane_at, uint32_t at) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_at + at, 0, 0));
}
}  // namespace llmops
