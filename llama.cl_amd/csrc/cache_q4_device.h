// Rows of a key/value cache in 4 bits: 128 values in 80 bytes, four groups of 32 values x one behind the other.
//   u the smallest power of two from 2^-24 on with max |x| <= 2032 u,  lo = round(min x / u),  hi = round(max x / u),  s = ceil((hi - lo) / 15);
//   d = s u and m = lo u,  a value's code round((x / u - lo) / s), 0 .. 15 (rounding to even);  the code stands for d code + m.
// s and lo are whole numbers, |lo + 15 s| <= 2046, so that d, m and all sixteen values are halves: d code + m is exact in a half, a group is
// an operand of the fp16 matrix cores as it is, and reading a cache back as halves loses nothing.  With the offset on the grid of the group's
// largest magnitude d may be up to a 1016th of that larger than (max - min) / 15 would be.
// Bytes 16 g .. of a row: the codes of group g, eight in a word, code i at bit 4 (i / 2) + 16 (i % 2): masks of 0x000f000f and 0x00f000f0
// take out neighbours, as the two halves of an operand's register.  Bytes 64 + 4 g ..: d and m of group g.
// A row that holds NaN or a magnitude above 65024 reads back as NaN throughout (d = 0, m = NaN in all four groups).
#pragma once

#include "attn_device.h"

namespace llmops {

constexpr int kQ4Row = 80;

// cos and sin of f * pos in 64 bits, right to 1e-15 for angles below 2^50 (Taylor's polynomials of degree 16 and 15 on [-pi/4, pi/4]): in fp32
// every millionth code would be another than the definition's
__device__ __forceinline__ double2 turn64(float f, int pos) {
    const double angle = (double)f * (double)pos, n = rint(angle * 0.6366197723675814);
    double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, angle));  // pi / 2 in two parts
    r = fabs(r) > 1.0 ? 0.0 : r;  // (angles that are not known to a turn)
    const double x = r * r;
    double c = 1.0 / 20922789888000.0, s = -1.0 / 1307674368000.0;
    c = fma(c, x, -1.0 / 87178291200.0), s = fma(s, x, 1.0 / 6227020800.0);
    c = fma(c, x, 1.0 / 479001600.0), s = fma(s, x, -1.0 / 39916800.0);
    c = fma(c, x, -1.0 / 3628800.0), s = fma(s, x, 1.0 / 362880.0);
    c = fma(c, x, 1.0 / 40320.0), s = fma(s, x, -1.0 / 5040.0);
    c = fma(c, x, -1.0 / 720.0), s = fma(s, x, 1.0 / 120.0);
    c = fma(c, x, 1.0 / 24.0), s = fma(s, x, -1.0 / 6.0);
    c = fma(c, x, -0.5), s = fma(s * x, r, r);
    c = fma(c, x, 1.0);
    const int quarter = (int)(n - 4.0 * floor(n * 0.25));  // 0 .. 3
    const double a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    return make_double2(quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b);
}

__device__ __forceinline__ float real_max(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double real_max(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float real_min(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double real_min(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ int exponent_of(float x) { int e; (void)frexpf(x, &e); return e; }
__device__ __forceinline__ int exponent_of(double x) { int e; (void)frexp(x, &e); return e; }
__device__ __forceinline__ float scaled(float x, int e) { return ldexpf(x, e); }
__device__ __forceinline__ double scaled(double x, int e) { return ldexp(x, e); }

// Sixteen lanes to a row, eight values to a lane (dims 8 * (lane % 16) ..), R float or double: the lane's word of codes, and d | m << 16 of its
// group (the same in its four lanes)
template <typename R>
__device__ __forceinline__ uint2 quantise8(const R (&x)[8]) {
    R top = x[0], low = x[0];
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        top = real_max(top, x[e]), low = real_min(low, x[e]);
        fine &= fabs(x[e]) <= (R)65024.0;  // (not NaN)
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) top = real_max(top, __shfl_xor(top, o, 64)), low = real_min(low, __shfl_xor(low, o, 64));
    // (the row's sixteen lanes: a bad value spoils all of it)
    const uint64_t bad = __ballot(!fine);
    const bool spoilt = (bad >> (threadIdx.x & 48) & 0xffff) != 0;
    const R most = real_max(top, -low);
    int e = exponent_of(most);  // 2^(e - 1) <= most < 2^e: u = 2^(e - 11), or twice that
    e += most > scaled((R)2032.0, e - 11);
    e = spoilt ? 0 : max(e, 11 - 24);
    const float lo = (float)rint(scaled(low, 11 - e)) + 0.0f, hi = (float)rint(scaled(top, 11 - e));
    const int step = ((int)(hi - lo) + 14) / 15;  // (lo is no -0: zeros of either sign are stored alike)
    const float s = (float)step, half = 0.5f * s, inv = step > 0 ? 1.0f / s : 0.0f, scale = ldexpf(1.0f, 11 - e);
    uint32_t word = 0;
    if constexpr (sizeof(R) == 4) {
        // The code or one less, from (x / u - lo) / s less 2^-10 (fp32 is off by less than 2^-12 there), then put right by the border above it,
        // lo + (code + 1/2) s, which is exact, as is the sign of what x / u is away from it; on the border itself odd codes go up
        const float slope = scale * inv, from = fmaf(-lo, inv, -0x1p-10f), border = lo + half;
        const int most_code = step > 0 ? 15 : 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float c = rintf(fmaf(x[i], slope, from)), past = fmaf(x[i], scale, -fmaf(c, s, border)), odd = __builtin_amdgcn_fractf(0.5f * c);
            const int code = (int)c + (fmaf(odd, 0x1p-99f, past) > 0.0f ? 1 : 0);
            word |= (uint32_t)min(code, most_code) << (4 * (i >> 1) + 16 * (i & 1));
        }
    } else {
        // in fp32, which is off by less than 2^-12 of a unit here, unless a value is nearer than 2^-11 to a border (in one of some hundred rows)
        float farthest = -1.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float t = (float)x[i] * scale, c = rintf(fminf(fmaxf((t - lo) * inv, 0.0f), 15.0f));
            farthest = fmaxf(farthest, fabsf(t - fmaf(c, s, lo)));
            word |= (uint32_t)c << (4 * (i >> 1) + 16 * (i & 1));
        }
        if (__any(farthest > half - 0x1p-11f && step > 0)) {
            word = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // a first guess, put right by the borders on either side of it, which are exact: lo + (c - 1/2) s and lo + (c + 1/2) s
                const R t = scaled(x[i], 11 - e);
                const float c = fminf(fmaxf(rintf(((float)t - lo) * inv), 0.0f), 15.0f), level = fmaf(c, s, lo);
                const bool odd = (int)c & 1;
                const R above = (R)(level + half), below = (R)(level - half);
                int code = (int)c + ((t > above || (t == above && odd)) ? 1 : 0) - ((t < below || (t == below && odd)) ? 1 : 0);
                code = step > 0 ? min(max(code, 0), 15) : 0;
                word |= (uint32_t)code << (4 * (i >> 1) + 16 * (i & 1));
            }
        }
    }
    const uint32_t d = f32_to_f16_bits(ldexpf(s, e - 11)), m = f32_to_f16_bits(ldexpf(lo, e - 11));
    return spoilt ? make_uint2(0u, 0x7e000000u) : make_uint2(word, d | m << 16);
}

template <typename T, typename R>
__device__ __forceinline__ void load8(const T* __restrict__ p, R (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const v8h h = as_v8h(*reinterpret_cast<const uint4*>(p));
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (R)(float)h[e];
    }
}

// A lane's eight values of a row, dims 8 j .., and those that they turn with where all dims turn (asked for together)
struct RowPair {
    float x[8], y[8];
    template <typename T>
    __device__ __forceinline__ void load(const T* __restrict__ row, int j) {
        load8(row + 8 * j, x);
        load8(row + (8 * j ^ 64), y);
    }
};
// .. turned: pairs (at, at + half), the dims behind them as they are.  R double or float
template <typename R, typename T>
__device__ __forceinline__ void turn_row(const RowPair& p, const T* __restrict__ row, int j, const double2* turn, int half, R (&out)[8]) {
    if (half == 64) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double2 t = turn[(8 * j & 63) + e];
            out[e] = fma((R)t.x, (R)p.x[e], (j < 8 ? -(R)t.y : (R)t.y) * (R)p.y[e]);
        }
    } else {
        const int first = 8 * (int)unseen(j);  // (so that no loop keeps these addresses in registers)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int at = first + e;
            out[e] = p.x[e];
            if (at < half) out[e] = fma((R)turn[at].x, (R)p.x[e], -(R)turn[at].y * (R)(float)row[at + half]);
            else if (at < 2 * half) out[e] = fma((R)turn[at - half].x, (R)p.x[e], (R)turn[at - half].y * (R)(float)row[at - half]);
        }
    }
}

// the row that sixteen lanes have quantised
__device__ __forceinline__ void store_q4(uint8_t* row, uint2 q, int j) {
    reinterpret_cast<uint32_t*>(row)[j] = q.x;
    if ((j & 3) == 0) reinterpret_cast<uint32_t*>(row)[16 + (j >> 2)] = q.y;
}

// eight codes as halves: two and two, codes 0 1, 2 3, 4 5, 6 7 of a word.  (The bits of a code below those of 1024, or four places up below
// those of 64, are a half that is 1024 or 64 more.)  The masks and what goes above them in registers of their own, one scalar: an instruction can
// have one scalar operand and no constants beside it, and with constants the compiler takes two (v_and, v_or).
struct Codes {
    uint32_t low_mask = 0x000f000fu, high_mask = 0x00f000f0u, of_1024 = 0x64006400u, of_64 = 0x54005400u;
    __device__ __forceinline__ Codes() { asm volatile("" : "+s"(low_mask), "+s"(high_mask), "+v"(of_1024), "+v"(of_64)); }
    __device__ __forceinline__ v2h low(uint32_t x) const { return __builtin_bit_cast(v2h, (x & low_mask) | of_1024) - (_Float16)1024.0f; }
    __device__ __forceinline__ v2h high(uint32_t x) const { return __builtin_bit_cast(v2h, (x & high_mask) | of_64) - (_Float16)64.0f; }
    __device__ __forceinline__ v8h values(uint32_t word, uint32_t dm) const {
        const v2h p = __builtin_bit_cast(v2h, dm), d = {p[0], p[0]}, m = {p[1], p[1]};
        const v2h a = __builtin_elementwise_fma(low(word), d, m), b = __builtin_elementwise_fma(high(word), d, m), c = __builtin_elementwise_fma(low(word >> 8), d, m),
                  e = __builtin_elementwise_fma(high(word >> 8), d, m);
        return v8h{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
    }
};

}  // namespace llmops
