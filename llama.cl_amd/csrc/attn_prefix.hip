// Attention of a batch whose sequences share a long prefix: the prefix's keys and values are held once and read once for all
// of the batch's queries; behind it every sequence has rows of its own.  (Beside attention_rope2 of attn.hip, whose cache
// belongs to one batch row from the first token on.)
//
// For sequence b with len[b] own rows and n[b] new tokens, token l < n[b], head h on kv head h / G, G = H / Hkv:
//   pos = P + len[b] + l,  q' = rot(q, pos),  own row len[b] + l = (rot(k, pos), v) in the cache's type,
//   out = sum_r e_r V_r / sum_r e_r,  e_r = exp(q' . K_r / sqrt(S) - max),  r over the P prefix rows and own rows 0 .. len[b] + l.
//
//   1. prefix_prep_kernel   rotates, writes the new cache rows and leaves q' as operands of the matrix instructions (part of 2 where that is one round)
//   2. prefix_apart_kernel  softmax(q'K^T)V of a piece of the rows for a tile of queries: running maximum and sum, one pass; the prefix
//      prefix_sweep_kernel  and the own rows apart, or in one sweep where a sequence has queries to fill tiles of its own, or where
//      prefix_brief_kernel  there are few rows
//   3. prefix_merge_kernel  joins the pieces of a query, where there are several
//
// Queries of a kv head are numbered m = (b*qL + l)*G + g, so that the queries that see the prefix, those of all sequences, and
// those of one sequence are both runs of m.  Rows are numbered through: r < P is the prefix's, P + i is the sequence's own row i.
//
// Arithmetic.  Products run on the fp16 matrix cores (v_mfma_f32_16x16x32_f16, fp32 sums) with fp32 values carried as two halves:
//   q'  scaled by a power of two of its row so that its largest value is in [2^13, 2^14): hi + lo, 22 bits of that (rows below 2^-110 scaled
//       by 2^123: 2^-148 at least)
//   K,V hi + lo / 2048, hi truncated and lo = (x - hi) * 2048 in a half: 21 bits of x from 2^-14 on, 2^-36 below (a cache of
//       halves is hi alone: all of x from 2^-14 on, 2^-38 in the sums below)
//   e   times 2^14: hi + lo, so that weights down to 2^-28 of the largest keep their bits
// A product is hi*hi + lo*hi + hi*lo/2048; what is dropped is below 2^-21 of it.  Values outside the halves' range, infinities
// and NaN are seen while a tile is cut up, and so is a piece whose K or whose V is below 2^-14 throughout; such a piece is multiplied on the
// vector ALU in full width instead, row by row of those that a query sees, so that what a mask hides has no effect whatever it holds.  (Values
// below 2^-14 beside larger ones of their piece are not seen: they are right to 2^-36, not to a part of themselves.)
#include "attn_device.h"
#include "extents.h"

namespace llmops {

typedef unsigned short v2us __attribute__((ext_vector_type(2)));

struct PrefixArgs {
    _Float16 *qh, *ql;                  // [Hkv][M][128]
    float* cq;                          // [Hkv][M]: score = cq * (q' . k), in units of log2
    const void *pk, *pv, *ok, *ov;      // [Hkv][pmax][128], [B][Hkv][maxlen][128]
    const int32_t *lengths, *q_lens;    // [B]; q_lens may be null
    float* rec_out;                     // [Hkv*M][nrec][128]
    float2* rec_stat;                   // [Hkv*M][nrec]: max (log2), sum
    float* out;                         // [B][qL][H*128]
    int64_t pmax, maxlen;
    int B, qL, G, Hkv, P, M, Mq;        // M = B*qL*G, Mq = qL*G
    int ptiles, ppieces, prows;         // prefix: tiles of queries, pieces of rows, rows of a piece
    int otiles, opieces, ostep;         // own rows (or all rows): tiles of a sequence's queries, pieces, least rows of one
    int nrec;
    unsigned pitems;
};

// ---- 1. rotation, cache rows, operands ----
// cos and sin of inv_freq * pos: the product is exact in 64 bits, and so reduced to [-pi, pi] there (in fp32 it is off by 1.2e-4 at position
// 4000, by up to 0.5 at 2^23); what its rounding to fp32 leaves out is put back to first order, 2^-24 being all that it can be
__device__ __forceinline__ void turn_of(float f, int pos, float& c, float& s) {
    const double angle = (double)f * (double)pos, whole = rint(angle * 0.15915494309189535);
    const double rest = fma(-whole, 2.4492935982947064e-16, fma(-whole, 6.283185307179586, angle));  // 2 pi in two parts
    const float hi = (float)rest, lo = (float)(rest - (double)hi);
    float s0, c0;
    sincosf(hi, &s0, &c0);
    c = fmaf(-lo, s0, c0);
    s = fmaf(lo, c0, s0);
}

__device__ __forceinline__ void store_row4(float* dst, const float* v) { *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_row4(__half* dst, const float* v) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(dst) = u;
}

struct PrepArgs {
    const float *q, *k, *v, *inv_freq;
    int64_t qsb, qsl, ksb, ksl, vsb, vsl;
    int half, groups;
};

// Sixteen lanes to a row of 128: dims d .. d+3 and 64+d .. +3 to a lane, d = 4 * (lane % 16)
__device__ __forceinline__ void load_row(const float* __restrict__ src, int d, float (&x)[8]) {
    const float4 lo = *reinterpret_cast<const float4*>(src + d), hi = *reinterpret_cast<const float4*>(src + 64 + d);
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
}
__device__ __forceinline__ void turn_row(const float* __restrict__ src, int d, const float2* turn, int half, float (&x)[8]) {
    if (half == 64) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float c = turn[d + e].x, s = turn[d + e].y, x0 = x[e], x1 = x[4 + e];
            x[e] = c * x0 - s * x1;
            x[4 + e] = s * x0 + c * x1;
        }
    } else {  // pairs (at, at + half), the other dims as they are
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int at = (e < 4 ? d : 60 + d) + e;
            if (at < half) x[e] = turn[at].x * x[e] - turn[at].y * src[at + half];
            else if (at < 2 * half) x[e] = turn[at - half].y * src[at - half] + turn[at - half].x * x[e];
        }
    }
}
template <typename T>
__device__ __forceinline__ void store_row(T* dst, int d, const float (&x)[8]) {
    store_row4(dst + d, x);
    store_row4(dst + 64 + d, x + 4);
}

// Before the launches whose workgroups do not rotate for themselves.  A workgroup per token and 16 of its H + 2*Hkv rows of 128.  Bound by latency
// at few tokens (64 of 48 rows: 5 us) and by memory at many (4 x 300 of 96 rows, a quarter padding: 20 us, 76 MB to and from HBM).
template <typename T>
__global__ __launch_bounds__(256) void prefix_prep_kernel(PrefixArgs a, PrepArgs p) {
    __shared__ float2 turn[64];
    const int bl = blockIdx.x / p.groups, group = blockIdx.x - bl * p.groups, b = bl / a.qL, l = bl - b * a.qL;
    const int H = a.G * a.Hkv, row = group * 16 + (threadIdx.x >> 4), d = 4 * (threadIdx.x & 15);
    const bool is_q = row < H, is_k = !is_q && row < H + a.Hkv, none = row >= H + 2 * a.Hkv;
    const float* src = is_q ? p.q + b * p.qsb + l * p.qsl + (int64_t)row * kS
                            : is_k ? p.k + b * p.ksb + l * p.ksl + (int64_t)(row - H) * kS : p.v + b * p.vsb + l * p.vsl + (int64_t)(row - H - a.Hkv) * kS;
    // (the row is on its way while the length is fetched and the angles are formed, also where the token turns out to be padding)
    float x[8] = {};
    if (!none) load_row(src, d, x);
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    const bool live = l < n;
    if (live && (int)threadIdx.x < p.half) turn_of(p.inv_freq[threadIdx.x], a.P + len + l, turn[threadIdx.x].x, turn[threadIdx.x].y);
    __syncthreads();
    if (none || (!live && !is_q)) return;
    if (live && (is_q || is_k)) turn_row(src, d, turn, p.half, x);
    if (!is_q) {
        const int hk = is_k ? row - H : row - H - a.Hkv;
        store_row(reinterpret_cast<T*>(const_cast<void*>(is_k ? a.ok : a.ov)) + (((int64_t)b * a.Hkv + hk) * a.maxlen + len + l) * kS, d, x);
        return;
    }
    const int64_t m = (int64_t)(row / a.G) * a.M + (int64_t)bl * a.G + row % a.G;
    const QueryRow r = query_row(x, live);
    *reinterpret_cast<uint2*>(a.qh + m * kS + d) = make_uint2(r.hi.x, r.hi.y);
    *reinterpret_cast<uint2*>(a.qh + m * kS + 64 + d) = make_uint2(r.hi.z, r.hi.w);
    *reinterpret_cast<uint2*>(a.ql + m * kS + d) = make_uint2(r.lo.x, r.lo.y);
    *reinterpret_cast<uint2*>(a.ql + m * kS + 64 + d) = make_uint2(r.lo.z, r.lo.w);
    if ((threadIdx.x & 15) == 0) a.cq[m] = r.c;
}

// ---- 2. a piece of the rows for a tile of queries ----
// Lanes of v_mfma_f32_16x16x32_f16: operand A row lane % 16, B column lane % 16, eight k-values 8 * (lane / 16) .. +7 of either;
// result column lane % 16, rows 4 * (lane / 16) + v.  With g = lane / 16 and i = lane % 16, 32 cache rows from t on:
//   S^T = K Q^T   A: rows t + 16*tt + i, dims 32*step + 8*g .. +7.  B: query i.  Result: query i, rows t + 16*tt + 4*g + v.
//   O^T = V^T e^T k-value j of lane group g stands for row t + 16*(j/4) + 4*g + j%4, so that B is the scores as they lie.
//                 A: column 64*(c/4) + 4*i + c%4 of product c, so that a lane's rows are loaded 16 bytes at a time.
//                 Result of product c: query i, dim 64*(c/4) + 16*g + 4*v + c%4.
// K or V of one head, rows 0 .. end: a run of the prefix or of a sequence's own
template <typename T>
struct Rows {
    const T* p;
    int end;
    // 32 rows from t on (the same t in the whole wave) as a descriptor that ends with the run: rows behind read as zero
    __device__ __forceinline__ buffer_rsrc from(int t) const {
        return make_rsrc(p + (int64_t)t * kS, (uint32_t)__builtin_amdgcn_readfirstlane(max(0, min(32, end - t))) * (uint32_t)(kS * sizeof(T)));
    }
};

struct Halves {
    v8h hi, lo;
};
__device__ __forceinline__ uint32_t cut2(float x, float y, uint32_t& lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const v2h hv = *reinterpret_cast<const v2h*>(&h);
    v2h l;
    l[0] = (_Float16)fmaf((float)hv[0], -2048.0f, x * 2048.0f);
    l[1] = (_Float16)fmaf((float)hv[1], -2048.0f, y * 2048.0f);
    lo = *reinterpret_cast<const uint32_t*>(&l);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The largest magnitude seen of K or V so far, NaN above all else: of fp32 values (an instruction for two), of halves as bits
template <typename T>
struct Seen;
template <>
struct Seen<float> {
    float top = 0.0f;
    __device__ __forceinline__ void note(float x, float y) { top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, fabsf(x)), fabsf(y)); }
    __device__ __forceinline__ void note(float4 x) {
        note(x.x, x.y), note(x.z, x.w);
        asm volatile("" : "+v"(top));  // here and now: put off to the loop's end, a tile's 64 operands stay in registers till then
    }
    // 2 if there are values outside the halves' range (those that truncate to the largest half, infinities, NaN), 1 if there are some in their
    // normal range; 0 if all are below 2^-14, where the low halves no longer hold 21 bits of the largest
    __device__ __forceinline__ int range() const { return !(top < 65504.0f) ? 2 : top >= 0x1p-14f ? 1 : 0; }
};
template <>
struct Seen<__half> {
    v2us top = {0, 0};
    __device__ __forceinline__ void note(uint32_t halves) {
        const uint32_t u = halves & 0x7fff7fffu;
        top = __builtin_elementwise_max(top, *reinterpret_cast<const v2us*>(&u));
    }
    __device__ __forceinline__ void note(uint4 h) {
        note(h.x), note(h.y), note(h.z), note(h.w);
        asm volatile("" : "+v"(top));  // (as above)
    }
    // (0 as above: sums of halves below 2^-14 come out of the matrix cores right to 2^-38, 3e-5 of values near 1e-7)
    __device__ __forceinline__ int range() const {
        const unsigned short most = top[0] > top[1] ? top[0] : top[1];
        return most >= 0x7c00 ? 2 : most >= 0x0400 ? 1 : 0;
    }
};

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const __half* p) { return __half2float(*p); }

// their operands: in registers for sixteen queries, in LDS for more (the four waves share them)
template <int RT>
struct QueryOps;
template <>
struct QueryOps<1> {
    v8h h[4], l[4];
    __device__ __forceinline__ void take(const uint4* lds, int lane) {
#pragma unroll
        for (int step = 0; step < 4; step++) h[step] = as_v8h(lds[step * 64 + lane]), l[step] = as_v8h(lds[(4 + step) * 64 + lane]);
    }
    __device__ __forceinline__ void load(const PrefixArgs& a, uint4*, int hk, int m0, int m_end, int lane) {
        const int64_t at = ((int64_t)hk * a.M + min(m0 + (lane & 15), m_end - 1)) * kS + 8 * (lane >> 4);
#pragma unroll
        for (int step = 0; step < 4; step++) {
            h[step] = as_v8h(*reinterpret_cast<const uint4*>(a.qh + at + 32 * step));
            l[step] = as_v8h(*reinterpret_cast<const uint4*>(a.ql + at + 32 * step));
        }
    }
    __device__ __forceinline__ v8h hi(int, int step) const { return h[step]; }
    __device__ __forceinline__ v8h lo(int, int step) const { return l[step]; }
};
template <>
struct QueryOps<2> {
    const uint4* mine;
    __device__ __forceinline__ void load(const PrefixArgs& a, uint4* lds, int hk, int m0, int m_end, int lane) {
        const int wave = threadIdx.x >> 6;  // a step to a wave
#pragma unroll
        for (int rt = 0; rt < 2; rt++) {
            const int64_t at = ((int64_t)hk * a.M + min(m0 + 16 * rt + (lane & 15), m_end - 1)) * kS + 8 * (lane >> 4) + 32 * wave;
            lds[(rt * 8 + wave) * 64 + lane] = *reinterpret_cast<const uint4*>(a.qh + at);
            lds[(rt * 8 + 4 + wave) * 64 + lane] = *reinterpret_cast<const uint4*>(a.ql + at);
        }
        mine = lds + lane;
        __syncthreads();
    }
    __device__ __forceinline__ v8h hi(int rt, int step) const { return as_v8h(mine[(rt * 8 + step) * 64]); }
    __device__ __forceinline__ v8h lo(int rt, int step) const { return as_v8h(mine[(rt * 8 + 4 + step) * 64]); }
};

// S^T of 16 rows, one step; `low` collects what the low halves of K add, times 2048
template <typename T>
__device__ __forceinline__ void score_step(v4f& acc, v4f& low, const Halves& k, v8h qh, v8h ql) {
    acc = mfma(k.hi, qh, acc);
    if constexpr (sizeof(T) == 4) low = mfma(k.lo, qh, low);
    acc = mfma(k.hi, ql, acc);
}

template <typename T>
__device__ __forceinline__ v4f add_rows(v4f o, const Halves& v, const Weights& w) {
    o = mfma(v.hi, w.hi, o);
    o = mfma(v.hi, w.lo, o);
    if constexpr (sizeof(T) == 4) o = mfma(v.lo, w.low, o);
    return o;
}

// Four dims from d on of what piece `piece` has for query m: a record, or the answer where there is one piece (live: the query is no padding)
__device__ __forceinline__ void leave(const PrefixArgs& a, int hk, int m, int piece, int d, float4 o, float sum, bool live) {
    if (a.nrec > 1) {
        *reinterpret_cast<float4*>(a.rec_out + (((int64_t)hk * a.M + m) * a.nrec + piece) * kS + d) = o;
        return;
    }
    const float f = live ? 1.0f / sum : 0.0f;
    const int bl = m / a.G;
    *reinterpret_cast<float4*>(a.out + ((int64_t)bl * a.G * a.Hkv + (int64_t)hk * a.G + (m - bl * a.G)) * kS + d) =
        live ? make_float4(o.x * f, o.y * f, o.z * f, o.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void leave_stat(const PrefixArgs& a, int hk, int m, int piece, float top, float sum) {
    if (a.nrec > 1) a.rec_stat[((int64_t)hk * a.M + m) * a.nrec + piece] = make_float2(top, sum);
}

// the row below which query m of sequence b sees its own rows
__device__ __forceinline__ int rows_seen(const PrefixArgs& a, int m, int b, int len, int n) {
    const int l = (m - b * a.Mq) / a.G;
    return l < n ? len + l + 1 : 0;
}

// The same in full width, for rows that hold values outside the halves' range: the workgroup starts again, half a wave to a query and
// four dims to a lane, only the rows that the query sees, in up to two runs (prefix, own).  Slow, and not met in a model's caches: with one value
// outside in the prefix a call takes 56 us instead of 16 (2 sequences behind 130 rows), 1.9 ms instead of 59 us (16 of 5 tokens behind 1500), 0.9 ms
// instead of 43 us (32 behind 2048, halves), 13 ms instead of 193 us (4 of 300 tokens behind 1000).
// sixteen queries in LDS: hi of step 0..3, lo of step 0..3, 16 bytes to a lane; where (in halves) the hi of dims d .. of query i is
__device__ __forceinline__ int held_at(int i, int d) { return ((d >> 5) * 64 + ((d >> 3) & 3) * 16 + i) * 8 + (d & 7); }
struct HeldQueries {  // in LDS: (16-byte pieces as the operands lie, factors), or null: in memory
    const uint4* q;
    const float* c;
};
template <typename T>
__device__ __forceinline__ void full_width(const PrefixArgs& a, HeldQueries held, int hk, int m0, int m_end, Rows<T> K0, Rows<T> V0, int from0, Rows<T> K1, Rows<T> V1, int from1,
                                           bool own, int b, int len, int n, int piece) {
    const int d = 4 * (threadIdx.x & 31);
#pragma unroll 1
    for (int m = m0 + (threadIdx.x >> 5); m < m_end; m += 8) {
        const int64_t at = (int64_t)hk * a.M + m;
        const int in = held_at(m - m0, d);
        const _Float16 *hi = held.q != nullptr ? reinterpret_cast<const _Float16*>(held.q) + in : a.qh + at * kS + d,
                       *lo = held.q != nullptr ? reinterpret_cast<const _Float16*>(held.q + 4 * 64) + in : a.ql + at * kS + d;
        double q[4];
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] = (double)(float)hi[e] + (double)(float)lo[e];
        const double c = (double)(held.q != nullptr ? held.c[m - m0] : a.cq[at]);
        const int see = own ? rows_seen(a, m, b, len, n) : 0;
        float top = -INFINITY, sum = 0.0f;
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int run = 0; run < 2; run++) {
            const T* k = run ? K1.p : K0.p;
            const T* v = run ? V1.p : V0.p;
            const int end = run ? min(K1.end, see) : see > 0 || !own ? K0.end : 0;
#pragma unroll 1
            for (int r = run ? from1 : from0; r < end; r++) {
                double x = 0.0;
#pragma unroll
                for (int e = 0; e < 4; e++) x += q[e] * (double)value(k + (int64_t)r * kS + d + e);
#pragma unroll
                for (int w = 16; w > 0; w >>= 1) x += __shfl_xor(x, w, 64);
                const float s = (float)(x * c), up = fmaxf(top, s), shrink = top == up ? 1.0f : __builtin_amdgcn_exp2f(top - up);
                const float w = s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - up + kLift);
                top = up;
                sum = fmaf(sum, shrink, w);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = fmaf(w, value(v + (int64_t)r * kS + d + e), o[e] * shrink);
            }
        }
        if (d == 0) leave_stat(a, hk, m, piece, top, sum);
        leave(a, hk, m, piece, d, make_float4(o[0], o[1], o[2], o[3]), sum, see > 0);
    }
}

// a piece without rows
__device__ __forceinline__ void nothing(const PrefixArgs& a, int hk, int m0, int m_end, int piece) {
    for (int m = m0 + threadIdx.x; m < m_end; m += 256) leave_stat(a, hk, m, piece, -INFINITY, 0.0f);
    if (a.nrec == 1)  // (then the queries are padding)
        for (int e = threadIdx.x; e < (m_end - m0) * 32; e += 256) leave(a, hk, m0 + (e >> 5), piece, 4 * (e & 31), make_float4(0.f, 0.f, 0.f, 0.f), 1.0f, false);
}

// a wave's say, and the workgroup's decision
template <typename T>
__device__ __forceinline__ void note_range(const Seen<T>& ktop, const Seen<T>& vtop, int (&range)[2], int lane) {
    const int k = ktop.range(), v = vtop.range();
    const int ks = __any(k == 2) ? 2 : __any(k == 1) ? 1 : 0, vs = __any(v == 2) ? 2 : __any(v == 1) ? 1 : 0;
    if (lane == 0) range[0] = ks, range[1] = vs;
}
template <typename T>
__device__ __forceinline__ bool all_zero(Rows<T> x, int from) {
    int some = 0;
    for (int64_t e = (int64_t)from * kS + threadIdx.x; e < (int64_t)x.end * kS; e += 256) some |= value(x.p + e) != 0.0f;
    return !__syncthreads_or(some);
}
template <typename T>
__device__ __forceinline__ bool needs_full_width(const int (&range)[4][2], Rows<T> K, Rows<T> V, int from, Rows<T> K1, Rows<T> V1, int from1) {
    const int k = max(max(range[0][0], range[1][0]), max(range[2][0], range[3][0])), v = max(max(range[0][1], range[1][1]), max(range[2][1], range[3][1]));
    return k == 2 || v == 2 || (k == 0 && !(all_zero(K, from) && all_zero(K1, from1))) || (v == 0 && !(all_zero(V, from) && all_zero(V1, from1)));
}

// Few queries to a workgroup (16 * RT): bound by reading rows of halves (32 sequences of 32 heads behind 2048 rows, 512 of their own at most: 170 MB in
// 38 us, 4.4 TB/s) and by cutting up those of fp32 (2 us for a wave's 32).  The four waves take 32 rows each of every 128; operands come
// straight from memory, K of the next rows asked for when K of these is used up, and so V; the waves' sums meet in LDS.
constexpr int kMeetRow = 132;  // floats (16 queries' rows on different banks)
struct MeetSmem {
    float m[4][32], l[4][32], sum[16];
    int range[4][2];
    union {
        float o[4][16][kMeetRow];
        struct {
            uint4 q[16 * 64];
            float c[16];
            float2 turn[16][64];
        } in;
    };
};

__device__ __forceinline__ uint2 ask8(buffer_rsrc r, uint32_t lane_at, uint32_t at) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_at + at, 0, 0));
}

template <typename T>
struct RowRegs;
template <>
struct RowRegs<float> {
    float4 k[2][4][2], v[8][2];
    __device__ __forceinline__ void load_k(Rows<float> K, int t, int i, int g) {
        const buffer_rsrc r = K.from(t);
        const uint32_t mine = unseen((uint32_t)(i * kS + 8 * g) * 4);
#pragma unroll
        for (int tt = 0; tt < 2; tt++)
#pragma unroll
            for (int step = 0; step < 4; step++)
#pragma unroll
                for (int h = 0; h < 2; h++) k[tt][step][h] = __builtin_bit_cast(float4, ask16(r, mine, (16 * tt * kS + 32 * step + 4 * h) * 4));
    }
    __device__ __forceinline__ void load_v(Rows<float> V, int t, int i, int g) {
        const buffer_rsrc r = V.from(t);
        const uint32_t mine = unseen((uint32_t)(4 * g * kS + 4 * i) * 4);
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) v[j][h] = __builtin_bit_cast(float4, ask16(r, mine, ((16 * (j >> 2) + (j & 3)) * kS + 64 * h) * 4));
    }
    __device__ __forceinline__ Halves k_op(int tt, int step, Seen<float>& top) const {
        const float4 x = k[tt][step][0], y = k[tt][step][1];
        top.note(x), top.note(y);
        uint4 h, l;
        h.x = cut2(x.x, x.y, l.x), h.y = cut2(x.z, x.w, l.y), h.z = cut2(y.x, y.y, l.z), h.w = cut2(y.z, y.w, l.w);
        return {as_v8h(h), as_v8h(l)};
    }
    __device__ __forceinline__ Halves v_op(int c, Seen<float>& top) const {
        auto f = [&](int j) { return reinterpret_cast<const float*>(&v[j][c >> 2])[c & 3]; };
        uint4 h, l;
        h.x = cut2(f(0), f(1), l.x), h.y = cut2(f(2), f(3), l.y), h.z = cut2(f(4), f(5), l.z), h.w = cut2(f(6), f(7), l.w);
        top.note(make_float4(f(0), f(1), f(2), f(3))), top.note(make_float4(f(4), f(5), f(6), f(7)));
        return {as_v8h(h), as_v8h(l)};
    }
};
template <>
struct RowRegs<__half> {
    uint4 k[2][4];
    uint2 v[8][2];
    __device__ __forceinline__ void load_k(Rows<__half> K, int t, int i, int g) {
        const buffer_rsrc r = K.from(t);
        const uint32_t mine = unseen((uint32_t)(i * kS + 8 * g) * 2);
#pragma unroll
        for (int tt = 0; tt < 2; tt++)
#pragma unroll
            for (int step = 0; step < 4; step++) k[tt][step] = ask16(r, mine, (16 * tt * kS + 32 * step) * 2);
    }
    __device__ __forceinline__ void load_v(Rows<__half> V, int t, int i, int g) {
        const buffer_rsrc r = V.from(t);
        const uint32_t mine = unseen((uint32_t)(4 * g * kS + 4 * i) * 2);
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) v[j][h] = ask8(r, mine, ((16 * (j >> 2) + (j & 3)) * kS + 64 * h) * 2);
    }
    __device__ __forceinline__ Halves k_op(int tt, int step, Seen<__half>& top) const {
        const uint4 h = k[tt][step];
        top.note(h);
        return {as_v8h(h), v8h{}};
    }
    __device__ __forceinline__ Halves v_op(int c, Seen<__half>& top) const {
        uint32_t h[4];
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint2 x = v[2 * p][c >> 2], y = v[2 * p + 1][c >> 2];
            const uint32_t a = (c & 2) ? x.y : x.x, b = (c & 2) ? y.y : y.x;
            h[p] = __builtin_amdgcn_perm(b, a, (c & 1) ? 0x07060302u : 0x05040100u);
        }
        const uint4 all = make_uint4(h[0], h[1], h[2], h[3]);
        top.note(all);
        return {as_v8h(all), v8h{}};
    }
};

// SELF: there is no launch before this one (prefix_prep_kernel).  A workgroup rotates its queries itself, and the rows that are new among a
// sequence's own (they are in one workgroup's piece).
// The queries of a workgroup, sixteen at most, asked for; their tokens' angles
struct OwnQueries {
    float x[8];
    const float* src;
    bool live;
    int token;
    __device__ __forceinline__ void load(const PrefixArgs& a, const PrepArgs& p, int hk, int m0, int m_end, MeetSmem& sm) {
        const int first = m0 / a.G, last = (m_end - 1) / a.G, m = min(m0 + (int)(threadIdx.x >> 4), m_end - 1), mine = m / a.G, b = mine / a.qL,
                  l = mine - b * a.qL;
        int len, n;
        own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
        live = l < n;
        token = mine - first;
        src = p.q + b * p.qsb + l * p.qsl + ((int64_t)hk * a.G + (m - mine * a.G)) * kS;
        load_row(src, 4 * (threadIdx.x & 15), x);
        const int f = threadIdx.x & 63;
        for (int bl = first + (int)(threadIdx.x >> 6); bl <= last; bl += 4) {
            const int c = bl / a.qL, lc = bl - c * a.qL;
            own_extent(a.lengths, a.q_lens, c, a.qL, a.maxlen, len, n);
            if (lc < n && f < p.half) turn_of(p.inv_freq[f], a.P + len + lc, sm.in.turn[bl - first][f].x, sm.in.turn[bl - first][f].y);
        }
        __syncthreads();
    }
    // rotated, as operands
    __device__ __forceinline__ void put(const PrepArgs& p, MeetSmem& sm) {
        const int i = threadIdx.x >> 4, d = 4 * (threadIdx.x & 15);
        if (live) turn_row(src, d, sm.in.turn[token], p.half, x);
        const QueryRow r = query_row(x, live);
        _Float16* hi = reinterpret_cast<_Float16*>(sm.in.q);
        _Float16* lo = hi + 4 * 64 * 8;
        *reinterpret_cast<uint2*>(hi + held_at(i, d)) = make_uint2(r.hi.x, r.hi.y);
        *reinterpret_cast<uint2*>(hi + held_at(i, 64 + d)) = make_uint2(r.hi.z, r.hi.w);
        *reinterpret_cast<uint2*>(lo + held_at(i, d)) = make_uint2(r.lo.x, r.lo.y);
        *reinterpret_cast<uint2*>(lo + held_at(i, 64 + d)) = make_uint2(r.lo.z, r.lo.w);
        if (d == 0) sm.in.c[i] = r.c;
    }
};
// the new rows among a sequence's own from r0 on (K.end: their end), whose first new token is token `first` of the workgroup's
template <typename T>
__device__ __forceinline__ void new_rows(const PrefixArgs& a, const PrepArgs& p, Rows<T> K, Rows<T> V, int hk, int b, int len, int r0, const MeetSmem& sm) {
    const int d = 4 * (threadIdx.x & 15);
    for (int r = max(r0, len) + (int)(threadIdx.x >> 4); r < K.end; r += 16) {
        const int l = r - len;
        const float *k = p.k + b * p.ksb + l * p.ksl + (int64_t)hk * kS, *v = p.v + b * p.vsb + l * p.vsl + (int64_t)hk * kS;
        float x[8], y[8];
        load_row(k, d, x);
        load_row(v, d, y);
        turn_row(k, d, sm.in.turn[l], p.half, x);
        store_row(const_cast<T*>(K.p) + (int64_t)r * kS, d, x);
        store_row(const_cast<T*>(V.p) + (int64_t)r * kS, d, y);
    }
}

// Tiles of 32 rows j0 .. j1-1: those below np are the prefix's (K0, V0), the others the sequence's own.
template <typename T, int RT, bool SELF>
__device__ __forceinline__ void few_queries(const PrefixArgs& a, const PrepArgs& p, int hk, int m0, int m_end, Rows<T> K0, Rows<T> V0, Rows<T> K1, Rows<T> V1,
                                            int np, int j0, int j1, bool own, int b, int len, int n, int piece, MeetSmem& sm) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    m_end = min(m_end, m0 + 16 * RT);
    if (j0 >= j1) {
        nothing(a, hk, m0, m_end, piece);
        return;
    }
    RowRegs<T> x;
    auto load_k = [&](int j) { x.load_k(j >= np ? K1 : K0, 32 * (j >= np ? j - np : j), i, g); };
    auto load_v = [&](int j) { x.load_v(j >= np ? V1 : V0, 32 * (j >= np ? j - np : j), i, g); };
    int j = j0 + wave;
    QueryOps<RT> q;
    Queries<RT> s;
    if constexpr (SELF) {
        static_assert(RT == 1, "");
        OwnQueries mine;
        mine.load(a, p, hk, m0, m_end, sm);
        const bool late = own && 32 * (j - np + 1) > len;  // (rows that are about to be written among them)
        if (j < j1 && !late) load_k(j), load_v(j);
        mine.put(p, sm);
        if (own) new_rows<T>(a, p, K1, V1, hk, b, len, 32 * max(0, j0 - np), sm);
        __syncthreads();
        if (j < j1 && late) load_k(j), load_v(j);
        q.take(sm.in.q, lane);
        s.start(sm.in.c, m0, m_end, i);
    } else {
        if (j < j1) load_k(j), load_v(j);
        q.load(a, sm.in.q, hk, m0, m_end, lane);
        s.start(a.cq + (int64_t)hk * a.M + m0, m0, m_end, i);
    }
    int see[RT], see_min = INT_MAX;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        see[rt] = own ? min(K1.end, rows_seen(a, min(m0 + 16 * rt + i, m_end - 1), b, len, n)) : 0;
        see_min = min(see_min, see[rt]);
    }
    Seen<T> ktop, vtop;
    for (; j < j1; j += 4) {
        const bool mine = j >= np;
        const int t = 32 * (mine ? j - np : j);
        const bool masked = __any(t + 32 > (mine ? see_min : K0.end));
#pragma unroll
        for (int rt = 0; rt < RT; rt++) s.see[rt] = mine ? see[rt] : K0.end;
        v4f sc[RT][2], low[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) sc[rt][0] = sc[rt][1] = low[rt][0] = low[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int step = 0; step < 4; step++) {
#pragma unroll
            for (int tt = 0; tt < 2; tt++) {
                const Halves h = x.k_op(tt, step, ktop);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) score_step<T>(sc[rt][tt], low[rt][tt], h, q.hi(rt, step), q.lo(rt, step));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (sizeof(T) == 4)
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int tt = 0; tt < 2; tt++)
#pragma unroll
                    for (int v = 0; v < 4; v++) sc[rt][tt][v] = fmaf(low[rt][tt][v], 1.0f / 2048.0f, sc[rt][tt][v]);
        if (j + 4 < j1) load_k(j + 4);
        Weights w[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            weigh(s, rt, sc[rt], t, g, masked);
            w[rt] = weights_of<T>(sc[rt]);
        }
#pragma unroll
        for (int c = 0; c < 8; c++) {
            const Halves h = x.v_op(c, vtop);
#pragma unroll
            for (int rt = 0; rt < RT; rt++) s.o[rt][c] = add_rows<T>(s.o[rt][c], h, w[rt]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (j + 4 < j1) load_v(j + 4);
    }
    // the four waves' sums
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        s.l[rt] += __shfl_xor(s.l[rt], 16, 64);
        s.l[rt] += __shfl_xor(s.l[rt], 32, 64);
        if (g == 0) sm.m[wave][16 * rt + i] = s.m[rt], sm.l[wave][16 * rt + i] = s.l[rt];
    }
    note_range<T>(ktop, vtop, sm.range[wave], lane);
    __syncthreads();
    const Rows<T> k0{K0.p, min(K0.end, 32 * min(j1, np))}, v0{V0.p, k0.end}, k1{K1.p, K1.end}, v1{V1.p, K1.end};
    const int from0 = 32 * j0, from1 = 32 * max(0, j0 - np);
    if (needs_full_width(sm.range, k0, v0, from0, k1, v1, from1)) {
        full_width<T>(a, SELF ? HeldQueries{sm.in.q, sm.in.c} : HeldQueries{nullptr, nullptr}, hk, m0, m_end, k0, v0, from0, k1, v1, from1, own, b, len, n, piece);
        return;
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float M = sm.m[0][16 * rt + i];
#pragma unroll
        for (int w = 1; w < 4; w++) M = fmaxf(M, sm.m[w][16 * rt + i]);
        const float f = s.m[rt] == M ? 1.0f : __builtin_amdgcn_exp2f(s.m[rt] - M);  // (equal: also both -inf)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                *reinterpret_cast<float4*>(&sm.o[wave][i][64 * h + 16 * g + 4 * v]) =
                    make_float4(s.o[rt][4 * h][v] * f, s.o[rt][4 * h + 1][v] * f, s.o[rt][4 * h + 2][v] * f, s.o[rt][4 * h + 3][v] * f);
        if (wave == 0 && g == 0) {
            float L = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float mw = sm.m[w][16 * rt + i];
                L += sm.l[w][16 * rt + i] * (mw == M ? 1.0f : __builtin_amdgcn_exp2f(mw - M));
            }
            sm.sum[i] = !own || see[rt] > 0 ? L : -1.0f;
            if (m0 + 16 * rt + i < m_end) leave_stat(a, hk, m0 + 16 * rt + i, piece, M, L);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int at = threadIdx.x + 256 * u, q = at >> 5, d = 4 * (at & 31);
            if (m0 + 16 * rt + q < m_end) {
                float4 r = *reinterpret_cast<const float4*>(&sm.o[0][q][d]);
#pragma unroll
                for (int w = 1; w < 4; w++) {
                    const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][q][d]);
                    r.x += y.x, r.y += y.y, r.z += y.z, r.w += y.w;
                }
                leave(a, hk, m0 + 16 * rt + q, piece, d, r, sm.sum[q], sm.sum[q] != -1.0f);
            }
        }
        __syncthreads();
    }
}

// Many queries (64 * RT to a workgroup, 16 * RT to a wave): bound by issuing instructions to three units that overlap in part.  (4 x 300 tokens of 32
// heads behind 1000 rows, a quarter padding, fp32, RT 1: 110 to 126 us, of which the vector ALU, weighing and cutting, would take 50 at 2.3 GHz, LDS
// reads 35, the matrix cores 29; waves wait for memory a quarter of the time.  RT 2 halves the reads.  A single buffer and three workgroups to a compute unit
// instead of two buffers and two: 151 us a call for 144.)  All waves multiply the same 32 rows, which the workgroup cuts up once and leaves in LDS in the order of the
// operands (a read is 16 bytes to a lane, in lane order); two buffers: while a tile is multiplied the next is cut up and the one behind
// it is on its way from memory.  Tiles 0 .. np-1 are the prefix's, those from np on the sequence's own.
template <typename T>
struct TileSmem {
    static constexpr int kPieces = sizeof(T) == 4 ? 2 : 1;
    uint4 k[2][kPieces][8][64], v[2][kPieces][8][64];
    int range[4][2];
};
template <typename T>
struct TileRegs;
template <>
struct TileRegs<float> {
    float4 k[2][2], v[4];
    // K: rows 16*tt + i, dims 32*step + 8*g .. of the wave's two (tt, step).  V: rows 16*(wave/2) + 4*g + 0..3, dims 64*(wave%2) + 4*i ..
    __device__ __forceinline__ void load(buffer_rsrc K, buffer_rsrc V, int wave, int i, int g) {
        const uint32_t k_at = unseen((uint32_t)((16 * (wave >> 1) + i) * kS + 64 * (wave & 1) + 8 * g) * 4),
                       v_at = unseen((uint32_t)((16 * (wave >> 1) + 4 * g) * kS + 64 * (wave & 1) + 4 * i) * 4);
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) k[c][h] = __builtin_bit_cast(float4, ask16(K, k_at, (32 * c + 4 * h) * 4));
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = __builtin_bit_cast(float4, ask16(V, v_at, r * kS * 4));
    }
    __device__ __forceinline__ void write(TileSmem<float>& sm, int buf, int wave, int lane, Seen<float>& ktop, Seen<float>& vtop) const {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float4 x = k[c][0], y = k[c][1];
            uint4 h, l;
            h.x = cut2(x.x, x.y, l.x), h.y = cut2(x.z, x.w, l.y), h.z = cut2(y.x, y.y, l.z), h.w = cut2(y.z, y.w, l.w);
            ktop.note(x), ktop.note(y);
            sm.k[buf][0][2 * wave + c][lane] = h;
            sm.k[buf][1][2 * wave + c][lane] = l;
        }
        const int tt = wave >> 1;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            auto f = [&](int r) { return reinterpret_cast<const float*>(&v[r])[c]; };
            uint2 h, l;
            h.x = cut2(f(0), f(1), l.x), h.y = cut2(f(2), f(3), l.y);
            vtop.note(make_float4(f(0), f(1), f(2), f(3)));
            reinterpret_cast<uint2*>(&sm.v[buf][0][4 * (wave & 1) + c][lane])[tt] = h;
            reinterpret_cast<uint2*>(&sm.v[buf][1][4 * (wave & 1) + c][lane])[tt] = l;
        }
    }
};
template <>
struct TileRegs<__half> {
    uint4 k[2];
    uint2 v[4];
    __device__ __forceinline__ void load(buffer_rsrc K, buffer_rsrc V, int wave, int i, int g) {
        const uint32_t k_at = unseen((uint32_t)((16 * (wave >> 1) + i) * kS + 64 * (wave & 1) + 8 * g) * 2),
                       v_at = unseen((uint32_t)((16 * (wave >> 1) + 4 * g) * kS + 64 * (wave & 1) + 4 * i) * 2);
#pragma unroll
        for (int c = 0; c < 2; c++) k[c] = ask16(K, k_at, 32 * c * 2);
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = ask8(V, v_at, r * kS * 2);
    }
    __device__ __forceinline__ void write(TileSmem<__half>& sm, int buf, int wave, int lane, Seen<__half>& ktop, Seen<__half>& vtop) const {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            ktop.note(k[c]);
            sm.k[buf][0][2 * wave + c][lane] = k[c];
        }
        const int tt = wave >> 1;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            auto f = [&](int r) { return (c & 2) ? v[r].y : v[r].x; };
            const uint32_t pick = (c & 1) ? 0x07060302u : 0x05040100u;
            const uint2 h = make_uint2(__builtin_amdgcn_perm(f(1), f(0), pick), __builtin_amdgcn_perm(f(3), f(2), pick));
            vtop.note(make_uint4(h.x, h.y, 0u, 0u));
            reinterpret_cast<uint2*>(&sm.v[buf][0][4 * (wave & 1) + c][lane])[tt] = h;
        }
    }
};

template <typename T, int RT>
__device__ __forceinline__ void many_queries(const PrefixArgs& a, int hk, int m0, int m_end, Rows<T> K0, Rows<T> V0, Rows<T> K1, Rows<T> V1, int np, int j0,
                                             int j1, bool own, int b, int len, int n, int piece, TileSmem<T>& sm) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    m_end = min(m_end, m0 + 64 * RT);
    if (j0 >= j1) {
        nothing(a, hk, m0, m_end, piece);
        return;
    }
    TileRegs<T> x;
    auto load = [&](int j) {
        const bool mine = j >= np;
        const int t = 32 * (mine ? j - np : j);
        x.load((mine ? K1 : K0).from(t), (mine ? V1 : V0).from(t), wave, i, g);
    };
    load(j0);
    v8h qh[RT][4], ql[RT][4];
    Queries<RT> s;
    const int mw = m0 + 16 * RT * wave;
    s.start(a.cq + (int64_t)hk * a.M + mw, mw, m_end, i);
    int see[RT], see_min = INT_MAX;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int m = min(mw + 16 * rt + i, m_end - 1);
        const int64_t at = ((int64_t)hk * a.M + m) * kS + 8 * g;
#pragma unroll
        for (int step = 0; step < 4; step++) {
            qh[rt][step] = as_v8h(*reinterpret_cast<const uint4*>(a.qh + at + 32 * step));
            ql[rt][step] = as_v8h(*reinterpret_cast<const uint4*>(a.ql + at + 32 * step));
        }
        see[rt] = own ? min(K1.end, rows_seen(a, m, b, len, n)) : 0;
        see_min = min(see_min, see[rt]);
    }
    Seen<T> ktop, vtop;
    x.write(sm, 0, wave, lane, ktop, vtop);
    load(min(j0 + 1, j1 - 1));
    __syncthreads();
#pragma unroll 1
    for (int j = j0; j < j1; j++) {
        const int buf = (j - j0) & 1;
        x.write(sm, buf ^ 1, wave, lane, ktop, vtop);  // (behind the last tile that one again: nobody reads it)
        load(min(j + 2, j1 - 1));
        __builtin_amdgcn_sched_barrier(0);  // (asked for now: behind the scores' products they come late)
        const bool mine = j >= np;
        const int t = 32 * (mine ? j - np : j);
        const bool masked = __any(t + 32 > (mine ? see_min : K0.end));
        v4f sc[RT][2], low[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            sc[rt][0] = sc[rt][1] = low[rt][0] = low[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
            s.see[rt] = mine ? see[rt] : K0.end;
        }
#pragma unroll
        for (int step = 0; step < 4; step++)
#pragma unroll
            for (int tt = 0; tt < 2; tt++) {
                Halves h{as_v8h(sm.k[buf][0][4 * tt + step][lane]), v8h{}};
                if constexpr (sizeof(T) == 4) h.lo = as_v8h(sm.k[buf][TileSmem<T>::kPieces - 1][4 * tt + step][lane]);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) score_step<T>(sc[rt][tt], low[rt][tt], h, qh[rt][step], ql[rt][step]);
            }
        Weights w[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            if constexpr (sizeof(T) == 4)
#pragma unroll
                for (int tt = 0; tt < 2; tt++)
#pragma unroll
                    for (int v = 0; v < 4; v++) sc[rt][tt][v] = fmaf(low[rt][tt][v], 1.0f / 2048.0f, sc[rt][tt][v]);
            weigh(s, rt, sc[rt], t, g, masked);
            w[rt] = weights_of<T>(sc[rt]);
        }
#pragma unroll
        for (int c0 = 0; c0 < 8; c0 += 4) {
            Halves h[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                h[c].hi = as_v8h(sm.v[buf][0][c0 + c][lane]);
                if constexpr (sizeof(T) == 4) h[c].lo = as_v8h(sm.v[buf][TileSmem<T>::kPieces - 1][c0 + c][lane]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                for (int c = 0; c < 4; c++) s.o[rt][c0 + c] = mfma(h[c].hi, w[rt].hi, s.o[rt][c0 + c]);
#pragma unroll
                for (int c = 0; c < 4; c++) s.o[rt][c0 + c] = mfma(h[c].hi, w[rt].lo, s.o[rt][c0 + c]);
                if constexpr (sizeof(T) == 4)
#pragma unroll
                    for (int c = 0; c < 4; c++) s.o[rt][c0 + c] = mfma(h[c].lo, w[rt].low, s.o[rt][c0 + c]);
            }
        }
        __syncthreads();
    }
    note_range<T>(ktop, vtop, sm.range[wave], lane);
    __syncthreads();
    const Rows<T> k0{K0.p, min(K0.end, 32 * min(j1, np))}, v0{V0.p, k0.end}, k1{K1.p, min(K1.end, 32 * (j1 - np))}, v1{V1.p, k1.end};
    const int from0 = 32 * j0, from1 = 32 * max(0, j0 - np);
    if (needs_full_width(sm.range, k0, v0, from0, k1, v1, from1)) {
        full_width<T>(a, HeldQueries{nullptr, nullptr}, hk, m0, m_end, k0, v0, from0, k1, v1, from1, own, b, len, n, piece);
        return;
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        s.l[rt] += __shfl_xor(s.l[rt], 16, 64);
        s.l[rt] += __shfl_xor(s.l[rt], 32, 64);
        const int m = mw + 16 * rt + i;
        if (m >= m_end) continue;
        if (g == 0) leave_stat(a, hk, m, piece, s.m[rt], s.l[rt]);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                leave(a, hk, m, piece, 64 * h + 16 * g + 4 * v, make_float4(s.o[rt][4 * h][v], s.o[rt][4 * h + 1][v], s.o[rt][4 * h + 2][v], s.o[rt][4 * h + 3][v]),
                      s.l[rt], see[rt] > 0);
    }
}

// Item `at` of groups * each: the items of a group, which read the same rows, follow each other on one XCD (consecutive workgroups go to
// the eight in turn), so that its L2 serves all but the first
__device__ __forceinline__ void item_of(unsigned at, unsigned groups, unsigned each, int& group, int& sub) {
    const unsigned whole = groups & ~7u;
    if (at < whole * each) {
        const unsigned eight = at / (8 * each), in = at - eight * 8 * each;
        group = (int)(eight * 8 + (in & 7)), sub = (int)(in >> 3);
    } else {
        const unsigned in = at - whole * each;
        group = (int)(whole + in / each), sub = (int)(in % each);
    }
}

// The prefix for the queries of all sequences, RTP times 16 of them (MANY: 64) to a workgroup, then every sequence's own rows for its
// queries, 16 to a workgroup
template <typename T, int RTP, bool MANY, bool SELF>
__global__ __launch_bounds__(256, 2) void prefix_apart_kernel(PrefixArgs a, PrepArgs p) {
    __shared__ union {
        MeetSmem few;
        TileSmem<T> many;
    } sm;
    if (blockIdx.x < a.pitems) {
        int group, tile;  // (a group: a head's piece of the prefix)
        item_of(blockIdx.x, a.Hkv * a.ppieces, a.ptiles, group, tile);
        const int piece = group % a.ppieces, hk = group / a.ppieces;
        const int64_t plane = (int64_t)hk * a.pmax * kS;
        if constexpr (MANY) {
            const Rows<T> K{(const T*)a.pk + plane, a.P}, V{(const T*)a.pv + plane, a.P}, none{(const T*)a.pk, 0};
            const int tiles = (a.P + 31) / 32;
            many_queries<T, RTP>(a, hk, tile * 64 * RTP, a.M, K, V, none, none, tiles, piece * (a.prows / 32), min(tiles, (piece + 1) * (a.prows / 32)), false, 0,
                                 0, 0, piece, sm.many);
        } else {
            const Rows<T> K{(const T*)a.pk + plane, a.P}, V{(const T*)a.pv + plane, a.P}, none{(const T*)a.pk, 0};
            const int tiles = (a.P + 31) / 32;
            few_queries<T, RTP, SELF>(a, p, hk, tile * 16 * RTP, a.M, K, V, none, none, tiles, piece * (a.prows / 32), min(tiles, (piece + 1) * (a.prows / 32)), false,
                                      0, 0, 0, piece, sm.few);
        }
    } else {
        int group, sub;  // (a group: a sequence's head)
        item_of(blockIdx.x - a.pitems, a.B * a.Hkv, a.otiles * a.opieces, group, sub);
        const int hk = group % a.Hkv, b = group / a.Hkv, tile = sub % a.otiles, piece = sub / a.otiles;
        int len, n;
        own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
        const int first = tile * 16, m0 = b * a.Mq + first, m_end = (b + 1) * a.Mq;
        // rows that the tile's last live query sees, in pieces of whole 128
        const int last = min(n, (first + 15) / a.G + 1), rows = first < n * a.G ? len + last : 0;
        const int step = max(a.ostep, (rows + 128 * a.opieces - 1) / (128 * a.opieces) * 128);
        const int64_t plane = ((int64_t)b * a.Hkv + hk) * a.maxlen * kS;
        const int end = min(rows, (piece + 1) * step);
        const Rows<T> none{(const T*)a.ok, 0}, K{(const T*)a.ok + plane, end}, V{(const T*)a.ov + plane, end};
        few_queries<T, 1, SELF>(a, p, hk, m0, m_end, none, none, K, V, 0, piece * (step / 32), (end + 31) / 32, true, b, len, n, a.ppieces + piece, sm.few);
    }
}

// Few rows: the prefix and the sequence's own in one go, sixteen queries of a sequence to a workgroup
template <typename T>
__global__ __launch_bounds__(256, 2) void prefix_brief_kernel(PrefixArgs a, PrepArgs p) {
    __shared__ MeetSmem sm;
    const int hk = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv;
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    const int rows = n > 0 ? len + n : 0, np = (a.P + 31) / 32, tiles = rows > 0 ? np + (rows + 31) / 32 : 0;
    const int64_t pplane = (int64_t)hk * a.pmax * kS, oplane = ((int64_t)b * a.Hkv + hk) * a.maxlen * kS;
    const Rows<T> K0{(const T*)a.pk + pplane, a.P}, V0{(const T*)a.pv + pplane, a.P}, K1{(const T*)a.ok + oplane, rows}, V1{(const T*)a.ov + oplane, rows};
    few_queries<T, 1, true>(a, p, hk, b * a.Mq, (b + 1) * a.Mq, K0, V0, K1, V1, np, 0, tiles, true, b, len, n, 0, sm);
}

// The prefix and the sequence's own rows in one sweep, or in pieces of it, for 64 * RT of a sequence's queries to a workgroup
template <typename T, int RT>
__global__ __launch_bounds__(256, 2) void prefix_sweep_kernel(PrefixArgs a) {
    __shared__ TileSmem<T> sm;
    int group, sub;
    item_of(blockIdx.x, a.B * a.Hkv, a.otiles * a.opieces, group, sub);
    const int hk = group % a.Hkv, b = group / a.Hkv, tile = a.otiles - 1 - sub / a.opieces, piece = sub % a.opieces;
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    const int first = tile * 64 * RT, last = min(n, (first + 64 * RT - 1) / a.G + 1), rows = first < n * a.G ? len + last : 0;
    const int np = (a.P + 31) / 32, tiles = rows > 0 ? np + (rows + 31) / 32 : 0, step = (tiles + a.opieces - 1) / a.opieces;
    const int64_t pplane = (int64_t)hk * a.pmax * kS, oplane = ((int64_t)b * a.Hkv + hk) * a.maxlen * kS;
    const Rows<T> K0{(const T*)a.pk + pplane, a.P}, V0{(const T*)a.pv + pplane, a.P}, K1{(const T*)a.ok + oplane, rows}, V1{(const T*)a.ov + oplane, rows};
    many_queries<T, RT>(a, hk, b * a.Mq + first, (b + 1) * a.Mq, K0, V0, K1, V1, np, piece * step, min(tiles, (piece + 1) * step), true, b, len, n, piece, sm);
}

// ---- 3. the pieces of a query ----
// half a wave to a query, 16 bytes to a lane.  Bound by latency: 4 us for two chats, 5 for 64 sequences of 32 heads (8 MB)
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixArgs a) {
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int d = 4 * (threadIdx.x & 31);
    if (r >= (int64_t)a.Hkv * a.M) return;
    const int hk = (int)(r / a.M), m = (int)(r - (int64_t)hk * a.M), bl = m / a.G, b = bl / a.qL, l = bl - b * a.qL;
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    float* out = a.out + ((int64_t)bl * a.G * a.Hkv + (int64_t)hk * a.G + (m - bl * a.G)) * kS + d;
    // eight records at a time, asked for together, with the length that tells whether the query is padding; a piece that the query sees nothing of has sum 0 and may have written nothing else
    const float2* stat = a.rec_stat + r * a.nrec;
    const float* rec = a.rec_out + r * a.nrec * kS + d;
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < a.nrec; c0 += 8) {
        float2 st[8];
        float4 x[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int c = min(c0 + u, a.nrec - 1);
            st[u] = stat[c];
            x[u] = *reinterpret_cast<const float4*>(rec + (int64_t)c * kS);
        }
        float up = M;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (c0 + u >= a.nrec) st[u] = make_float2(-INFINITY, 0.0f);
            up = fmaxf(up, st[u].x);
        }
        const float shrink = M == up ? 1.0f : __builtin_amdgcn_exp2f(M - up);
        M = up;
        L *= shrink, o.x *= shrink, o.y *= shrink, o.z *= shrink, o.w *= shrink;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const bool none = st[u].y == 0.0f;
            const float w = none ? 0.0f : st[u].x == M ? 1.0f : __builtin_amdgcn_exp2f(st[u].x - M);
            if (none) x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            L = fmaf(w, st[u].y, L);
            o.x = fmaf(w, x[u].x, o.x), o.y = fmaf(w, x[u].y, o.y), o.z = fmaf(w, x[u].z, o.z), o.w = fmaf(w, x[u].w, o.w);
        }
    }
    const float inv = 1.0f / L;
    *reinterpret_cast<float4*>(out) = l < n ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
}

struct PrefixPlan {
    bool brief, sweep, many, self;  // one sweep for a sequence's tiles; the prefix by many_queries; workgroups rotate their queries themselves
    int rt, ptiles, ppieces, prows, otiles, opieces, ostep;
};
// pieces of `rows`: some `wanted` of them, none below `least` rows
static int pieces_of(int64_t wanted, int64_t rows, int64_t least) {
    const int64_t most = (rows + least - 1) / least, n = wanted < most ? wanted : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
static PrefixPlan plan_prefix(int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t P, int64_t maxlen, bool half, bool ragged) {
    PrefixPlan p{};
    const int64_t Mq = qL * (H / Hkv), M = B * Mq;
    // (16 sequences of 32 heads behind 1500 rows, apart / sweep: 32 tokens 106 / 144, 77 / 92; 48 tokens
    // 155 / 142, 110 / 93; 64 tokens 181 / 154, 131 / 102.)
    // (All figures: us a call, fp32 caches and then halves.)  Few rows: one workgroup goes through all of a sequence's, 128 at a time, 2 us each time of
    // fp32 and 1 of halves, and nothing is to be joined.  In pieces / in one go, 32 heads: 1 sequence behind 20 rows, 30 of its own 10.4 / 7.5, 9.6 / 6.7;
    // 8 behind 130, 64 14.8 / 12.8, 11.8 / 8.8; 16 behind 200, 64 18.3 / 20.5, 15.6 / 13.4; 1 behind 400, 100 12.4 / 18.6, 10.3 / 11.3.
    p.brief = Mq <= 16 && P + maxlen <= (half ? 384 : 128) && B * Hkv <= 512;
    if (p.brief) {
        p.self = true;
        p.otiles = p.opieces = p.ostep = 1;
        return p;
    }
    p.sweep = Mq >= 48;
    if (p.sweep) {
        // 64 queries to a workgroup, or 128, which read the cut rows half as often: where the tiles are as full and there are workgroups enough, which
        // matters more for halves (nothing to cut).  64 / 128: 8 sequences of 256 tokens 222 / 187, 143 / 136; 4 of 300 170 / 160, 102 / 117; 4 of 160
        // 100 / 100, 66 / 75; 2 of 128 with 4 heads to a kv head 44 / 48, 39 / 43.  4 of 150 to 300, the rest padding: 129 / 169, so 64 where lengths differ.
        const int64_t t64 = (Mq + 63) / 64, t128 = (Mq + 127) / 128, items2 = B * Hkv * t128;
        const bool two = !ragged && (half ? 20 * t64 >= 38 * t128 && items2 >= 512 : 100 * t64 > 164 * t128 && items2 >= 128);
        p.rt = two ? 2 : 1;
        p.otiles = (int)(two ? t128 : t64);
        const int64_t items = B * Hkv * p.otiles;
        // (Pieces where that leaves the chip empty, until there are some 512 workgroups; until 256 / 512 / 1024: one sequence of 300 tokens 64 / 51 / 59.)
        p.opieces = pieces_of((512 + items / 2) / items, P + maxlen, 256);
        p.ostep = 1;
        return p;
    }
    const int64_t oitems = B * Hkv * ((Mq + 15) / 16);
    // many_queries cuts a row up once for 64 queries, few_queries goes through a piece four times as fast.  (Few / many behind 2000 rows: 128 queries of
    // each of 8 kv heads 30 / 37, 23 / 29; 256 of 8 45 / 41, 29 / 31; 48 of 32 39 / 42, 25 / 30; 128 of 32 64 / 53, 40 / 35.)
    p.many = M > 32 && M * Hkv > 1536;
    // many_queries with 128 queries as above, for fp32 rows and where they leave workgroups enough (64 / 128, 80 queries of 32 heads behind 2000 rows 107 / 102,
    // halves 63 / 65; 256 of 8 41 / 52).
    const bool wide = !half && 100 * ((M + 63) / 64) > 164 * ((M + 127) / 128) && Hkv * ((M + 127) / 128) * ((P + 511) / 512) >= 96;
    // few_queries with 32 queries reads rows half as often, with 16 there are more workgroups.  (16 / 32 behind 2000 rows: 128 of 8 27 / 30, 23 / 24; 40 of 32
    // 37 / 33, 26 / 24.)  Own rows always by 16: for 20 tokens of 8 sequences 32 took 67 instead of 67, 46 instead of 41.
    p.rt = (p.many ? wide : M > 16 && Hkv * ((M + 31) / 32) * ((P + 511) / 512) + oitems >= 320) ? 2 : 1;
    const int64_t tile = (p.many ? 64 : 16) * p.rt;
    p.ptiles = (int)((M + tile - 1) / tile);
    p.otiles = (int)((Mq + 15) / 16);
    // Pieces of 512 rows of the prefix and 1024 of the own rows, so that none is the last at work; smaller ones, down to 128, until there are
    // the 512 workgroups that the chip holds.  (Prefix in pieces of 256 / 512 / 1024 / 2048 rows: 64 sequences with 4 heads to a kv head behind 4001 rows
    // 77 / 68 / 71 / 115, 49 / 39 / 50 / 78; 16 of 5 tokens behind 1500 70 / 62 / 64 / 94.  Own rows, some 3000, in pieces of 512 / 1024 / 2048: 32 sequences
    // 289 / 296 / 344.)
    const int64_t pitems = Hkv * p.ptiles, all = (P > 0 ? pitems : 0) + oitems;
    const int64_t fill = (512 + all - 1) / all;
    if (P > 0) {
        const int64_t large = (P + 511) / 512, n = pieces_of(fill > large ? fill : large, P, 128);
        p.prows = (int)((P + 128 * n - 1) / (128 * n) * 128);
        p.ppieces = (int)((P + p.prows - 1) / p.prows);
    }
    p.ostep = fill > 1 ? 128 : 1024;
    p.opieces = pieces_of(fill > 1 ? fill : (maxlen + 1023) / 1024, maxlen, p.ostep);
    // A launch less where the workgroups are at work at once and have sixteen queries.  (Two / one launch before the pieces are joined: 2 sequences behind
    // 130 rows 13.2 / 11.8, 10.9 / 9.9; 8 behind 500 19.8 / 18.9, 15.5 / 14.3; 32 behind 2048, whose 1152 workgroups take turns and rotate in each,
    // 46.7 / 48.7 for halves; 8 with 32 queries to a workgroup 24.3 / 26.1, 19.3 / 18.6.)
    p.self = M <= 16 && pitems * p.ppieces + oitems * p.opieces <= 512;
    return p;
}

static size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
struct PrefixLayout {
    size_t qh, ql, cq, stat, rec, total;
};
static PrefixLayout layout_prefix(const PrefixPlan& plan, int64_t rows) {
    PrefixLayout w{};
    const size_t nrec = plan.ppieces + plan.opieces, held = plan.self ? 0 : rows;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes, 256);
        return here;
    };
    w.qh = take(held * kS * 2);
    w.ql = take(held * kS * 2);
    w.cq = take(held * 4);
    w.stat = take((size_t)rows * nrec * 8);
    w.rec = take((size_t)rows * nrec * kS * 4);
    w.total = at;
    return w;
}

template <typename T>
static int prefix_launch(PrefixArgs a, PrepArgs p, const PrefixPlan& plan, hipStream_t st) {
    const int64_t prep = (int64_t)a.B * a.qL * p.groups, items = (int64_t)a.pitems + (int64_t)a.B * a.Hkv * a.otiles * a.opieces,
                  merge = ((int64_t)a.Hkv * a.M + 7) / 8, most = (int64_t)1 << 24;  // (a launch has fewer than 2^32 threads)
    LLMOPS_REQUIRE(prep < most && items < most && merge < most);
    // (a workgroup reads its q, k and v while others may have written their rows and results)
    const Wide heads = (Wide)a.G * a.Hkv * kS * 4, kv_heads = (Wide)a.Hkv * kS * 4, plane = (Wide)a.Hkv * kS * sizeof(T);
    const Extent q(p.q, a.B, (Wide)p.qsb * 4, a.qL, (Wide)p.qsl * 4, heads), k(p.k, a.B, (Wide)p.ksb * 4, a.qL, (Wide)p.ksl * 4, kv_heads),
        v(p.v, a.B, (Wide)p.vsb * 4, a.qL, (Wide)p.vsl * 4, kv_heads), out(a.out, (Wide)a.B * a.qL * heads), own(a.ok, 2 * a.B * a.maxlen * plane),
        prefix(a.pk, a.P > 0 ? 2 * a.pmax * plane : 0);
    LLMOPS_REQUIRE(apart(own, q) && apart(own, k) && apart(own, v));
    LLMOPS_REQUIRE(apart(out, q) && apart(out, k) && apart(out, v) && apart(out, own) && apart(out, prefix));
    if (!plan.self) prefix_prep_kernel<T><<<(unsigned)prep, 256, 0, st>>>(a, p);
    LLMOPS_LAUNCH_CHECK();
    const unsigned grid = (unsigned)items;
#define LLMOPS_APART(RTP, MANY, SELF) prefix_apart_kernel<T, RTP, MANY, SELF><<<grid, 256, 0, st>>>(a, p)
    if (plan.brief) prefix_brief_kernel<T><<<grid, 256, 0, st>>>(a, p);
    else if (plan.sweep && plan.rt == 1) prefix_sweep_kernel<T, 1><<<grid, 256, 0, st>>>(a);
    else if (plan.sweep) prefix_sweep_kernel<T, 2><<<grid, 256, 0, st>>>(a);
    else if (plan.many && plan.rt == 2) LLMOPS_APART(sizeof(T) == 4 ? 2 : 1, true, false);
    else if (plan.many) LLMOPS_APART(1, true, false);
    else if (plan.self) LLMOPS_APART(1, false, true);
    else if (plan.rt == 1) LLMOPS_APART(1, false, false);
    else LLMOPS_APART(2, false, false);
#undef LLMOPS_APART
    LLMOPS_LAUNCH_CHECK();
    if (a.nrec > 1) prefix_merge_kernel<<<(unsigned)merge, 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}

}  // namespace llmops

using namespace llmops;

static bool prefix_sizes_fit(int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t prefix_len, int64_t maxlen) {
    const int64_t most = (int64_t)1 << 24;  // positions are exact in fp32
    return B > 0 && qL > 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && prefix_len >= 0 && maxlen > 0 && B < most && qL < most && H < most && prefix_len <= most &&
           maxlen <= most && prefix_len + maxlen <= most && B * qL < ((int64_t)1 << 31) / H;
}

extern "C" size_t llmops_attention_prefix_workspace_bytes(int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t S, int64_t prefix_len, int64_t maxlen) {
    if (S != kS || !prefix_sizes_fit(B, qL, H, Hkv, prefix_len, maxlen)) return 0;
    size_t most = 0;
    for (int kind = 0; kind < 4; kind++) {
        const size_t need = layout_prefix(plan_prefix(B, qL, H, Hkv, prefix_len, maxlen, kind & 1, kind & 2), B * qL * H).total;
        most = need > most ? need : most;
    }
    return most;
}

extern "C" int llmops_attention_rope_prefix(const float* q, int64_t q_stride_b, int64_t q_stride_l, const float* k, int64_t k_stride_b, int64_t k_stride_l,
                                            const float* v, int64_t v_stride_b, int64_t v_stride_l, int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t S,
                                            const float* inv_freq, int64_t half, const void* prefix_cache, int64_t prefix_planes, int64_t prefix_maxlen,
                                            int64_t prefix_len, void* kv_cache, int cache_dtype, int64_t planes, int64_t maxlen, const int32_t* lengths,
                                            const int32_t* q_lens, int layer_id, float* out, void* workspace, size_t workspace_bytes,
                                            llmops_stream_t stream) {
    LLMOPS_REQUIRE(q != nullptr && k != nullptr && v != nullptr && inv_freq != nullptr && kv_cache != nullptr && lengths != nullptr);
    LLMOPS_REQUIRE(out != nullptr && workspace != nullptr && (prefix_cache != nullptr || prefix_len == 0));
    LLMOPS_REQUIRE(S == 128);  // head size of every supported model shape
    LLMOPS_REQUIRE(prefix_sizes_fit(B, qL, H, Hkv, prefix_len, maxlen));
    LLMOPS_REQUIRE(half > 0 && 2 * half <= S);
    LLMOPS_REQUIRE(prefix_len == 0 || prefix_len <= prefix_maxlen);
    LLMOPS_REQUIRE(layer_id >= 0 && 2 * (int64_t)layer_id + 1 < planes && (prefix_len == 0 || 2 * (int64_t)layer_id + 1 < prefix_planes));
    LLMOPS_REQUIRE(cache_dtype == LLMOPS_CACHE_F32 || cache_dtype == LLMOPS_CACHE_F16);
    LLMOPS_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(prefix_cache, 16) && aligned(kv_cache, 16) &&
                   aligned(workspace, 256));
    LLMOPS_REQUIRE(q_stride_b % 4 == 0 && q_stride_l % 4 == 0 && k_stride_b % 4 == 0 && k_stride_l % 4 == 0 && v_stride_b % 4 == 0 && v_stride_l % 4 == 0);
    const size_t e = cache_dtype == LLMOPS_CACHE_F32 ? 4 : 2, row = (size_t)Hkv * kS * e;
    const uintptr_t p0 = reinterpret_cast<uintptr_t>(prefix_cache), p1 = p0 + (size_t)prefix_planes * prefix_maxlen * row,
                    o0 = reinterpret_cast<uintptr_t>(kv_cache), o1 = o0 + (size_t)planes * B * maxlen * row;
    LLMOPS_REQUIRE(prefix_len == 0 || p1 <= o0 || o1 <= p0);  // the caches do not overlap
    const PrefixPlan plan = plan_prefix(B, qL, H, Hkv, prefix_len, maxlen, cache_dtype == LLMOPS_CACHE_F16, q_lens != nullptr);
    const PrefixLayout w = layout_prefix(plan, B * qL * H);
    const size_t need = llmops_attention_prefix_workspace_bytes(B, qL, H, Hkv, S, prefix_len, maxlen);
    if (workspace_bytes < need) return fail(LLMOPS_EWORKSPACE, "attention_rope_prefix needs %zu workspace bytes, got %zu", need, workspace_bytes);
    char* ws = reinterpret_cast<char*>(workspace);
    PrefixArgs a{};
    a.qh = reinterpret_cast<_Float16*>(ws + w.qh), a.ql = reinterpret_cast<_Float16*>(ws + w.ql), a.cq = reinterpret_cast<float*>(ws + w.cq);
    a.rec_out = reinterpret_cast<float*>(ws + w.rec), a.rec_stat = reinterpret_cast<float2*>(ws + w.stat);
    const size_t pplane = (size_t)prefix_maxlen * row, oplane = (size_t)B * maxlen * row;
    a.pk = reinterpret_cast<const char*>(prefix_cache) + 2 * layer_id * pplane, a.pv = reinterpret_cast<const char*>(a.pk) + pplane;
    a.ok = reinterpret_cast<const char*>(kv_cache) + 2 * layer_id * oplane, a.ov = reinterpret_cast<const char*>(a.ok) + oplane;
    a.lengths = lengths, a.q_lens = q_lens, a.out = out;
    a.pmax = prefix_maxlen, a.maxlen = maxlen;
    a.B = (int)B, a.qL = (int)qL, a.G = (int)(H / Hkv), a.Hkv = (int)Hkv, a.P = (int)prefix_len, a.Mq = (int)(qL * a.G), a.M = (int)(B * a.Mq);
    a.ptiles = plan.ptiles, a.ppieces = plan.ppieces, a.prows = plan.prows, a.otiles = plan.otiles, a.opieces = plan.opieces, a.ostep = plan.ostep;
    a.nrec = plan.ppieces + plan.opieces;
    const int64_t pitems = Hkv * plan.ptiles * plan.ppieces;
    LLMOPS_REQUIRE(pitems < ((int64_t)1 << 24));
    a.pitems = (unsigned)pitems;
    const PrepArgs p{q, k, v, inv_freq, q_stride_b, q_stride_l, k_stride_b, k_stride_l, v_stride_b, v_stride_l, (int)half, (int)((H + 2 * Hkv + 15) / 16)};
    hipStream_t st = as_stream(stream);
    return cache_dtype == LLMOPS_CACHE_F32 ? prefix_launch<float>(a, p, plan, st) : prefix_launch<__half>(a, p, plan, st);
}
