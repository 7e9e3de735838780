// Attention of a batch over a cache that is held in 4 bits (its rows: cache_q4_device.h).  For sequence b with len[b] rows and n[b] new tokens,
// token l < n[b], head h on kv head h / G, G = H / Hkv:
//   pos = len[b] + l,  q' = rot(q, pos),  row pos of the cache = the codes of (rot(k, pos), v),
//   out = sum_r e_r V_r / sum_r e_r,  e_r = exp(q' . K_r / sqrt(S) - max),  r = 0 .. pos,  K and V as the cache holds them
//
//   1. q4_prep_kernel   rotates, writes the new rows and leaves q' as operands of the matrix instructions (part of 2 where caches are short)
//   2. q4_few_kernel or q4_many_kernel   softmax(q'K^T)V, running maximum and sum, one pass: rows shared out among workgroups by the lengths
//   3. q4_join_kernel   joins what several workgroups have of a query, unless each has all rows of its queries
//
// A sequence's queries of a kv head are numbered l*G + g.
//
// Arithmetic.  The cache's values are halves, so that they are operands of v_mfma_f32_16x16x32_f16 (fp32 sums) without any loss; q' and the weights
// are two halves each: q' scaled by a power of two of its row so that its largest value is in [2^13, 2^14), 22 bits of that, the weights times
// 2^14, so that those down to 2^-28 of the largest keep their bits.
#include "cache_q4_device.h"
#include "extents.h"

namespace llmops {

constexpr int kUnit = 128;  // rows that a workgroup's four waves read at a time

struct Q4Args {
    const float *q, *k, *v, *inv_freq;
    int64_t qsb, qsl, ksb, ksl, vsb, vsl;
    _Float16 *qh, *ql;                  // [Hkv][M][128]: rotated queries (M = B*Mq)
    float* cq;                          // [Hkv][M]: score = cq * (q' . k), in units of log2
    uint8_t *ck, *cv;                   // the layer's planes [B][Hkv][maxlen][80]
    const int32_t *lengths, *q_lens;    // [B]; q_lens may be null
    float* rec_out;                     // [groups][2][queries of a tile][128]
    float2* rec_stat;                   // [groups][2][queries of a tile]: max (log2), sum (-1: padding)
    int2* parts;                        // [B][Hkv][tiles]: the first and the last workgroup that have rows of a tile
    float* out;                         // [B][qL][H*128]
    int64_t maxlen;
    int B, qL, G, Hkv, M, Mq, half;     // Mq = qL*G
    int tile, tiles, groups, turns;     // queries of a tile, tiles of a sequence's queries for a kv head; workgroups, to a compute unit
    int join;                           // queries that a workgroup joins
    int row_groups;                     // workgroups to a token that rotate its rows
};
// query `in` of a sequence for kv head hk: token in / G, head hk*G + in % G
__device__ __forceinline__ const float* query_at(const Q4Args& a, int b, int hk, int in) {
    const int l = in / a.G;
    return a.q + b * a.qsb + l * a.qsl + (int64_t)(hk * a.G + in - l * a.G) * kS;
}

// ---- 1. ----
// Sixteen lanes to a row of k or v, dims 8 * (lane % 16) .. to a lane: k turned and its codes chosen in 64 bits, v in fp32; the row written
__device__ __forceinline__ void write_row(const Q4Args& a, const RowPair& p, const float* src, bool is_k, int b, int hk, int64_t row, int j, const double2* turn) {
    uint8_t* dst = (is_k ? a.ck : a.cv) + (((int64_t)b * a.Hkv + hk) * a.maxlen + row) * kQ4Row;
    if (is_k) {
        double x[8];
        turn_row(p, src, j, turn, a.half, x);
        store_q4(dst, quantise8(x), j);
    } else {
        store_q4(dst, quantise8(p.x), j);
    }
}
// .. of a query: turned in fp32
__device__ __forceinline__ QueryRow turned_query(const RowPair& p, const float* src, int j, const double2* turn, int half, bool live) {
    float x[8];
    if (live) turn_row(p, src, j, turn, half, x);
    else
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.0f;
    return query_row(x, live);
}
__device__ __forceinline__ const float* new_row_at(const Q4Args& a, bool is_k, int b, int hk, int l) {
    return is_k ? a.k + b * a.ksb + l * a.ksl + (int64_t)hk * kS : a.v + b * a.vsb + l * a.vsl + (int64_t)hk * kS;
}

// A workgroup per token and 16 of its H + 2*Hkv rows of 128, sixteen lanes to a row.  By itself and not in the workgroups of step 2: many of these share a
// query and each would turn it again (4 turns of 300 tokens: step 2 takes 62 us as it is, 73 with that).
// Latency with few tokens (32 of 96 rows 5.0 us: the length, the row and the frequency in one round trip, the sincos in 64 bits, the codes), memory with many
// (1200 tokens, 59 MB in, padding's rows among them, and 21 out, 18 us, 4.4 TB/s; two or three rows one behind the other to sixteen lanes: the same).
__global__ __launch_bounds__(256) void q4_prep_kernel(Q4Args a) {
    __shared__ double2 turn[64];
    const int bl = blockIdx.x / a.row_groups, group = blockIdx.x - bl * a.row_groups, b = bl / a.qL, l = bl - b * a.qL;
    const int H = a.G * a.Hkv, row = group * 16 + (threadIdx.x >> 4), j = threadIdx.x & 15;
    const bool is_q = row < H, is_k = !is_q && row < H + a.Hkv, none = row >= H + 2 * a.Hkv;
    const int hk = is_k ? row - H : row - H - a.Hkv;
    const float* src = is_q ? a.q + b * a.qsb + l * a.qsl + (int64_t)row * kS : new_row_at(a, is_k, b, hk, l);
    // (the row is on its way while the length is fetched and the angles are formed, also where the token turns out to be padding)
    RowPair p = {};
    if (!none) p.load(src, j);
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    if (l >= n) return;
    if ((int)threadIdx.x < a.half) turn[threadIdx.x] = turn64(a.inv_freq[threadIdx.x], len + l);
    __syncthreads();
    if (is_q) {
        const int64_t m = (int64_t)(row / a.G) * a.M + (int64_t)bl * a.G + row % a.G;
        const QueryRow r = turned_query(p, src, j, turn, a.half, true);
        *reinterpret_cast<uint4*>(a.qh + m * kS + 8 * j) = r.hi;
        *reinterpret_cast<uint4*>(a.ql + m * kS + 8 * j) = r.lo;
        if (j == 0) a.cq[m] = r.c;
    } else if (!none) {
        write_row(a, p, src, is_k, b, hk, len + l, j, turn);
    }
}

// ---- 2. rows for a tile of queries ----
// Lanes of v_mfma_f32_16x16x32_f16: operand A row lane % 16, B column lane % 16, eight k-values 8 * (lane / 16) .. +7 of either;
// result column lane % 16, rows 4 * (lane / 16) + v.  With g = lane / 16 and i = lane % 16, 32 cache rows from t on:
//   S^T = K Q^T   A: rows t + 16*tt + i, dims 32*g + 8*step .. +7: one group of the cache's to a lane, 16 bytes of codes.  B: query i.
//                 Result: query i, rows t + 16*tt + 4*g + v.
//   O^T = V^T e^T k-value j of lane group g stands for row t + 16*(j/4) + 4*g + j%4, so that B is the scores as they lie.
//                 A: dim 8*i + c of product c: a lane loads word i of its eight rows, which holds the eight products' codes, and turns the
//                 8 x 8 codes over in its registers.  Result of product c: query i, dim 8*(4*g + v) + c.
__device__ __forceinline__ uint32_t ask4(buffer_rsrc r, uint32_t lane_at, uint32_t at) { return __builtin_amdgcn_raw_buffer_load_b32(r, lane_at + at, 0, 0); }

// N rows from t on (the same t in the whole wave) as a descriptor that ends with the rows: those behind read as zero
template <int N = 32>
__device__ __forceinline__ buffer_rsrc q4_rows(const uint8_t* p, int t, int end) {
    return make_rsrc(p + (int64_t)t * kQ4Row, (uint32_t)__builtin_amdgcn_readfirstlane(max(0, min(N, end - t))) * (uint32_t)kQ4Row);
}
struct Q4Regs {
    uint4 k[2];
    uint32_t kdm[2], v[8], vdm[8];
    __device__ __forceinline__ void load_k(buffer_rsrc r, int i, int g) {
        const uint32_t codes = unseen((uint32_t)(i * kQ4Row + 16 * g)), pairs = unseen((uint32_t)(i * kQ4Row + 64 + 4 * g));
#pragma unroll
        for (int tt = 0; tt < 2; tt++) k[tt] = ask16(r, codes, 16 * tt * kQ4Row), kdm[tt] = ask4(r, pairs, 16 * tt * kQ4Row);
    }
    __device__ __forceinline__ void load_v(buffer_rsrc r, int i, int g) {
        const uint32_t codes = unseen((uint32_t)(4 * g * kQ4Row + 4 * i)), pairs = unseen((uint32_t)(4 * g * kQ4Row + 64 + (i & 12)));
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = ask4(r, codes, (16 * (j >> 2) + (j & 3)) * kQ4Row);
            vdm[j] = ask4(r, pairs, (16 * (j >> 2) + (j & 3)) * kQ4Row);
        }
    }
    __device__ __forceinline__ v8h k_op(const Codes& codes, int tt, int step) const {
        return codes.values(step == 0 ? k[tt].x : step == 1 ? k[tt].y : step == 2 ? k[tt].z : k[tt].w, kdm[tt]);
    }
    // the operands of two products from byte y of the eight words: codes 0 2, 4 6, 1 3, 5 7
    __device__ __forceinline__ void v_ops(const Codes& codes, int y, v8h& low, v8h& high) const {
        const uint32_t pick = 0x0c000c00u | (uint32_t)(4 + y) << 16 | (uint32_t)y;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint32_t x = __builtin_amdgcn_perm(v[2 * p + 1], v[2 * p], pick);
            const v2h d = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(vdm[2 * p + 1], vdm[2 * p], 0x05040100u)),
                      m = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(vdm[2 * p + 1], vdm[2 * p], 0x07060302u));
            const v2h lo = __builtin_elementwise_fma(codes.low(x), d, m), hi = __builtin_elementwise_fma(codes.high(x), d, m);
            low[2 * p] = lo[0], low[2 * p + 1] = lo[1], high[2 * p] = hi[0], high[2 * p + 1] = hi[1];
        }
    }
    // a V row that holds NaN (m tells, in every group) among rows that not every query sees: NaN in the scores of those that do, and nothing in
    // the operand, where it would reach the others as 0 * NaN
    __device__ __forceinline__ void hide_nan(uint32_t& hidden) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if ((vdm[j] & 0x7fff0000u) > 0x7c000000u) vdm[j] = 0, hidden |= 1u << j;
    }
};
__device__ __forceinline__ constexpr int first_code(int y) { return y == 0 ? 0 : y == 1 ? 4 : y == 2 ? 1 : 5; }  // of byte y; the other is 2 more

// A tile's rotated queries as operands in LDS (the four waves share them, and leave registers for a fourth wave on a SIMD), with their factors
template <int RT>
struct Q4FewIn {
    uint4 q[RT * 8 * 64];
    double2 turn[16 * RT][64];  // of the sequence's tokens
};
template <int RT>
__device__ __forceinline__ void q4_take(const Q4Args& a, Q4FewIn<RT>& sm, float* factors, int b, int hk, int n, int lane) {
    const int wave = threadIdx.x >> 6;  // a step to a wave
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int64_t m = (int64_t)hk * a.M + (int64_t)b * a.Mq + min(16 * rt + (lane & 15), a.Mq - 1), at = m * kS + 32 * (lane >> 4) + 8 * wave;
        sm.q[(rt * 8 + wave) * 64 + lane] = *reinterpret_cast<const uint4*>(a.qh + at);
        sm.q[(rt * 8 + 4 + wave) * 64 + lane] = *reinterpret_cast<const uint4*>(a.ql + at);
        if (wave == 0 && lane < 16) factors[16 * rt + lane] = min(16 * rt + lane, a.Mq - 1) / a.G < n ? a.cq[m] : 0.0f;  // (padding's queries hold anything)
    }
    __syncthreads();
}
// The same from q itself, and the sequence's new rows of k and v written (a launch less).  All of it by the workgroup, sixteen lanes to a row, 16 rows at a time.
// Loads that wait for each other: where many workgroups keep the memory busy the launch is the better way (32 sequences of up to 4096 rows 88 us with
// it, 109 without; two of up to 200 14.9 and 9.7).
// What it needs of memory is asked for with the length (q, first_new: a row of k or v, f); queries from the first sixteen lanes on, new rows from the last, so
// that one query and its row are turned by different waves at a time.
struct Q4Asked {
    RowPair first_new;
    float f;
};
template <int RT>
__device__ __forceinline__ void q4_begin(const Q4Args& a, Q4FewIn<RT>& sm, float* factors, int b, int hk, int len, int n, const RowPair (&q)[RT], const Q4Asked& asked) {
    const int thread = (int)unseen(threadIdx.x), i = thread >> 4, j = thread & 15;
    if ((thread & 63) < a.half)
#pragma unroll 1
        for (int l = thread >> 6; l < n; l += 4) sm.turn[l][thread & 63] = turn64(asked.f, len + l);
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int in = 16 * rt + i, at = rt * 8 * 64 + (j & 3) * 64 + 16 * (j >> 2) + i;  // dims 32*g + 8*step .. of query i
        QueryRow r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0), 0.0f};
        if (in < a.Mq) r = turned_query(q[rt], query_at(a, b, hk, in), j, sm.turn[min(in / a.G, max(n - 1, 0))], a.half, in / a.G < n);
        sm.q[at] = r.hi;
        sm.q[at + 4 * 64] = r.lo;
        if (j == 0) factors[16 * rt + i] = r.c;
    }
    RowPair p = asked.first_new;
#pragma unroll 1
    for (int r = 15 - i; r < 2 * n; r += 16) {  // (k and v of a row in turn)
        const float* src = new_row_at(a, (r & 1) == 0, b, hk, r >> 1);
        if (r >= 16) p.load(src, j);
        write_row(a, p, src, (r & 1) == 0, b, hk, len + (r >> 1), j, sm.turn[r >> 1]);
    }
    __syncthreads();
}

// Units of 128 rows are numbered through: sequence after sequence, in each kv head after kv head, in each tile after tile.  Behind the units of a tile
// there are kStart more without rows, for what it costs to begin with queries and to bring the waves' sums together, so that workgroups with short
// sequences have no more to do.  A tile that is all padding has one unit, in which its zeros are written.
constexpr int kStart = 1;
struct UnitsOf {
    int tile, live, head;  // units of a tile that is not all padding, such tiles, units of a kv head
};
__device__ __forceinline__ UnitsOf units_of(const Q4Args& a, int b) {
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    UnitsOf u;
    u.live = (n * a.G + a.tile - 1) / a.tile;
    u.tile = n > 0 ? (len + n + kUnit - 1) / kUnit + kStart : 1;
    u.head = u.live * u.tile + a.tiles - u.live;
    return u;
}
// the tile of unit `in` of a kv head, its units, and how many are before this one
__device__ __forceinline__ void tile_of(const UnitsOf& u, int in, int& tile, int& units, int& at) {
    const bool live = in < u.live * u.tile;
    tile = live ? in / u.tile : u.live + in - u.live * u.tile;
    units = live ? u.tile : 1;
    at = live ? in - tile * u.tile : 0;
}
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        v += lane >= o ? u : 0;
    }
    return v;
}
// Units first .. last-1 of a workgroup's, out of `all`.  Where the chip is full, a.turns workgroups to a compute unit, those that come first have the
// waves that are served first when several wait: with equal shares they were done in half the time of those that come last.  So shares fall from 1.25
// to 0.75 of the mean (32 sequences of up to 4096 rows 86.2 us with equal shares, 86.3 / 84.2 / 87.4 with 0.15 / 0.25 / 0.35; 64 with grouped heads 88.2, 85.3 / 83.6 /
// 85.4; 16 of 5 tokens 39.8, 37.5 / 37.1 / 37.0; 4 turns 86.4, 86.3 / 83.8 / 85.6).
constexpr int kSlope = 25;  // hundredths
__device__ __forceinline__ int64_t share_at(const Q4Args& a, int w, int64_t all) {
    // (few units: one to a workgroup, or as many to each, until there are none.  None may be left out between two that have rows of a tile)
    if (a.turns == 1 || all < 4 * (int64_t)a.groups) return min(all, (all + a.groups - 1) / a.groups * w);
    const int each = a.groups / a.turns, turn = w / each, in = w - turn * each;
    // shares of turn 0, 1, ..: 100 + kSlope * (1 - 2 turn / (turns - 1)), in all 100 * turns
    const int64_t steps = a.turns - 1, before = turn * (100 + kSlope) * steps - kSlope * (int64_t)turn * (turn - 1), its = (100 + kSlope) * steps - 2 * kSlope * turn;
    return all * (before * each + its * in) / (100 * steps * a.groups);
}
// Every wave for itself: a workgroup's units, and the sequence that has the first of them (-1: it has none), with the units before that sequence
struct UnitPlace {
    int first, last, b, before;
};
__device__ __forceinline__ UnitPlace place_of(const Q4Args& a, int lane) {
    int all = 0, its = 0, upto = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        its = b0 + lane < a.B ? units_of(a, b0 + lane).head * a.Hkv : 0;
        upto = all + wave_scan(its, lane);
        all = __builtin_amdgcn_readlane(upto, 63);
    }
    UnitPlace p{(int)share_at(a, blockIdx.x, all), (int)share_at(a, blockIdx.x + 1, all), -1, 0};
    if (p.first >= p.last) return p;
    int before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (a.B > 64) {
            its = b0 + lane < a.B ? units_of(a, b0 + lane).head * a.Hkv : 0;
            upto = before + wave_scan(its, lane);
        }
        const uint64_t hit = __ballot(upto > p.first);
        if (hit != 0) {
            const int at = __builtin_ctzll(hit);
            p.b = b0 + at;
            p.before = __builtin_amdgcn_readlane(upto - its, at);
            break;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return p;
}

__device__ __forceinline__ void q4_leave(const Q4Args& a, int b, int hk, int in, int d, float4 o, float sum, bool live) {
    const float f = live ? 1.0f / sum : 0.0f;
    const int l = in / a.G;
    *reinterpret_cast<float4*>(a.out + (((int64_t)b * a.qL + l) * a.G * a.Hkv + (int64_t)hk * a.G + (in - l * a.G)) * kS + d) =
        live ? make_float4(o.x * f, o.y * f, o.z * f, o.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
}

constexpr int kQ4MeetRow = 132;  // floats (16 queries' rows on different banks)
template <int RT>
struct Q4MeetSmem {
    float m[4][32], l[4][32], sum[16], factors[16 * RT];
    union {
        float o[4][16][kQ4MeetRow];
        Q4FewIn<RT> in;
    };
};

// Few queries to a workgroup (16 * RT).  The four waves take 32 rows each of every 128; operands come straight from memory, the next rows asked
// for when these are used up; the waves' sums meet in LDS.
// Memory bounds it: a row's 80 bytes of K are read in 16-byte pieces by the lanes that multiply them, V's in words.  32 sequences of up to 4096 rows, 32 heads: 335 MB
// in 74 us, 4.5 TB/s (a kernel that only reads them, in one order: 51 us; this one with its products taken out: 65); the vector ALU is busy half of
// the time, mostly with making halves of codes.  One sequence of 50000 rows, 8 kv heads: 64 MB
// in 23 us, three or four times 128 rows to a workgroup, so that beginning and end are as long as the stream.  Not faster: copies to LDS by the DMA
// engine, one or two stages ahead (87 us for the call, 87 and 93); waves' priorities by turn (91 to 97); more workgroups than the chip holds (87).
template <int RT, bool WHOLE>
__global__ __launch_bounds__(256, RT == 1 && !WHOLE ? 4 : 2) void q4_few_kernel(Q4Args a) {
    __shared__ Q4MeetSmem<RT> sm;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Codes codes;
    int b, before, first, last;
    if constexpr (WHOLE) {  // a kv head of a sequence to a workgroup
        b = blockIdx.x / a.Hkv, before = 0;
        const int units = units_of(a, b).head;
        first = (blockIdx.x - b * a.Hkv) * units, last = first + units;
    } else {
        const UnitPlace start = place_of(a, threadIdx.x & 63);
        if (start.b < 0) return;
        b = start.b, before = start.before, first = start.first, last = start.last;
    }
    RowPair q_rows[WHOLE ? RT : 1];
    Q4Asked asked;
    if constexpr (WHOLE) {  // (asked for with the length)
        const int i = threadIdx.x >> 4, r = 15 - i, j = threadIdx.x & 15, hk = blockIdx.x - b * a.Hkv;
        asked.f = a.inv_freq[min((int)threadIdx.x & 63, a.half - 1)];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) q_rows[rt].load(query_at(a, b, hk, min(16 * rt + i, a.Mq - 1)), j);
        if (r < 2 * a.qL) asked.first_new.load(new_row_at(a, (r & 1) == 0, b, hk, r >> 1), j);
    }
    UnitsOf its = units_of(a, b);
#pragma unroll 1
    for (int at = first; at < last;) {
        if (at >= before + its.head * a.Hkv) {  // (the next sequence)
            before += its.head * a.Hkv;
            its = units_of(a, ++b);
        }
        const int hk = (at - before) / its.head;
        int tile, units, u0;  // (one tile)
        tile_of(its, at - before - hk * its.head, tile, units, u0);
        const int u1 = min(units, u0 + (last - at)), real = units > kStart ? units - kStart : units;
        if (!WHOLE && (u0 == 0 || u1 >= real) && threadIdx.x == 0) {
            int2* parts = a.parts + ((int64_t)b * a.Hkv + hk) * a.tiles + tile;
            if (u0 == 0) parts->x = blockIdx.x;
            if (u0 < real && u1 >= real) parts->y = blockIdx.x;
        }
        at += u1 - u0;
        if (u0 >= real) continue;
        const int lane = (int)unseen(threadIdx.x & 63), i = lane & 15, g = lane >> 4;
        int len, n;
        own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
        const int rows = n > 0 ? len + n : 0;
        const int64_t plane = ((int64_t)b * a.Hkv + hk) * a.maxlen * kQ4Row;
        const uint8_t *K = a.ck + plane, *V = a.cv + plane;
        Q4Regs x;
        const int j0 = 4 * u0 + wave, j1 = min(4 * u1, (rows + 31) / 32);
        // (rows that were there before this call are asked for before the queries are turned, new ones when they are written)
        const bool old = !WHOLE || 32 * j0 + 32 <= len;
        if (j0 < j1 && old) x.load_k(q4_rows(K, 32 * j0, rows), i, g), x.load_v(q4_rows(V, 32 * j0, rows), i, g);
        if constexpr (WHOLE) {
            q4_begin<RT>(a, sm.in, sm.factors, b, hk, len, n, q_rows, asked);
            if (j0 < j1 && !old) x.load_k(q4_rows(K, 32 * j0, rows), i, g), x.load_v(q4_rows(V, 32 * j0, rows), i, g);
        }
        if constexpr (!WHOLE) q4_take<RT>(a, sm.in, sm.factors, b, hk, n, lane);
        Queries<RT> s;
        bool live[RT];
        int see_min = INT_MAX;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int l = min(16 * rt + i, a.Mq - 1) / a.G;
            s.c[rt] = sm.factors[16 * rt + i], s.m[rt] = -INFINITY, s.l[rt] = 0.0f;
#pragma unroll
            for (int c = 0; c < 8; c++) s.o[rt][c] = v4f{0.f, 0.f, 0.f, 0.f};
            live[rt] = l < n;
            s.see[rt] = live[rt] ? len + l + 1 : INT_MAX;  // (what padding sees is thrown away)
            see_min = min(see_min, s.see[rt]);
        }
#pragma unroll 1
        for (int j = j0; j < j1; j += 4) {
            const int t = 32 * j;
            const bool masked = __any(t + 32 > see_min);
            const uint4* q = sm.in.q + unseen(lane);  // (read here and now: kept from one time to the next, operands take registers)
            v4f sc[RT][2];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) sc[rt][0] = sc[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int step = 0; step < 4; step++) {
                const v8h k0 = x.k_op(codes, 0, step), k1 = x.k_op(codes, 1, step);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    const v8h hi = as_v8h(q[(rt * 8 + step) * 64]), lo = as_v8h(q[(rt * 8 + 4 + step) * 64]);
                    sc[rt][0] = mfma(k0, hi, sc[rt][0]);
                    sc[rt][1] = mfma(k1, hi, sc[rt][1]);
                    sc[rt][0] = mfma(k0, lo, sc[rt][0]);
                    sc[rt][1] = mfma(k1, lo, sc[rt][1]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            x.load_k(q4_rows(K, t + 128, rows), i, g);  // (behind the last rows too, where nothing is read: with a branch around them all loads would be waited for)
            uint32_t hidden = 0;
            if (masked) x.hide_nan(hidden);
            Weights w[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                if (hidden != 0)
#pragma unroll
                    for (int r = 0; r < 8; r++)
                        if (hidden >> r & 1) sc[rt][r >> 2][r & 3] = NAN;
                weigh<true>(s, rt, sc[rt], t, g, masked);
                w[rt] = weights_of<__half>(sc[rt]);
            }
#pragma unroll
            for (int y = 0; y < 4; y++) {
                v8h low, high;
                x.v_ops(codes, y, low, high);
                const int c = first_code(y);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    s.o[rt][c] = mfma(low, w[rt].hi, s.o[rt][c]);
                    s.o[rt][c + 2] = mfma(high, w[rt].hi, s.o[rt][c + 2]);
                    s.o[rt][c] = mfma(low, w[rt].lo, s.o[rt][c]);
                    s.o[rt][c + 2] = mfma(high, w[rt].lo, s.o[rt][c + 2]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            x.load_v(q4_rows(V, t + 128, rows), i, g);
        }
        // the four waves' sums
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            s.l[rt] += __shfl_xor(s.l[rt], 16, 64);
            s.l[rt] += __shfl_xor(s.l[rt], 32, 64);
            if (g == 0) sm.m[wave][16 * rt + i] = s.m[rt], sm.l[wave][16 * rt + i] = s.l[rt];
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 >= real;
        const int64_t record = ((int64_t)blockIdx.x * 2 + (u0 == 0)) * (16 * RT);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float M = sm.m[0][16 * rt + i];
#pragma unroll
            for (int w = 1; w < 4; w++) M = fmaxf(M, sm.m[w][16 * rt + i]);
            const float f = s.m[rt] == M ? 1.0f : __builtin_amdgcn_exp2f(s.m[rt] - M);  // (equal: also both -inf)
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    *reinterpret_cast<float4*>(&sm.o[wave][i][8 * (4 * g + v) + 4 * h]) =
                        make_float4(s.o[rt][4 * h][v] * f, s.o[rt][4 * h + 1][v] * f, s.o[rt][4 * h + 2][v] * f, s.o[rt][4 * h + 3][v] * f);
            if (wave == 0 && g == 0) {
                float L = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const float mw = sm.m[w][16 * rt + i];
                    L += sm.l[w][16 * rt + i] * (mw == M ? 1.0f : __builtin_amdgcn_exp2f(mw - M));
                }
                sm.sum[i] = live[rt] ? L : -1.0f;
                if (!whole) a.rec_stat[record + 16 * rt + i] = make_float2(M, sm.sum[i]);
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int e = lane + 64 * wave + 256 * u, query = e >> 5, d = 4 * (e & 31), in = 16 * rt + query;
                if (in < a.Mq) {
                    float4 r = *reinterpret_cast<const float4*>(&sm.o[0][query][d]);
#pragma unroll
                    for (int w = 1; w < 4; w++) {
                        const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][query][d]);
                        r.x += y.x, r.y += y.y, r.z += y.z, r.w += y.w;
                    }
                    if (whole) q4_leave(a, b, hk, in, d, r, sm.sum[query], sm.sum[query] != -1.0f);
                    else *reinterpret_cast<float4*>(a.rec_out + (record + 16 * rt + query) * kS + d) = r;
                }
            }
            __syncthreads();
        }
    }
}

// Many queries (64 to a workgroup, 16 to a wave).  All waves multiply the same 64 rows, whose values the workgroup forms once and leaves in LDS in the
// order of the operands (a read is 16 bytes to a lane, in lane order); two buffers: while a tile is multiplied the next one's values are formed and the one
// behind it is on its way from memory.
// Instructions bound it, and what two waves to a SIMD leave uncovered: 4 turns of 300 tokens behind up to 1777 rows, 32 heads, 61 us, of which the vector ALU is
// busy 22, the matrix cores 12 and LDS reads, 32 KB to a wave and tile of 64 rows, 12; waves wait for data 28 % of the time and for a turn to issue 36 %.  Not faster: 128 queries to four
// waves (fewer workgroups than places, twice the registers), 128 to eight waves (the call 104 us instead of 86; 2048 tokens of one sequence, 194 instead of 211),
// one buffer and three workgroups to a compute unit (85 instead of 83).
struct Q4TileSmem {
    uint4 k[2][16][64], v[2][16][64];
    uint32_t bad[2][4];  // of 16 rows each: V rows that hold NaN, among those that are new
};
struct Q4TileRegs {
    uint4 k;
    uint32_t kdm, v[4], vdm[4];
    // rows 16*wave .. of 64 to a wave.  K: row i, group g.  V: word i of rows 4*g + 0..3
    __device__ __forceinline__ void load(buffer_rsrc K, buffer_rsrc V, int wave, int i, int g) {
        const uint32_t k_at = (uint32_t)((16 * wave + i) * kQ4Row), v_at = (uint32_t)((16 * wave + 4 * g) * kQ4Row);
        k = ask16(K, k_at + 16 * g, 0);
        kdm = ask4(K, k_at + 64 + 4 * g, 0);
        const uint32_t codes = unseen(v_at + 4 * i), pairs = unseen(v_at + 64 + (i & 12));
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = ask4(V, codes, r * kQ4Row), vdm[r] = ask4(V, pairs, r * kQ4Row);
    }
    __device__ __forceinline__ void write(const Codes& codes, Q4TileSmem& sm, int buf, int wave, int lane, bool fresh) {
        sm.k[buf][4 * wave][lane] = __builtin_bit_cast(uint4, codes.values(k.x, kdm));
        sm.k[buf][4 * wave + 1][lane] = __builtin_bit_cast(uint4, codes.values(k.y, kdm));
        sm.k[buf][4 * wave + 2][lane] = __builtin_bit_cast(uint4, codes.values(k.z, kdm));
        sm.k[buf][4 * wave + 3][lane] = __builtin_bit_cast(uint4, codes.values(k.w, kdm));
        if (fresh) {
            uint32_t bad = 0;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const bool nan = (vdm[r] & 0x7fff0000u) > 0x7c000000u;
                const uint64_t rows = __ballot(nan);
                if (nan) vdm[r] = 0;
#pragma unroll
                for (int g = 0; g < 4; g++) bad |= (uint32_t)(rows >> (16 * g) & 1) << (4 * g + r);
            }
            if (lane == 0) sm.bad[buf][wave] = bad;
        }
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const uint32_t pick = 0x0c000c00u | (uint32_t)(4 + y) << 16 | (uint32_t)y;
            uint2 low, high;
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const uint32_t x = __builtin_amdgcn_perm(v[2 * p + 1], v[2 * p], pick);
                const v2h d = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(vdm[2 * p + 1], vdm[2 * p], 0x05040100u)),
                          m = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(vdm[2 * p + 1], vdm[2 * p], 0x07060302u));
                (p ? low.y : low.x) = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(codes.low(x), d, m));
                (p ? high.y : high.x) = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(codes.high(x), d, m));
            }
            // (rows 0 .. 31 are the first eight operands' first and second halves, rows 32 .. 63 the others')
            const int c = 8 * (wave >> 1) + first_code(y);
            reinterpret_cast<uint2*>(&sm.v[buf][c][lane])[wave & 1] = low;
            reinterpret_cast<uint2*>(&sm.v[buf][c + 2][lane])[wave & 1] = high;
        }
    }
};

__global__ __launch_bounds__(256, 2) void q4_many_kernel(Q4Args a) {
    __shared__ Q4TileSmem sm;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const Codes codes;
    const UnitPlace start = place_of(a, lane);
    if (start.b < 0) return;
    const int first = start.first, last = start.last;
    int b = start.b, before = start.before;
    UnitsOf its = units_of(a, b);
#pragma unroll 1
    for (int at = first; at < last;) {
        if (at >= before + its.head * a.Hkv) {  // (the next sequence)
            before += its.head * a.Hkv;
            its = units_of(a, ++b);
        }
        const int hk = (at - before) / its.head;
        int tile, units, u0;
        tile_of(its, at - before - hk * its.head, tile, units, u0);
        const int u1 = min(units, u0 + (last - at)), real = units > kStart ? units - kStart : units;
        if ((u0 == 0 || u1 >= real) && threadIdx.x == 0) {
            int2* parts = a.parts + ((int64_t)b * a.Hkv + hk) * a.tiles + tile;
            if (u0 == 0) parts->x = blockIdx.x;
            if (u0 < real && u1 >= real) parts->y = blockIdx.x;
        }
        at += u1 - u0;
        if (u0 >= real) continue;
        int len, n;
        own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
        const int in0 = tile * 64, in_end = min(a.Mq, in0 + 64);
        // rows that the tile's last live query sees
        const int rows = in0 < n * a.G ? len + min(n, (in_end - 1) / a.G + 1) : 0;
        const int64_t plane = ((int64_t)b * a.Hkv + hk) * a.maxlen * kQ4Row;
        const uint8_t *K = a.ck + plane, *V = a.cv + plane;
        const int j0 = 2 * u0, j1 = min(2 * u1, (rows + 63) / 64);
        Q4TileRegs x;
        auto load = [&](int j) { x.load(q4_rows<64>(K, 64 * j, rows), q4_rows<64>(V, 64 * j, rows), wave, i, g); };
        if (j0 < j1) load(j0);
        v8h qh[4], ql[4];
        Queries<1> s;
        const int mine = min(in0 + 16 * wave + i, in_end - 1), l = mine / a.G;
        const bool live = l < n;
        const int64_t m = (int64_t)hk * a.M + (int64_t)b * a.Mq + mine, from = m * kS + 32 * g;
#pragma unroll
        for (int step = 0; step < 4; step++) {
            qh[step] = as_v8h(*reinterpret_cast<const uint4*>(a.qh + from + 8 * step));
            ql[step] = as_v8h(*reinterpret_cast<const uint4*>(a.ql + from + 8 * step));
        }
        s.c[0] = live ? a.cq[m] : 0.0f, s.m[0] = -INFINITY, s.l[0] = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; c++) s.o[0][c] = v4f{0.f, 0.f, 0.f, 0.f};
        s.see[0] = live ? len + l + 1 : INT_MAX;  // (what padding sees is thrown away)
        if (j0 < j1) {
            x.write(codes, sm, 0, wave, lane, 64 * j0 + 64 > len);
            load(min(j0 + 1, j1 - 1));
        }
        __syncthreads();
#pragma unroll 1
        for (int j = j0; j < j1; j++) {
            const int buf = (j - j0) & 1, t = 64 * j;
            x.write(codes, sm, buf ^ 1, wave, lane, t + 128 > len);  // (behind the last tile that one again: nobody reads it)
            load(min(j + 2, j1 - 1));
            __builtin_amdgcn_sched_barrier(0);  // (asked for now: behind the scores' products they come late)
            const bool masked = __any(t + 64 > s.see[0]);
            v4f sc[4];
            sc[0] = sc[1] = sc[2] = sc[3] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int step = 0; step < 4; step++) {
                v8h k[4];
#pragma unroll
                for (int tt = 0; tt < 4; tt++) k[tt] = as_v8h(sm.k[buf][4 * tt + step][lane]);
#pragma unroll
                for (int tt = 0; tt < 4; tt++) sc[tt] = mfma(k[tt], qh[step], sc[tt]);
#pragma unroll
                for (int tt = 0; tt < 4; tt++) sc[tt] = mfma(k[tt], ql[step], sc[tt]);
            }
            Weights w[2];
            if (t + 64 > len) {
#pragma unroll
                for (int tt = 0; tt < 4; tt++) {
                    const uint32_t bad = __builtin_amdgcn_readfirstlane(sm.bad[buf][tt]);
                    if (bad != 0)
#pragma unroll
                        for (int v = 0; v < 4; v++)
                            if (bad >> (4 * g + v) & 1) sc[tt][v] = NAN;
                }
            }
            weigh<true>(s, 0, sc, t, g, masked);
            w[0] = weights_of<__half>({sc[0], sc[1]});
            w[1] = weights_of<__half>({sc[2], sc[3]});
#pragma unroll
            for (int c0 = 0; c0 < 16; c0 += 4) {
                v8h h[4];
#pragma unroll
                for (int c = 0; c < 4; c++) h[c] = as_v8h(sm.v[buf][c0 + c][lane]);
                const Weights& x2 = w[c0 >> 3];
#pragma unroll
                for (int c = 0; c < 4; c++) s.o[0][(c0 & 7) + c] = mfma(h[c], x2.hi, s.o[0][(c0 & 7) + c]);
#pragma unroll
                for (int c = 0; c < 4; c++) s.o[0][(c0 & 7) + c] = mfma(h[c], x2.lo, s.o[0][(c0 & 7) + c]);
            }
            __syncthreads();
        }
        const bool whole = u0 == 0 && u1 >= real;
        const int64_t record = ((int64_t)blockIdx.x * 2 + (u0 == 0)) * 64;
        s.l[0] += __shfl_xor(s.l[0], 16, 64);
        s.l[0] += __shfl_xor(s.l[0], 32, 64);
        const int in = 16 * wave + i;
        if (in0 + in >= in_end) continue;
        if (!whole && g == 0) a.rec_stat[record + in] = make_float2(s.m[0], live ? s.l[0] : -1.0f);
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float4 o = make_float4(s.o[0][4 * h][v], s.o[0][4 * h + 1][v], s.o[0][4 * h + 2][v], s.o[0][4 * h + 3][v]);
                const int d = 8 * (4 * g + v) + 4 * h;
                if (whole) q4_leave(a, b, hk, in0 + in, d, o, s.l[0], live);
                else *reinterpret_cast<float4*>(a.rec_out + (record + in) * kS + d) = o;
            }
    }
}

// ---- 3. what several workgroups have of a query ----
// A workgroup to a.join (1, 2, 4, 8) queries of a tile, 8 / a.join half waves to a query, each to as many records from the other, 16 bytes to a lane.  Latency: 5 us
// with one or two records to a query, 6.2 with 128, 9.7 with 38400 queries (20 MB of records, 20 MB out).  Joined by the last workgroup to arrive
// instead, records written through to memory: 32 sequences 90 us instead of 89, 64 with grouped heads 87.5 and 89.4, one of 50000 rows 41 and 32.
__global__ __launch_bounds__(256) void q4_join_kernel(Q4Args a) {
    __shared__ float stat[8][2];
    __shared__ float4 part[8][32];
    const int parts = (min(a.tile, a.Mq) + a.join - 1) / a.join, item = blockIdx.x / parts, in0 = a.join * (blockIdx.x - item * parts);
    const int each = a.Hkv * a.tiles, b = item / each, hk = (item - b * each) / a.tiles, tile = item % a.tiles;
    const int2 of = a.parts[item];
    const int w0 = of.x, w1 = of.y;
    const int queries = min(a.join, min(a.tile, a.Mq - tile * a.tile) - in0);
    if (w0 == w1 || queries <= 0) return;
    const int halves = 8 / a.join;
    const int half = threadIdx.x >> 5, turn = half & (halves - 1), query = in0 + half / halves, d = 4 * (threadIdx.x & 31);
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (query < in0 + queries) {
#pragma unroll 1
        for (int w = w0 + turn; w <= w1; w += 4 * halves) {
            float2 st[4];
            float4 x[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int64_t wg = min(w + halves * u, w1), record = (wg * 2 + (wg == w0)) * a.tile + query;
                st[u] = a.rec_stat[record];
                x[u] = *reinterpret_cast<const float4*>(a.rec_out + record * kS + d);
            }
            float up = M;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (w + halves * u > w1) st[u] = make_float2(-INFINITY, 0.0f);
                up = fmaxf(up, st[u].x);
            }
            const float shrink = M == up ? 1.0f : __builtin_amdgcn_exp2f(M - up);
            M = up;
            L *= shrink, o.x *= shrink, o.y *= shrink, o.z *= shrink, o.w *= shrink;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const bool none = st[u].y == 0.0f;
                const float f = none ? 0.0f : st[u].x == M ? 1.0f : __builtin_amdgcn_exp2f(st[u].x - M);
                if (none) x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                L = fmaf(f, st[u].y, L);
                o.x = fmaf(f, x[u].x, o.x), o.y = fmaf(f, x[u].y, o.y), o.z = fmaf(f, x[u].z, o.z), o.w = fmaf(f, x[u].w, o.w);
            }
        }
    }
    if (halves > 1) {
        if (d == 0) stat[half][0] = M, stat[half][1] = L;
        part[half][threadIdx.x & 31] = o;
        __syncthreads();
        if (turn != 0 || query >= in0 + queries) return;
        M = stat[half][0];
        for (int h = 1; h < halves; h++) M = fmaxf(M, stat[half + h][0]);
        L = 0.0f, o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int h = 0; h < halves; h++) {
            const float sum = stat[half + h][1], f = sum == 0.0f ? 0.0f : stat[half + h][0] == M ? 1.0f : __builtin_amdgcn_exp2f(stat[half + h][0] - M);
            const float4 x = part[half + h][threadIdx.x & 31];
            L = fmaf(f, sum, L);
            o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
        }
    }
    const int in = tile * a.tile + query;
    if (query < in0 + queries) q4_leave(a, b, hk, in, d, o, L, !(L < 0.0f));
}

struct Q4Plan {
    bool many;
    int rt, tile, tiles, groups, turns, join;
};
static Q4Plan plan_q4(int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t maxlen) {
    Q4Plan p{};
    const int64_t Mq = qL * (H / Hkv);
    // (us with few and with many: 16 sequences of 20 queries to a kv head 59 and 66, of 30 62 and 72; 2 of 20 28 and 32.  Above 32 queries the few would read rows twice)
    p.many = Mq > 32;
    p.rt = !p.many && Mq > 16 ? 2 : 1;  // (of the few)
    p.tile = p.many ? 64 : 16 * p.rt;
    p.tiles = (int)((Mq + p.tile - 1) / p.tile);
    const int64_t items = B * Hkv * p.tiles;
    // One launch where a workgroup can have all rows of a kv head in the time of the two others' launches, or the chip is busy with one to each anyway;
    // not where so many queries and new rows wait for memory at once (us with three launches and with one: 2 sequences of 32 kv heads and 300 rows 14.8 and 9.8,
    // 1000 rows 16.5 and 14.3; 2 of 8 kv heads and 1500 rows 14.9 and 16.5; 16 of 32 and 500 rows 22.6 and 14.7, 1500 rows 30.5 and 24.4;
    // 16 of 32 and 1 token, up to 2200 rows, 36.0 and 31.6, 5 tokens 37.8 and 33.2; 24 of 32 and 2200 rows 45.1 and 45.6; 40 of 8 and 2200 rows 32.3 and 33.6, 100 of 8 52.2 and 58.5;
    // 32 of 32 and 1500 rows 44.4 and 44.3; 64 of 32 and 300 rows 35.1 and 39.1).  Above 2048 rows some numbers of sequences gain and others lose: those stay with three.
    // With more than 16 queries to a kv head a workgroup takes longer for its rows, and two fit a compute unit: (4 of 32 kv heads and 20 tokens, 300 rows 20.5 and 17.0, 700
    // rows 24.4 and 22.9; 2 of 32 and 30 tokens, 1000 rows 23.6 and 27.1, 1 and 32 tokens, 100 rows 15.0 and 17.6; 1 of 8 and 8 tokens of 4 heads each, 400 rows 16.3 and 14.1, 1000
    // 16.5 and 17.6; 40 of 8 and 8 tokens, 900 rows 34.3 and 30.7, 1500 37.5 and 41.0; 10 of 32 and 20 tokens, 900 rows 33.9 and 27.4; 20 of 32, 2000 rows 71.9 and 60.5)
    // (there by tokens, not queries: new rows and angles are by token, and a workgroup has those of its kv head all to itself)
    const int one_launch = p.rt == 1 ? (items >= 256 ? 16 : 8) : items >= 512 ? 16 : items >= 256 ? 8 : qL <= 24 ? 4 : 0;  // units
    if (!p.many && items <= 1024 && maxlen <= one_launch * kUnit) {
        p.groups = (int)items;
        return p;
    }
    const int64_t most = items * ((maxlen + kUnit - 1) / kUnit + kStart), held = p.many || p.rt == 2 ? 512 : 1024;  // (workgroups that the chip holds)
    p.groups = (int)(most < held ? most : held);
    p.turns = most < held ? 1 : (int)(held / 256);
    const int64_t queries = B * Hkv * Mq;  // (workgroups enough to fill the chip, then queries to each)
    p.join = queries >= 8192 ? 8 : queries >= 4096 ? 4 : queries >= 2048 ? 2 : 1;
    return p;
}
struct Q4Layout {
    size_t qh, ql, cq, parts, stat, rec, total;
};
static Q4Layout layout_q4(const Q4Plan& plan, int64_t rows, int64_t items) {
    Q4Layout w{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t records = plan.join > 0 ? (size_t)plan.groups * 2 * plan.tile : 0, held = plan.join > 0 ? rows : 0;
    w.qh = take(held * kS * 2);
    w.ql = take(held * kS * 2);
    w.cq = take(held * 4);
    w.parts = take(plan.join > 0 ? items * 8 : 0);
    w.stat = take(records * 8);
    w.rec = take(records * kS * 4);
    w.total = at > 0 ? at : 256;  // (0 stands for sizes that are refused)
    return w;
}

static int q4_launch(const Q4Args& a, const Q4Plan& plan, hipStream_t st) {
    const unsigned prep = (unsigned)((int64_t)a.B * a.qL * a.row_groups);
    if (plan.join > 0) q4_prep_kernel<<<prep, 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    const unsigned groups = (unsigned)plan.groups;
    if (plan.many) q4_many_kernel<<<groups, 256, 0, st>>>(a);
    else if (plan.join == 0 && plan.rt == 2) q4_few_kernel<2, true><<<groups, 256, 0, st>>>(a);
    else if (plan.join == 0) q4_few_kernel<1, true><<<groups, 256, 0, st>>>(a);
    else if (plan.rt == 2) q4_few_kernel<2, false><<<groups, 256, 0, st>>>(a);
    else q4_few_kernel<1, false><<<groups, 256, 0, st>>>(a);
    LLMOPS_LAUNCH_CHECK();
    if (plan.join > 0) {
        const int64_t parts = ((plan.tile < a.Mq ? plan.tile : a.Mq) + plan.join - 1) / plan.join;
        q4_join_kernel<<<(unsigned)((int64_t)a.B * a.Hkv * plan.tiles * parts), 256, 0, st>>>(a);
    }
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}

}  // namespace llmops

using namespace llmops;

static bool q4_sizes_fit(int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t maxlen) {
    const int64_t most = (int64_t)1 << 24;  // (a launch has fewer than 2^32 threads)
    if (!(B > 0 && qL > 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && maxlen > 0 && B < most && qL < most && H < most && maxlen <= most && B * qL < most && B * qL * H < most)) return false;
    // (units are numbered in 32 bits; of fewer than 64 queries there is one tile)
    const int64_t tiles = (qL * (H / Hkv) + 63) / 64, units = (maxlen + kUnit - 1) / kUnit + kStart;
    return (Wide)B * Hkv * tiles * units < ((Wide)1 << 31);
}

extern "C" size_t llmops_attention_q4_workspace_bytes(int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t S, int64_t maxlen) {
    if (S != kS || !q4_sizes_fit(B, qL, H, Hkv, maxlen)) return 0;
    const Q4Plan plan = plan_q4(B, qL, H, Hkv, maxlen);
    return layout_q4(plan, B * qL * H, B * Hkv * plan.tiles).total;
}

extern "C" int llmops_attention_rope_q4(const float* q, int64_t q_stride_b, int64_t q_stride_l, const float* k, int64_t k_stride_b, int64_t k_stride_l,
                                        const float* v, int64_t v_stride_b, int64_t v_stride_l, int64_t B, int64_t qL, int64_t H, int64_t Hkv, int64_t S,
                                        const float* inv_freq, int64_t half, void* kv_cache, int64_t planes, int64_t maxlen, const int32_t* lengths,
                                        const int32_t* q_lens, int layer_id, float* out, void* workspace, size_t workspace_bytes, llmops_stream_t stream) {
    LLMOPS_REQUIRE(q != nullptr && k != nullptr && v != nullptr && inv_freq != nullptr && kv_cache != nullptr && lengths != nullptr);
    LLMOPS_REQUIRE(out != nullptr && workspace != nullptr);
    LLMOPS_REQUIRE(S == 128);  // head size of every supported model shape
    LLMOPS_REQUIRE(q4_sizes_fit(B, qL, H, Hkv, maxlen));
    LLMOPS_REQUIRE(half > 0 && 2 * half <= S);
    LLMOPS_REQUIRE(layer_id >= 0 && 2 * (int64_t)layer_id + 1 < planes);
    LLMOPS_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(kv_cache, 16) && aligned(workspace, 256));
    LLMOPS_REQUIRE(aligned(inv_freq, 4) && aligned(lengths, 4) && aligned(q_lens, 4));
    LLMOPS_REQUIRE(q_stride_b % 4 == 0 && q_stride_l % 4 == 0 && k_stride_b % 4 == 0 && k_stride_l % 4 == 0 && v_stride_b % 4 == 0 && v_stride_l % 4 == 0);
    const int64_t G = H / Hkv;
    LLMOPS_REQUIRE((Wide)B * qL * ((H + 2 * Hkv + 15) / 16) < ((Wide)1 << 24));
    const Wide heads = (Wide)H * kS * 4, kv_heads = (Wide)Hkv * kS * 4, plane = (Wide)B * Hkv * maxlen * kQ4Row;
    LLMOPS_REQUIRE((Wide)planes * plane < ((Wide)1 << 62));
    const Q4Plan plan = plan_q4(B, qL, H, Hkv, maxlen);
    const Q4Layout w = layout_q4(plan, B * qL * H, B * Hkv * plan.tiles);
    if (workspace_bytes < w.total) return fail(LLMOPS_EWORKSPACE, "attention_rope_q4 needs %zu workspace bytes, got %zu", w.total, workspace_bytes);
    char* ws = reinterpret_cast<char*>(workspace);
    Q4Args a{};
    a.q = q, a.k = k, a.v = v, a.inv_freq = inv_freq;
    a.qsb = q_stride_b, a.qsl = q_stride_l, a.ksb = k_stride_b, a.ksl = k_stride_l, a.vsb = v_stride_b, a.vsl = v_stride_l;
    a.qh = reinterpret_cast<_Float16*>(ws + w.qh), a.ql = reinterpret_cast<_Float16*>(ws + w.ql), a.cq = reinterpret_cast<float*>(ws + w.cq);
    a.rec_out = reinterpret_cast<float*>(ws + w.rec), a.rec_stat = reinterpret_cast<float2*>(ws + w.stat), a.parts = reinterpret_cast<int2*>(ws + w.parts);
    a.ck = reinterpret_cast<uint8_t*>(kv_cache) + 2 * layer_id * (int64_t)plane, a.cv = a.ck + (int64_t)plane;
    a.lengths = lengths, a.q_lens = q_lens, a.out = out, a.maxlen = maxlen;
    a.B = (int)B, a.qL = (int)qL, a.G = (int)G, a.Hkv = (int)Hkv, a.Mq = (int)(qL * G), a.M = (int)(B * qL * G), a.half = (int)half, a.row_groups = (int)((H + 2 * Hkv + 15) / 16);
    a.tile = plan.tile, a.tiles = plan.tiles, a.groups = plan.groups, a.turns = plan.turns, a.join = plan.join;
    // (a workgroup reads its q, k and v while others may have written their rows and results)
    const Extent q_at(q, B, (Wide)q_stride_b * 4, qL, (Wide)q_stride_l * 4, heads), k_at(k, B, (Wide)k_stride_b * 4, qL, (Wide)k_stride_l * 4, kv_heads),
        v_at(v, B, (Wide)v_stride_b * 4, qL, (Wide)v_stride_l * 4, kv_heads), out_at(out, (Wide)B * qL * heads), written(a.ck, 2 * plane);
    LLMOPS_REQUIRE(apart(written, q_at) && apart(written, k_at) && apart(written, v_at));
    LLMOPS_REQUIRE(apart(out_at, q_at) && apart(out_at, k_at) && apart(out_at, v_at) && apart(out_at, written));
    const Extent lengths_at(lengths, (Wide)B * 4), q_lens_at(q_lens, q_lens != nullptr ? (Wide)B * 4 : 0), inv_freq_at(inv_freq, (Wide)half * 4);
    LLMOPS_REQUIRE(apart(written, lengths_at) && apart(written, q_lens_at) && apart(written, inv_freq_at));
    LLMOPS_REQUIRE(apart(out_at, lengths_at) && apart(out_at, q_lens_at) && apart(out_at, inv_freq_at));
    hipStream_t st = as_stream(stream);
    return q4_launch(a, plan, st);
}
