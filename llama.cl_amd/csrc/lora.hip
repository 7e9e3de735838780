// Low-rank adapters of several requests beside a shared projection: out = y + scale[a] * (x A_a^T) B_a^T, the adapter a chosen by
// sequence (none: out = y).  (The reference has no adapters; the projection is fc_Q4A, whose output y is.)
//
//   1. lora_down_kernel  t = x A^T, K cut into runs: partial sums, fp32
//   2. lora_up_kernel    sums t in the runs' order, t B^T, scale, add
//
// Sixteen tokens to a tile, in the order they come, whatever their adapters: a wave goes through the adapters that occur among its
// tokens and takes over results only for the tokens of the one at hand, so that a weight that is no number stays with its own
// requests.  One adapter in a tile is read once for all; sixteen are read once each, which they must be anyway.
//
// Products run on the bf16 matrix cores (v_mfma_f32_16x16x32_bf16, fp32 sums) on exact pieces: an fp32 value is three bf16 values
// (8 bits each, cut off), an fp16 weight two, a bf16 weight itself.  Products of pieces whose places (0 to 2) sum to two or less are
// formed.  A piece is below 2^-7 of the one before it, the third below 2^-15 of the first: what is dropped is below 2 * 2^-22 of a product with
// fp32 weights, 2^-22 with fp16, nothing with bf16.
#include <algorithm>

#include "common.h"
#include "extents.h"

namespace llmops {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct LoraArgs {
    const float *x, *y, *scales;
    const void *A, *B;   // [adapters][R][K], [adapters][N][R]
    const int32_t* ids;  // [batch]
    float *out, *part;   // part [splits][rows][rank_stride(R)]
    int64_t xsb, xsl, ysb, ysl, osb, osl;
    int rows, tokens, K, N, R, adapters, splits, chunk;
    int share;  // workgroups among which the adapters of a tile are dealt out, by number
    int tiles;  // of a sequence; 0: tiles go on over the sequences' ends
};

// A row of partial sums takes up whole fours
__host__ __device__ __forceinline__ int rank_stride(int R) { return (R + 3) & ~3; }
struct __attribute__((packed, aligned(4))) Four32 {
    float x[4];
};

// The tokens of a tile: numbers first .. end - 1.  Sequences of a tile's tokens or more have tiles of their own, so that a tile has one
// adapter; of shorter ones several share a tile
struct Tile {
    int first, end;
    __device__ __forceinline__ Tile(const LoraArgs& a, int tile, int size) {
        if (a.tiles > 0) {
            const int b = tile / a.tiles;
            first = b * a.tokens + (tile - b * a.tiles) * size;
            end = min(first + size, (b + 1) * a.tokens);
        } else {
            first = tile * size;
            end = min(first + size, a.rows);
        }
    }
};

template <int N>
struct Pieces {
    v8bf p[N];
};
__device__ __forceinline__ v8bf as_v8bf(uint4 u) { return __builtin_bit_cast(v8bf, u); }
__device__ __forceinline__ uint32_t upper(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// eight fp32 values as N bf16 pieces each (an infinity leaves NaN behind it)
template <int N>
__device__ __forceinline__ Pieces<N> cut8(const float (&x)[8]) {
    Pieces<N> r;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e++) rest[e] = x[e];
#pragma unroll
    for (int n = 0; n < N; n++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = upper(__float_as_uint(rest[2 * e]), __float_as_uint(rest[2 * e + 1]));
#pragma unroll
        for (int e = 0; e < 8; e++) rest[e] -= __uint_as_float(__float_as_uint(rest[e]) & 0xffff0000u);
        r.p[n] = as_v8bf(make_uint4(w[0], w[1], w[2], w[3]));
    }
    return r;
}

// Eight neighbours of a row, wherever it starts (global loads need no alignment)
struct __attribute__((packed, aligned(4))) Eight32 {
    float x[8];
};
struct __attribute__((packed, aligned(2))) Eight16 {
    uint16_t x[8];
};
// The eight that a lane takes at the end of a row: where fewer are left, those that end with it, and the other operand's are zero where they
// are before `at` (another lane's, or nobody's)
__device__ __forceinline__ int eight_from(int at, int end) { return max(0, min(at, end - 8)); }

// a weight's type: eight of a row as they are in memory, and their pieces
struct Half16 {
    uint16_t u;
};
struct Bf16 {
    uint16_t u;
};
template <typename W>
struct Weight;
template <>
struct Weight<float> {
    typedef Eight32 Raw;
    typedef float Bits;
    static __device__ __forceinline__ Pieces<3> cut(const Raw& r) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = r.x[e];
        return cut8<3>(x);
    }
};
template <>
struct Weight<Half16> {
    typedef Eight16 Raw;
    typedef uint16_t Bits;
    static __device__ __forceinline__ Pieces<2> cut(const Raw& r) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = f16_bits_to_f32(r.x[e]);
        return cut8<2>(x);
    }
};
template <>
struct Weight<Bf16> {
    typedef Eight16 Raw;
    typedef uint16_t Bits;
    static __device__ __forceinline__ Pieces<1> cut(const Raw& r) { return {{__builtin_bit_cast(v8bf, r)}}; }
};
template <typename W>
__device__ __forceinline__ typename Weight<W>::Raw load8(const W* row, int at) {
    return *reinterpret_cast<const typename Weight<W>::Raw*>(row + at);
}
// the same at a row's end; SHORT: the whole row is fewer than eight
template <bool SHORT, typename W>
__device__ __forceinline__ typename Weight<W>::Raw load8_end(const W* row, int at, int end) {
    if constexpr (!SHORT) {
        return load8(row, eight_from(at, end));
    } else {
        typename Weight<W>::Raw r{};
        const auto* from = reinterpret_cast<const typename Weight<W>::Bits*>(row);
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < end) r.x[e] = from[e];
        return r;
    }
}
__device__ __forceinline__ Pieces<3> cut_end(const Eight32& r, int at, int end) {
    const int from = eight_from(at, end);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = from + e < at ? 0.0f : r.x[e];
    return cut8<3>(x);
}

template <int NW>
__device__ __forceinline__ v4f times(const Pieces<NW>& w, const Pieces<3>& x, v4f acc) {
#pragma unroll
    for (int n = 0; n < NW; n++)
#pragma unroll
        for (int m = 0; m < 3 && n + m < 3; m++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[n], x.p[m], acc, 0, 0, 0);
    return acc;
}
__device__ __forceinline__ v4f keep(bool match, v4f sum, v4f acc) {
#pragma unroll
    for (int v = 0; v < 4; v++) acc[v] = match ? sum[v] : acc[v];
    return acc;
}

constexpr int kDownWaves = 8;

// token `row`'s adapter, -1 for none
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int row, int end) {
    const int id = a.ids[min(row, end - 1) / a.tokens];
    return row < end && id >= 0 && id < a.adapters ? id : -1;
}
// The adapters that occur among a wave's tokens (token t's in lane t), each once, in the order of their first token
struct Adapters {
    int of_lane;
    uint64_t todo;
    __device__ __forceinline__ explicit Adapters(int ids) : of_lane(ids), todo(__ballot(ids >= 0)) {}
    __device__ __forceinline__ int next() {
        const int id = __builtin_amdgcn_readlane(of_lane, __builtin_ctzll(todo));
        todo &= ~__ballot(of_lane == id);
        return id;
    }
    // up to U of them; past the last, that one again.  Returns how many
    template <int U>
    __device__ __forceinline__ int next(int (&id)[U]) {
        int n = 1;
        id[0] = next();
#pragma unroll
        for (int u = 1; u < U; u++) {
            id[u] = id[u - 1];
            if (todo != 0) id[u] = next(), n = u + 1;
        }
        return n;
    }
};

// A workgroup: 16 * TT tokens (of several adapters: those whose number is its own among `share`), a run of K (its eight waves an eighth of
// every 256 each), 16 * NR rows of A.  Bound by latency with few tokens (1 x 4096, rank 8: 2.8 us) and by issuing instructions with many, those
// that cut x and A up most of all (4 x 300 x 11008, rank 64: 29 us, 1.9 TB/s); so the operands of two steps are asked for before those of the two before them are used, or those
// of four adapters at a time.
// A operand: row of A lane % 16, eight k; B operand: token lane % 16, the same k; result: token lane % 16, rows 4 * (lane / 16) + v.
template <typename W, int NR, int TT, bool SHORT>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(LoraArgs a) {
    constexpr int kStep = 32 * kDownWaves, U = 2, UA = sizeof(W) == 4 && NR * TT > 2 ? 2 : 4;
    typedef typename Weight<W>::Raw Raw;
    __shared__ v4f meet[kDownWaves][NR * TT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const Tile tile(a, blockIdx.x, 16 * TT);
    const int row0 = tile.first, r0 = blockIdx.z / a.share * 16 * NR, part = blockIdx.z % a.share;
    const int k0 = blockIdx.y * a.chunk, k1 = min(a.K, k0 + a.chunk);
    int of_lane = adapter_of(a, row0 + (lane & (16 * TT - 1)), tile.end);
    if (of_lane % a.share != part) of_lane = -1;
    const float* x[TT];
#pragma unroll
    for (int tt = 0; tt < TT; tt++) {
        const int row = min(row0 + 16 * tt + i, tile.end - 1), b = row / a.tokens;
        x[tt] = a.x + b * a.xsb + (row - b * a.tokens) * a.xsl;
    }
    const W* A[NR];  // rows of the adapter with number 0; past the last rank that rank again (not stored)
#pragma unroll
    for (int n = 0; n < NR; n++) A[n] = reinterpret_cast<const W*>(a.A) + (int64_t)min(r0 + 16 * n + i, a.R - 1) * a.K;
    const int64_t adapter = (int64_t)a.R * a.K;
    v4f acc[NR][TT];
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int tt = 0; tt < TT; tt++) acc[n][tt] = v4f{0.f, 0.f, 0.f, 0.f};
    Adapters all(lane < 16 * TT ? of_lane : -1);
    if (all.todo == 0) return;  // (nobody reads these sums)
    const int only = all.next();
    int k = k0 + 32 * wave;
    if (all.todo == 0) {
        const int64_t at = only * adapter;
        struct Stage {
            Raw w[U][NR];
            Eight32 x[U][TT];
        } s0, s1;
        auto ask = [&](Stage& s, int from) {
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int tt = 0; tt < TT; tt++) s.x[u][tt] = load8(x[tt], from + kStep * u + 8 * g);
#pragma unroll
                for (int n = 0; n < NR; n++) s.w[u][n] = load8(A[n] + at, from + kStep * u + 8 * g);
            }
        };
        auto use = [&](const Stage& s) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                Pieces<3> xp[TT];
#pragma unroll
                for (int tt = 0; tt < TT; tt++) xp[tt] = Weight<float>::cut(s.x[u][tt]);
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    const auto wp = Weight<W>::cut(s.w[u][n]);
#pragma unroll
                    for (int tt = 0; tt < TT; tt++) acc[n][tt] = times(wp, xp[tt], acc[n][tt]);
                }
            }
        };
        // (past the last stage that one is asked for again: a wave that may or may not have asked waits for everything)
        const int reach = kStep * (U - 1) + 32, stages = k1 - k >= reach ? (k1 - k - reach) / (kStep * U) + 1 : 0;
        const int last = k + (stages - 1) * kStep * U;
        if (stages > 0) {
            ask(s0, k);
            for (int n = 0; n < stages; n += 2) {
                ask(s1, min(k + kStep * U, last));
                use(s0);
                ask(s0, min(k + 2 * kStep * U, last));
                if (n + 1 < stages) use(s1);
                k += 2 * kStep * U;
            }
            k = last + kStep * U;
        }
        for (; k < k1; k += kStep) {
            Pieces<3> xp[TT];
#pragma unroll
            for (int tt = 0; tt < TT; tt++) xp[tt] = cut_end(load8_end<SHORT>(x[tt], k + 8 * g, k1), k + 8 * g, k1);
#pragma unroll
            for (int n = 0; n < NR; n++) {
                const auto wp = Weight<W>::cut(load8_end<SHORT>(A[n] + at, k + 8 * g, k1));
#pragma unroll
                for (int tt = 0; tt < TT; tt++) acc[n][tt] = times(wp, xp[tt], acc[n][tt]);
            }
        }
    } else {
        int mine[TT];
#pragma unroll
        for (int tt = 0; tt < TT; tt++) mine[tt] = __shfl(of_lane, 16 * tt + i, 64);
        Adapters some(lane < 16 * TT ? of_lane : -1);
        struct Stage {
            int k, n, id[UA];
            Raw w[UA][NR];
            Eight32 x[TT];
        } s0, s1;
        // the next adapters of this step, or the first of the next; past the last step its first again (not used)
        auto ask = [&](Stage& s) {
            if (some.todo == 0) some = Adapters(lane < 16 * TT ? of_lane : -1), k += kStep;
            s.n = some.next(s.id);
            s.k = k;
            const int at = (k < k1 ? k : k - kStep) + 8 * g;
#pragma unroll
            for (int tt = 0; tt < TT; tt++) s.x[tt] = load8_end<SHORT>(x[tt], at, k1);
#pragma unroll
            for (int u = 0; u < UA; u++)
#pragma unroll
                for (int n = 0; n < NR; n++) s.w[u][n] = load8_end<SHORT>(A[n] + s.id[u] * adapter, at, k1);
        };
        auto use = [&](const Stage& s) {
            Pieces<3> xp[TT];
#pragma unroll
            for (int tt = 0; tt < TT; tt++) xp[tt] = cut_end(s.x[tt], s.k + 8 * g, k1);
#pragma unroll
            for (int u = 0; u < UA; u++) {
                if (u >= s.n) break;
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    const auto wp = Weight<W>::cut(s.w[u][n]);
#pragma unroll
                    for (int tt = 0; tt < TT; tt++) acc[n][tt] = keep(mine[tt] == s.id[u], times(wp, xp[tt], acc[n][tt]), acc[n][tt]);
                }
            }
        };
        if (k < k1) {
            ask(s0);
            while (true) {
                ask(s1);
                use(s0);
                if (s1.k >= k1) break;
                ask(s0);
                use(s1);
                if (s0.k >= k1) break;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int tt = 0; tt < TT; tt++) meet[wave][n * TT + tt][lane] = acc[n][tt];
    __syncthreads();
    for (int m = wave; m < NR * TT; m += kDownWaves) {
        const int n = m / TT, row = row0 + 16 * (m - n * TT) + i, r = r0 + 16 * n + 4 * g;
        v4f s = meet[0][m][lane];
#pragma unroll
        for (int w = 1; w < kDownWaves; w++) s += meet[w][m][lane];
        const bool mine = __shfl(of_lane, row - row0, 64) >= 0;
        if (!mine) continue;
        const int stride = rank_stride(a.R);  // (behind the last rank stands that one again, which nobody takes)
        if (r < stride) *reinterpret_cast<Four32*>(a.part + ((int64_t)blockIdx.y * a.rows + row) * stride + r) = Four32{{s[0], s[1], s[2], s[3]}};
    }
}

// A workgroup: 16 * TT tokens (as above; those without an adapter with part 0), 64 * CT columns (16 * CT to a wave), ranks 128 at a time.  Bound by
// latency (one token, 4096 columns: 4.5 us; 4 x 300, rank 64: 25 us, 1.6 TB/s, 12 of it until the sums are there): what does not depend on
// anything (adapters, y, the first partial sums) is asked for at once, and the first weights before the sums are used.
// A operand: column lane % 16 of B, eight ranks; B operand: token lane % 16, the same ranks; result: token lane % 16, columns 4 * (lane / 16) + v.
template <typename W, int CT, int TT, bool SHORT>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a, bool vec_out) {
    constexpr int kRanks = 128, kStride = kRanks + 4, U = CT == 1 ? 4 : 1;
    typedef typename Weight<W>::Raw Raw;
    __shared__ __align__(16) float t[16 * TT][kStride];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const Tile tile(a, blockIdx.y, 16 * TT);
    const int row0 = tile.first, n0 = (blockIdx.x * 4 + wave) * 16 * CT;
    int of_lane = adapter_of(a, row0 + (lane & (16 * TT - 1)), tile.end);
    const uint64_t here = __ballot((of_lane < 0 ? 0 : of_lane % a.share) == (int)blockIdx.z);  // its tokens, and part 0 those without an adapter
    if (!(here >> lane & 1)) of_lane = -1;
    const float* y[TT];
    float* out[TT];
    float4 yv[CT][TT];
#pragma unroll
    for (int tt = 0; tt < TT; tt++) {
        const int row = min(row0 + 16 * tt + i, tile.end - 1), b = row / a.tokens, l = row - b * a.tokens;
        y[tt] = a.y + b * a.ysb + l * a.ysl;
        out[tt] = a.out + b * a.osb + l * a.osl;
    }
    if (vec_out) {  // (a lane past the last column reads the last four again, and stores nothing)
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int c = 0; c < CT; c++) yv[c][tt] = *reinterpret_cast<const float4*>(y[tt] + min(n0 + 16 * c + 4 * g, a.N - 4));
    } else {
#pragma unroll
        for (int tt = 0; tt < TT; tt++)
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int v = 0; v < 4; v++) reinterpret_cast<float*>(&yv[c][tt])[v] = y[tt][min(n0 + 16 * c + 4 * g + v, a.N - 1)];
    }
    const W* B[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) B[c] = reinterpret_cast<const W*>(a.B) + (int64_t)min(n0 + 16 * c + i, a.N - 1) * a.R;
    const int64_t adapter = (int64_t)a.N * a.R;
    v4f acc[CT][TT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int tt = 0; tt < TT; tt++) acc[c][tt] = v4f{0.f, 0.f, 0.f, 0.f};
    const bool any = __ballot(lane < 16 * TT && of_lane >= 0) != 0;  // (the same in the four waves)
    int mine[TT];
#pragma unroll
    for (int tt = 0; tt < TT; tt++) mine[tt] = __shfl(of_lane, 16 * tt + i, 64);
    for (int r0 = 0; r0 < a.R && any; r0 += kRanks) {
        const int ranks = min(kRanks, a.R - r0), padded = (ranks + 31) & ~31;
        if (r0 > 0) __syncthreads();
        // (four neighbours and eight runs at a time, all on their way together; value by value they were two thirds of a prompt's launch)
        const int fours = padded / 4;
        for (int e = threadIdx.x; e < 16 * TT * fours; e += 256) {
            const int token = e / fours, r = 4 * (e - token * fours), stride = rank_stride(a.R);
            const bool there = r < ranks && row0 + token < tile.end;
            const float* from = a.part + (there ? (int64_t)(row0 + token) * stride + r0 + r : 0);
            const int64_t run = (int64_t)a.rows * stride;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < a.splits; c += 8) {
                Four32 x[8];
#pragma unroll
                for (int u = 0; u < 8; u++) x[u] = *reinterpret_cast<const Four32*>(from + min(c + u, a.splits - 1) * run);
#pragma unroll
                for (int u = 0; u < 8; u++)
#pragma unroll
                    for (int v = 0; v < 4; v++) sum[v] += c + u < a.splits ? x[u].x[v] : 0.0f;
            }
#pragma unroll
            for (int v = 0; v < 4; v++) sum[v] = there && r + v < ranks ? sum[v] : 0.0f;
            *reinterpret_cast<float4*>(&t[token][r]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
        }
        Adapters some(lane < 16 * TT ? of_lane : -1);
        struct Stage {
            int step, n, id[U];
            Raw w[U][CT];
        } s0, s1;
        int step = 0;
        auto ask = [&](Stage& s) {  // as above
            if (some.todo == 0) some = Adapters(lane < 16 * TT ? of_lane : -1), step += 32;
            s.n = some.next(s.id);
            s.step = step;
            const int at = r0 + (step < padded ? step : step - 32) + 8 * g;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int c = 0; c < CT; c++) s.w[u][c] = load8_end<SHORT>(B[c] + s.id[u] * adapter, at, a.R);
        };
        int cut = -1;
        Pieces<3> tp[TT];
        auto use = [&](const Stage& s) {
            if (s.step != cut) {
                cut = s.step;
#pragma unroll
                for (int tt = 0; tt < TT; tt++) {
                    // (t holds zeros behind the last rank, so that the operand may start anywhere)
                    float x[8];
                    const int at = r0 + s.step + 8 * g, from = eight_from(at, a.R) - r0;
                    if (a.R % 8 == 0) {
                        const float* here = &t[16 * tt + i][s.step + 8 * g];
                        const float4 lo = *reinterpret_cast<const float4*>(here), hi = *reinterpret_cast<const float4*>(here + 4);
                        x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = r0 + from + e < at || from + e < 0 ? 0.0f : t[16 * tt + i][max(from + e, 0)];
                    }
                    tp[tt] = cut8<3>(x);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (u >= s.n) break;
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    const auto wp = Weight<W>::cut(s.w[u][c]);
#pragma unroll
                    for (int tt = 0; tt < TT; tt++) acc[c][tt] = keep(mine[tt] == s.id[u], times(wp, tp[tt], acc[c][tt]), acc[c][tt]);
                }
            }
        };
        ask(s0);
        __syncthreads();
        while (true) {
            ask(s1);
            use(s0);
            if (s1.step >= padded) break;
            ask(s0);
            use(s1);
            if (s0.step >= padded) break;
        }
    }
#pragma unroll
    for (int tt = 0; tt < TT; tt++) {
        if (row0 + 16 * tt + i >= tile.end || !(here >> (16 * tt + i) & 1)) continue;
        const float scale = mine[tt] >= 0 ? a.scales[mine[tt]] : 0.0f;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const int col = n0 + 16 * c + 4 * g;
            float4 u = yv[c][tt];
            if (mine[tt] >= 0)
                u = make_float4(fmaf(scale, acc[c][tt][0], u.x), fmaf(scale, acc[c][tt][1], u.y), fmaf(scale, acc[c][tt][2], u.z), fmaf(scale, acc[c][tt][3], u.w));
            if (vec_out) {
                if (col < a.N) *reinterpret_cast<float4*>(out[tt] + col) = u;
            } else {
                const float* from = reinterpret_cast<const float*>(&u);
#pragma unroll
                for (int v = 0; v < 4; v++)
                    if (col + v < a.N) out[tt][col + v] = from[v];
            }
        }
    }
}

// Tokens to a tile: 32 where there are enough of them to fill the chip so.  (us a call, 16 / 32, fp16 and then fp32 weights: 320 tokens 15.4 / 19.2, 22.0 / 21.0;
// 384 16.0 / 15.6, 20.3 / 16.2; 512 of rank 64 31 / 23, 42 / 24.)
static int lora_tile(int64_t rows) { return rows > 320 ? 32 : 16; }
static int64_t lora_tiles(int64_t batch, int64_t tokens) {
    const int64_t tile = lora_tile(batch * tokens);
    return tokens >= tile ? batch * ((tokens + tile - 1) / tile) : (batch * tokens + tile - 1) / tile;
}
// K in runs of whole steps, until there are some 256 workgroups.  (128 / 256 / 512 of them: 4 x 300 tokens, 11008 -> 4096, rank 64 58 / 52 / 56; runs of at
// least 256 / 1024, 4 x 16 tokens, 4096 -> 4096, rank 16 7.8 / 10.5: a step waits once, however few there are.)
static int lora_chunk(int64_t batch, int64_t tokens, int64_t K, int64_t R) {
    const int64_t groups = lora_tiles(batch, tokens) * ((R + 63) / 64), step = 32 * kDownWaves, n = step * ((256 + groups - 1) / groups);
    return (int)((K + n - 1) / n * step);
}

template <typename W>
static int lora_launch(LoraArgs a, bool vec_out, hipStream_t st) {
    const int tile = lora_tile(a.rows), tt = tile / 16, nr = a.R <= 16 ? 1 : a.R <= 32 ? 2 : 4;
    const unsigned tiles = (unsigned)lora_tiles(a.rows / a.tokens, a.tokens);
    a.tiles = a.tokens >= tile ? (a.tokens + tile - 1) / tile : 0;
    // Tiles with several adapters: dealt out while there are fewer than 256 workgroups.  (us a call, the first launch with 1 / 2 / 4 / 8 for each, fp16: 32
    // tokens, 20 adapters 4096 -> 11008, rank 16 16.4 / 14.9 / 14.0 / 13.6; 3 tokens, 3 adapters 4096 -> 4096 8.8 / 7.4; 32 x 5 tokens, which have 160 workgroups,
    // 12.4 / 14.9 / 13.7 / 13.1.  The second, until there are 128 / 256 / 1024: 32 tokens, 32 adapters 4096 -> 4096 11.7 / 10.9 / 12.0.)
    auto shares = [&](int64_t groups) { return a.tokens < tile && a.rows > a.tokens ? std::max(1, std::min(a.adapters, (int)(256 / groups))) : 1; };
    const unsigned nz = (unsigned)((a.R + 16 * nr - 1) / (16 * nr));
    a.share = shares((int64_t)tiles * a.splits * nz);
    const dim3 down(tiles, (unsigned)a.splits, nz * (unsigned)a.share);
#define LLMOPS_DOWN(NR, TT) lora_down_kernel<W, NR, TT, false><<<down, 64 * kDownWaves, 0, st>>>(a)
    const dim3 narrow(tiles, 1, (unsigned)((a.R + 15) / 16) * (unsigned)a.share);
    if (a.K < 8 && tt == 1) lora_down_kernel<W, 1, 1, true><<<narrow, 64 * kDownWaves, 0, st>>>(a);
    else if (a.K < 8) lora_down_kernel<W, 1, 2, true><<<narrow, 64 * kDownWaves, 0, st>>>(a);
    else if (tt == 1 && nr == 1) LLMOPS_DOWN(1, 1);
    else if (tt == 1 && nr == 2) LLMOPS_DOWN(2, 1);
    else if (tt == 1) LLMOPS_DOWN(4, 1);
    else if (nr == 1) LLMOPS_DOWN(1, 2);
    else if (nr == 2) LLMOPS_DOWN(2, 2);
    else LLMOPS_DOWN(4, 2);
#undef LLMOPS_DOWN
    LLMOPS_LAUNCH_CHECK();
    // few tokens: 64 columns to a workgroup, so that there are enough of them, and the weights of eight adapters on their way; many: 256, so that a
    // token's sums are read by fewer
    const int ct = tt == 1 ? 1 : 4;
    const unsigned columns = (unsigned)((a.N + 64 * ct - 1) / (64 * ct));
    a.share = shares((int64_t)columns * tiles);
    const dim3 up(columns, tiles, (unsigned)a.share);
    if (tt == 1 && a.R < 8) lora_up_kernel<W, 1, 1, true><<<up, 256, 0, st>>>(a, vec_out);
    else if (tt == 1) lora_up_kernel<W, 1, 1, false><<<up, 256, 0, st>>>(a, vec_out);
    else if (a.R < 8) lora_up_kernel<W, 4, 2, true><<<up, 256, 0, st>>>(a, vec_out);
    else lora_up_kernel<W, 4, 2, false><<<up, 256, 0, st>>>(a, vec_out);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}

}  // namespace llmops

using namespace llmops;

static bool lora_sizes_fit(int64_t batch, int64_t tokens, int64_t N, int64_t K, int64_t R) {
    const int64_t most = (int64_t)1 << 29;  // (a launch has fewer than 2^32 threads, four to a column; K + what a step reaches fits 31 bits)
    return batch > 0 && tokens > 0 && N > 0 && K > 0 && R > 0 && batch < most && tokens < most && N < most && K < most && R <= 4096 &&
           batch * tokens <= ((int64_t)1 << 20) && lora_tiles(batch, tokens) <= 65535;
}

extern "C" size_t llmops_lora_workspace_bytes(int64_t batch, int64_t tokens, int64_t N, int64_t K, int64_t R, int64_t adapters) {
    if (!lora_sizes_fit(batch, tokens, N, K, R) || adapters <= 0) return 0;
    const int64_t chunk = lora_chunk(batch, tokens, K, R);
    return (size_t)((K + chunk - 1) / chunk) * (size_t)(batch * tokens) * (size_t)rank_stride((int)R) * sizeof(float);
}

extern "C" int llmops_lora_add(const float* y, int64_t y_stride_b, int64_t y_stride_l, const float* x, int64_t x_stride_b, int64_t x_stride_l, int64_t batch,
                               int64_t tokens, int64_t N, int64_t K, const void* lora_A, const void* lora_B, int weight_dtype, int64_t R, int64_t adapters,
                               const int32_t* ids, const float* scales, float* out, int64_t out_stride_b, int64_t out_stride_l, void* workspace,
                               size_t workspace_bytes, llmops_stream_t stream) {
    LLMOPS_REQUIRE(y != nullptr && x != nullptr && lora_A != nullptr && lora_B != nullptr && ids != nullptr && scales != nullptr && out != nullptr);
    LLMOPS_REQUIRE(lora_sizes_fit(batch, tokens, N, K, R));
    LLMOPS_REQUIRE(adapters > 0 && adapters < ((int64_t)1 << 31));
    LLMOPS_REQUIRE(weight_dtype == LLMOPS_F32 || weight_dtype == LLMOPS_F16 || weight_dtype == LLMOPS_BF16);
    const size_t e = weight_dtype == LLMOPS_F32 ? 4 : 2;
    LLMOPS_REQUIRE(aligned(y, 4) && aligned(x, 4) && aligned(out, 4) && aligned(lora_A, e) && aligned(lora_B, e));
    const size_t need = llmops_lora_workspace_bytes(batch, tokens, N, K, R, adapters);
    if (workspace == nullptr || workspace_bytes < need)
        return fail(LLMOPS_EWORKSPACE, "lora_add needs %zu workspace bytes, got %zu", need, workspace == nullptr ? (size_t)0 : workspace_bytes);
    LLMOPS_REQUIRE(aligned(workspace, 4));
    // (a workgroup reads its x and y while others may have written their out)
    const Extent out_rows(out, batch, (Wide)out_stride_b * 4, tokens, (Wide)out_stride_l * 4, (Wide)N * 4),
        y_rows(y, batch, (Wide)y_stride_b * 4, tokens, (Wide)y_stride_l * 4, (Wide)N * 4), x_rows(x, batch, (Wide)x_stride_b * 4, tokens, (Wide)x_stride_l * 4, (Wide)K * 4);
    const bool in_place = out == y && (batch == 1 || out_stride_b == y_stride_b) && (tokens == 1 || out_stride_l == y_stride_l);
    LLMOPS_REQUIRE(rows_apart(out_rows));
    LLMOPS_REQUIRE(apart(out_rows, x_rows));
    LLMOPS_REQUIRE(in_place || apart(out_rows, y_rows));
    LoraArgs a{};
    a.x = x, a.y = y, a.scales = scales, a.A = lora_A, a.B = lora_B, a.ids = ids, a.out = out, a.part = reinterpret_cast<float*>(workspace);
    a.xsb = x_stride_b, a.xsl = x_stride_l, a.ysb = y_stride_b, a.ysl = y_stride_l, a.osb = out_stride_b, a.osl = out_stride_l;
    a.rows = (int)(batch * tokens), a.tokens = (int)tokens, a.K = (int)K, a.N = (int)N, a.R = (int)R, a.adapters = (int)adapters;
    a.chunk = lora_chunk(batch, tokens, K, R);
    a.splits = (int)((K + a.chunk - 1) / a.chunk);
    const bool vec_out = N % 4 == 0 && aligned(y, 16) && aligned(out, 16) && y_stride_b % 4 == 0 && y_stride_l % 4 == 0 && out_stride_b % 4 == 0 && out_stride_l % 4 == 0;
    hipStream_t st = as_stream(stream);
    if (weight_dtype == LLMOPS_F32) return lora_launch<float>(a, vec_out, st);
    if (weight_dtype == LLMOPS_F16) return lora_launch<Half16>(a, vec_out, st);
    return lora_launch<Bf16>(a, vec_out, st);
}
