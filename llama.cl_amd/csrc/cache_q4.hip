// A key/value cache in 4 bits as it is written and as it is read back (its rows: cache_q4_device.h; the attention that reads it: attn_q4.hip).
#include "cache_q4_device.h"
#include "extents.h"

namespace llmops {

struct WriteArgs {
    const void *k, *v;
    const float* inv_freq;
    int64_t ksb, ksl, ksh, vsb, vsl, vsh;  // elements
    uint8_t *ck, *cv;                      // planes [B][Hkv][maxlen][80]
    const int32_t *lengths, *q_lens;
    int64_t maxlen;
    int B, qL, Hkv, half, groups, shared;  // shared: every sequence is given the same rows
};

// A workgroup per token and 16 of its 2*Hkv rows, sixteen lanes to a row.  k is rotated, and its codes chosen, in 64 bits.
// Latency: one token 3.0 us, 5 times 77 tokens of 8 heads 4.2 (3.2 MB in, 0.5 out; 64-bit instructions are some 2 us of that on the waves that turn k).
template <typename T>
__global__ __launch_bounds__(256) void q4_write_turned_kernel(WriteArgs a) {
    __shared__ double2 turn[64];
    const int bl = blockIdx.x / a.groups, group = blockIdx.x - bl * a.groups, b = bl / a.qL, l = bl - b * a.qL;
    const int row = group * 16 + (threadIdx.x >> 4), j = threadIdx.x & 15;
    int len, n;
    own_extent(a.lengths, a.q_lens, b, a.qL, a.maxlen, len, n);
    if (l >= n) return;
    if ((int)threadIdx.x < a.half) turn[threadIdx.x] = turn64(a.inv_freq[threadIdx.x], len + l);
    __syncthreads();
    if (row >= 2 * a.Hkv) return;
    const bool is_k = row < a.Hkv;
    const int hk = is_k ? row : row - a.Hkv;
    const T* src = is_k ? (const T*)a.k + b * a.ksb + l * a.ksl + hk * a.ksh : (const T*)a.v + b * a.vsb + l * a.vsl + hk * a.vsh;
    uint8_t* dst = (is_k ? a.ck : a.cv) + (((int64_t)b * a.Hkv + hk) * a.maxlen + len + l) * kQ4Row;
    if (is_k) {
        RowPair p;
        p.load(src, j);
        double x[8];
        turn_row(p, src, j, turn, a.half, x);
        store_q4(dst, quantise8(x), j);
    } else {
        float x[8];
        load8(src + 8 * j, x);
        store_q4(dst, quantise8(x), j);
    }
}

// Rows that need no turning, in fp32: a workgroup per 16 tokens and one of the 2*Hkv rows of each.  Rows that all sequences are given (a system
// prompt) are quantised once.  The rows meet in LDS and are stored 16 bytes at a time, 1280 bytes on end: word by word, as the lanes have them, 2048 rows of 32
// heads for eight sequences took 42 us, of which the stores' partial lines were most; now 34.6: 34 MB in and 84 out, 3.4 TB/s, a chain of row, LDS and stores in each
// of four rounds of workgroups.  (Stores past the caches: 33, but reading the rows back then takes 65 instead of 60.)
template <typename T>
__global__ __launch_bounds__(256) void q4_write_kernel(WriteArgs a) {
    __shared__ uint4 rows[16 * kQ4Row / 16];
    const int tiles = (a.qL + 15) / 16, plane_row = blockIdx.x % (2 * a.Hkv), rest = blockIdx.x / (2 * a.Hkv), tile = rest % tiles, b0 = rest / tiles;
    const bool is_k = plane_row < a.Hkv;
    const int hk = is_k ? plane_row : plane_row - a.Hkv, row = threadIdx.x >> 4, j = threadIdx.x & 15, from = min(tile * 16 + row, a.qL - 1);
    const T* src = is_k ? (const T*)a.k + b0 * a.ksb + from * a.ksl + hk * a.ksh : (const T*)a.v + b0 * a.vsb + from * a.vsl + hk * a.vsh;
    float x[8];
    load8(src + 8 * j, x);
    // (three sequences at a time, 80 lanes to each; their extents asked for with the rows)
    const int piece = threadIdx.x % 80, l = tile * 16 + piece / 5, b_end = a.shared ? a.B : b0 + 1;
    int b = b0 + (int)threadIdx.x / 80, len[4], n[4];
    auto extents = [&] {
#pragma unroll
        for (int u = 0; u < 4; u++) own_extent(a.lengths, a.q_lens, min(b + 3 * u, a.B - 1), a.qL, a.maxlen, len[u], n[u]);
    };
    extents();
    store_q4(reinterpret_cast<uint8_t*>(rows) + row * kQ4Row, quantise8(x), j);
    __syncthreads();
    if (threadIdx.x >= 240) return;
    const uint4 mine = rows[piece];
    uint8_t* plane = is_k ? a.ck : a.cv;
    while (b < b_end) {
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (b + 3 * u < b_end && l < n[u])
                *reinterpret_cast<uint4*>(plane + (((int64_t)(b + 3 * u) * a.Hkv + hk) * a.maxlen + len[u] + tile * 16) * kQ4Row + 16 * piece) = mine;
        b += 12;
        if (b < b_end) extents();
    }
}

// Sixteen lanes to a row: rows starts[b] .. of every plane, sequence and head; rows outside the cache are 0.  Bound by its stores: 2048 rows of 8 sequences
// and 32 heads, 84 MB in and 268 out as halves, 60 us, 5.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void q4_read_kernel(const uint8_t* __restrict__ cache, int64_t heads, int B, int Hkv, int64_t maxlen, const int32_t* __restrict__ starts,
                                                      int64_t rows, T* __restrict__ out) {
    const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int j = threadIdx.x & 15;
    if (at >= heads * rows) return;
    const int64_t head = at / rows, r = at - head * rows;  // (plane, sequence, head)
    const int64_t row = r + (starts != nullptr ? starts[(int)(head / Hkv % B)] : 0);
    v8h x = {};
    if (row >= 0 && row < maxlen) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(cache + (head * maxlen + row) * kQ4Row);
        x = Codes().values(src[j], src[16 + (j >> 2)]);
    }
    T* dst = out + at * kS + 8 * j;
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4((float)x[4], (float)x[5], (float)x[6], (float)x[7]);
    } else {
        *reinterpret_cast<uint4*>(dst) = __builtin_bit_cast(uint4, x);
    }
}

}  // namespace llmops

using namespace llmops;

extern "C" int llmops_cache_write_q4(const void* k, int64_t k_stride_b, int64_t k_stride_l, int64_t k_stride_h, const void* v, int64_t v_stride_b,
                                     int64_t v_stride_l, int64_t v_stride_h, int dtype, int64_t B, int64_t qL, int64_t Hkv, int64_t S, const float* inv_freq,
                                     int64_t half, void* kv_cache, int64_t planes, int64_t maxlen, const int32_t* lengths, const int32_t* q_lens, int layer_id,
                                     llmops_stream_t stream) {
    const int64_t most = (int64_t)1 << 24;
    LLMOPS_REQUIRE(k != nullptr && v != nullptr && kv_cache != nullptr && lengths != nullptr);
    LLMOPS_REQUIRE(S == 128);  // head size of every supported model shape
    LLMOPS_REQUIRE(dtype == LLMOPS_F32 || dtype == LLMOPS_F16);
    LLMOPS_REQUIRE(B > 0 && qL > 0 && Hkv > 0 && maxlen > 0 && B < most && qL < most && Hkv < most && maxlen <= most);
    LLMOPS_REQUIRE(inv_freq == nullptr || (half > 0 && 2 * half <= S));
    LLMOPS_REQUIRE(layer_id >= 0 && 2 * (int64_t)layer_id + 1 < planes);
    const int64_t e = dtype == LLMOPS_F32 ? 4 : 2, per = 16 / e;
    LLMOPS_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(kv_cache, 16) && aligned(lengths, 4) && aligned(q_lens, 4) && aligned(inv_freq, 4));
    LLMOPS_REQUIRE(k_stride_b % per == 0 && k_stride_l % per == 0 && k_stride_h % per == 0 && v_stride_b % per == 0 && v_stride_l % per == 0 && v_stride_h % per == 0);
    WriteArgs a{k, v, inv_freq, k_stride_b, k_stride_l, k_stride_h, v_stride_b, v_stride_l, v_stride_h};
    const Wide plane = (Wide)B * Hkv * maxlen * kQ4Row;
    LLMOPS_REQUIRE((Wide)planes * plane < ((Wide)1 << 62));
    a.ck = reinterpret_cast<uint8_t*>(kv_cache) + 2 * layer_id * (int64_t)plane, a.cv = a.ck + (int64_t)plane;
    // (a workgroup reads its rows while others have written theirs)
    const Extent written(a.ck, 2 * plane);
    const bool dense = k_stride_h == kS && v_stride_h == kS;  // (a token's heads one behind the other: looked at together)
    for (int64_t h = 0; h < (dense ? 1 : Hkv); h++) {
        const Wide width = (Wide)(dense ? Hkv : 1) * kS * e;
        const Extent kh(reinterpret_cast<const char*>(k) + h * k_stride_h * e, B, (Wide)k_stride_b * e, qL, (Wide)k_stride_l * e, width),
            vh(reinterpret_cast<const char*>(v) + h * v_stride_h * e, B, (Wide)v_stride_b * e, qL, (Wide)v_stride_l * e, width);
        LLMOPS_REQUIRE(apart(written, kh) && apart(written, vh));
    }
    const Extent lengths_at(lengths, (Wide)B * 4), q_lens_at(q_lens, q_lens != nullptr ? (Wide)B * 4 : 0), inv_freq_at(inv_freq, inv_freq != nullptr ? (Wide)half * 4 : 0);
    LLMOPS_REQUIRE(apart(written, lengths_at) && apart(written, q_lens_at) && apart(written, inv_freq_at));
    a.lengths = lengths, a.q_lens = q_lens, a.maxlen = maxlen;
    a.B = (int)B, a.qL = (int)qL, a.Hkv = (int)Hkv, a.half = (int)half, a.groups = (int)((2 * Hkv + 15) / 16);
    a.shared = B > 1 && k_stride_b == 0 && v_stride_b == 0;
    const int64_t grid = inv_freq != nullptr ? B * qL * a.groups : (a.shared ? 1 : B) * ((qL + 15) / 16) * 2 * Hkv;
    LLMOPS_REQUIRE((Wide)B * qL * 2 * Hkv < ((Wide)1 << 40) && grid < most);  // (a launch has fewer than 2^32 threads)
    hipStream_t st = as_stream(stream);
    if (inv_freq != nullptr) {
        if (dtype == LLMOPS_F32) q4_write_turned_kernel<float><<<(unsigned)grid, 256, 0, st>>>(a);
        else q4_write_turned_kernel<_Float16><<<(unsigned)grid, 256, 0, st>>>(a);
    } else {
        if (dtype == LLMOPS_F32) q4_write_kernel<float><<<(unsigned)grid, 256, 0, st>>>(a);
        else q4_write_kernel<_Float16><<<(unsigned)grid, 256, 0, st>>>(a);
    }
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}

extern "C" int llmops_cache_read_q4(const void* kv_cache, int64_t planes, int64_t B, int64_t Hkv, int64_t maxlen, int64_t S, const int32_t* starts, int64_t rows,
                                    void* out, int dtype, llmops_stream_t stream) {
    const int64_t most = (int64_t)1 << 24;
    LLMOPS_REQUIRE(kv_cache != nullptr && out != nullptr);
    LLMOPS_REQUIRE(S == 128);
    LLMOPS_REQUIRE(dtype == LLMOPS_F32 || dtype == LLMOPS_F16);
    LLMOPS_REQUIRE(planes > 0 && B > 0 && Hkv > 0 && maxlen > 0 && rows > 0 && planes < most && B < most && Hkv < most && maxlen <= most && rows <= most);
    LLMOPS_REQUIRE(aligned(kv_cache, 16) && aligned(out, 16) && aligned(starts, 4));
    const Wide heads = (Wide)planes * B * Hkv;
    LLMOPS_REQUIRE(heads * maxlen * kQ4Row < ((Wide)1 << 62) && (heads * rows + 15) / 16 < most);  // (a launch has fewer than 2^32 threads)
    const Extent cache_at(kv_cache, heads * maxlen * kQ4Row), out_at(out, heads * rows * kS * (dtype == LLMOPS_F32 ? 4 : 2)),
        starts_at(starts, starts != nullptr ? B * 4 : 0);
    LLMOPS_REQUIRE(apart(out_at, cache_at) && apart(out_at, starts_at));
    const unsigned grid = (unsigned)((heads * rows + 15) / 16);
    hipStream_t st = as_stream(stream);
    const uint8_t* cache = reinterpret_cast<const uint8_t*>(kv_cache);
    if (dtype == LLMOPS_F32) q4_read_kernel<float><<<grid, 256, 0, st>>>(cache, (int64_t)heads, (int)B, (int)Hkv, maxlen, starts, rows, (float*)out);
    else q4_read_kernel<_Float16><<<grid, 256, 0, st>>>(cache, (int64_t)heads, (int)B, (int)Hkv, maxlen, starts, rows, (_Float16*)out);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}
