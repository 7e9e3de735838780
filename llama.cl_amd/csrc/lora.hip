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
// (8 bits each, cut off), an fp16 weight two, a bf16 weight itself.  Products of pieces whose places sum to three or less are
// formed; what is dropped is below 2^-22 of a product.
#include "common.h"

namespace llmops {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct LoraArgs {
    const float *x, *y, *scales;
    const void *A, *B;   // [adapters][R][K], [adapters][N][R]
    const int32_t* ids;  // [batch]
    float *out, *part;   // part [splits][rows][R]
    int64_t xsb, xsl, ysb, ysl, osb, osl;
    int rows, tokens, K, N, R, adapters, splits, chunk;
};

template <int N>
struct Pieces {
    v8bf p[N];
};
__device__ __forceinline__ v8bf as_v8bf(uint4 u) { return __builtin_bit_cast(v8bf, u); }
__device__ __forceinline__ uint32_t upper(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// eight fp32 values as N bf16 pieces each (infinities and NaN in the first)
template <int N>
__device__ __forceinline__ Pieces<N> cut8(const float (&x)[8]) {
    Pieces<N> r;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e++) rest[e] = x[e];
#pragma unroll
    for (int n = 0; n < N; n++) {
        uint32_t u[8], w[4];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            u[e] = __float_as_uint(rest[e]);
            const float left = rest[e] - __uint_as_float(u[e] & 0xffff0000u);
            rest[e] = (u[e] << 1) == 0xff000000u ? 0.0f : left;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = upper(u[2 * e], u[2 * e + 1]);
        r.p[n] = as_v8bf(make_uint4(w[0], w[1], w[2], w[3]));
    }
    return r;
}

// a weight's type: its pieces, and eight of a row from `at` on, zeros from `end` on
template <typename W>
struct Weight;
template <>
struct Weight<float> {
    static constexpr int kPieces = 3;
    template <bool VEC>
    static __device__ __forceinline__ Pieces<3> load(const float* row, int at, int end) {
        float x[8];
        if (VEC && at + 8 <= end) {
            const float4 a = *reinterpret_cast<const float4*>(row + at), b = *reinterpret_cast<const float4*>(row + at + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = at + e < end ? row[at + e] : 0.0f;
        }
        return cut8<3>(x);
    }
};
struct Half16 {
    uint16_t u;
};
struct Bf16 {
    uint16_t u;
};
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int at, int end) {
    if (VEC && at + 8 <= end) return *reinterpret_cast<const uint4*>(row + at);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        w[e] = (at + 2 * e < end ? row[at + 2 * e] : 0u) | (at + 2 * e + 1 < end ? (uint32_t)row[at + 2 * e + 1] << 16 : 0u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
struct Weight<Half16> {
    static constexpr int kPieces = 2;
    template <bool VEC>
    static __device__ __forceinline__ Pieces<2> load(const Half16* row, int at, int end) {
        const uint4 u = load8<VEC>(reinterpret_cast<const uint16_t*>(row), at, end);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = f16_bits_to_f32((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
        return cut8<2>(x);
    }
};
template <>
struct Weight<Bf16> {
    static constexpr int kPieces = 1;
    template <bool VEC>
    static __device__ __forceinline__ Pieces<1> load(const Bf16* row, int at, int end) {
        return {{as_v8bf(load8<VEC>(reinterpret_cast<const uint16_t*>(row), at, end))}};
    }
};

template <int NW>
__device__ __forceinline__ v4f times(const Pieces<NW>& w, const Pieces<3>& x, v4f acc) {
#pragma unroll
    for (int n = 0; n < NW; n++)
#pragma unroll
        for (int m = 0; m < 3 && n + m < 3; m++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[n], x.p[m], acc, 0, 0, 0);
    return acc;
}

// token `row`'s adapter, -1 for none
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int row) {
    if (row >= a.rows) return -1;
    const int id = a.ids[row / a.tokens];
    return id >= 0 && id < a.adapters ? id : -1;
}
// calls f(adapter, whether this lane's token is one of its) for every adapter among the sixteen tokens (token lane % 16)
template <typename F>
__device__ __forceinline__ void each_adapter(int mine, F f) {
    uint32_t todo = (uint32_t)__ballot(mine >= 0) & 0xffffu;
    while (todo != 0) {
        const int id = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
        f(id, mine == id);
        todo &= ~(uint32_t)__ballot(mine == id);
    }
}

// A workgroup: sixteen tokens, a run of K (its four waves a quarter of every 128 each), 16 * NR rows of A.
// A operand: row of A lane % 16, eight k; B operand: token lane % 16, the same k; result: token lane % 16, rows 4 * (lane / 16) + v.
template <typename W, int NR, bool VEC>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    __shared__ v4f meet[4][NR][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16, r0 = blockIdx.z * 16 * NR, row = row0 + i;
    const int k0 = blockIdx.y * a.chunk, k1 = min(a.K, k0 + a.chunk);
    const int mine = adapter_of(a, row);
    const int safe = min(row, a.rows - 1), b = safe / a.tokens;
    const float* x = a.x + b * a.xsb + (safe - b * a.tokens) * a.xsl;
    v4f acc[NR];
#pragma unroll
    for (int n = 0; n < NR; n++) acc[n] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int k = k0 + 32 * wave; k < k1; k += 128) {
        const Pieces<3> xp = Weight<float>::load<VEC>(x, k + 8 * g, k1);
        each_adapter(mine, [&](int id, bool match) {
            const W* A = reinterpret_cast<const W*>(a.A) + (int64_t)id * a.R * a.K;
#pragma unroll
            for (int n = 0; n < NR; n++) {
                const int r = r0 + 16 * n + i;
                const auto w = Weight<W>::template load<VEC>(A + (int64_t)min(r, a.R - 1) * a.K, k + 8 * g, k1);
                const v4f sum = times(w, xp, acc[n]);
#pragma unroll
                for (int v = 0; v < 4; v++) acc[n][v] = match ? sum[v] : acc[n][v];
            }
        });
    }
#pragma unroll
    for (int n = 0; n < NR; n++) meet[wave][n][lane] = acc[n];
    __syncthreads();
    for (int n = wave; n < NR; n += 4) {
        const v4f s = (meet[0][n][lane] + meet[1][n][lane]) + (meet[2][n][lane] + meet[3][n][lane]);
        if (row >= a.rows) continue;
        float* to = a.part + ((int64_t)blockIdx.y * a.rows + row) * a.R;
#pragma unroll
        for (int v = 0; v < 4; v++)
            if (r0 + 16 * n + 4 * g + v < a.R) to[r0 + 16 * n + 4 * g + v] = s[v];
    }
}

// A workgroup: sixteen tokens, 256 columns (64 to a wave), ranks 128 at a time.
// A operand: column lane % 16 of B, eight ranks; B operand: token lane % 16, the same ranks; result: token lane % 16, columns 4 * (lane / 16) + v.
template <typename W, bool VEC>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a, bool vec_out) {
    constexpr int kRanks = 128, kStride = kRanks + 4;
    __shared__ __align__(16) float t[16][kStride];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.y * 16, n0 = blockIdx.x * 256 + 64 * wave, row = row0 + i;
    const int mine = adapter_of(a, row);
    v4f acc[4];
#pragma unroll
    for (int n = 0; n < 4; n++) acc[n] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < a.R; r0 += kRanks) {
        const int ranks = min(kRanks, a.R - r0), padded = (ranks + 31) & ~31;
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * padded; e += 256) {
            const int token = e / padded, r = e - token * padded;
            float s = 0.0f;
            if (r < ranks && row0 + token < a.rows) {
                const float* from = a.part + (int64_t)(row0 + token) * a.R + r0 + r;
                for (int c = 0; c < a.splits; c++) s += from[(int64_t)c * a.rows * a.R];
            }
            t[token][r] = s;
        }
        __syncthreads();
        for (int step = 0; step < padded; step += 32) {
            float x[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float4 u = *reinterpret_cast<const float4*>(&t[i][step + 8 * g + 4 * h]);
                x[4 * h] = u.x, x[4 * h + 1] = u.y, x[4 * h + 2] = u.z, x[4 * h + 3] = u.w;
            }
            const Pieces<3> tp = cut8<3>(x);
            each_adapter(mine, [&](int id, bool match) {
                const W* B = reinterpret_cast<const W*>(a.B) + (int64_t)id * a.N * a.R;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int col = min(n0 + 16 * n + i, a.N - 1);
                    const auto w = Weight<W>::template load<VEC>(B + (int64_t)col * a.R, r0 + step + 8 * g, a.R);
                    const v4f sum = times(w, tp, acc[n]);
#pragma unroll
                    for (int v = 0; v < 4; v++) acc[n][v] = match ? sum[v] : acc[n][v];
                }
            });
        }
    }
    if (row >= a.rows) return;
    const int b = row / a.tokens, l = row - b * a.tokens;
    const float* y = a.y + b * a.ysb + l * a.ysl;
    float* out = a.out + b * a.osb + l * a.osl;
    const float scale = mine >= 0 ? a.scales[mine] : 0.0f;
#pragma unroll
    for (int n = 0; n < 4; n++) {
        const int col = n0 + 16 * n + 4 * g;
        if (vec_out && col + 4 <= a.N) {
            float4 u = *reinterpret_cast<const float4*>(y + col);
            if (mine >= 0) u = make_float4(fmaf(scale, acc[n][0], u.x), fmaf(scale, acc[n][1], u.y), fmaf(scale, acc[n][2], u.z), fmaf(scale, acc[n][3], u.w));
            *reinterpret_cast<float4*>(out + col) = u;
        } else {
#pragma unroll
            for (int v = 0; v < 4; v++)
                if (col + v < a.N) out[col + v] = mine >= 0 ? fmaf(scale, acc[n][v], y[col + v]) : y[col + v];
        }
    }
}

// K in runs: until there are some 512 workgroups, a run at least 128
static int lora_splits(int64_t rows, int64_t K, int64_t R) {
    const int64_t groups = (rows + 15) / 16 * ((R + 63) / 64), most = (K + 127) / 128;
    int64_t n = (512 + groups - 1) / groups;
    n = n < most ? n : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

template <typename W>
static int lora_launch(LoraArgs a, bool vec_down, bool vec_up, bool vec_out, hipStream_t st) {
    const unsigned tiles = (unsigned)((a.rows + 15) / 16);
    const int nr = a.R <= 16 ? 1 : a.R <= 32 ? 2 : 4;
    const dim3 down(tiles, (unsigned)a.splits, (unsigned)((a.R + 16 * nr - 1) / (16 * nr)));
#define LLMOPS_DOWN(NR)                                                          \
    if (vec_down) lora_down_kernel<W, NR, true><<<down, 256, 0, st>>>(a);        \
    else lora_down_kernel<W, NR, false><<<down, 256, 0, st>>>(a)
    if (nr == 1) {
        LLMOPS_DOWN(1);
    } else if (nr == 2) {
        LLMOPS_DOWN(2);
    } else {
        LLMOPS_DOWN(4);
    }
#undef LLMOPS_DOWN
    LLMOPS_LAUNCH_CHECK();
    const dim3 up((unsigned)((a.N + 255) / 256), tiles);
    if (vec_up) lora_up_kernel<W, true><<<up, 256, 0, st>>>(a, vec_out);
    else lora_up_kernel<W, false><<<up, 256, 0, st>>>(a, vec_out);
    LLMOPS_LAUNCH_CHECK();
    return LLMOPS_OK;
}

}  // namespace llmops

using namespace llmops;

static bool lora_sizes_fit(int64_t batch, int64_t tokens, int64_t N, int64_t K, int64_t R) {
    const int64_t most = (int64_t)1 << 30;
    return batch > 0 && tokens > 0 && N > 0 && K > 0 && R > 0 && batch < most && tokens < most && N < most && K < most && R <= 4096 &&
           batch * tokens <= 65535 * 16;
}

extern "C" size_t llmops_lora_workspace_bytes(int64_t batch, int64_t tokens, int64_t N, int64_t K, int64_t R) {
    if (!lora_sizes_fit(batch, tokens, N, K, R)) return 0;
    return (size_t)lora_splits(batch * tokens, K, R) * (size_t)(batch * tokens) * (size_t)R * sizeof(float);
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
    const size_t need = llmops_lora_workspace_bytes(batch, tokens, N, K, R);
    if (workspace == nullptr || workspace_bytes < need)
        return fail(LLMOPS_EWORKSPACE, "lora_add needs %zu workspace bytes, got %zu", need, workspace == nullptr ? (size_t)0 : workspace_bytes);
    LLMOPS_REQUIRE(aligned(workspace, 4));
    LoraArgs a{};
    a.x = x, a.y = y, a.scales = scales, a.A = lora_A, a.B = lora_B, a.ids = ids, a.out = out, a.part = reinterpret_cast<float*>(workspace);
    a.xsb = x_stride_b, a.xsl = x_stride_l, a.ysb = y_stride_b, a.ysl = y_stride_l, a.osb = out_stride_b, a.osl = out_stride_l;
    a.rows = (int)(batch * tokens), a.tokens = (int)tokens, a.K = (int)K, a.N = (int)N, a.R = (int)R, a.adapters = (int)adapters;
    a.splits = lora_splits(a.rows, K, R);
    a.chunk = (int)((K + 128 * a.splits - 1) / (128 * a.splits) * 128);
    a.splits = (int)((K + a.chunk - 1) / a.chunk);
    const bool vec_down = K % 8 == 0 && aligned(x, 16) && x_stride_b % 4 == 0 && x_stride_l % 4 == 0 && aligned(lora_A, 16),
               vec_up = R % 8 == 0 && aligned(lora_B, 16),
               vec_out = aligned(y, 16) && aligned(out, 16) && y_stride_b % 4 == 0 && y_stride_l % 4 == 0 && out_stride_b % 4 == 0 && out_stride_l % 4 == 0;
    hipStream_t st = as_stream(stream);
    if (weight_dtype == LLMOPS_F32) return lora_launch<float>(a, vec_down, vec_up, vec_out, st);
    if (weight_dtype == LLMOPS_F16) return lora_launch<Half16>(a, vec_down, vec_up, vec_out, st);
    return lora_launch<Bf16>(a, vec_down, vec_up, vec_out, st);
}
