// The int8 inner product of few tokens: the weights' bytes are the work, each is read once.
//
//   block      MT * 16 output channels and all of K; its warps take blocks of 128 bytes of K in turn, and their int32 sums meet in
//              shared memory.  16 channels' rows of 4096 bytes fit the registers of eight warps, so all of a block's loads are in flight at once.
//   product    mma.sync m16n8k32 on bytes that go from memory straight to registers: a thread's 16 bytes of a weight row and of a token's
//              row are the operands of two MMAs, which so take the 64 bytes of four threads in an order of K of their own -- the same
//              one for both operands, which is all that a sum needs.  (With up to 32 tokens the MMAs of a block take a fraction of its loads' time,
//              tcgen05 would only add its set-up.)
//   tokens     int8 rows, read like the weights; or floating rows of which every block quantizes all in shared memory, while its
//              weights are on their way
#include "inner_prod_i8.h"

#include <algorithm>

namespace tsb {
namespace few {
namespace {

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bytes [k, k + 16) of a row of `cols` bytes; those behind its end are zero.
__device__ __forceinline__ uint4 load16(const int8_t *row, int k, int cols) {
    if (k + 16 <= cols) return __ldg(reinterpret_cast<const uint4 *>(row + k));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll 1
    for (int i = 0; i < cols - k; ++i) w[i >> 2] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int NT, int MT>
struct Shape {
    static constexpr int kTokens = 8 * NT, kChannels = 16 * MT;
    static constexpr int kPitch = kChannels + 4;             // words between two tokens' sums: a warp's writes meet 32 banks
    static constexpr int kAhead = NT * MT <= 2 ? 4 : 2;      // blocks of 128 bytes a warp loads before it multiplies
};

// Quantizes the block's M floating rows into shared memory, `pitch` bytes apart and zero up to there.
template <typename X>
__device__ void quantize_tokens(const InnerProdParams &p, const X *x, int8_t *rows, int pitch, float *scales, uint32_t *part) {
    constexpr int kN = Vec16<X>::kN;
    const int threads = blockDim.x;
    for (int m = 0; m < (int)p.m; ++m) {
        const X *row = x + m * p.x_pitch;
        const bool vec = reinterpret_cast<uintptr_t>(row) % 16 == 0;
        const int whole = vec ? p.k / kN : 0;
        uint32_t most = 0;
        for (int u = threadIdx.x; u < whole; u += threads) {
            float v[kN];
            Vec16<X>::get(__ldg(reinterpret_cast<const uint4 *>(row) + u), v);
#pragma unroll
            for (int i = 0; i < kN; ++i) most = max(most, magnitude(v[i]));
        }
        for (int c = whole * kN + threadIdx.x; c < p.k; c += threads) most = max(most, magnitude(to_f32(row[c])));
        most = __reduce_max_sync(0xffffffffu, most);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
        __syncthreads();
        most = 0;
        for (int i = 0; i < threads / 32; ++i) most = max(most, part[i]);
        const RowScale q(most);
        if (threadIdx.x == 0) scales[m] = q.scale;
        int8_t *out = rows + m * pitch;
        for (int u = threadIdx.x; u < whole; u += threads) {
            float v[kN];
            Vec16<X>::get(__ldg(reinterpret_cast<const uint4 *>(row) + u), v);
            uint32_t w[kN / 4];
#pragma unroll
            for (int i = 0; i < kN / 4; ++i)
                w[i] = (uint32_t)(uint8_t)q(v[4 * i]) | (uint32_t)(uint8_t)q(v[4 * i + 1]) << 8 | (uint32_t)(uint8_t)q(v[4 * i + 2]) << 16 | (uint32_t)(uint8_t)q(v[4 * i + 3]) << 24;
#pragma unroll
            for (int i = 0; i < kN / 4; ++i) reinterpret_cast<uint32_t *>(out)[u * (kN / 4) + i] = w[i];
        }
        for (int c = whole * kN + threadIdx.x; c < pitch; c += threads) out[c] = c < p.k ? (int8_t)q(to_f32(row[c])) : (int8_t)0;
        __syncthreads();
    }
}

// X: the type of floating rows, or int8_t.  early: the weights may be read before the kernel in front has completed.
template <typename T, typename X, int NT, int MT, int W>
__global__ void __launch_bounds__(32 * W)
inner_prod_i8_few_kernel(const __grid_constant__ InnerProdParams p, int early, int x_rows_pitch) {
    using S = Shape<NT, MT>;
    constexpr bool kQuantize = sizeof(X) > 1;
    constexpr int kAhead = S::kAhead;
    extern __shared__ __align__(16) uint8_t smem[];
    int *sums = reinterpret_cast<int *>(smem);                                    // [warp][token][channel]
    float *scales = reinterpret_cast<float *>(smem + W * S::kTokens * S::kPitch * 4);
    uint32_t *part = reinterpret_cast<uint32_t *>(scales + S::kTokens);
    int8_t *x_rows = reinterpret_cast<int8_t *>(part + W);
    if (!early) pdl_sync();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * S::kChannels;
    const int8_t *w[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[i][h] = p.w + (int64_t)min(n0 + i * 16 + h * 8 + g, p.n - 1) * p.w_pitch;   // (channels behind the last are not written)
    int acc[MT][NT][4] = {};
    uint4 a[kAhead][MT][2][2];
    auto load_weights = [&](int k0) {
#pragma unroll
        for (int b = 0; b < kAhead; ++b)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int k = k0 + b * W * 128 + s * 64 + t * 16;
                        a[b][i][h][s] = k < p.k ? load16(w[i][h], k, p.k) : make_uint4(0, 0, 0, 0);
                    }
    };
    load_weights(warp * 128);
    if (early) pdl_sync();
    if constexpr (kQuantize) quantize_tokens<X>(p, reinterpret_cast<const X *>(p.x), x_rows, x_rows_pitch, scales, part);

    for (int k0 = warp * 128; k0 < p.k; k0 += kAhead * W * 128) {
        if (k0 > warp * 128) load_weights(k0);
        uint4 x[kAhead][NT][2];
#pragma unroll
        for (int b = 0; b < kAhead; ++b)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int k = k0 + b * W * 128 + s * 64 + t * 16, m = j * 8 + g;
                    x[b][j][s] = make_uint4(0, 0, 0, 0);
                    if (m < p.m && k < p.k) {
                        if constexpr (kQuantize) x[b][j][s] = *reinterpret_cast<const uint4 *>(x_rows + m * x_rows_pitch + k);
                        else x[b][j][s] = load16(p.x + m * p.x_pitch, k, p.k);
                    }
                }
#pragma unroll
        for (int b = 0; b < kAhead; ++b)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const uint4 r0 = a[b][i][0][s], r1 = a[b][i][1][s];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const uint4 v = x[b][j][s];
                        mma_s8(acc[i][j], r0.x, r1.x, r0.y, r1.y, v.x, v.y);
                        mma_s8(acc[i][j], r0.z, r1.z, r0.w, r1.w, v.z, v.w);
                    }
                }
    }

    int *mine = sums + warp * S::kTokens * S::kPitch;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) mine[(j * 8 + t * 2 + (q & 1)) * S::kPitch + i * 16 + (q >> 1) * 8 + g] = acc[i][j][q];
    __syncthreads();
    for (int o = threadIdx.x; o < S::kTokens * S::kChannels; o += 32 * W) {
        const int m = o / S::kChannels, c = o % S::kChannels, n = n0 + c;
        if (m >= p.m || n >= p.n) continue;
        int sum[1] = {0};
#pragma unroll
        for (int i = 0; i < W; ++i) sum[0] += sums[(i * S::kTokens + m) * S::kPitch + c];
        float v[1];
        inner_prod_values<T>(p, sum, kQuantize ? scales[m] : p.x_scales[m * p.xs_stride], [&](int) { return p.w_scales[n]; }, [&](int) { return p.bias ? p.bias[n] : 0.0f; },
                             [&](int) { return to_f32(static_cast<const T *>(p.residual)[m * p.residual_pitch + n]); }, v);
        static_cast<T *>(p.y)[m * p.y_pitch + n] = from_f32<T>(v[0]);
    }
}

template <typename T, typename X, int NT, int MT, int W>
int launch(const InnerProdParams &p, int early, cudaStream_t stream) {
    using S = Shape<NT, MT>;
    const int pitch = round_up(p.k, 128) + 64;      // (64 bytes more: two tokens' reads fall into different banks)
    const size_t smem = (size_t)W * S::kTokens * S::kPitch * 4 + S::kTokens * 4 + W * 4 + (sizeof(X) > 1 ? (size_t)p.m * pitch : 0);
    TSB_CUDA(launch_pdl(inner_prod_i8_few_kernel<T, X, NT, MT, W>, dim3(ceil_div(p.n, S::kChannels)), dim3(32 * W), smem, stream, p, early, pitch));
    TSB_LAUNCHED("inner_prod_i8_few_kernel");
    return TSB_OK;
}

template <typename T>
int pick(const InnerProdParams &p, int early, cudaStream_t stream) {
    if (p.m <= 8) return launch<T, int8_t, 1, 1, 8>(p, early, stream);
    if (p.m <= 16) return launch<T, int8_t, 2, 1, 8>(p, early, stream);
    return launch<T, int8_t, 4, 1, 8>(p, early, stream);
}

template <typename T>
int pick_float(const InnerProdParams &p, cudaStream_t stream) { return launch<T, T, 1, 1, 8>(p, 0, stream); }

}  // namespace

// Up to 32 tokens of int8 rows.
int inner_prod(const InnerProdParams &p, int y_type, int early, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick<float>(p, early, stream);
        case TSB_TYPE_F16: return pick<__half>(p, early, stream);
        default: return pick<__nv_bfloat16>(p, early, stream);
    }
}

bool can_quantize(const InnerProdParams &p, int x_type, int y_type) { return x_type == y_type && p.m <= 8 && p.m * (round_up(p.k, 128) + 64) <= 32768; }

// Up to 8 tokens of floating rows, of y's type, 32 KB of int8 rows.
int inner_prod_quantize(const InnerProdParams &p, int y_type, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick_float<float>(p, stream);
        case TSB_TYPE_F16: return pick_float<__half>(p, stream);
        default: return pick_float<__nv_bfloat16>(p, stream);
    }
}

}  // namespace few
}  // namespace tsb
