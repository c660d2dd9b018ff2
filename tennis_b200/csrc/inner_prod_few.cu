// The int8 inner product of few tokens: the weights' bytes are the work, each is read once.
//
//   block      16 output channels and all of K; its warps take blocks of 128 bytes of K in turn, and their int32 sums meet in shared memory
//   loads      cp.async into a ring of the warp's own, kDepth blocks of K ahead; a thread reads back what it loaded itself, so a ring needs
//              no barrier.  The sixteen warps on a multiprocessor have 128 KB of weights under way for up to 8 tokens, 96 KB for up to 16, 64 KB for
//              up to 32, whose own loads take the rest of the rings
//   product    mma.sync m16n8k32: a thread's 16 bytes of a weight row and of a token's row are the operands of two MMAs, which so take
//              the 64 bytes of four threads in an order of K of their own -- the same one for both operands, which is all that a sum
//              needs.  (The MMAs of up to 32 tokens take a fraction of the loads' time; tcgen05 would only add its set-up.)
//   tokens     int8 rows, read like the weights; or one floating row, which every block quantizes in shared memory while its weights
//              are on their way (two rows or more are quantized sooner by quantize_rows, a block each)
// Bound by the weights' bytes on large layers (one token through 8192 x 8192 14.6 us, 4.6 TB/s), by the chain of load, product and
// meeting on small ones (through 4096 x 4096 5.0 us, quantized inside 5.9; 16 tokens through 2048 x 8192 6.4).
#include "inner_prod_i8.h"

#include <algorithm>
#include <type_traits>

namespace tsb {
namespace few {
namespace {

constexpr int kMaxQuantized = 32768;      // bytes of a quantized row that a block keeps

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes to shared memory, of which `size` come from memory and the rest are zero
__device__ __forceinline__ void load16(uint32_t to, const int8_t *from, int size) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ uint4 read16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// NT: groups of eight tokens; X: int8_t, or the type of one floating row
template <typename X, int NT>
struct Shape {
    static constexpr bool kQuantize = sizeof(X) > 1;
    static constexpr int kTokens = 8 * NT, kChannels = 16;
    static constexpr int kPitch = kChannels + 4;                  // words between two tokens' sums: a warp's writes meet 32 banks
    static constexpr int kSlots = 4 + (kQuantize ? 0 : 2 * NT);   // 16-byte pieces a thread loads for a block of K
    static constexpr int kDepth = NT == 1 ? 4 : NT == 2 ? 3 : 2;
    static constexpr uint32_t kRing = kDepth * kSlots * 512;      // a warp's; its sums lie there afterwards
    static_assert(kTokens * kPitch * 4 <= kRing, "the sums fit the ring");
};

// Quantizes the one floating row into shared memory, zero up to `pitch`: held in registers between the maximum and the rounding as far
// as it fits eight vectors a thread.  start() loads, finish() ends with a barrier.
template <typename X, int W>
struct TokenQuantizer {
    static constexpr int kN = Vec16<X>::kN, kHeld = 8;
    const X *row;
    int k, whole;                 // whole: 16-byte vectors that are read as such
    uint4 held[kHeld];

    __device__ __forceinline__ TokenQuantizer(const InnerProdParams &p) : row(reinterpret_cast<const X *>(p.x)), k(p.k) {
        whole = reinterpret_cast<uintptr_t>(row) % 16 == 0 ? k / kN : 0;
    }
    __device__ __forceinline__ uint4 vector(int u) const { return __ldg(reinterpret_cast<const uint4 *>(row) + u); }
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int u = threadIdx.x + i * 32 * W;
            held[i] = u < whole ? vector(u) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ float finish(int8_t *out, int pitch, uint32_t *part) {
        Largest<X> largest;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) largest.add(held[i]);
        for (int u = threadIdx.x + kHeld * 32 * W; u < whole; u += 32 * W) largest.add(vector(u));
        for (int c = whole * kN + threadIdx.x; c < k; c += 32 * W) largest.add(row[c]);
        uint32_t most = largest.bits();
        most = __reduce_max_sync(0xffffffffu, most);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
        __syncthreads();
        most = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) most = max(most, part[i]);
        const RowScale q(most);
        auto put = [&](const uint4 &from, int u) {
            uint32_t w[kN / 4];
            quantize16<X>(q, from, w);
#pragma unroll
            for (int i = 0; i < kN / 4; ++i) reinterpret_cast<uint32_t *>(out)[u * (kN / 4) + i] = w[i];
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int u = threadIdx.x + i * 32 * W;
            if (u < whole) put(held[i], u);
        }
        for (int u = threadIdx.x + kHeld * 32 * W; u < whole; u += 32 * W) put(vector(u), u);
        for (int c = whole * kN + threadIdx.x; c < pitch; c += 32 * W) out[c] = c < k ? (int8_t)q(to_f32(row[c])) : (int8_t)0;
        __syncthreads();
        return q.scale;
    }
};

// early: the weights may be read before the kernel in front has completed.
template <typename T, typename X, int NT, int W>
__global__ void __launch_bounds__(32 * W)
inner_prod_i8_few_kernel(const __grid_constant__ InnerProdParams p, int early, int x_row_bytes) {
    using S = Shape<X, NT>;
    extern __shared__ __align__(16) uint8_t smem[];
    int8_t *x_rows = reinterpret_cast<int8_t *>(smem + W * S::kRing);              // floating rows: quantized
    uint32_t *part = reinterpret_cast<uint32_t *>(x_rows + (S::kQuantize ? x_row_bytes : 0));
    float scale = 0.0f;                                                            // of the floating row
    if (!early) pdl_sync();
    TokenQuantizer<std::conditional_t<S::kQuantize, X, float>, W> quantizer(p);
    if constexpr (S::kQuantize) quantizer.start();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * S::kChannels;
    const int8_t *w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = p.w + (int64_t)min(n0 + h * 8 + g, p.n - 1) * p.w_pitch;   // (channels behind the last are not written)
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * S::kRing + lane * 16;
    const int blocks = (p.k + 127) / 128, mine = blocks > warp ? (blocks - warp + W - 1) / W : 0;   // this warp's blocks of K: warp, warp + W, ...
    auto load_weights = [&](int i) {
        const uint32_t to = ring + (uint32_t)(i % S::kDepth) * (S::kSlots * 512);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k = (warp + i * W) * 128 + s * 64 + t * 16, size = max(0, min(16, p.k - k)), at = size ? k : 0;
            load16(to + (s * 2 + 0) * 512, w[0] + at, size);
            load16(to + (s * 2 + 1) * 512, w[1] + at, size);
        }
    };
    auto load_tokens = [&](int i) {
        if constexpr (!S::kQuantize) {
            const uint32_t to = ring + (uint32_t)(i % S::kDepth) * (S::kSlots * 512) + 4 * 512;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int m = j * 8 + g;
                const int8_t *row = p.x + (m < p.m ? m : 0) * p.x_pitch;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int k = (warp + i * W) * 128 + s * 64 + t * 16, size = m < p.m ? max(0, min(16, p.k - k)) : 0;
                    load16(to + (j * 2 + s) * 512, row + (size ? k : 0), size);
                }
            }
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    // A group of loads a block of K: block i is there once no more than kDepth - 1 younger groups are under way.  (Weights that are
    // loaded early, ahead of the kernel in front, all belong to the first group.)
    if (early) {
#pragma unroll
        for (int i = 0; i < S::kDepth; ++i)
            if (i < mine) load_weights(i);
        pdl_sync();
    }
#pragma unroll
    for (int i = 0; i < S::kDepth; ++i) {
        if (i < mine) {
            if (!early) load_weights(i);
            load_tokens(i);
        }
        commit();
    }
    if constexpr (S::kQuantize) scale = quantizer.finish(x_rows, x_row_bytes, part);

    int acc[NT][4] = {};
    for (int i = 0; i < mine; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kDepth - 1) : "memory");
        const uint32_t at = ring + (uint32_t)(i % S::kDepth) * (S::kSlots * 512);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint4 r0 = read16(at + (s * 2 + 0) * 512), r1 = read16(at + (s * 2 + 1) * 512);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if constexpr (S::kQuantize) {
                    if (g == 0) v = *reinterpret_cast<const uint4 *>(x_rows + (warp + i * W) * 128 + s * 64 + t * 16);
                } else {
                    v = read16(at + (4 + j * 2 + s) * 512);
                }
                mma_s8(acc[j], r0.x, r1.x, r0.y, r1.y, v.x, v.y);
                mma_s8(acc[j], r0.z, r1.z, r0.w, r1.w, v.z, v.w);
            }
        }
        if (i + S::kDepth < mine) {
            load_weights(i + S::kDepth);
            load_tokens(i + S::kDepth);
        }
        commit();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // a warp's sums [token][channel] where its ring was (every lane's reads and loads are done)
    __syncwarp();
    int *sums = reinterpret_cast<int *>(smem + warp * S::kRing);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) sums[(j * 8 + t * 2 + (q & 1)) * S::kPitch + (q >> 1) * 8 + g] = acc[j][q];
    __syncthreads();
    for (int o = threadIdx.x; o < S::kTokens * S::kChannels; o += 32 * W) {
        const int m = o / S::kChannels, c = o % S::kChannels, n = n0 + c;
        if (m >= p.m || n >= p.n) continue;
        int sum[1] = {0};
#pragma unroll
        for (int i = 0; i < W; ++i) sum[0] += reinterpret_cast<const int *>(smem + i * S::kRing)[m * S::kPitch + c];
        float v[1];
        const float xs = S::kQuantize ? scale : p.x_scales[m * p.xs_stride];
        inner_prod_values<T>(p, sum, [&](int) { return PairScales{make_float2(p.w_scales[n], 0.0f), xs, make_float2(p.bias ? p.bias[n] : 0.0f, 0.0f)}; },
                             [&](int) { return to_f32(static_cast<const T *>(p.residual)[m * p.residual_pitch + n]); }, v);
        static_cast<T *>(p.y)[m * p.y_pitch + n] = from_f32<T>(v[0]);
    }
}

template <typename T, typename X, int NT, int W>
int launch(const InnerProdParams &p, int early, cudaStream_t stream) {
    using S = Shape<X, NT>;
    const int x_row_bytes = round_up(p.k, 128);
    const size_t smem = W * S::kRing + (S::kQuantize ? x_row_bytes : 0) + W * 4;
    auto kernel = inner_prod_i8_few_kernel<T, X, NT, W>;
    static DeviceOnce raised;
    if (raised.first()) {
        TSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(W * S::kRing + kMaxQuantized + W * 4)));
        raised.done();
    }
    TSB_CUDA(launch_pdl(kernel, dim3(ceil_div(p.n, S::kChannels)), dim3(32 * W), smem, stream, p, early, x_row_bytes));
    TSB_LAUNCHED("inner_prod_i8_few_kernel");
    return TSB_OK;
}

template <typename T, typename X, int NT>
int pick_warps(const InnerProdParams &p, int early, cudaStream_t stream) {
    // Two blocks of eight warps a multiprocessor, or four of four where there are more blocks than that (8192 channels x 2048: 6.3 us
    // by eights, 5.5 by fours; 2048 x 8192: 5.3 and 6.4).
    return ceil_div(p.n, 16) > 2 * 148 ? launch<T, X, NT, 4>(p, early, stream) : launch<T, X, NT, 8>(p, early, stream);
}

template <typename T>
int pick(const InnerProdParams &p, int early, cudaStream_t stream) {
    if (p.m <= 8) return pick_warps<T, int8_t, 1>(p, early, stream);
    if (p.m <= 16) return pick_warps<T, int8_t, 2>(p, early, stream);
    return pick_warps<T, int8_t, 4>(p, early, stream);
}

}  // namespace

// Up to 32 tokens of int8 rows.
int inner_prod(const InnerProdParams &p, int y_type, int early, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick<float>(p, early, stream);
        case TSB_TYPE_F16: return pick<__half>(p, early, stream);
        default: return pick<__nv_bfloat16>(p, early, stream);
    }
}

bool can_quantize(const InnerProdParams &p, int x_type, int y_type) { return x_type == y_type && p.m == 1 && p.k <= kMaxQuantized; }

// One floating row of y's type.
int inner_prod_quantize(const InnerProdParams &p, int y_type, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick_warps<float, float, 1>(p, 0, stream);
        case TSB_TYPE_F16: return pick_warps<__half, __half, 1>(p, 0, stream);
        default: return pick_warps<__nv_bfloat16, __nv_bfloat16, 1>(p, 0, stream);
    }
}

}  // namespace few
}  // namespace tsb
