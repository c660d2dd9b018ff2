// What the kernels of the int8 inner product share: the operands as the kernels see them.
#pragma once

#include "typed.cuh"

#include <type_traits>

namespace tsb {

struct InnerProdParams {
    const int8_t *x, *w;
    int64_t x_pitch, w_pitch;         // elements between rows
    const float *x_scales, *w_scales;
    int64_t xs_stride;
    const float *bias;                // or NULL
    const void *residual;             // of the output's type, or NULL
    void *y;
    int64_t residual_pitch, y_pitch;
    int64_t m;
    int n, k;
    int activation;
    float leaky;
    int residual_after;
};

#ifdef __CUDACC__
// A sum as fp32.  SHORT: sums of at most 255 products, below 2^22 in magnitude, by an addition to the bits of 1.5 * 2^23 (the
// conversion instruction is done 16 times a clock on a multiprocessor, an eighth as often).
constexpr int kShortSum = 255;
template <bool SHORT>
__device__ __forceinline__ float sum_to_f32(int acc) {
    return SHORT ? __fadd_rn(__int_as_float(acc + 0x4b400000), -12582912.0f) : __int2float_rn(acc);
}

// N values: sum -> fp32, times the output channel's scale, times the token's, + bias (a missing one is 0), + residual, activation
// (+ residual); every step is rounded by itself, so the values do not depend on which kernel computed them.
// of(i): values i and i + 1's scales of their channels (one value: .x alone), their token's scale, their biases, their residuals.
struct PairScales {
    float2 ws;
    float xs;
    float2 bias;
};
// RES: false where there is certainly no residual.
template <typename T, bool RES = true, int N, typename Of, typename Res>
__device__ __forceinline__ void inner_prod_values(const InnerProdParams &p, const int (&acc)[N], const Of &of, const Res &res, float (&v)[N]) {
    auto scale = [&](auto is_short) {
        constexpr bool kShort = decltype(is_short)::value;
        if constexpr (N > 1) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                // (products by twos, sums one by one: the assembler makes fused operations of a packed product and a packed sum)
                const PairScales s = of(i);
                const float2 r = mul2(mul2(make_float2(sum_to_f32<kShort>(acc[i]), sum_to_f32<kShort>(acc[i + 1])), s.ws), make_float2(s.xs, s.xs));
                v[i] = __fadd_rn(r.x, s.bias.x);
                v[i + 1] = __fadd_rn(r.y, s.bias.y);
            }
        } else {
            const PairScales s = of(0);
            v[0] = __fadd_rn(__fmul_rn(__fmul_rn(sum_to_f32<kShort>(acc[0]), s.ws.x), s.xs), s.bias.x);
        }
    };
    if (N >= 16 && p.k <= kShortSum) scale(std::true_type());
    else scale(std::false_type());
    if (RES && p.residual && !p.residual_after) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fadd_rn(v[i], res(i));
    }
    by_activation(p.activation, [&](auto act) { activate<decltype(act)::value, T>(v, p.leaky); });
    if (RES && p.residual && p.residual_after) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fadd_rn(v[i], res(i));
    }
}
#endif

// inner_prod_tc.cu: the tensor-core kernel
namespace tc {
bool inner_prod_can(const InnerProdParams &p, const char **why);     // whether it (and the one below) takes these operands, and if not, why
bool weights_fit(const InnerProdParams &p);                           // the part of that that concerns w
int inner_prod(const InnerProdParams &p, int y_type, cudaStream_t stream);
int inner_prod_status(cudaStream_t stream);
int inner_prod_status_decode(int word);
}  // namespace tc

// inner_prod_few.cu: the kernel of few tokens
namespace few {
constexpr int kMaxTokens = 32;
int inner_prod(const InnerProdParams &p, int y_type, int early, cudaStream_t stream);      // early: weights may be read before the kernel in front is done
bool can_quantize(const InnerProdParams &p, int x_type, int y_type);                       // whether the next one takes these floating rows
int inner_prod_quantize(const InnerProdParams &p, int y_type, cudaStream_t stream);
}  // namespace few

}  // namespace tsb
