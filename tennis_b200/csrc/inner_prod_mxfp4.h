// What the kernels of the 4-bit inner product share: the operands as the kernels see them.
#pragma once

#include "mxfp4.cuh"

namespace tsb {

struct InnerProdMxfp4Params {
    const uint8_t *x, *w;
    int64_t x_pitch, w_pitch;         // bytes between rows
    const uint8_t *x_scales, *w_scales;
    const float *bias;                // or NULL
    const void *residual;             // of the output's type, or NULL
    void *y;
    int64_t residual_pitch, y_pitch;
    int64_t m;
    int n, groups;                    // groups of 32 values a row
    int activation;
    float leaky;
    int residual_after;
};

#ifdef __CUDACC__
// N sums: + bias (a missing one is 0), + residual, activation (+ residual); every step is rounded by itself.
// bias(i), res(i): value i's.  RES: false where there is certainly no residual.
template <typename T, bool RES = true, int N, typename Bias, typename Res>
__device__ __forceinline__ void finish_values(const InnerProdMxfp4Params &p, const Bias &bias, const Res &res, float (&v)[N]) {
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fadd_rn(v[i], bias(i));
    }
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

// inner_prod_mxfp4_tc.cu: the tensor-core kernel
namespace tc {
bool inner_prod_can(const InnerProdMxfp4Params &p, const char **why);     // whether it takes these operands, and if not, why
bool weights_fit(const InnerProdMxfp4Params &p);                           // the part of that that concerns w
int inner_prod(const InnerProdMxfp4Params &p, int y_type, cudaStream_t stream);
int mxfp4_status_word(int **at);                                          // of the current device, for the kernels of few tokens too
int inner_prod_mxfp4_status(cudaStream_t stream);
int inner_prod_mxfp4_status_decode(int word);
}  // namespace tc

// inner_prod_mxfp4_few.cu: the kernel of few tokens
namespace few {
constexpr int kMaxMxfp4Tokens = 64;
int inner_prod(const InnerProdMxfp4Params &p, int y_type, int early, cudaStream_t stream);       // early: weights may be read before the kernel in front is done
bool can_quantize(const InnerProdMxfp4Params &p, int x_type, int y_type);                        // whether the next one takes these floating rows
int inner_prod_quantize(const InnerProdMxfp4Params &p, int y_type, int64_t x_pitch, int cols, cudaStream_t stream);
}  // namespace few

}  // namespace tsb
