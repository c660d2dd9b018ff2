// What the kernels of the int8 inner product share: the operands as the kernels see them.
#pragma once

#include "typed.cuh"

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
// One value: sum -> fp32, times the output channel's scale, times the token's, + bias, + residual, activation (+ residual); every step
// is rounded by itself, so the value does not depend on which kernel computed it.
__device__ __forceinline__ float inner_prod_value(int acc, float ws, float xs, float bias, bool has_bias, float residual, bool has_residual,
                                                  bool residual_after, int activation, float leaky) {
    float v = __fmul_rn(__fmul_rn(__int2float_rn(acc), ws), xs);
    if (has_bias) v = __fadd_rn(v, bias);
    if (has_residual && !residual_after) v = __fadd_rn(v, residual);
    v = activate(v, activation, leaky);
    if (has_residual && residual_after) v = __fadd_rn(v, residual);
    return v;
}
#endif

// inner_prod_tc.cu: the tensor-core kernel
namespace tc {
bool inner_prod_can(const InnerProdParams &p, const char **why);     // whether it takes these operands, and if not, why
int inner_prod(const InnerProdParams &p, int y_type, cudaStream_t stream);
int inner_prod_status(cudaStream_t stream);
}  // namespace tc

}  // namespace tsb
