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
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// gelu of values that become results of 16 bits: v / 2 + |v| / 2 - |v| / 2 erfc(|v| / sqrt(2)).  With b = |v| sqrt(log2(e) / 2) and t = 1 / (b + 2.451) that is exp2(-b^2) b t P(t), a polynomial of
// degree six that was fitted by linear programming, so that erfc is off by 5.3e-8 at most and by 6.7e-6 of itself: below zero, where the result is the last term alone, the second counts.  With
// the roundings of fp32 the result is off by 2^-16 of itself at most (2^-19 from v = -1 on), a sixteenth of half a step of fp16 at most, down to v = -13, and is zero below -13.3.  (erff and the rest are some
// 60 instructions a value, these 12: 333 x 777 x 1021 with a residual 6.1 -> 5.4 us.)
__device__ __forceinline__ float2 gelu_short(float2 v) {
    const float2 w = mul2(make_float2(fabsf(v.x), fabsf(v.y)), both(0.849321783f));
    const float2 b = make_float2(fminf(w.x, 13.6f), fminf(w.y, 13.6f));      // (erfc is 0 there; an infinity's would be infinity times 0)
    const float2 d = add2(b, both(2.4512701f));
    const float2 t = make_float2(reciprocal_approx(d.x), reciprocal_approx(d.y));
    const float2 q = mul2(b, b);
    const float2 e = make_float2(exp2_approx(-q.x), exp2_approx(-q.y));
    float2 p = fma2(both(-27.3318176f), t, both(47.4502983f));
    p = fma2(p, t, both(-23.1390343f));
    p = fma2(p, t, both(-0.0789856464f));
    p = fma2(p, t, both(-2.50978255f));
    p = fma2(p, t, both(-0.955673873f));
    p = fma2(p, t, both(-0.399428397f));
    // (a NaN is one here, whatever the minimum above made of it, and minus infinity becomes one)
    const float2 rising = fma2(make_float2(fabsf(v.x), fabsf(v.y)), both(0.5f), mul2(v, both(0.5f)));
    return fma2(mul2(mul2(p, t), e), b, rising);
}
// The activation as activate() takes it, gelu of 16-bit results as above.
template <int ACT, typename T, int N>
__device__ __forceinline__ void activate_sums(float (&v)[N], float leaky) {
    if constexpr (ACT == TSB_ACT_GELU && sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 y = gelu_short(make_float2(v[i], v[i + 1]));
            v[i] = y.x;
            v[i + 1] = y.y;
        }
    } else {
        activate<ACT, T>(v, leaky);
    }
}

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
    by_activation(p.activation, [&](auto act) { activate_sums<decltype(act)::value, T>(v, p.leaky); });
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
// Whether it is the sooner one: up to 32 tokens, and up to 64 of more than 1024 values each (64 tokens, by it and by tiles: 300 x 300 3.7 and 3.2 us, 8000 x 300 4.3 and 3.8,
// 2000 x 4000 4.7 and 5.1, 300 x 8192 5.1 and 7.9; 32 tokens 2.7 and 3.1, 3.2 and 3.8, 3.8 and 5.3, 4.3 and 7.8).
inline bool takes(const InnerProdMxfp4Params &p) { return p.m <= 32 || (p.m <= 64 && p.groups > 32); }
int inner_prod(const InnerProdMxfp4Params &p, int y_type, int early, cudaStream_t stream);       // early: weights may be read before the kernel in front is done
bool can_quantize(const InnerProdMxfp4Params &p, int x_type, int y_type);                        // whether the next one takes these floating rows
int inner_prod_quantize(const InnerProdMxfp4Params &p, int y_type, int64_t x_pitch, int cols, cudaStream_t stream);
}  // namespace few

}  // namespace tsb
