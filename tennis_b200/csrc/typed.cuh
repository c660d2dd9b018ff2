// Element types of the operators that take fp32, fp16 and bf16 tensors: 16-byte vectors to and from fp32, and the activations
// that follow a product or a norm.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tsb {

inline size_t type_bytes(int type) { return type == TSB_TYPE_F32 ? 4 : (type == TSB_TYPE_I8 ? 1 : 2); }
inline bool is_float_type(int type) { return type == TSB_TYPE_F32 || type == TSB_TYPE_F16 || type == TSB_TYPE_BF16; }
inline bool aligned16(const void *p, int64_t pitch, int type) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (pitch * (int64_t)type_bytes(type)) % 16 == 0;
}
// One past the last byte of `rows` rows of `cols` elements, as an offset; -1 where it does not fit 62 bits.
inline int64_t extent_bytes(int64_t rows, int64_t pitch, int64_t cols, int type) {
    const __int128 e = ((__int128)(rows - 1) * pitch + cols) * (int64_t)type_bytes(type);
    return e >> 62 ? -1 : (int64_t)e;
}

#ifdef __CUDACC__

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// The one rounding to a narrower output: to nearest, ties to even.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The activations after a product or a norm.  relu and leaky_relu are the operators' own (a NaN gives 0 and NaN).
__device__ __forceinline__ float activate(float v, int activation, float leaky) {
    switch (activation) {
        case TSB_ACT_RELU: return v > 0.0f ? v : 0.0f;
        case TSB_ACT_LEAKY_RELU: return v > 0.0f ? v : __fmul_rn(v, leaky);
        case TSB_ACT_SILU: return __fdiv_rn(v, __fadd_rn(1.0f, expf(-v)));
        case TSB_ACT_GELU: return __fmul_rn(__fmul_rn(0.5f, v), __fadd_rn(1.0f, erff(__fmul_rn(v, 0.70710678118654752f))));
        default: return v;
    }
}

#endif  // __CUDACC__

}  // namespace tsb
