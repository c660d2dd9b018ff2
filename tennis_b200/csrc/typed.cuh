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

template <typename T> struct Vec16;        // 16 bytes of a type as fp32 values, and back
template <> struct Vec16<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void get(const uint4 &q, float (&v)[4]) {
        v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 put(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Vec16<__half> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void get(const uint4 &q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Vec16<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void get(const uint4 &q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// ---- int8 rows with a scale taken from the row
// The largest magnitude of a row as the bits of an fp32 value: magnitudes order as their bits do, infinity lies above every number
// and NaN above infinity, so an integer maximum carries both through to the scale.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The same of many values of type T, 16 bytes at a time (of 16-bit types by their own bits, two in one operation).
template <typename T>
class Largest {
public:
    __device__ __forceinline__ void add(const uint4 &q) {
        if constexpr (sizeof(T) == 2) {
            bits_ = __vimax3_u16x2(bits_, q.x & 0x7fff7fffu, q.y & 0x7fff7fffu);
            bits_ = __vimax3_u16x2(bits_, q.z & 0x7fff7fffu, q.w & 0x7fff7fffu);
        } else {
            bits_ = max(bits_, max(max(q.x & 0x7fffffffu, q.y & 0x7fffffffu), max(q.z & 0x7fffffffu, q.w & 0x7fffffffu)));
        }
    }
    __device__ __forceinline__ void add(T v) { single_ = max(single_, magnitude(to_f32(v))); }
    __device__ __forceinline__ uint32_t bits() const {
        if constexpr (sizeof(T) == 2) {
            const uint16_t top = (uint16_t)max(bits_ & 0xffffu, bits_ >> 16);
            return max(single_, magnitude(to_f32(*reinterpret_cast<const T *>(&top))));
        } else {
            return max(single_, bits_);
        }
    }

private:
    uint32_t bits_ = 0, single_ = 0;
};

// Rows below 2^-100 count as zero: the factor 127 / a stays a finite number and the scale a / 127 a normal one.
struct RowScale {
    float by, scale;
    bool finite;
    __device__ __forceinline__ explicit RowScale(uint32_t largest_bits) {
        const float a = __uint_as_float(largest_bits);
        const bool zero = a < 7.888609052210118e-31f;
        by = zero ? 0.0f : __fdiv_rn(127.0f, a);
        scale = zero ? 0.0f : __fdiv_rn(a, 127.0f);
        finite = largest_bits < 0x7f800000u;
    }
    __device__ __forceinline__ int operator()(float v) const { return q8_half_even(__fmul_rn(v, by)); }
};
// 16 bytes of a floating row as int8.  The products of a row of numbers are at most 127 (1 + 2^-23), so nothing is to be clamped, and a
// sum with 1.5 * 2^23 rounds them, half to even, to whole numbers that its low byte holds (a conversion is done an eighth as often).
template <typename X>
__device__ __forceinline__ void quantize16(const RowScale &q, const uint4 &from, uint32_t *to) {
    constexpr int kN = Vec16<X>::kN;
    float v[kN];
    Vec16<X>::get(from, v);
    uint32_t r[kN];
    if (q.finite) {
#pragma unroll
        for (int i = 0; i < kN; ++i) r[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], q.by), 12582912.0f));
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) r[i] = (uint32_t)q(v[i]);
    }
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) to[i] = __byte_perm(__byte_perm(r[4 * i], r[4 * i + 1], 0x0040), __byte_perm(r[4 * i + 2], r[4 * i + 3], 0x0040), 0x5410);
}

// ---- two fp32 values in one instruction (each half is rounded by itself)
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float exp2_approx(float t) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return e;
}
__device__ __forceinline__ float reciprocal_approx(float v) {
    float q;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(v));
    return q;
}

// silu, v / (1 + exp(-v)), by the hardware's exp2 and reciprocal (relative errors of 2^-22 and 2^-23).  For fp32 results the rounding
// error of -v log2(e), which exp2 would turn into a relative error of |v| 2^-24, is computed by a fused multiply-add and put back
// to first order: 8 half steps of the result in all.  (expf and a division take some 40 instructions a value.)
__device__ __forceinline__ float silu(float v) {
    const float c = fminf(fmaxf(v, -200.0f), 200.0f);        // (exp2 is infinite or 0 at either end)
    const float t = __fmul_rn(c, -1.44269502f);
    const float r = fmaf(c, -1.92596303e-8f, fmaf(c, -1.44269502f, -t));   // log2(e) = 1.44269502 (fp32) + 1.92596303e-8
    return __fmul_rn(v, reciprocal_approx(__fadd_rn(1.0f, __fmul_rn(exp2_approx(t), fmaf(r, 0.693147182f, 1.0f)))));
}
// Two values that become results of 16 bits, whose half step is 2^13 times that of fp32 or more: without that correction.  Each is a function of
// itself alone, so its bits do not depend on what it is paired with.  (One reciprocal for both, 1 / a = b (1 / ab), saves one of the four
// functions, of which a multiprocessor does 16 a clock; but then they do.)
__device__ __forceinline__ float2 silu_short(float2 v) {
    const float2 t = mul2(v, make_float2(-1.44269504f, -1.44269504f));
    const float2 a = add2(make_float2(exp2_approx(t.x), exp2_approx(t.y)), make_float2(1.0f, 1.0f));
    return mul2(v, make_float2(reciprocal_approx(a.x), reciprocal_approx(a.y)));
}
__device__ __forceinline__ float gelu(float v) {
    return __fmul_rn(__fmul_rn(0.5f, v), __fadd_rn(1.0f, erff(__fmul_rn(v, 0.70710678118654752f))));
}

// The activation of N values that become results of type T (relu and leaky_relu are the operators' own: a NaN gives 0 and NaN).
template <int ACT, typename T, int N>
__device__ __forceinline__ void activate(float (&v)[N], float leaky) {
    if constexpr (ACT == TSB_ACT_SILU && sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 y = silu_short(make_float2(v[i], i + 1 < N ? v[i + (i + 1 < N)] : 0.0f));
            v[i] = y.x;
            if (i + 1 < N) v[i + (i + 1 < N)] = y.y;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (ACT == TSB_ACT_RELU) v[i] = v[i] > 0.0f ? v[i] : 0.0f;
        if (ACT == TSB_ACT_LEAKY_RELU) v[i] = v[i] > 0.0f ? v[i] : __fmul_rn(v[i], leaky);
        if (ACT == TSB_ACT_SILU) v[i] = silu(v[i]);
        if (ACT == TSB_ACT_GELU) v[i] = gelu(v[i]);
    }
}
// body(a constant of the activation's number): one branch for all values of a loop.  (With the choice made value by value, the unrolled
// code of all five did not fit the instruction cache.)
template <int ACT> struct Activation { static constexpr int value = ACT; };
template <typename Body>
__device__ __forceinline__ void by_activation(int activation, const Body &body) {
    switch (activation) {
        case TSB_ACT_NONE: body(Activation<TSB_ACT_NONE>()); break;
        case TSB_ACT_RELU: body(Activation<TSB_ACT_RELU>()); break;
        case TSB_ACT_LEAKY_RELU: body(Activation<TSB_ACT_LEAKY_RELU>()); break;
        case TSB_ACT_SILU: body(Activation<TSB_ACT_SILU>()); break;
        default: body(Activation<TSB_ACT_GELU>());
    }
}

#endif  // __CUDACC__

}  // namespace tsb
