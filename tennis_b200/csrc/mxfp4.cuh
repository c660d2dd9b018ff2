// Microscaled 4-bit floating point: codes, scales, and where a scale lies.
#pragma once

#include "typed.cuh"

#include <type_traits>

namespace tsb {
namespace mx {

constexpr int kGroup = 32;                // values that share a scale
constexpr int kTileRows = 128, kTileGroups = 4, kTileBytes = kTileRows * kTileGroups;

inline int64_t row_bytes(int64_t cols) { return (cols + kGroup - 1) / kGroup * (kGroup / 2); }
inline int64_t tiles_of(int64_t cols) { return (cols + kGroup * kTileGroups - 1) / (kGroup * kTileGroups); }
inline int64_t scale_bytes(int64_t rows, int64_t cols) { return (rows + kTileRows - 1) / kTileRows * tiles_of(cols) * kTileBytes; }

// The four scales of row r's tile t (`tiles` of them a row): where they lie, four neighbouring bytes.
__host__ __device__ __forceinline__ int64_t word_at(int64_t r, int64_t t, int64_t tiles) {
    return (r / kTileRows * tiles + t) * kTileBytes + r % 32 * 16 + r % kTileRows / 32 * 4;
}

#ifdef __CUDACC__

// The scale of a group whose largest magnitude has these bits (fp32): its power of two two lower, and 255 of infinities and NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest_bits) {
    const int e = (int)(largest_bits >> 23);
    return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// The factor that a group's values are divided by, as a product: 2^(127 - byte); exact, bytes are at most 252 (of 255 it is any number).
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float(byte == 255 ? 0x3f800000u : (254u - byte) << 23); }
// 2^(byte - 127); NaN of 255
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return __uint_as_float(byte == 255 ? 0x7fffffffu : byte == 0 ? 0x00400000u : byte << 23);
}

// N values, scaled already, as codes: value i in bits 4 i to 4 i + 3
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
__device__ __forceinline__ uint32_t codes4(const float (&v)[4]) {
    const float w[8] = {v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f};
    return codes8(w);
}
// The values of N codes.  A code's three bits at an fp32 number's lowest bits of exponent and highest of mantissa are 2^-126 times its value, 0.5 as a
// subnormal number too.  (The conversion instruction from pairs, of bytes picked out of a word, took the wrong byte as compiled here.)
template <int N>
__device__ __forceinline__ void values_of(uint32_t codes, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t c = codes >> (4 * i);
        v[i] = __fmul_rn(__uint_as_float((c & 7u) << 22 | (c & 8u) << 28), 8.507059173023462e37f);
    }
}

// A warp whose lanes hold neighbouring runs of kN values of a row (kN = 4 or 8, values that do not exist are zero) quantizes them: the lane's
// codes, and the word of scales of its tile, the same in all lanes of the tile.  most: the largest magnitude's bits of the lane's values.  All lanes take part.
template <int kN>
__device__ __forceinline__ uint32_t quantize_lanes(const float (&v)[kN], uint32_t most, uint32_t *scales) {
    constexpr int kLanes = kGroup / kN;          // of a group
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
    const uint32_t byte = scale_byte(most);
    const float by = inverse_scale(byte);
    float t[kN];
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
        const float2 r = mul2(make_float2(v[i], v[i + 1]), make_float2(by, by));
        t[i] = r.x;
        t[i + 1] = r.y;
    }
    uint32_t word = byte << (8 * ((threadIdx.x & 31) / kLanes % kTileGroups));
    word |= __shfl_xor_sync(0xffffffffu, word, kLanes);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanes);
    *scales = word;
    if constexpr (kN == 8) return codes8(t);
    else return codes4(t);
}
// The same of 16 bytes of a floating row, and of 32 neighbouring ones.
template <typename T>
__device__ __forceinline__ uint32_t quantize_vector(const uint4 &q, uint32_t *scales) {
    Largest<T> largest;
    largest.add(q);
    float v[Vec16<T>::kN];
    Vec16<T>::get(q, v);
    return quantize_lanes<Vec16<T>::kN>(v, largest.bits(), scales);
}
template <typename T>
__device__ __forceinline__ void quantize_bytes(const uint4 (&q)[2], uint32_t (&codes)[4 / sizeof(T)], uint32_t *scales) {
    constexpr int kHalf = Vec16<T>::kN, kLanes = kGroup / (2 * kHalf);
    Largest<T> largest;
    largest.add(q[0]);
    largest.add(q[1]);
    uint32_t most = largest.bits();
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
    const uint32_t byte = scale_byte(most);
    const float by = inverse_scale(byte);
    float t[2 * kHalf];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[kHalf];
        Vec16<T>::get(q[h], v);
#pragma unroll
        for (int i = 0; i < kHalf; i += 2) {
            const float2 r = mul2(make_float2(v[i], v[i + 1]), make_float2(by, by));
            t[h * kHalf + i] = r.x;
            t[h * kHalf + i + 1] = r.y;
        }
    }
    uint32_t word = byte << (8 * ((threadIdx.x & 31) / kLanes % kTileGroups));
    word |= __shfl_xor_sync(0xffffffffu, word, kLanes);
    word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanes);
    *scales = word;
#pragma unroll
    for (int h = 0; h < kHalf / 4; ++h) {
        const float some[8] = {t[8 * h], t[8 * h + 1], t[8 * h + 2], t[8 * h + 3], t[8 * h + 4], t[8 * h + 5], t[8 * h + 6], t[8 * h + 7]};
        codes[h] = codes8(some);
    }
}
// Eight codes as bf16 values (fp16: their upper bytes differ, their lower ones are zero), pairs of them: bytes out of tables by the codes themselves, a sign from a table whose
// every byte has its highest bit set, which a selector with the code's sign bit repeats.
template <typename T>
__device__ __forceinline__ void short_values8(uint32_t codes, uint32_t (&pairs)[4]) {
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t four = codes >> (16 * h), at = four & 0x7777u;
        uint32_t sign;                                       // 0x80, and 0xff of a negative code
        asm("prmt.b32 %0, %1, %1, %2;" : "=r"(sign) : "r"(0x80808080u), "r"(four));
        const uint32_t upper = (sign << 7 & 0x80808080u) | (kBf16 ? __byte_perm(0x3f3f3f00u, 0x40404040u, at) : __byte_perm(0x3e3c3800u, 0x46444240u, at));
        const uint32_t lower = kBf16 ? __byte_perm(0xc0800000u, 0xc0804000u, at) : 0u;
        pairs[2 * h] = __byte_perm(lower, upper, 0x5140);
        pairs[2 * h + 1] = __byte_perm(lower, upper, 0x7362);
    }
}
// 16 bytes of values of type T of a group with a scale: one rounding, to T
template <typename T>
__device__ __forceinline__ uint4 values_vector(uint32_t codes, uint32_t byte) {
    if constexpr (sizeof(T) == 4) {
        uint32_t pairs[4];
        short_values8<__nv_bfloat16>(codes, pairs);      // (four of the eight)
        const float by = scale_value(byte);
        float v[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 r = mul2(make_float2(__uint_as_float(pairs[i] << 16), __uint_as_float(pairs[i] & 0xffff0000u)), make_float2(by, by));
            v[2 * i] = r.x;
            v[2 * i + 1] = r.y;
        }
        return Vec16<T>::put(v);
    } else {
        uint32_t pairs[4];
        short_values8<T>(codes, pairs);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            // (every scale is a bf16 number)
            const uint32_t one = byte == 255 ? 0x7fffu : byte == 0 ? 0x0040u : byte << 7, by = one | one << 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&pairs[i]), *reinterpret_cast<const __nv_bfloat162 *>(&by));
                pairs[i] = *reinterpret_cast<const uint32_t *>(&r);
            }
        } else if (byte >= 113 && byte <= 142) {
            // (2^-14 to 2^15 are fp16's normal powers of two)
            const uint32_t one = (byte - 112) << 10, by = one | one << 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&pairs[i]), *reinterpret_cast<const __half2 *>(&by));
                pairs[i] = *reinterpret_cast<const uint32_t *>(&r);
            }
        } else {
            const float by = scale_value(byte);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&pairs[i]));
                const __half2 r = __floats2half2_rn(__fmul_rn(v.x, by), __fmul_rn(v.y, by));
                pairs[i] = *reinterpret_cast<const uint32_t *>(&r);
            }
        }
        return make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
    }
}
// Such a lane's codes to `to`, kN / 2 bytes
template <int kN>
__device__ __forceinline__ void store_codes(uint8_t *to, uint32_t codes, bool aligned) {
    if (aligned) {
        if constexpr (kN == 8) *reinterpret_cast<uint32_t *>(to) = codes;
        else *reinterpret_cast<uint16_t *>(to) = (uint16_t)codes;
    } else {
#pragma unroll
        for (int i = 0; i < kN / 2; ++i) to[i] = (uint8_t)(codes >> (8 * i));
    }
}
__device__ __forceinline__ void store_scales(uint8_t *to, uint32_t word, bool aligned) {
    if (aligned) *reinterpret_cast<uint32_t *>(to) = word;
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = (uint8_t)(word >> (8 * i));
}

// 16 bytes of a floating row from value c on: one load where `aligned`, else value by value; zeros at and behind the row's end
template <typename T>
__device__ __forceinline__ uint4 load_values(const T *row, int64_t c, int64_t cols, bool aligned) {
    constexpr int kN = Vec16<T>::kN;
    if (aligned && c + kN <= cols) return *reinterpret_cast<const uint4 *>(row + c);
    uint4 out = make_uint4(0, 0, 0, 0);
    T *v = reinterpret_cast<T *>(&out);
#pragma unroll
    for (int i = 0; i < kN; ++i)
        if (c + i < cols) v[i] = row[c + i];
    return out;
}

#endif  // __CUDACC__

}  // namespace mx
}  // namespace tsb
