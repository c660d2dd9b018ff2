// Root-mean-square norm of rows: the residual's addition in front of it, int8 or 4-bit rows for a product behind it, in one pass.
//
// Bound by memory: a row is read once (two tensors of it with a residual), held in registers as the sums' own type while the squares are added up, and written
// with its sum.  Squares are added in 64 bits: how a row is shared out, which goes by the number of rows and by alignment too, shows in the mean's 50th bit, and in the fp32
// reciprocal deviation, and so in the results, of fewer than one row in a million.  A row belongs to a warp, which needs no barrier, or to a block of as many warps as it needs: of many rows, threads with four
// vectors each (loads in flight), of few, more threads with one (a short way from load to store).
// Measured, bf16 rows of 16384 x 8192: 92 us (5.8 TB/s), with a residual 158 (6.8), to int8 143 (6.6; for seconds, at the power limit, 155 to 163), to 4 bits 136 (6.5), without a
// residual to int8 108 (3.7: instructions, two passes over gamma); 2048 x 4096 with a residual to 4 bits 12.7 us; 1 x 4096 2.5 us.
#include "mxfp4.cuh"

#include <algorithm>
#include <type_traits>

namespace tsb {
namespace {

constexpr int kWarpRowThreads = 128;      // rows of a warp each: threads of a block
constexpr int kMost = 1024;               // threads of a row, at most

enum Out { kSame, kInt8, kMxfp4 };

struct NormParams {
    const void *x, *residual;
    void *sum;
    const float *gamma;
    void *y, *scales;
    int64_t x_pitch, residual_pitch, sum_pitch, y_pitch, rows;
    double eps;
    int cols, tiles;                      // of scales in 4 bits
    int aligned, sum_aligned, y_aligned, gamma_aligned, scales_aligned;      // aligned: of what is read
};

// Where vector u of a row lies, N elements each.  WHOLE: such rows have 4 * kMost vectors at most, and an address and an unsigned offset of 32 bits are one instruction's
// operands; other rows may be longer than 2^32 bytes.
template <bool WHOLE, int N, typename E>
__device__ __forceinline__ E *vector_at(E *row, int u) {
    return WHOLE ? reinterpret_cast<E *>(reinterpret_cast<uintptr_t>(row) + (uint32_t)u * (uint32_t)(N * sizeof(E))) : row + (int64_t)u * N;
}

// Vector u of gamma; ones where there is none, and where a row has ended.  WHOLE: vectors are whole and lie on 16 bytes.
template <bool WHOLE, int N>
__device__ __forceinline__ void load_gamma(const NormParams &p, int u, float (&g)[N]) {
    if (p.gamma && (WHOLE || (p.gamma_aligned && u * N + N <= p.cols))) {
        const float4 *from = reinterpret_cast<const float4 *>(vector_at<WHOLE, N>(p.gamma, u));
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = from[i / 4];
            g[i] = v.x; g[i + 1] = v.y; g[i + 2] = v.z; g[i + 3] = v.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = !WHOLE && p.gamma && u * N + i < p.cols ? p.gamma[u * N + i] : 1.0f;
}

template <bool WHOLE, typename T>
__device__ __forceinline__ uint4 load_vector(const T *row, int u, int cols, bool aligned) {
    return WHOLE ? *reinterpret_cast<const uint4 *>(vector_at<WHOLE, Vec16<T>::kN>(row, u)) : mx::load_values(row, (int64_t)u * Vec16<T>::kN, cols, aligned);
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store_vector(T *row, int u, int cols, const uint4 &values, bool aligned) {
    constexpr int kN = Vec16<T>::kN;
    if (WHOLE || (aligned && u * kN + kN <= cols)) {
        *reinterpret_cast<uint4 *>(vector_at<WHOLE, kN>(row, u)) = values;
    } else {
        const T *v = reinterpret_cast<const T *>(&values);
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (u * kN + i < cols) row[u * kN + i] = v[i];
    }
}

template <typename T>
__device__ __forceinline__ uint4 add_rounded(const uint4 &a, const uint4 &b) {
    constexpr int kN = Vec16<T>::kN;
    float x[kN], r[kN];
    Vec16<T>::get(a, x);
    Vec16<T>::get(b, r);
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
        const float2 s = add2(make_float2(x[i], x[i + 1]), make_float2(r[i], r[i + 1]));
        x[i] = s.x;
        x[i + 1] = s.y;
    }
    return Vec16<T>::put(x);
}

// s + the squares of a vector, in 64 bits
template <typename T>
__device__ __forceinline__ double squares(const uint4 &h, double s) {
    constexpr int kN = Vec16<T>::kN;
    float x[kN];
    Vec16<T>::get(h, x);
#pragma unroll
    for (int i = 0; i < kN; ++i) s = fma((double)x[i], (double)x[i], s);
    return s;
}

// The reciprocal deviation from the squares' sums of the row's threads: of a warp, or of the block by way of `part` and `result`, where one warp alone takes
// the root and divides (in 64 bits these are some hundred instructions: done by all, a fifth of the kernel's).
template <bool WARP>
__device__ __forceinline__ float reciprocal_deviation(double s, const NormParams &p, double *part, float *result) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    if constexpr (WARP) return (float)(1.0 / sqrt(s / (double)p.cols + p.eps));
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = lane < warps ? part[lane] : 0.0;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) *result = (float)(1.0 / sqrt(s / (double)p.cols + p.eps));
    }
    __syncthreads();
    return *result;
}
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t most, uint32_t *part) {
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (!WARP) {
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) part[threadIdx.x >> 5] = most;
        __syncthreads();
        most = __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0);
    }
    return most;
}

// V: vectors a thread holds; 0: any number, read again for each use.  WARP: a row belongs to a warp, else to the block.  WHOLE: rows are whole 16-byte vectors that lie on
// 16 bytes, their results likewise (an instance of its own: checks of every vector are half of the instructions of the general one).
template <typename T, Out OUT, bool RES, int V, bool WARP, bool WHOLE>
__global__ void __launch_bounds__(WARP ? kWarpRowThreads : kMost)
rms_norm_kernel(const __grid_constant__ NormParams p) {
    constexpr int kN = Vec16<T>::kN;
    __shared__ double sums[kMost / 32];
    __shared__ uint32_t maxima[kMost / 32];
    __shared__ float deviation;
    pdl_sync();
    const int warps = blockDim.x >> 5, at = WARP ? threadIdx.x & 31 : threadIdx.x, step = WARP ? 32 : blockDim.x;
    // (4 bits: whole tiles of scales, so that all lanes of a warp that has any of a row take part)
    const int vectors = (p.cols + kN - 1) / kN, turns = (vectors + step - 1) / step;
    const int64_t first = WARP ? (int64_t)blockIdx.x * warps + (threadIdx.x >> 5) : blockIdx.x, stride = WARP ? (int64_t)gridDim.x * warps : gridDim.x;
    // (4 bits: the last 128 rows' scales have room for 128 rows, and what no row has is zero)
    const int64_t room_rows = OUT == kMxfp4 ? (p.rows + mx::kTileRows - 1) / mx::kTileRows * mx::kTileRows : p.rows;
    for (int64_t r = first; r < room_rows; r += stride) {
        if (OUT == kMxfp4 && r >= p.rows) {
            for (int t = at; t < p.tiles; t += step) mx::store_scales(static_cast<uint8_t *>(p.scales) + mx::word_at(r, t, p.tiles), 0, p.scales_aligned);
            continue;
        }
        const T *xr = static_cast<const T *>(p.x) + r * p.x_pitch;
        const T *rr = RES ? static_cast<const T *>(p.residual) + r * p.residual_pitch : nullptr;
        T *hr = RES && p.sum ? static_cast<T *>(p.sum) + r * p.sum_pitch : nullptr;
        // h from x and the residual, and h again where it is not held: of the sum, which may have taken the place of one of them
        auto fresh = [&](int u) {
            uint4 h = load_vector<WHOLE>(xr, u, p.cols, p.aligned);
            if constexpr (RES) h = add_rounded<T>(h, load_vector<WHOLE>(rr, u, p.cols, p.aligned));
            return h;
        };
        auto again = [&](int u) { return RES && hr ? load_vector<WHOLE>(const_cast<const T *>(hr), u, p.cols, p.sum_aligned) : fresh(u); };
        uint4 held[V > 0 ? V : 1];
        double s = 0.0;
        if constexpr (V > 0) {
            uint4 res[RES ? V : 1];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                held[i] = make_uint4(0, 0, 0, 0);
                if (at + i * step < vectors) held[i] = load_vector<WHOLE>(xr, at + i * step, p.cols, p.aligned);
                if constexpr (RES) {
                    res[i] = make_uint4(0, 0, 0, 0);
                    if (at + i * step < vectors) res[i] = load_vector<WHOLE>(rr, at + i * step, p.cols, p.aligned);
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if constexpr (RES) {
                    held[i] = add_rounded<T>(held[i], res[i]);
                    if (hr && at + i * step < vectors) store_vector<WHOLE>(hr, at + i * step, p.cols, held[i], p.sum_aligned);
                }
                s = squares<T>(held[i], s);
            }
        } else {
            for (int u = at; u < vectors; u += step) {
                const uint4 h = fresh(u);
                if (RES && hr) store_vector<WHOLE>(hr, u, p.cols, h, p.sum_aligned);
                s = squares<T>(h, s);
            }
        }
        const float by = reciprocal_deviation<WARP>(s, p, sums, &deviation);
        auto normed = [&](const uint4 &h, int u, float (&v)[kN]) {
            float g[kN];
            load_gamma<WHOLE>(p, u, g);
            Vec16<T>::get(h, v);
#pragma unroll
            for (int i = 0; i < kN; i += 2) {
                const float2 r = mul2(mul2(make_float2(v[i], v[i + 1]), make_float2(by, by)), make_float2(g[i], g[i + 1]));
                v[i] = r.x;
                v[i + 1] = r.y;
            }
        };
        // (a row that is not finite: what lies behind its end is NaN)
        auto clear_behind = [&](int u, float (&v)[kN]) {
            if (!WHOLE && (int64_t)u * kN + kN > p.cols)
#pragma unroll
                for (int i = 0; i < kN; ++i)
                    if ((int64_t)u * kN + i >= p.cols) v[i] = 0.0f;
        };
        auto largest = [&](const float (&v)[kN], float most) {
#pragma unroll
            for (int i = 0; i < kN; i += 2) most = max_magnitude(most, v[i], v[i + 1]);
            return most;
        };
        // body(turn, vector, its h): of all vectors; ALL: and of as many behind the row's end as the other lanes of a warp have
        auto each = [&](auto all, const auto &body) {
            if constexpr (V > 0) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (decltype(all)::value ? i < turns : at + i * step < vectors) body(i, at + i * step, held[i]);
            } else {
                for (int i = 0; i < turns; ++i) {
                    const int u = at + i * step;
                    if (decltype(all)::value || u < vectors) body(0, u, u < vectors ? again(u) : make_uint4(0, 0, 0, 0));
                }
            }
        };
        using Live = std::false_type;
        using All = std::true_type;
        if constexpr (OUT == kSame) {
            each(Live(), [&](int, int u, const uint4 &h) {
                float v[kN];
                normed(h, u, v);
                store_vector<WHOLE>(static_cast<T *>(p.y) + r * p.y_pitch, u, p.cols, Vec16<T>::put(v), p.y_aligned);
            });
        } else if constexpr (OUT == kInt8) {
            // (up to sixteen values are kept between the maximum and the rounding, so that gamma is read once; 32 of a thread's 64 registers would be too many)
            constexpr bool kKeep = V > 0 && V * kN <= 16;
            float most = 0.0f, kept[kKeep ? V : 1][kN];
            each(Live(), [&](int i, int u, const uint4 &h) {
                float (&v)[kN] = kept[kKeep ? i : 0];
                normed(h, u, v);
                clear_behind(u, v);
                most = largest(v, most);
            });
            const RowScale scale(row_max<WARP>(__float_as_uint(most), maxima));
            if (at == 0) static_cast<float *>(p.scales)[r] = scale.scale;
            int8_t *yr = static_cast<int8_t *>(p.y) + r * p.y_pitch;
            auto write = [&](auto finite, int i, int u, const uint4 &h) {
                float (&v)[kN] = kept[kKeep ? i : 0];
                if (!kKeep) normed(h, u, v);
                uint32_t w[kN / 4];
                quantize_values<decltype(finite)::value>(scale, v, w);
                int8_t *to = yr + (uint32_t)(u * kN);
                if (WHOLE || (p.y_aligned && u * kN + kN <= p.cols)) {
                    if constexpr (kN == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
                    else *reinterpret_cast<uint32_t *>(to) = w[0];
                } else {
#pragma unroll
                    for (int i = 0; i < kN; ++i)
                        if (u * kN + i < p.cols) to[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
                }
            };
            // (chosen once for a row)
            if (scale.finite) each(Live(), [&](int i, int u, const uint4 &h) { write(std::true_type(), i, u, h); });
            else each(Live(), [&](int i, int u, const uint4 &h) { write(std::false_type(), i, u, h); });
        } else {
            const int used = (p.cols + mx::kGroup - 1) / mx::kGroup * mx::kGroup;
            uint8_t *yr = static_cast<uint8_t *>(p.y) + r * p.y_pitch, *scales = static_cast<uint8_t *>(p.scales) + mx::word_at(r, 0, p.tiles);
            constexpr int kLanes = 128 / kN;      // of a tile of scales
            each(All(), [&](int, int u, const uint4 &h) {
                // (behind the row's end there is nothing of gamma to read)
                float v[kN] = {};
                if (u < vectors) {
                    normed(h, u, v);
                    clear_behind(u, v);
                }
                uint32_t word;
                const uint32_t codes = mx::quantize_lanes<kN>(v, __float_as_uint(largest(v, 0.0f)), &word);
                if (u * kN < used) mx::store_codes<kN>(yr + u * (kN / 2), codes, WHOLE || p.y_aligned);
                if (u % kLanes == 0 && u / kLanes < p.tiles) mx::store_scales(scales + u / kLanes * (int64_t)mx::kTileBytes, word, WHOLE || p.scales_aligned);
            });
        }
        if constexpr (!WARP) __syncthreads();      // (the next row's sums)
    }
}

template <typename T, Out OUT, bool RES>
int launch(const NormParams &p, cudaStream_t stream) {
    constexpr int kN = Vec16<T>::kN;
    const int vectors = ceil_div(p.cols, kN);
    const int64_t rows = OUT == kMxfp4 ? ceil_div64(p.rows, mx::kTileRows) * mx::kTileRows : p.rows;
    auto go = [&](auto kernel, int64_t blocks, int threads) {
        TSB_CUDA(launch_pdl(kernel, dim3((int)std::min<int64_t>(blocks, 148 * 64)), dim3(threads), 0, stream, p));
        TSB_LAUNCHED("rms_norm_kernel");
        return TSB_OK;
    };
    const bool whole = p.cols % kN == 0 && p.aligned && p.y_aligned && (p.sum_aligned || !p.sum) && p.gamma_aligned && p.scales_aligned;
    auto pick = [&](auto is_whole) {
        constexpr bool kWhole = decltype(is_whole)::value;
        if (vectors <= 32) return go(rms_norm_kernel<T, OUT, RES, 1, true, kWhole>, ceil_div64(rows, kWarpRowThreads / 32), kWarpRowThreads);
        if (vectors <= 64) return go(rms_norm_kernel<T, OUT, RES, 2, true, kWhole>, ceil_div64(rows, kWarpRowThreads / 32), kWarpRowThreads);
        if (vectors <= kMost && p.rows <= 148 * 2) return go(rms_norm_kernel<T, OUT, RES, 1, false, kWhole>, rows, round_up(vectors, 32));
        return go(rms_norm_kernel<T, OUT, RES, 4, false, kWhole>, rows, round_up(ceil_div(vectors, 4), 32));
    };
    if (vectors > 4 * kMost) return go(rms_norm_kernel<T, OUT, RES, 0, false, false>, rows, kMost);
    return whole ? pick(std::true_type()) : pick(std::false_type());
}

template <typename T, Out OUT>
int launch(const NormParams &p, cudaStream_t stream) { return p.residual ? launch<T, OUT, true>(p, stream) : launch<T, OUT, false>(p, stream); }
template <typename T>
int launch(const NormParams &p, int y_type, cudaStream_t stream) {
    return y_type == TSB_TYPE_I8 ? launch<T, kInt8>(p, stream) : y_type == TSB_TYPE_MXFP4 ? launch<T, kMxfp4>(p, stream) : launch<T, kSame>(p, stream);
}

}  // namespace

int rms_norm(const tsb_rms_norm_desc *d, cudaStream_t stream) {
    if (!d) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: null arguments");
    if (!is_float_type(d->x_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: x_type %d is no floating type", d->x_type);
    const bool int8 = d->y_type == TSB_TYPE_I8, mxfp4 = d->y_type == TSB_TYPE_MXFP4;
    if (!int8 && !mxfp4 && d->y_type != d->x_type) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: y_type %d is neither x's nor int8 nor 4 bits", d->y_type);
    if (d->rows < 0 || d->cols < 1 || d->cols > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: bad shape [%lld, %lld]", (long long)d->rows, (long long)d->cols);
    if (!(d->eps >= 0.0) || d->eps > 1.7976931348623157e308) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: eps is a number, not negative");
    if (d->sum && !d->residual) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: a sum without a residual is x itself");
    if (d->rows == 0) return TSB_OK;
    if (!d->x || !d->y || ((int8 || mxfp4) && !d->scales)) return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: null pointer");
    const size_t element = type_bytes(d->x_type);
    if ((reinterpret_cast<uintptr_t>(d->x) | reinterpret_cast<uintptr_t>(d->residual) | reinterpret_cast<uintptr_t>(d->sum)) % element || reinterpret_cast<uintptr_t>(d->gamma) % 4 ||
        (!int8 && !mxfp4 && reinterpret_cast<uintptr_t>(d->y) % element) || (int8 && reinterpret_cast<uintptr_t>(d->scales) % 4))
        return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: tensors must be aligned to their element");
    const int64_t y_cols = mxfp4 ? mx::row_bytes(d->cols) : d->cols;
    const int y_type = mxfp4 ? TSB_TYPE_I8 : d->y_type;
    if (d->rows > 1 && (d->x_pitch < 0 || (d->residual && d->residual_pitch < 0) || (d->sum && d->sum_pitch < d->cols) || d->y_pitch < y_cols))
        return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: rows overlap (pitch)");
    const bool many = d->rows > 1;
    if (extent_bytes(d->rows, many ? d->x_pitch : 0, d->cols, d->x_type) < 0 || (d->residual && extent_bytes(d->rows, many ? d->residual_pitch : 0, d->cols, d->x_type) < 0) ||
        (d->sum && extent_bytes(d->rows, many ? d->sum_pitch : 0, d->cols, d->x_type) < 0) || extent_bytes(d->rows, many ? d->y_pitch : 0, y_cols, y_type) < 0 ||
        d->rows > (int64_t)1 << 38)
        return fail(TSB_ERR_INVALID_ARGUMENT, "rms_norm: extent beyond the address range");
    NormParams p = {};
    p.x = d->x;
    p.residual = d->residual;
    p.sum = d->sum;
    p.gamma = d->gamma;
    p.y = d->y;
    p.scales = d->scales;
    p.x_pitch = many ? d->x_pitch : 0;      // (of a single row, never stepped by)
    p.residual_pitch = many ? d->residual_pitch : 0;
    p.sum_pitch = many ? d->sum_pitch : 0;
    p.y_pitch = many ? d->y_pitch : 0;
    p.rows = d->rows;
    p.eps = d->eps;
    p.cols = (int)d->cols;
    p.tiles = (int)mx::tiles_of(d->cols);
    p.aligned = aligned16(d->x, p.x_pitch, d->x_type) && (!d->residual || aligned16(d->residual, p.residual_pitch, d->x_type));
    p.sum_aligned = d->sum && aligned16(d->sum, p.sum_pitch, d->x_type);
    const int64_t unit = mxfp4 ? 4 : 16 / (int64_t)element;      // of a store to y, in elements (4 bits: bytes)
    p.y_aligned = reinterpret_cast<uintptr_t>(d->y) % (int8 || mxfp4 ? unit : 16) == 0 && p.y_pitch % unit == 0;
    p.gamma_aligned = reinterpret_cast<uintptr_t>(d->gamma) % 16 == 0;
    p.scales_aligned = reinterpret_cast<uintptr_t>(d->scales) % 4 == 0;
    switch (d->x_type) {
        case TSB_TYPE_F32: return launch<float>(p, d->y_type, stream);
        case TSB_TYPE_F16: return launch<__half>(p, d->y_type, stream);
        default: return launch<__nv_bfloat16>(p, d->y_type, stream);
    }
}

}  // namespace tsb
