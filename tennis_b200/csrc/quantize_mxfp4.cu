// Rows in microscaled 4-bit floating point, and back.
//
// Bound by memory.  A warp takes neighbouring tiles of a row's 128 values, a 16-byte vector a lane: the largest magnitude of a group is found among the
// four or eight lanes that hold it, so nothing goes through shared memory.
#include "mxfp4.cuh"

#include <algorithm>

namespace tsb {
namespace {

constexpr int kThreads = 256;

// A warp's tiles: kLanes lanes each, kTurns times 32 / kLanes of them, one behind the other through rows of `tiles`
template <int kN>
struct Tiles {
    static constexpr int kLanes = 128 / kN, kAtOnce = 32 / kLanes, kTurns = 4;
    int64_t row;
    int tile;
    __device__ __forceinline__ explicit Tiles(int tiles) {
        const int64_t first = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (kAtOnce * kTurns) + (threadIdx.x & 31) / kLanes;
        row = first / tiles;
        tile = (int)(first - row * tiles);
    }
    __device__ __forceinline__ void next(int tiles) {
        tile += kAtOnce;
        while (tile >= tiles) {
            tile -= tiles;
            ++row;
        }
    }
};
template <int kN>
int64_t blocks_of(int64_t rows, int64_t tiles) {
    return ceil_div64(rows * tiles, (int64_t)Tiles<kN>::kAtOnce * Tiles<kN>::kTurns * (kThreads / 32));
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_mxfp4_kernel(const T *x, int64_t x_pitch, uint8_t *q, int64_t q_pitch, uint8_t *scales, int64_t rows, int64_t room_rows,
                           int64_t cols, int tiles, int x_aligned, int q_aligned, int s_aligned) {
    constexpr int kN = Vec16<T>::kN;
    using W = Tiles<kN>;
    pdl_sync();
    const int lane = threadIdx.x & 31;
    const int64_t used = (cols + mx::kGroup - 1) / mx::kGroup * mx::kGroup;      // values of a row with those that fill up its last group
    uint4 held[W::kTurns];
    W at(tiles);
#pragma unroll
    for (int i = 0; i < W::kTurns; ++i, at.next(tiles)) {
        held[i] = make_uint4(0, 0, 0, 0);
        if (at.row < rows) held[i] = mx::load_values(x + at.row * x_pitch, (int64_t)at.tile * 128 + lane % W::kLanes * kN, cols, x_aligned);
    }
    at = W(tiles);
#pragma unroll
    for (int i = 0; i < W::kTurns; ++i, at.next(tiles)) {
        float v[kN];
        Vec16<T>::get(held[i], v);
        uint32_t word;
        const uint32_t codes = mx::quantize_lanes<kN>(v, &word);
        const int64_t c = (int64_t)at.tile * 128 + lane % W::kLanes * kN;
        if (at.row < rows && c < used) mx::store_codes<kN>(q + at.row * q_pitch + c / 2, codes, q_aligned);
        if (at.row < room_rows && lane % W::kLanes == 0) mx::store_scales(scales + mx::word_at(at.row, at.tile, tiles), word, s_aligned);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
dequantize_rows_mxfp4_kernel(const uint8_t *q, int64_t q_pitch, const uint8_t *scales, T *y, int64_t y_pitch, int64_t rows, int64_t cols,
                             int tiles, int q_aligned, int y_aligned) {
    constexpr int kN = Vec16<T>::kN;
    using W = Tiles<kN>;
    pdl_sync();
    const int lane = threadIdx.x & 31;
    uint32_t codes[W::kTurns];
    uint8_t byte[W::kTurns];
    W at(tiles);
#pragma unroll
    for (int i = 0; i < W::kTurns; ++i, at.next(tiles)) {
        const int64_t c = (int64_t)at.tile * 128 + lane % W::kLanes * kN;
        codes[i] = byte[i] = 0;
        if (at.row < rows && c < cols) {
            const uint8_t *from = q + at.row * q_pitch + c / 2;
            if (q_aligned) {
                if constexpr (kN == 8) codes[i] = *reinterpret_cast<const uint32_t *>(from);
                else codes[i] = *reinterpret_cast<const uint16_t *>(from);
            } else {
#pragma unroll
                for (int b = 0; b < kN / 2; ++b) codes[i] |= (uint32_t)from[b] << (8 * b);
            }
            byte[i] = scales[mx::word_at(at.row, at.tile, tiles) + lane % W::kLanes * kN / mx::kGroup];
        }
    }
    at = W(tiles);
#pragma unroll
    for (int i = 0; i < W::kTurns; ++i, at.next(tiles)) {
        const int64_t c = (int64_t)at.tile * 128 + lane % W::kLanes * kN;
        if (at.row >= rows || c >= cols) continue;
        float v[kN];
        mx::values_of<kN>(codes[i], v);
        const float by = mx::scale_value(byte[i]);
#pragma unroll
        for (int j = 0; j < kN; ++j) v[j] = __fmul_rn(v[j], by);
        T *to = y + at.row * y_pitch + c;
        const uint4 out = Vec16<T>::put(v);
        if (y_aligned && c + kN <= cols) {
            *reinterpret_cast<uint4 *>(to) = out;
        } else {
            const T *o = reinterpret_cast<const T *>(&out);
#pragma unroll
            for (int j = 0; j < kN; ++j)
                if (c + j < cols) to[j] = o[j];
        }
    }
}

template <typename T>
int launch_quantize(const void *x, int64_t x_pitch, uint8_t *q, int64_t q_pitch, uint8_t *scales, int64_t rows, int64_t cols, cudaStream_t stream) {
    constexpr int kN = Vec16<T>::kN;
    const int64_t tiles = mx::tiles_of(cols), room_rows = ceil_div64(rows, mx::kTileRows) * mx::kTileRows, blocks = blocks_of<kN>(room_rows, tiles);
    if (blocks > INT32_MAX) return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows_mxfp4: too many values");
    const int x_aligned = aligned16(x, x_pitch, sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16);
    const int q_aligned = reinterpret_cast<uintptr_t>(q) % 4 == 0 && q_pitch % 4 == 0, s_aligned = reinterpret_cast<uintptr_t>(scales) % 4 == 0;
    TSB_CUDA(launch_pdl(quantize_rows_mxfp4_kernel<T>, dim3((int)blocks), dim3(kThreads), 0, stream, static_cast<const T *>(x), x_pitch, q, q_pitch, scales, rows, room_rows, cols,
                        (int)tiles, x_aligned, q_aligned, s_aligned));
    TSB_LAUNCHED("quantize_rows_mxfp4_kernel");
    return TSB_OK;
}

template <typename T>
int launch_dequantize(const uint8_t *q, int64_t q_pitch, const uint8_t *scales, void *y, int64_t y_pitch, int64_t rows, int64_t cols, cudaStream_t stream) {
    constexpr int kN = Vec16<T>::kN;
    const int64_t tiles = mx::tiles_of(cols), blocks = blocks_of<kN>(rows, tiles);
    if (blocks > INT32_MAX) return fail(TSB_ERR_INVALID_ARGUMENT, "dequantize_rows_mxfp4: too many values");
    const int q_aligned = reinterpret_cast<uintptr_t>(q) % 4 == 0 && q_pitch % 4 == 0, y_aligned = aligned16(y, y_pitch, sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16);
    TSB_CUDA(launch_pdl(dequantize_rows_mxfp4_kernel<T>, dim3((int)blocks), dim3(kThreads), 0, stream, q, q_pitch, scales, static_cast<T *>(y), y_pitch, rows, cols, (int)tiles,
                        q_aligned, y_aligned));
    TSB_LAUNCHED("dequantize_rows_mxfp4_kernel");
    return TSB_OK;
}

// What both directions ask of a 4-bit matrix and the floating one beside it (f: that one)
int check(const char *name, const void *q, int64_t q_pitch, const void *scales, const void *f, int type, int64_t f_pitch, bool f_is_read, int64_t rows, int64_t cols) {
    if (!is_float_type(type)) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: type %d is no floating type", name, type);
    if (rows < 0 || cols < 1 || cols > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: bad shape [%lld, %lld]", name, (long long)rows, (long long)cols);
    if (rows == 0) return TSB_OK;
    if (!q || !scales || !f) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (reinterpret_cast<uintptr_t>(f) % type_bytes(type)) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: tensors must be aligned to their element", name);
    if (rows > 1 && (f_pitch < (f_is_read ? 0 : cols) || q_pitch < (f_is_read ? mx::row_bytes(cols) : 0)))
        return fail(TSB_ERR_INVALID_ARGUMENT, "%s: rows overlap (pitch)", name);
    if (extent_bytes(rows, rows > 1 ? f_pitch : 0, cols, type) < 0 || extent_bytes(rows, rows > 1 ? q_pitch : 0, mx::row_bytes(cols), TSB_TYPE_I8) < 0 || rows > (int64_t)1 << 38)
        return fail(TSB_ERR_INVALID_ARGUMENT, "%s: extent beyond the address range", name);
    return TSB_OK;
}

}  // namespace

// Sizes that are none have no bytes.
int64_t mxfp4_row_bytes(int64_t cols) { return cols > 0 && cols <= INT32_MAX ? mx::row_bytes(cols) : 0; }
int64_t mxfp4_scale_bytes(int64_t rows, int64_t cols) { return rows > 0 && cols > 0 && rows <= (int64_t)1 << 38 && cols <= INT32_MAX ? mx::scale_bytes(rows, cols) : 0; }

int quantize_rows_mxfp4(const void *x, int x_type, int64_t x_pitch, void *q, int64_t q_pitch, void *scales, int64_t rows, int64_t cols, cudaStream_t stream) {
    const int st = check("quantize_rows_mxfp4", q, q_pitch, scales, x, x_type, x_pitch, true, rows, cols);
    if (st != TSB_OK || rows == 0) return st;
    if (rows == 1) x_pitch = q_pitch = 0;      // (never stepped by)
    uint8_t *to = static_cast<uint8_t *>(q), *s = static_cast<uint8_t *>(scales);
    switch (x_type) {
        case TSB_TYPE_F32: return launch_quantize<float>(x, x_pitch, to, q_pitch, s, rows, cols, stream);
        case TSB_TYPE_F16: return launch_quantize<__half>(x, x_pitch, to, q_pitch, s, rows, cols, stream);
        default: return launch_quantize<__nv_bfloat16>(x, x_pitch, to, q_pitch, s, rows, cols, stream);
    }
}

int dequantize_rows_mxfp4(const void *q, int64_t q_pitch, const void *scales, void *y, int y_type, int64_t y_pitch, int64_t rows, int64_t cols, cudaStream_t stream) {
    const int st = check("dequantize_rows_mxfp4", q, q_pitch, scales, y, y_type, y_pitch, false, rows, cols);
    if (st != TSB_OK || rows == 0) return st;
    if (rows == 1) y_pitch = q_pitch = 0;
    const uint8_t *from = static_cast<const uint8_t *>(q), *s = static_cast<const uint8_t *>(scales);
    switch (y_type) {
        case TSB_TYPE_F32: return launch_dequantize<float>(from, q_pitch, s, y, y_pitch, rows, cols, stream);
        case TSB_TYPE_F16: return launch_dequantize<__half>(from, q_pitch, s, y, y_pitch, rows, cols, stream);
        default: return launch_dequantize<__nv_bfloat16>(from, q_pitch, s, y, y_pitch, rows, cols, stream);
    }
}

}  // namespace tsb
