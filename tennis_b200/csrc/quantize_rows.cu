// quantize with a scale for each row that is taken from the row (no counterpart in the reference, whose scales are attributes).
//
// Bound by memory: a row is read once, held in registers while its largest magnitude is found, and written as int8.  A row belongs to
// a warp, whose lanes hold up to two 16-byte vectors and need no barrier; or, where it is longer, to a block of as many warps as
// it needs -- of many rows, threads with four vectors each (loads in flight), of few, more threads with one (a short way from load to store).
// Measured: 32768 x 4096 fp16 67 us (6.0 TB/s), 16384 x 8192 fp32 122 us (5.5 TB/s), 1 x 2048 bf16 1.1 us.
#include "typed.cuh"

#include <algorithm>

namespace tsb {
namespace {

constexpr int kWarpRowThreads = 128;      // rows of a warp each: threads of a block
constexpr int kMost = 1024;               // threads of a row, at most

// Vector u of a row: one 16-byte load, or value by value where rows do not start on 16 bytes and at the row's end (zeros behind it,
// which change neither the maximum nor what is written).
template <typename T>
__device__ __forceinline__ uint4 load_vector(const T *row, int u, int cols, bool aligned) {
    constexpr int kN = Vec16<T>::kN;
    if (aligned && u * kN + kN <= cols) return __ldg(reinterpret_cast<const uint4 *>(row) + u);
    uint4 out = make_uint4(0, 0, 0, 0);
    T *v = reinterpret_cast<T *>(&out);
#pragma unroll
    for (int i = 0; i < kN; ++i)
        if (u * kN + i < cols) v[i] = row[u * kN + i];
    return out;
}

// Vector u as int8, in one store where the row starts on a multiple of its bytes.
template <typename T>
__device__ __forceinline__ void store_vector(const RowScale &scale, const uint4 &q, int8_t *row, int u, int cols, bool aligned) {
    constexpr int kN = Vec16<T>::kN;
    uint32_t w[kN / 4];
    quantize16<T>(scale, q, w);
    int8_t *to = row + u * kN;
    if (aligned && u * kN + kN <= cols) {
        if constexpr (kN == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(to) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (u * kN + i < cols) to[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
    }
}

// V: vectors a thread holds; 0: any number, read a second time.  WARP: a row belongs to a warp, else to the block.
template <typename T, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRowThreads : kMost)
quantize_rows_kernel(const T *__restrict__ x, int64_t x_pitch, int8_t *__restrict__ y, int64_t y_pitch, float *__restrict__ scales,
                     int64_t rows, int cols, int x_aligned, int y_aligned) {
    __shared__ uint32_t part[kMost / 32];
    pdl_sync();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int at = WARP ? lane : threadIdx.x, step = WARP ? 32 : blockDim.x;
    const int vectors = (cols + Vec16<T>::kN - 1) / Vec16<T>::kN;
    const int64_t first = WARP ? (int64_t)blockIdx.x * warps + warp : blockIdx.x, stride = WARP ? (int64_t)gridDim.x * warps : gridDim.x;
    for (int64_t r = first; r < rows; r += stride) {
        const T *xr = x + r * x_pitch;
        int8_t *yr = y + r * y_pitch;
        uint4 held[V > 0 ? V : 1];
        Largest<T> largest;
        if constexpr (V > 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                held[i] = make_uint4(0, 0, 0, 0);
                if (at + i * step < vectors) held[i] = load_vector(xr, at + i * step, cols, x_aligned);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) largest.add(held[i]);
        } else {
#pragma unroll 4
            for (int u = at; u < vectors; u += step) largest.add(load_vector(xr, u, cols, x_aligned));
        }
        uint32_t most = __reduce_max_sync(0xffffffffu, largest.bits());
        if constexpr (!WARP) {
            if (lane == 0) part[warp] = most;
            __syncthreads();
            most = __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0);
        }
        const RowScale scale(most);
        if (at == 0) scales[r] = scale.scale;
        if constexpr (V > 0) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (at + i * step < vectors) store_vector<T>(scale, held[i], yr, at + i * step, cols, y_aligned);
        } else {
#pragma unroll 4
            for (int u = at; u < vectors; u += step) store_vector<T>(scale, load_vector(xr, u, cols, x_aligned), yr, u, cols, y_aligned);
        }
        if constexpr (!WARP) __syncthreads();      // (the next row's maxima)
    }
}

template <typename T>
int launch(const void *x, int64_t x_pitch, int8_t *y, int64_t y_pitch, float *scales, int64_t rows, int cols, cudaStream_t stream) {
    constexpr int kN = Vec16<T>::kN;
    const int x_aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (x_pitch * (int64_t)sizeof(T)) % 16 == 0;
    const int y_aligned = reinterpret_cast<uintptr_t>(y) % kN == 0 && y_pitch % kN == 0;
    const int vectors = ceil_div(cols, kN);
    auto go = [&](auto kernel, int64_t blocks, int threads) {
        TSB_CUDA(launch_pdl(kernel, dim3((int)std::min<int64_t>(blocks, 148 * 64)), dim3(threads), 0, stream, static_cast<const T *>(x), x_pitch, y, y_pitch,
                            scales, rows, cols, x_aligned, y_aligned));
        TSB_LAUNCHED("quantize_rows_kernel");
        return TSB_OK;
    };
    // A warp a row, which needs no barrier, where a row is two vectors a lane or less (262144 x 256 fp32 57 us, by blocks 74; of longer rows
    // blocks are as fast or faster: 65536 x 1024 fp32 55 us, by warps 92, whose registers hold too few rows)
    if (vectors <= 32) return go(quantize_rows_kernel<T, 1, true>, ceil_div64(rows, kWarpRowThreads / 32), kWarpRowThreads);
    if (vectors <= 64) return go(quantize_rows_kernel<T, 2, true>, ceil_div64(rows, kWarpRowThreads / 32), kWarpRowThreads);
    if (vectors <= kMost && rows <= 148 * 2) return go(quantize_rows_kernel<T, 1, false>, rows, round_up(vectors, 32));
    if (vectors <= 4 * kMost) return go(quantize_rows_kernel<T, 4, false>, rows, round_up(ceil_div(vectors, 4), 32));
    return go(quantize_rows_kernel<T, 0, false>, rows, kMost);
}

}  // namespace

int quantize_rows_i8(const void *x, int x_type, int64_t x_pitch, int8_t *y, int64_t y_pitch, float *scales, int64_t rows, int64_t cols,
                     cudaStream_t stream) {
    if (!is_float_type(x_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows: x_type %d is no floating type", x_type);
    if (rows < 0 || cols < 1 || cols > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows: bad shape [%lld, %lld]", (long long)rows, (long long)cols);
    if (rows == 0) return TSB_OK;
    if (!x || !y || !scales) return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows: null pointer");
    if (reinterpret_cast<uintptr_t>(x) % type_bytes(x_type) || reinterpret_cast<uintptr_t>(scales) % 4)
        return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows: tensors must be aligned to their element");
    if (rows > 1 && (x_pitch < 0 || y_pitch < cols)) return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows: rows overlap (pitch below %lld)", (long long)cols);
    if (rows == 1) x_pitch = y_pitch = 0;      // (never stepped by)
    if (extent_bytes(rows, x_pitch, cols, x_type) < 0 || extent_bytes(rows, y_pitch, cols, TSB_TYPE_I8) < 0)
        return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows: extent beyond the address range");
    switch (x_type) {
        case TSB_TYPE_F32: return launch<float>(x, x_pitch, y, y_pitch, scales, rows, (int)cols, stream);
        case TSB_TYPE_F16: return launch<__half>(x, x_pitch, y, y_pitch, scales, rows, (int)cols, stream);
        default: return launch<__nv_bfloat16>(x, x_pitch, y, y_pitch, scales, rows, (int)cols, stream);
    }
}

}  // namespace tsb
