// quantize with a scale for each row that is taken from the row (no counterpart in the reference, whose scales are attributes).
#include "typed.cuh"

namespace tsb {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T *__restrict__ x, int64_t x_pitch, int8_t *__restrict__ y, int64_t y_pitch, float *__restrict__ scales,
                     int64_t rows, int cols) {
    __shared__ uint32_t part[kThreads / 32];
    pdl_sync();
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * x_pitch;
        uint32_t m = 0;
        for (int c = threadIdx.x; c < cols; c += kThreads) m = max(m, magnitude(to_f32(xr[c])));
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) m = max(m, part[i]);
        __syncthreads();
        const RowScale row(m);
        if (threadIdx.x == 0) scales[r] = row.scale;
        int8_t *yr = y + r * y_pitch;
        for (int c = threadIdx.x; c < cols; c += kThreads) yr[c] = (int8_t)row(to_f32(xr[c]));
    }
}

template <typename T>
int launch(const void *x, int64_t x_pitch, int8_t *y, int64_t y_pitch, float *scales, int64_t rows, int cols, cudaStream_t stream) {
    const int grid = (int)(rows < 148 * 64 ? rows : 148 * 64);
    TSB_CUDA(launch_pdl(quantize_rows_kernel<T>, dim3(grid), dim3(kThreads), 0, stream, static_cast<const T *>(x), x_pitch, y, y_pitch, scales, rows,
                        cols));
    TSB_LAUNCHED("quantize_rows_kernel");
    return TSB_OK;
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
