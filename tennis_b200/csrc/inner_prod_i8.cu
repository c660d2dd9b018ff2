// int8 x int8 -> int32 inner product with a scale per token and per output channel (operator "inner_prod" of the reference,
// src/kernels/gpu/inner_prod.cu, on int8 operands).
#include "inner_prod_i8.h"

#include <algorithm>
#include <cstdio>

namespace tsb {
namespace {

// ---- CUDA-core kernel: any alignment, any pitch -----------------------------------------------------------------------
// A block computes 64 tokens x 64 output channels, 16 values a thread (4 x 4), 64 bytes of K at a time from shared memory.  Bound by dp4a and the
// shared-memory reads that feed it (8192^3 10.5 ms, 0.1 POPS): for operands that the copies of the other kernels cannot read.
constexpr int kTile = 64, kTileK = 64, kThreads = 256;
constexpr int kRow = kTileK / 4 + 1;      // words of a staged row; odd, so that neighbouring rows lie in different banks

// 16 bytes of a row from column k on; what lies at or behind the row's end (or in a row that does not exist) is zero
__device__ __forceinline__ void load16(const int8_t *row, bool exists, int k, int k_end, bool vec, uint32_t (&v)[4]) {
    v[0] = v[1] = v[2] = v[3] = 0;
    if (!exists || k >= k_end) return;
    if (vec && k + 16 <= k_end) {
        const uint4 t = __ldg(reinterpret_cast<const uint4 *>(row + k));
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < k_end) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
inner_prod_i8_direct_kernel(InnerProdParams p, int vec_x, int vec_w) {
    __shared__ uint32_t sx[kTile][kRow], sw[kTile][kRow];
    pdl_sync();
    const int n_tiles = (p.n + kTile - 1) / kTile;
    const int64_t tiles = (p.m + kTile - 1) / kTile * n_tiles;
    const int lr = threadIdx.x / 4, lk = threadIdx.x % 4 * 16;       // the row and the 16 bytes that this thread stages
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;          // its values: tokens tm + 16 i, channels tn + 16 j
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t m0 = t / n_tiles * kTile;
        const int n0 = (int)(t % n_tiles) * kTile;
        const bool has_x = m0 + lr < p.m, has_w = n0 + lr < p.n;
        const int8_t *xr = p.x + (has_x ? m0 + lr : 0) * p.x_pitch, *wr = p.w + (int64_t)(has_w ? n0 + lr : 0) * p.w_pitch;
        int acc[4][4] = {};
        for (int k0 = 0; k0 < p.k; k0 += kTileK) {
            uint32_t vx[4], vw[4];
            load16(xr, has_x, k0 + lk, p.k, vec_x, vx);
            load16(wr, has_w, k0 + lk, p.k, vec_w, vw);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sx[lr][lk / 4 + i] = vx[i];
                sw[lr][lk / 4 + i] = vw[i];
            }
            __syncthreads();
#pragma unroll 4
            for (int q = 0; q < kTileK / 4; ++q) {
                int a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = (int)sx[tm + 16 * i][q];
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = (int)sw[tn + 16 * j][q];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + tm + 16 * i;
            if (m >= p.m) continue;
            // (a channel that does not exist reads the last one's vectors and is not written)
            const int last = p.n - 1;
            auto at = [&](int j) { return min(n0 + tn + 16 * j, last); };
            float v[4];
            const float xs = p.x_scales[m * p.xs_stride];
            inner_prod_values<T>(p, acc[i],
                                 [&](int j) {
                                     return PairScales{make_float2(p.w_scales[at(j)], p.w_scales[at(j + 1)]), xs,
                                                       p.bias ? make_float2(p.bias[at(j)], p.bias[at(j + 1)]) : make_float2(0.0f, 0.0f)};
                                 },
                                 [&](int j) { return to_f32(static_cast<const T *>(p.residual)[m * p.residual_pitch + at(j)]); }, v);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + tn + 16 * j < p.n) static_cast<T *>(p.y)[m * p.y_pitch + n0 + tn + 16 * j] = from_f32<T>(v[j]);
        }
    }
}

template <typename T>
int launch_direct(const InnerProdParams &p, cudaStream_t stream) {
    const int64_t tiles = ceil_div64(p.m, kTile) * ceil_div64(p.n, kTile);
    const int grid = (int)std::min<int64_t>(tiles, 148 * 64);
    TSB_CUDA(launch_pdl(inner_prod_i8_direct_kernel<T>, dim3(grid), dim3(kThreads), 0, stream, p, (int)aligned16(p.x, p.x_pitch, TSB_TYPE_I8),
                        (int)aligned16(p.w, p.w_pitch, TSB_TYPE_I8)));
    TSB_LAUNCHED("inner_prod_i8_direct_kernel");
    return TSB_OK;
}

int check_args(const tsb_inner_prod_args *a) {
    if (!a) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: null arguments");
    if (a->m < 0 || a->n < 0 || a->n > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: bad shape [%lld, %lld]", (long long)a->m, (long long)a->n);
    // 131071 products of -128 x -128 are the most that an int32 sum holds
    if (a->k < 1 || a->k > 131071) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: k = %lld is not in 1..131071, the products that an int32 sum holds", (long long)a->k);
    if (a->x_type != TSB_TYPE_I8 && !is_float_type(a->x_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: unknown x_type %d", a->x_type);
    if (!is_float_type(a->y_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: y_type %d is no floating type", a->y_type);
    if (a->activation < TSB_ACT_NONE || a->activation > TSB_ACT_GELU) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: unknown activation %d", a->activation);
    if (a->kernel != TSB_KERNEL_AUTO && a->kernel != TSB_KERNEL_DIRECT && a->kernel != TSB_KERNEL_TCGEN05)
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: unknown kernel %d", a->kernel);
    if (a->m == 0 || a->n == 0) return TSB_OK;
    if (!a->x || !a->w || !a->w_scales || !a->y) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: null pointer");
    if ((a->x_type == TSB_TYPE_I8) != (a->x_scales != nullptr)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: int8 rows come with x_scales, floating rows without");
    const size_t ya = type_bytes(a->y_type);
    if (reinterpret_cast<uintptr_t>(a->x) % type_bytes(a->x_type) || reinterpret_cast<uintptr_t>(a->y) % ya || reinterpret_cast<uintptr_t>(a->residual) % ya ||
        (reinterpret_cast<uintptr_t>(a->x_scales) | reinterpret_cast<uintptr_t>(a->w_scales) | reinterpret_cast<uintptr_t>(a->bias)) % 4)
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: tensors must be aligned to their element");
    if (a->x_scales && (a->x_scales_stride < 0 || a->x_scales_stride > 1)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: x_scales_stride is 0 or 1");
    if ((a->m > 1 && (a->x_pitch < 0 || a->y_pitch < a->n || (a->residual && a->residual_pitch < 0))) || (a->n > 1 && a->w_pitch < 0))
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: bad pitch");
    if (extent_bytes(a->m, a->m > 1 ? a->x_pitch : 0, a->k, a->x_type) < 0 || extent_bytes(a->n, a->n > 1 ? a->w_pitch : 0, a->k, TSB_TYPE_I8) < 0 ||
        extent_bytes(a->m, a->m > 1 ? a->y_pitch : 0, a->n, a->y_type) < 0 || (a->residual && extent_bytes(a->m, a->m > 1 ? a->residual_pitch : 0, a->n, a->y_type) < 0) ||
        a->m > (int64_t)1 << 46)
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: extent beyond the address range");
    return TSB_OK;
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
int64_t rows_pitch(int64_t k) { return (k + 15) / 16 * 16; }

int run(const InnerProdParams &p, int y_type, int kernel, int early, cudaStream_t stream) {
    const char *why = "";
    const bool tc_can = tc::inner_prod_can(p, &why);
    if (kernel == TSB_KERNEL_TCGEN05 && !tc_can) return fail(TSB_ERR_UNSUPPORTED, "inner_prod_i8: no tensor-core kernel: %s", why);
    if (kernel == TSB_KERNEL_AUTO && tc_can && p.m <= few::kMaxTokens) return few::inner_prod(p, y_type, early, stream);
    if (kernel == TSB_KERNEL_TCGEN05 || (kernel == TSB_KERNEL_AUTO && tc_can)) return tc::inner_prod(p, y_type, stream);
    switch (y_type) {
        case TSB_TYPE_F32: return launch_direct<float>(p, stream);
        case TSB_TYPE_F16: return launch_direct<__half>(p, stream);
        default: return launch_direct<__nv_bfloat16>(p, stream);
    }
}

InnerProdParams params_of(const tsb_inner_prod_args *a) {
    InnerProdParams p = {};
    p.x = static_cast<const int8_t *>(a->x);
    p.x_pitch = a->m > 1 ? a->x_pitch : 0;      // (of a single row, never stepped by)
    p.w = a->w;
    p.w_pitch = a->n > 1 ? a->w_pitch : 0;
    p.x_scales = a->x_scales;
    p.xs_stride = a->x_scales_stride;
    p.w_scales = a->w_scales;
    p.bias = a->bias;
    p.residual = a->residual;
    p.residual_pitch = a->m > 1 ? a->residual_pitch : 0;
    p.y = a->y;
    p.y_pitch = a->m > 1 ? a->y_pitch : 0;
    p.m = a->m;
    p.n = (int)a->n;
    p.k = (int)a->k;
    p.activation = a->activation;
    p.leaky = a->leaky_scale;
    p.residual_after = a->residual && a->residual_after_activation ? 1 : 0;
    return p;
}

// Whether floating rows are quantized by the kernel that multiplies them.
bool quantizes_inside(const tsb_inner_prod_args *a, const InnerProdParams &p) {
    return a->kernel == TSB_KERNEL_AUTO && tc::weights_fit(p) && few::can_quantize(p, a->x_type, a->y_type);
}

// Workspace of floating rows: the rows as int8 (16-byte pitch), then their scales.
size_t workspace_of(const tsb_inner_prod_args *a, const InnerProdParams &p) {
    if (a->x_type == TSB_TYPE_I8 || quantizes_inside(a, p)) return 0;
    return align256((size_t)(a->m * rows_pitch(a->k))) + align256((size_t)a->m * 4);
}

}  // namespace

int quantize_rows_i8(const void *, int, int64_t, int8_t *, int64_t, float *, int64_t, int64_t, cudaStream_t);

size_t inner_prod_i8_workspace_bytes(const tsb_inner_prod_args *a) {
    return check_args(a) != TSB_OK || a->m == 0 || a->n == 0 ? 0 : workspace_of(a, params_of(a));
}

int inner_prod_i8(const tsb_inner_prod_args *a, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    int st = check_args(a);
    if (st != TSB_OK || a->m == 0 || a->n == 0) return st;
    InnerProdParams p = params_of(a);
    if (a->x_type == TSB_TYPE_I8) return run(p, a->y_type, a->kernel, 0, stream);
    if (quantizes_inside(a, p)) return few::inner_prod_quantize(p, a->y_type, stream);
    const size_t need = workspace_of(a, p);
    if (!workspace || workspace_bytes < need) return fail(TSB_ERR_WORKSPACE_TOO_SMALL, "inner_prod_i8: %zu bytes of workspace, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_i8: the workspace must be 256-byte aligned");
    int8_t *q = static_cast<int8_t *>(workspace);
    float *s = reinterpret_cast<float *>(q + align256((size_t)(a->m * rows_pitch(a->k))));
    st = quantize_rows_i8(a->x, a->x_type, a->x_pitch, q, rows_pitch(a->k), s, a->m, a->k, stream);
    if (st != TSB_OK) return st;
    p.x = q;
    p.x_pitch = rows_pitch(a->k);
    p.x_scales = s;
    p.xs_stride = 1;
    // The weights may be read early: quantize_rows lets the next kernel start only after all in front of it, and so whatever
    // wrote the weights, has completed.
    return run(p, a->y_type, a->kernel, 1, stream);
}

}  // namespace tsb
