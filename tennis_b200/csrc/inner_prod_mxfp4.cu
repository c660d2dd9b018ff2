// Inner product on rows of 4-bit floating point with a scale for every 32 values (operator "inner_prod" of the reference,
// src/kernels/gpu/inner_prod.cu, on 4-bit operands).
#include "inner_prod_mxfp4.h"

#include <algorithm>

namespace tsb {
namespace {

// ---- CUDA-core kernel: any alignment, any pitch -----------------------------------------------------------------------
// A block computes 64 tokens x 64 output channels, 16 values a thread (4 x 4), two groups of K at a time as fp32 values in shared memory.  Bound by fused multiply-adds and
// the shared-memory reads that feed them (8192^3 43.7 ms): for operands that the copies of the other kernels cannot read.
// Under the two largest scales, 2^126 and 2^127, a value may lie beyond fp32 and its product with the other operand's not: where one of a block's groups has such a
// scale, values are staged without their scales, and a group's sum of products, which is exact then (at most 32 * 36, multiples of a quarter), joins the others times both scales.
constexpr int kTile = 64, kTileK = 64, kThreads = 256;
constexpr int kRow = kTileK + 1;         // words of a staged row; odd, so that neighbouring rows lie in different banks
constexpr int kTurnGroups = kTileK / mx::kGroup;      // of a turn of the loop over K
constexpr int kLarge = 253;              // the lowest byte of such a scale (255 is NaN, not one)

// Sixteen codes of a row, half of a group, and the byte of its scale; zeros where the row or the group does not exist.
struct Half {
    uint32_t codes[2] = {0, 0};
    int byte = 0;
    __device__ __forceinline__ Half(const uint8_t *q, int64_t pitch, const uint8_t *scales, int64_t r, bool exists, int k, int groups) {
        const int g = k / mx::kGroup;
        if (!exists || g >= groups) return;
        const uint8_t *from = q + r * pitch + k / 2;
        byte = scales[mx::word_at(r, g / mx::kTileGroups, (groups + mx::kTileGroups - 1) / mx::kTileGroups) + g % mx::kTileGroups];
#pragma unroll
        for (int b = 0; b < 8; ++b) codes[b / 4] |= (uint32_t)from[b] << (8 * (b % 4));
    }
    __device__ __forceinline__ bool large() const { return byte >= kLarge && byte < 255; }
    // its values, without their scale where they are kept `apart` from it, into a staged row
    __device__ __forceinline__ void stage(bool apart, float *to) const {
        const float by = mx::scale_value(apart && byte < 255 ? 127 : byte);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
            mx::values_of<8>(codes[h], v);
#pragma unroll
            for (int i = 0; i < 8; ++i) to[8 * h + i] = __fmul_rn(v[i], by);
        }
    }
};

// acc[i][j] + the products of values q0 to q1 - 1 of staged tokens tm + 16 i and channels tn + 16 j
__device__ __forceinline__ void multiply(const float (&sx)[kTile][kRow], const float (&sw)[kTile][kRow], int tm, int tn, int q0, int q1, float (&acc)[4][4]) {
#pragma unroll 4
    for (int q = q0; q < q1; ++q) {
        float a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = sx[tm + 16 * i][q];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = sw[tn + 16 * j][q];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
}

// sum + part * 2^e, one rounding.  part: 0, or from 2^-2 to 2^11 in magnitude (or NaN); beyond +-200 e is of no account: such a product is infinite, or nothing beside any sum.
__device__ __forceinline__ float add_scaled(float part, int e, float sum) {
    e = min(max(e, -200), 200);
    const int half = e >> 1;
    return fmaf(__fmul_rn(part, __int_as_float((half + 127) << 23)), __int_as_float((e - half + 127) << 23), sum);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
inner_prod_mxfp4_direct_kernel(const __grid_constant__ InnerProdMxfp4Params p) {
    __shared__ float sx[kTile][kRow], sw[kTile][kRow];
    __shared__ int ex[kTurnGroups][kTile], ew[kTurnGroups][kTile];   // exponents of the groups' scales, where values are staged without
    pdl_sync();
    const int n_tiles = (p.n + kTile - 1) / kTile;
    const int64_t tiles = (p.m + kTile - 1) / kTile * n_tiles;
    const int lr = threadIdx.x / 4, lk = threadIdx.x % 4 * 16;       // the row and the 16 values that this thread stages
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;          // its values: tokens tm + 16 i, channels tn + 16 j
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t m0 = t / n_tiles * kTile;
        const int n0 = (int)(t % n_tiles) * kTile;
        float acc[4][4] = {};
        for (int k0 = 0; k0 < p.groups * mx::kGroup; k0 += kTileK) {
            const Half x(p.x, p.x_pitch, p.x_scales, m0 + lr, m0 + lr < p.m, k0 + lk, p.groups), w(p.w, p.w_pitch, p.w_scales, n0 + lr, n0 + lr < p.n, k0 + lk, p.groups);
            const bool apart = __syncthreads_or(x.large() || w.large());      // (and nobody reads the staged values of the turn before any more)
            x.stage(apart, &sx[lr][lk]);
            w.stage(apart, &sw[lr][lk]);
            if (apart && lk % mx::kGroup == 0) {
                ex[lk / mx::kGroup][lr] = x.byte - 127;
                ew[lk / mx::kGroup][lr] = w.byte - 127;
            }
            __syncthreads();
            if (!apart) {
                multiply(sx, sw, tm, tn, 0, kTileK, acc);
                continue;
            }
#pragma unroll 1
            for (int g = 0; g < kTurnGroups; ++g) {
                float part[4][4] = {};
                multiply(sx, sw, tm, tn, g * mx::kGroup, (g + 1) * mx::kGroup, part);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = add_scaled(part[i][j], ex[g][tm + 16 * i] + ew[g][tn + 16 * j], acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + tm + 16 * i;
            if (m >= p.m) continue;
            // (a channel that does not exist reads the last one's bias and residual and is not written)
            auto at = [&](int j) { return min(n0 + tn + 16 * j, p.n - 1); };
            finish_values<T>(p, [&](int j) { return p.bias[at(j)]; }, [&](int j) { return to_f32(static_cast<const T *>(p.residual)[m * p.residual_pitch + at(j)]); }, acc[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + tn + 16 * j < p.n) static_cast<T *>(p.y)[m * p.y_pitch + n0 + tn + 16 * j] = from_f32<T>(acc[i][j]);
        }
    }
}

template <typename T>
int launch_direct(const InnerProdMxfp4Params &p, cudaStream_t stream) {
    const int64_t tiles = ceil_div64(p.m, kTile) * ceil_div64(p.n, kTile);
    const int grid = (int)std::min<int64_t>(tiles, 148 * 64);
    TSB_CUDA(launch_pdl(inner_prod_mxfp4_direct_kernel<T>, dim3(grid), dim3(kThreads), 0, stream, p));
    TSB_LAUNCHED("inner_prod_mxfp4_direct_kernel");
    return TSB_OK;
}

int check_args(const tsb_inner_prod_mxfp4_args *a) {
    if (!a) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: null arguments");
    if (a->m < 0 || a->n < 0 || a->n > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: bad shape [%lld, %lld]", (long long)a->m, (long long)a->n);
    if (a->k < 1 || a->k > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: bad k = %lld", (long long)a->k);
    if (a->x_type != TSB_TYPE_MXFP4 && !is_float_type(a->x_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: x_type %d is neither 4 bits nor a floating type", a->x_type);
    if (!is_float_type(a->y_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: y_type %d is no floating type", a->y_type);
    if (a->activation < TSB_ACT_NONE || a->activation > TSB_ACT_GELU) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: unknown activation %d", a->activation);
    if (a->kernel != TSB_KERNEL_AUTO && a->kernel != TSB_KERNEL_DIRECT && a->kernel != TSB_KERNEL_TCGEN05)
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: unknown kernel %d", a->kernel);
    if (a->m == 0 || a->n == 0) return TSB_OK;
    if (!a->x || !a->w || !a->w_scales || !a->y) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: null pointer");
    const bool floating = a->x_type != TSB_TYPE_MXFP4;
    if (floating == (a->x_scales != nullptr)) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: 4-bit rows come with x_scales, floating rows without");
    const size_t ya = type_bytes(a->y_type);
    if ((floating && reinterpret_cast<uintptr_t>(a->x) % type_bytes(a->x_type)) || reinterpret_cast<uintptr_t>(a->y) % ya || reinterpret_cast<uintptr_t>(a->residual) % ya ||
        reinterpret_cast<uintptr_t>(a->bias) % 4)
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: tensors must be aligned to their element");
    if ((a->m > 1 && (a->x_pitch < 0 || a->y_pitch < a->n || (a->residual && a->residual_pitch < 0))) || (a->n > 1 && a->w_pitch < 0))
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: bad pitch");
    const int64_t bytes = mx::row_bytes(a->k);
    if (extent_bytes(a->m, a->m > 1 ? a->x_pitch : 0, floating ? a->k : bytes, floating ? a->x_type : TSB_TYPE_I8) < 0 ||
        extent_bytes(a->n, a->n > 1 ? a->w_pitch : 0, bytes, TSB_TYPE_I8) < 0 || extent_bytes(a->m, a->m > 1 ? a->y_pitch : 0, a->n, a->y_type) < 0 ||
        (a->residual && extent_bytes(a->m, a->m > 1 ? a->residual_pitch : 0, a->n, a->y_type) < 0) || (floating && extent_bytes(a->m, bytes, bytes, TSB_TYPE_I8) < 0) ||
        a->m > (int64_t)1 << 38)
        return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: extent beyond the address range");
    return TSB_OK;
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

int run(const InnerProdMxfp4Params &p, int y_type, int kernel, int early, cudaStream_t stream) {
    const char *why = "";
    const bool tc_can = tc::inner_prod_can(p, &why);
    if (kernel == TSB_KERNEL_TCGEN05 && !tc_can) return fail(TSB_ERR_UNSUPPORTED, "inner_prod_mxfp4: no tensor-core kernel: %s", why);
    if (kernel == TSB_KERNEL_AUTO && tc_can && few::takes(p)) return few::inner_prod(p, y_type, early, stream);
    if (kernel != TSB_KERNEL_DIRECT && tc_can) return tc::inner_prod(p, y_type, stream);
    switch (y_type) {
        case TSB_TYPE_F32: return launch_direct<float>(p, stream);
        case TSB_TYPE_F16: return launch_direct<__half>(p, stream);
        default: return launch_direct<__nv_bfloat16>(p, stream);
    }
}

InnerProdMxfp4Params params_of(const tsb_inner_prod_mxfp4_args *a) {
    InnerProdMxfp4Params p = {};
    p.x = static_cast<const uint8_t *>(a->x);
    p.x_pitch = a->m > 1 ? a->x_pitch : 0;      // (of a single row, never stepped by)
    p.w = static_cast<const uint8_t *>(a->w);
    p.w_pitch = a->n > 1 ? a->w_pitch : 0;
    p.x_scales = static_cast<const uint8_t *>(a->x_scales);
    p.w_scales = static_cast<const uint8_t *>(a->w_scales);
    p.bias = a->bias;
    p.residual = a->residual;
    p.residual_pitch = a->m > 1 ? a->residual_pitch : 0;
    p.y = a->y;
    p.y_pitch = a->m > 1 ? a->y_pitch : 0;
    p.m = a->m;
    p.n = (int)a->n;
    p.groups = (int)((a->k + mx::kGroup - 1) / mx::kGroup);
    p.activation = a->activation;
    p.leaky = a->leaky_scale;
    p.residual_after = a->residual && a->residual_after_activation ? 1 : 0;
    return p;
}

// Whether floating rows are quantized by the kernel that multiplies them.
bool quantizes_inside(const tsb_inner_prod_mxfp4_args *a, const InnerProdMxfp4Params &p) {
    return a->kernel == TSB_KERNEL_AUTO && tc::weights_fit(p) && few::can_quantize(p, a->x_type, a->y_type);
}

// Workspace of floating rows: the rows in 4 bits, then their scales.
size_t workspace_of(const tsb_inner_prod_mxfp4_args *a, const InnerProdMxfp4Params &p) {
    if (a->x_type == TSB_TYPE_MXFP4 || quantizes_inside(a, p)) return 0;
    return align256((size_t)(a->m * mx::row_bytes(a->k))) + align256((size_t)mx::scale_bytes(a->m, a->k));
}

}  // namespace

int quantize_rows_mxfp4(const void *, int, int64_t, void *, int64_t, void *, int64_t, int64_t, cudaStream_t);

size_t inner_prod_mxfp4_workspace_bytes(const tsb_inner_prod_mxfp4_args *a) {
    return check_args(a) != TSB_OK || a->m == 0 || a->n == 0 ? 0 : workspace_of(a, params_of(a));
}

int inner_prod_mxfp4(const tsb_inner_prod_mxfp4_args *a, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    int st = check_args(a);
    if (st != TSB_OK || a->m == 0 || a->n == 0) return st;
    InnerProdMxfp4Params p = params_of(a);
    if (a->x_type == TSB_TYPE_MXFP4) return run(p, a->y_type, a->kernel, 0, stream);
    if (quantizes_inside(a, p)) return few::inner_prod_quantize(p, a->y_type, p.x_pitch, (int)a->k, stream);
    const size_t need = workspace_of(a, p);
    if (!workspace || workspace_bytes < need)
        return fail(TSB_ERR_WORKSPACE_TOO_SMALL, "inner_prod_mxfp4: %zu bytes of workspace, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TSB_ERR_INVALID_ARGUMENT, "inner_prod_mxfp4: the workspace must be 256-byte aligned");
    uint8_t *q = static_cast<uint8_t *>(workspace), *s = q + align256((size_t)(a->m * mx::row_bytes(a->k)));
    st = quantize_rows_mxfp4(a->x, a->x_type, a->x_pitch, q, mx::row_bytes(a->k), s, a->m, a->k, stream);
    if (st != TSB_OK) return st;
    p.x = q;
    p.x_pitch = a->m > 1 ? mx::row_bytes(a->k) : 0;
    p.x_scales = s;
    // The weights may be read early: quantize_rows_mxfp4 lets the next kernel start only after all in front of it, and so whatever wrote
    // the weights, has completed.
    return run(p, a->y_type, a->kernel, 1, stream);
}

}  // namespace tsb
