// Group norm with an activation on channels-last tensors (no counterpart in the reference).
#include "typed.cuh"

#include <algorithm>
#include <cmath>

namespace tsb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxSplits = 64;

struct GroupNormParams {
    const void *x;
    void *y;
    int64_t x_pixel, x_image, y_pixel, y_image;   // elements
    const float *gamma, *beta;                    // or NULL
    int n, channels, groups, per;                 // per = channels of a group
    int64_t pixels;
    int splits;
    double eps;
    int activation;
    float leaky;
    int out_channels;                             // channels written: int8 outputs are padded with zeros
    int64_t rne_limit;                            // int8: values below this (in channel-major order) round half to even
    int nscales;
    float scales[TSB_MAX_REQUANT_SCALES];
};

// sums[image][split][group] = {sum, sum of squares} of the split's pixels.  Both in 64 bits: with 53 bits the difference of the mean
// square and the squared mean keeps 32-bit accuracy for means up to 10^4 deviations, in one pass and any order of summation.
template <typename T>
__global__ void __launch_bounds__(kThreads)
group_norm_sums_kernel(GroupNormParams p, double2 *__restrict__ sums) {
    __shared__ double2 part[kThreads];
    pdl_sync();
    const int split = blockIdx.x % p.splits, image = blockIdx.x / p.splits;
    const int64_t p0 = p.pixels * split / p.splits, p1 = p.pixels * (split + 1) / p.splits;
    const int lanes = min(p.channels, kThreads), rows = kThreads / lanes;
    const int lane = threadIdx.x % lanes, row = threadIdx.x / lanes;
    double2 *out = sums + ((int64_t)image * p.splits + split) * p.groups;
    for (int g = threadIdx.x; g < p.groups; g += kThreads) out[g] = make_double2(0.0, 0.0);
    for (int c0 = 0; c0 < p.channels; c0 += lanes) {
        double s = 0.0, ss = 0.0;
        if (c0 + lane < p.channels && row < rows) {
            const T *col = static_cast<const T *>(p.x) + image * p.x_image + c0 + lane;
            for (int64_t q = p0 + row; q < p1; q += rows) {
                const double v = (double)to_f32(col[q * p.x_pixel]);
                s += v;
                ss = fma(v, v, ss);
            }
        }
        __syncthreads();
        part[threadIdx.x] = make_double2(s, ss);
        __syncthreads();
        // a group's channels in this block of channels, by the one thread that owns the group
        const int c1 = min(c0 + lanes, p.channels);
        for (int g = threadIdx.x; g < p.groups; g += kThreads) {
            const int a = max(c0, g * p.per), b = min(c1, (g + 1) * p.per);
            double2 t = out[g];
            for (int c = a; c < b; ++c)
                for (int r = 0; r < rows; ++r) {
                    t.x += part[r * lanes + c - c0].x;
                    t.y += part[r * lanes + c - c0].y;
                }
            out[g] = t;
        }
    }
}

// stats[image][group] = {mean, 1 / sqrt(variance + eps)}, each rounded once
__global__ void __launch_bounds__(kThreads)
group_norm_stats_kernel(GroupNormParams p, const double2 *__restrict__ sums, float2 *__restrict__ stats) {
    pdl_sync();
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= (int64_t)p.n * p.groups) return;
    const int64_t image = i / p.groups, g = i % p.groups;
    double s = 0.0, ss = 0.0;
    for (int k = 0; k < p.splits; ++k) {
        const double2 t = sums[(image * p.splits + k) * p.groups + g];
        s += t.x;
        ss += t.y;
    }
    const double count = (double)p.pixels * p.per;
    const double mean = s / count;
    double var = fma(-mean, mean, ss / count);
    var = var < 0.0 ? 0.0 : var;
    stats[i] = make_float2((float)mean, (float)(1.0 / sqrt(var + p.eps)));
}

template <typename T, typename Y>
__global__ void __launch_bounds__(kThreads)
group_norm_apply_kernel(GroupNormParams p, const float2 *__restrict__ stats) {
    pdl_sync();
    const int64_t total = (int64_t)p.n * p.pixels * p.out_channels;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int c = (int)(i % p.out_channels);
        const int64_t q = i / p.out_channels % p.pixels, image = i / p.out_channels / p.pixels;
        Y *y = static_cast<Y *>(p.y) + image * p.y_image + q * p.y_pixel + c;
        if (c >= p.channels) {
            *y = Y(0);
            continue;
        }
        const float2 st = stats[image * p.groups + c / p.per];
        float v = __fmul_rn(__fsub_rn(to_f32(static_cast<const T *>(p.x)[image * p.x_image + q * p.x_pixel + c]), st.x), st.y);
        if (p.gamma) v = __fmul_rn(v, p.gamma[c]);
        if (p.beta) v = __fadd_rn(v, p.beta[c]);
        float one[1] = {v};
        activate<Y>(one, p.activation, p.leaky);
        v = one[0];
        if constexpr (sizeof(Y) == 1) {
            const int64_t at = (image * p.channels + c) * p.pixels + q;
            *y = (Y)q8(v, p.scales[p.nscales == 1 ? 0 : image], at < p.rne_limit);
        } else {
            *y = from_f32<Y>(v);
        }
    }
}

int check_desc(const tsb_group_norm_desc *d) {
    if (!d) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: null descriptor");
    if (d->n < 0 || d->pixels < 0 || d->channels < 1 || d->groups < 1 || d->channels > 1 << 24 || d->n > 1 << 24 || d->pixels > (int64_t)1 << 40)
        return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: bad shape [%lld, %lld, %lld]", (long long)d->n, (long long)d->pixels, (long long)d->channels);
    if (d->channels % d->groups) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: %lld channels do not make %lld groups", (long long)d->channels, (long long)d->groups);
    if (!is_float_type(d->x_type)) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: x_type %d is no floating type", d->x_type);
    if (d->y_type != d->x_type && d->y_type != TSB_TYPE_I8) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: y_type is x_type or TSB_TYPE_I8");
    if (d->activation < TSB_ACT_NONE || d->activation > TSB_ACT_GELU) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: unknown activation %d", d->activation);
    if (!(d->eps >= 0.0) || std::isinf(d->eps)) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: eps must be a number of at least 0");
    const bool i8 = d->y_type == TSB_TYPE_I8;
    if (i8) {
        if (!d->requant_scales_host || d->n_requant_scales < 1) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: int8 output needs requant_scales");
        if (d->n_requant_scales != 1 && d->n_requant_scales != d->n) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: requant_scales: one, or one per image");
        if (d->n_requant_scales > TSB_MAX_REQUANT_SCALES) return fail(TSB_ERR_UNSUPPORTED, "group_norm: more than %d requant_scales", TSB_MAX_REQUANT_SCALES);
    }
    if (d->n == 0 || d->pixels == 0) return TSB_OK;
    if (!d->x || !d->y) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: null pointer");
    if (reinterpret_cast<uintptr_t>(d->x) % type_bytes(d->x_type) || reinterpret_cast<uintptr_t>(d->y) % (i8 ? 16 : type_bytes(d->y_type)) ||
        (reinterpret_cast<uintptr_t>(d->gamma) | reinterpret_cast<uintptr_t>(d->beta)) % 4)
        return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: tensors must be aligned to their element, int8 outputs to 16 bytes");
    if (d->x_pixel_stride < 0 || d->x_image_stride < 0) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: negative stride");
    if (!i8 && ((d->pixels > 1 && d->y_pixel_stride < d->channels) || (d->n > 1 && d->y_image_stride < (d->pixels - 1) * d->y_pixel_stride + d->channels)))
        return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: output pixels or images that overlap or interleave");
    if ((__int128)d->n * d->pixels * (d->channels + 64) >> 60) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: tensor too large");
    const int64_t span[2][2] = {{d->x_pixel_stride, d->x_image_stride}, {i8 ? 0 : d->y_pixel_stride, i8 ? 0 : d->y_image_stride}};
    for (auto &s : span)
        if (((__int128)(d->n - 1) * s[1] + (__int128)(d->pixels - 1) * s[0] + d->channels) >> 60) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: extent beyond the address range");
    return TSB_OK;
}

// Parts that an image's pixels are summed in: some four blocks a multiprocessor over the whole batch, 64 values a thread or more.
int choose_splits(const tsb_group_norm_desc *d) {
    const int64_t by_work = ceil_div64(d->pixels * d->channels, 64 * kThreads), by_blocks = ceil_div64(148 * 4, d->n);
    return (int)std::max<int64_t>(1, std::min<int64_t>({by_work, by_blocks, d->pixels, kMaxSplits}));
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
size_t sums_bytes(const tsb_group_norm_desc *d) { return align256((size_t)d->n * choose_splits(d) * d->groups * sizeof(double2)); }

template <typename T, typename Y>
int launch(const GroupNormParams &p, double2 *sums, float2 *stats, cudaStream_t stream) {
    TSB_CUDA(launch_pdl(group_norm_sums_kernel<T>, dim3(p.n * p.splits), dim3(kThreads), 0, stream, p, sums));
    TSB_LAUNCHED("group_norm_sums_kernel");
    TSB_CUDA(launch_pdl(group_norm_stats_kernel, dim3((int)ceil_div64((int64_t)p.n * p.groups, kThreads)), dim3(kThreads), 0, stream, p, sums, stats));
    TSB_LAUNCHED("group_norm_stats_kernel");
    const int64_t values = (int64_t)p.n * p.pixels * p.out_channels;
    TSB_CUDA(launch_pdl(group_norm_apply_kernel<T, Y>, dim3((int)std::min<int64_t>(ceil_div64(values, kThreads), 148 * 64)), dim3(kThreads), 0, stream, p, stats));
    TSB_LAUNCHED("group_norm_apply_kernel");
    return TSB_OK;
}

}  // namespace

size_t group_norm_workspace_bytes(const tsb_group_norm_desc *d) {
    if (check_desc(d) != TSB_OK || d->n == 0 || d->pixels == 0) return 0;
    return sums_bytes(d) + align256((size_t)d->n * d->groups * sizeof(float2));
}

int group_norm_nhwc(const tsb_group_norm_desc *d, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    int st = check_desc(d);
    if (st != TSB_OK || d->n == 0 || d->pixels == 0) return st;
    const size_t need = group_norm_workspace_bytes(d);
    if (!workspace || workspace_bytes < need) return fail(TSB_ERR_WORKSPACE_TOO_SMALL, "group_norm: %zu bytes of workspace, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: the workspace must be 256-byte aligned");
    const bool i8 = d->y_type == TSB_TYPE_I8;
    GroupNormParams p = {};
    p.x = d->x;
    p.y = d->y;
    p.x_pixel = d->x_pixel_stride;
    p.x_image = d->x_image_stride;
    p.gamma = d->gamma;
    p.beta = d->beta;
    p.n = (int)d->n;
    p.channels = (int)d->channels;
    p.groups = (int)d->groups;
    p.per = p.channels / p.groups;
    p.pixels = d->pixels;
    p.splits = choose_splits(d);
    p.eps = d->eps;
    p.activation = d->activation;
    p.leaky = d->leaky_scale;
    p.out_channels = i8 ? tsb_padded_channels(p.channels) : p.channels;
    p.y_pixel = i8 ? p.out_channels : d->y_pixel_stride;
    p.y_image = i8 ? p.out_channels * d->pixels : d->y_image_stride;
    if (i8) {
        p.nscales = d->n_requant_scales;
        p.rne_limit = p.nscales == 1 ? d->n * d->pixels * d->channels / 8 * 8 : 0;
        for (int i = 0; i < p.nscales; ++i) p.scales[i] = d->requant_scales_host[i];
    }
    double2 *sums = static_cast<double2 *>(workspace);
    float2 *stats = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + sums_bytes(d));
    switch (d->x_type) {
        case TSB_TYPE_F32: return i8 ? launch<float, int8_t>(p, sums, stats, stream) : launch<float, float>(p, sums, stats, stream);
        case TSB_TYPE_F16: return i8 ? launch<__half, int8_t>(p, sums, stats, stream) : launch<__half, __half>(p, sums, stats, stream);
        default: return i8 ? launch<__nv_bfloat16, int8_t>(p, sums, stats, stream) : launch<__nv_bfloat16, __nv_bfloat16>(p, sums, stats, stream);
    }
}

}  // namespace tsb
