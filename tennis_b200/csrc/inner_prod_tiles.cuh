// What the tensor-core kernels of the inner products share, whatever their operands' type: the walk over tiles, the staged outputs and
// residuals of a warp, and the tensor maps.  P: an operator's parameters, with y, its residual, their pitches, m and n.
#pragma once

#include "tc_ptx.cuh"
#include "typed.cuh"

#include <cudaTypedefs.h>

#include <algorithm>

namespace tsb {
namespace tc {
namespace {

constexpr int kKBytes = 128;                 // bytes of K a stage
constexpr int kGroupM = 16;                  // token tiles that neighbouring CTAs share
constexpr uint32_t kABytes = kBM * kKBytes;
constexpr int kCh = 32;                      // channels of a step of the epilogue
constexpr uint32_t kOutRows = 2048;          // bytes of a step of a warp's
constexpr uint32_t kSmem = 227 * 1024;
constexpr int kMaxStages = 8;
constexpr uint32_t kScales = 1024;           // bytes of a stage's scales of 128 rows in 4 bits

// Tiles in the order in which CTAs take them.
struct Walk {
    int tiles_m, tiles_n, kblocks;
    int group_m;                  // token tiles that neighbouring CTAs share: a power of two
    uint32_t per_group, inverse;  // tiles of such a group, 2^32 / that
};

inline Walk walk_of(int tiles_m, int tiles_n, int kblocks) {
    Walk t = {tiles_m, tiles_n, kblocks, 0, 0, 0};
    // (of few output channels, tiles of the same tokens follow each other: then a CTA of an even grid stays with its channels)
    t.group_m = t.tiles_n <= 4 ? 1 : kGroupM;
    t.per_group = (uint32_t)(t.group_m * t.tiles_n);
    t.inverse = (uint32_t)std::min<uint64_t>(UINT32_MAX, ((uint64_t)1 << 32) / t.per_group);
    return t;
}

__device__ __forceinline__ void tile_of(const Walk &t, int i, int &m_tile, int &n_tile) {
    // (every warp of the epilogue does this for every tile: no division but in the last group)
    int g = (int)__umulhi((uint32_t)i, t.inverse), r = i - g * (int)t.per_group;      // the quotient or one less
    if (r >= (int)t.per_group) {
        ++g;
        r -= (int)t.per_group;
    }
    const int rows = t.tiles_m - g * t.group_m;
    n_tile = rows >= t.group_m ? r >> (31 - __clz(t.group_m)) : r / rows;
    m_tile = g * t.group_m + r - n_tile * min(rows, t.group_m);
}

// A warp's staged outputs, rows of CH channels: in the order of a tensor map's 64- or 128-byte swizzle, so that the fragments' writes (eight
// rows at a time, a 16-byte unit each or half a unit to a lane) and the rows' reads meet a bank once or twice.
template <typename T, int CH = kCh>
struct Staged {
    static constexpr int kRowBytes = CH * sizeof(T), kUnits = kRowBytes / 16;
    static constexpr int kRows = 2048 / kRowBytes;            // tokens of a step: 32 in rows of 64 bytes, 16 in rows of 128 bytes
    static __device__ __forceinline__ uint32_t unit(int r, int u) { return (uint32_t)(r * kRowBytes + ((u ^ (kUnits == 4 ? (r >> 1) & 3 : r & 7)) << 4)); }
    static __device__ __forceinline__ uint32_t value(int r, int c) { return unit(r, c * (int)sizeof(T) / 16) + c * (uint32_t)sizeof(T) % 16; }
};

// The residual of such a step into `rows`, once the copy that reads these rows last has done so.
template <typename T, int CH = kCh, typename P>
__device__ __forceinline__ void fetch_residual(const P &p, int64_t m0, int live, int c0, uint8_t *rows, bool res_vec) {
    using S = Staged<T, CH>;
    const int lane = threadIdx.x & 31;
    if (lane == 0) bulk_wait_read();
    __syncwarp();
    if (res_vec && c0 + CH <= p.n) {
        constexpr int kN = Vec16<T>::kN, kStep = 32 / S::kUnits;
        const int r0 = lane / S::kUnits, u0 = lane % S::kUnits;
        const T *from = static_cast<const T *>(p.residual) + (m0 + r0) * p.residual_pitch + c0 + u0 * kN;
        const int64_t step = kStep * p.residual_pitch;
#pragma unroll
        for (int r = 0; r < S::kRows; r += kStep, from += step)
            if (r + r0 < live) *reinterpret_cast<uint4 *>(rows + S::unit(r + r0, u0)) = *reinterpret_cast<const uint4 *>(from);
    } else {
        // value by value, neighbouring lanes neighbouring channels, as many loads under way as registers allow
        constexpr int kPieces = CH / 32, kAtOnce = CH == kCh ? 8 : 16;
        const T *from = static_cast<const T *>(p.residual) + m0 * p.residual_pitch + c0 + lane;
        T some[kPieces][kAtOnce];
        for (int r = 0; r < live; r += kAtOnce) {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i, from += p.residual_pitch)
#pragma unroll
                for (int c = 0; c < kPieces; ++c)
                    if (r + i < live && c0 + 32 * c + lane < p.n) some[c][i] = from[32 * c];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int c = 0; c < kPieces; ++c)
                    if (r + i < live && c0 + 32 * c + lane < p.n) *reinterpret_cast<T *>(rows + S::value(r + i, 32 * c + lane)) = some[c][i];
        }
    }
    __syncwarp();
}

// The same without waiting for it: whole pieces alone (whole_residual), by asynchronous copies, a group of them in any case.  (Of wider steps, whose 16-byte units are eight
// values, pieces of whole units too.)
template <int CH = kCh, typename P>
__device__ __forceinline__ bool whole_residual(const P &p, int c0, bool res_vec) { return res_vec && (c0 + CH <= p.n || (CH != kCh && p.n % 8 == 0)); }
template <typename T, int CH = kCh, typename P>
__device__ __forceinline__ void start_residual(const P &p, int64_t m0, int live, int c0, uint8_t *rows, bool res_vec) {
    using S = Staged<T, CH>;
    const int lane = threadIdx.x & 31;
    if (lane == 0) bulk_wait_read();
    __syncwarp();
    if (live > 0 && whole_residual<CH>(p, c0, res_vec)) {
        constexpr int kStep = 32 / S::kUnits;
        const int r0 = lane / S::kUnits, u0 = lane % S::kUnits;
        const T *from = static_cast<const T *>(p.residual) + (m0 + r0) * p.residual_pitch + c0 + u0 * Vec16<T>::kN;
        const int64_t step = kStep * p.residual_pitch;
#pragma unroll
        for (int r = 0; r < S::kRows; r += kStep, from += step)
            if (r + r0 < live && (CH == kCh || c0 + u0 * Vec16<T>::kN < p.n)) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(rows + S::unit(r + r0, u0))), "l"(from) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// cuTensorMapEncodeTiled, looked up once
inline PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// Tiles of `box_rows` rows x 128 bytes of a matrix of bytes.  (Rows shorter than that lie several to a line of the L2; where it fetches two lines for each of them, 100352 x 256 x 64 in 4 bits takes
// 16.1 us, with one 14.1, and in int8 20.9 and 19.4; rows of 128 bytes and more take the same time either way.)
inline int encode(CUtensorMap *map, const void *at, int64_t rows, int cols, int64_t pitch, int box_rows) {
    const auto fn = encode_tiled();
    if (!fn) return fail(TSB_ERR_UNSUPPORTED, "driver lacks cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? pitch : (cols + 15) / 16 * 16)};
    cuuint32_t box[2] = {(cuuint32_t)kKBytes, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(at), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, cols < kKBytes ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TSB_ERR_UNSUPPORTED, "inner product: cuTensorMapEncodeTiled failed with %d", (int)r);
    return TSB_OK;
}

// The boxes that a warp writes
template <typename T, int CH = kCh, typename P>
int encode_output(CUtensorMap *map, const P &p) {
    const auto fn = encode_tiled();
    if (!fn) return fail(TSB_ERR_UNSUPPORTED, "driver lacks cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)p.n, (cuuint64_t)p.m};
    cuuint64_t strides[1] = {(cuuint64_t)(p.m > 1 ? p.y_pitch * (int64_t)sizeof(T) : ((int64_t)p.n * (int64_t)sizeof(T) + 15) / 16 * 16)};
    cuuint32_t box[2] = {CH, Staged<T, CH>::kRows}, estr[2] = {1, 1};
    const CUresult r = fn(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          Staged<T, CH>::kRowBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TSB_ERR_UNSUPPORTED, "inner product: cuTensorMapEncodeTiled(y) failed with %d", (int)r);
    return TSB_OK;
}

// The scales of a 4-bit matrix as words of four: `tiles` runs of 128 a row of 128 rows' tiles; a box holds two runs of `box_rows` such rows
inline int encode_scales(CUtensorMap *map, const uint8_t *at, int64_t rows, int64_t tiles, int box_rows) {
    const auto fn = encode_tiled();
    if (!fn) return fail(TSB_ERR_UNSUPPORTED, "driver lacks cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)tiles * 128, (cuuint64_t)ceil_div64(rows, 128)}, strides[1] = {(cuuint64_t)tiles * 512};
    cuuint32_t box[2] = {256, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 2, const_cast<uint8_t *>(at), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TSB_ERR_UNSUPPORTED, "inner product: cuTensorMapEncodeTiled failed with %d", (int)r);
    return TSB_OK;
}

}  // namespace
}  // namespace tc
}  // namespace tsb
