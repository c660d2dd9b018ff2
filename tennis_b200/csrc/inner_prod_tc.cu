// The int8 inner product on the sm_100a tensor cores: y [m, n] = x [m, k] . w [n, k], both operands K-major as they lie in memory.
//
//   tile       128 tokens x BN output channels, 128 bytes of K a stage: two TMA boxes (128-byte swizzle; rows and columns behind the
//              matrices' ends arrive as zeros) feed tcgen05.mma kind::i8, int32 sums in tensor memory, two buffers of them
//   roles      warp 0 loads, warp 1 issues the MMAs, sixteen warps (eight of narrow tiles) turn finished sums into outputs while the next
//              tile is computed
//   epilogue   a thread owns a token: tcgen05.ld gives it 64 bytes' worth of channels, the rows of a warp go through 2 KB of shared
//              memory so that residuals are read and outputs written in runs of 64 bytes
//   grid       persistent, one CTA per multiprocessor; neighbouring CTAs work on a block of kGroupM token tiles, whose operands
//              the L2 then serves
//
// Every wait on a barrier is bounded; one that runs out records a code in the status word, raises the CTA's abort flag, and
// all roles go to the common exit.
#include "inner_prod_i8.h"
#include "tc_ptx.cuh"

#include <cudaTypedefs.h>

#include <algorithm>

namespace tsb {
namespace tc {
namespace {

constexpr int kKBytes = 128;                 // bytes of K a stage
constexpr int kGroupM = 16;                  // token tiles that neighbouring CTAs share
constexpr uint32_t kABytes = kBM * kKBytes;
constexpr uint32_t kStageRow = 64;           // bytes of a staged output row: 32 channels of 2 bytes, 16 of 4
constexpr uint32_t kTableFloats = 64;        // a warp's scales and biases of as many channels
constexpr uint32_t kSmem = 227 * 1024;
constexpr int kMaxStages = 8;

// code of the wait that ran out: 1 stage free, 2 stage full, 3 sums free, 4 sums complete
__device__ int g_status;

struct TcParams {
    InnerProdParams p;
    int tiles_m, tiles_n, kblocks, stages;
};

template <int BN>
struct Layout {
    static constexpr int kEpiWarps = BN >= 128 ? 16 : 8;                          // four (or two) share the channels of a tile
    static constexpr int kThreads = 32 * (2 + kEpiWarps);
    static constexpr uint32_t kBBytes = BN * kKBytes;
    static constexpr uint32_t kStage = kABytes + kBBytes;
    static constexpr uint32_t kOut = kEpiWarps * 32 * kStageRow;                  // staged output rows
    static constexpr uint32_t kTables = kEpiWarps * kTableFloats * 4;
    static constexpr uint32_t kBars = 256;
    static constexpr int kStages = (int)((kSmem - 1024 - kOut - kTables - kBars) / kStage) < kMaxStages
                                       ? (int)((kSmem - 1024 - kOut - kTables - kBars) / kStage) : kMaxStages;
    static constexpr uint32_t kBytes = 1024 + kStages * kStage + kOut + kTables + kBars;
};

__device__ __forceinline__ void tile_of(const TcParams &t, int i, int &m_tile, int &n_tile) {
    const int per_group = kGroupM * t.tiles_n;
    const int g = i / per_group, r = i - g * per_group;
    const int rows = min(kGroupM, t.tiles_m - g * kGroupM);
    n_tile = r / rows;
    m_tile = g * kGroupM + r - n_tile * rows;
}

// The 16-byte unit u of row r of a warp's staged rows (four units): the units of eight neighbouring rows lie in different banks.
__device__ __forceinline__ uint32_t staged(int r, int u) { return (uint32_t)(r * kStageRow + ((u ^ ((r >> 1) & 3)) << 4)); }

// CH = 64 bytes of channels of a warp's 32 tokens: sums in tensor memory at `taddr` -> y.  m0, c0: the first token and channel.
template <typename T>
__device__ __forceinline__ void epilogue_chunk(const InnerProdParams &p, uint32_t taddr, int64_t m0, int c0, float xs, uint8_t *rows, float *table, bool y_vec, bool res_vec) {
    constexpr int kN = Vec16<T>::kN, CH = kStageRow / sizeof(T);        // values of a 16-byte unit, of a row
    const int lane = threadIdx.x & 31;
    const int live = (int)min((int64_t)32, p.m - m0), cols = min(CH, p.n - c0);
    if (lane < CH) {
        table[lane] = c0 + lane < p.n ? __ldg(p.w_scales + c0 + lane) : 0.0f;
        table[CH + lane] = c0 + lane < p.n && p.bias ? __ldg(p.bias + c0 + lane) : 0.0f;
    }
    int acc[CH];
    if constexpr (CH == 32) tmem_ld32(taddr, acc);
    else tmem_ld16(taddr, acc);
    if (p.residual) {
        const T *res = static_cast<const T *>(p.residual) + m0 * p.residual_pitch + c0;
        if (res_vec && cols == CH) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + lane / 4, u = lane % 4;
                if (r < live) *reinterpret_cast<uint4 *>(rows + staged(r, u)) = *reinterpret_cast<const uint4 *>(res + r * p.residual_pitch + u * kN);
            }
        } else {
            // value by value, neighbouring lanes neighbouring channels
            constexpr int kRows = 32 / CH;
            const int c = lane % CH;
#pragma unroll 4
            for (int r = lane / CH; r < live; r += kRows)
                if (c < cols) reinterpret_cast<T *>(rows + staged(r, c / kN))[c % kN] = res[r * p.residual_pitch + c];
        }
    }
    __syncwarp();
    float v[CH], res[CH];
    if (p.residual) {
#pragma unroll
        for (int u = 0; u < 4; ++u) Vec16<T>::get(*reinterpret_cast<const uint4 *>(rows + staged(lane, u)), *reinterpret_cast<float (*)[kN]>(&res[u * kN]));
    }
    tmem_ld_wait();
    inner_prod_values<T>(p, acc, xs, [&](int j) { return table[j]; }, [&](int j) { return table[CH + j]; }, [&](int j) { return res[j]; }, v);
#pragma unroll
    for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4 *>(rows + staged(lane, u)) = Vec16<T>::put(*reinterpret_cast<float (*)[kN]>(&v[u * kN]));
    __syncwarp();
    T *y = static_cast<T *>(p.y) + m0 * p.y_pitch + c0;
    if (y_vec && cols == CH) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + lane / 4, u = lane % 4;
            if (r < live) *reinterpret_cast<uint4 *>(y + r * p.y_pitch + u * kN) = *reinterpret_cast<const uint4 *>(rows + staged(r, u));
        }
    } else {
        constexpr int kRows = 32 / CH;
        const int c = lane % CH;
#pragma unroll 4
        for (int r = lane / CH; r < live; r += kRows)
            if (c < cols) y[r * p.y_pitch + c] = reinterpret_cast<const T *>(rows + staged(r, c / kN))[c % kN];
    }
    __syncwarp();
}

template <typename T, int BN>
__global__ void __launch_bounds__(Layout<BN>::kThreads, 1)
inner_prod_i8_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TcParams t,
                        int y_vec, int res_vec) {
    using L = Layout<BN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *out_rows = smem_raw + (base - raw) + L::kStages * L::kStage;
    float *tables = reinterpret_cast<float *>(out_rows + L::kOut);
    uint8_t *bars_ptr = out_rows + L::kOut + L::kTables;
    const uint32_t bar_full = smem_u32(bars_ptr), bar_empty = bar_full + 8 * kMaxStages, bar_tfull = bar_empty + 8 * kMaxStages, bar_tempty = bar_tfull + 16;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars_ptr + 8 * (2 * kMaxStages + 4));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars_ptr + 8 * (2 * kMaxStages + 4) + 4);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int tiles = t.tiles_m * t.tiles_n;

    if (warp == 0) {
        if (lane < L::kStages) {
            mbar_init(bar_full + 8 * lane, 1);
            mbar_init(bar_empty + 8 * lane, 1);
        }
        if (lane < 2) {
            mbar_init(bar_tfull + 8 * lane, 1);
            mbar_init(bar_tempty + 8 * lane, L::kEpiWarps);
        }
        if (lane == 0) {
            *abort_flag = 0;
            prefetch_tensormap(&map_x);
            prefetch_tensormap(&map_w);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_sync();
    auto give_up = [&](int code) {
        if (!*abort_flag) { *abort_flag = 1; atomicExch(&g_status, code); }
    };

    if (warp == 0) {
        uint32_t s = 0;
        for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
            int mt, nt;
            tile_of(t, i, mt, nt);
            for (int kb = 0; kb < t.kblocks; ++kb, ++s) {
                const uint32_t stage = s % L::kStages, round = s / L::kStages;
                if (!mbar_wait_warp(bar_empty + 8 * stage, (round & 1) ^ 1, abort_flag)) { give_up(1); goto done; }
                if (elect_one()) {
                    mbar_arrive_expect_tx(bar_full + 8 * stage, L::kStage);
                    tma_load_2d(base + stage * L::kStage, &map_x, bar_full + 8 * stage, kb * kKBytes, mt * kBM);
                    tma_load_2d(base + stage * L::kStage + kABytes, &map_w, bar_full + 8 * stage, kb * kKBytes, nt * BN);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        uint32_t s = 0, n = 0;
        constexpr uint64_t kDescHi = smem_desc_hi<kKBytes>(8 * kKBytes);
        for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++n) {
            const uint32_t acc = n & 1;
            if (!mbar_wait_warp(bar_tempty + 8 * acc, ((n >> 1) & 1) ^ 1, abort_flag)) { give_up(3); goto done; }
            tc_fence_after();
            for (int kb = 0; kb < t.kblocks; ++kb, ++s) {
                const uint32_t stage = s % L::kStages, round = s / L::kStages;
                if (!mbar_wait_warp(bar_full + 8 * stage, round & 1, abort_flag)) { give_up(2); goto done; }
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t a = kDescHi | ((base + stage * L::kStage) >> 4), b = kDescHi | ((base + stage * L::kStage + kABytes) >> 4);
#pragma unroll
                    for (int q = 0; q < kKBytes / 32; ++q) mma_i8(tmem + acc * BN, a + 2 * q, b + 2 * q, instr_desc<BN>(), kb > 0 || q > 0);
                    tc_commit(bar_empty + 8 * stage);
                    if (kb == t.kblocks - 1) tc_commit(bar_tfull + 8 * acc);
                }
                __syncwarp();
            }
        }
    } else {
        const int e = warp - 2, quarter = warp & 3;      // tensor memory lanes of this warp: 32 * (warp % 4)
        constexpr int kShare = BN / (L::kEpiWarps / 4), kCh = kStageRow / sizeof(T);
        const int share = e / 4 * kShare;                // its channels of the tile
        uint8_t *rows = out_rows + e * 32 * kStageRow;
        float *table = tables + e * kTableFloats;
        uint32_t n = 0;
        for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++n) {
            int mt, nt;
            tile_of(t, i, mt, nt);
            const uint32_t acc = n & 1;
            const int64_t m0 = (int64_t)mt * kBM + quarter * 32;
            const float xs = m0 + lane < t.p.m ? t.p.x_scales[(m0 + lane) * t.p.xs_stride] : 0.0f;
            if (!mbar_wait_warp(bar_tfull + 8 * acc, (n >> 1) & 1, abort_flag)) { give_up(4); goto done; }
            tc_fence_after();
            if (m0 < t.p.m)
                for (int c = share; c < share + kShare && nt * BN + c < t.p.n; c += kCh)
                    epilogue_chunk<T>(t.p, tmem + acc * BN + ((uint32_t)(quarter * 32) << 16) + c, m0, nt * BN + c, xs, rows, table, y_vec != 0, res_vec != 0);
            tc_fence_before();
            if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
            __syncwarp();
        }
    }
done:
    if (*abort_flag) {
        // copies that may still be in flight get time to land before shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// cuTensorMapEncodeTiled, looked up once
PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// Tiles of `box_rows` rows x 128 bytes of an int8 matrix
int encode(CUtensorMap *map, const int8_t *at, int64_t rows, int cols, int64_t pitch, int box_rows) {
    const auto fn = encode_tiled();
    if (!fn) return fail(TSB_ERR_UNSUPPORTED, "driver lacks cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? pitch : (cols + 15) / 16 * 16)};
    cuuint32_t box[2] = {(cuuint32_t)kKBytes, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(at), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TSB_ERR_UNSUPPORTED, "inner_prod_i8: cuTensorMapEncodeTiled failed with %d", (int)r);
    return TSB_OK;
}

template <typename T, int BN>
int launch(const InnerProdParams &p, cudaStream_t stream) {
    using L = Layout<BN>;
    CUtensorMap mx, mw;
    int st = encode(&mx, p.x, p.m, p.k, p.x_pitch, kBM);
    if (st == TSB_OK) st = encode(&mw, p.w, p.n, p.k, p.w_pitch, BN);
    if (st != TSB_OK) return st;
    auto kernel = inner_prod_i8_tc_kernel<T, BN>;
    static DeviceOnce raised;
    if (raised.first()) {
        TSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes));
        raised.done();
    }
    TcParams t = {p, (int)ceil_div64(p.m, kBM), ceil_div(p.n, BN), ceil_div(p.k, kKBytes), L::kStages};
    const int type = sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16;
    const int y_vec = aligned16(p.y, p.y_pitch, type), res_vec = p.residual && aligned16(p.residual, p.residual_pitch, type);
    const int grid = (int)std::min<int64_t>((int64_t)t.tiles_m * t.tiles_n, 148);
    TSB_CUDA(launch_pdl(kernel, dim3(grid), dim3(L::kThreads), L::kBytes, stream, mx, mw, t, y_vec, res_vec));
    TSB_LAUNCHED("inner_prod_i8_tc_kernel");
    return TSB_OK;
}

template <typename T>
int pick(const InnerProdParams &p, cudaStream_t stream) {
    if (p.n <= 64) return launch<T, 64>(p, stream);
    if (p.n <= 128 || ceil_div64(p.m, kBM) * ceil_div(p.n, 256) < 148) return launch<T, 128>(p, stream);
    return launch<T, 256>(p, stream);
}

}  // namespace

namespace {
bool operand_fits(const int8_t *at, int64_t rows, int64_t pitch, int k) {
    return reinterpret_cast<uintptr_t>(at) % 16 == 0 && (rows == 1 || (pitch % 16 == 0 && pitch >= k && pitch < (int64_t)1 << 40));
}
}  // namespace

bool weights_fit(const InnerProdParams &p) { return operand_fits(p.w, p.n, p.w_pitch, p.k); }

bool inner_prod_can(const InnerProdParams &p, const char **why) {
    if (!operand_fits(p.x, p.m, p.x_pitch, p.k) || !weights_fit(p)) { *why = "an operand's address or pitch is no multiple of 16 bytes, or its rows overlap"; return false; }
    if (ceil_div64(p.m, kBM) * ceil_div(p.n, 64) > INT32_MAX / 2) { *why = "too many tiles"; return false; }
    return true;
}

int inner_prod(const InnerProdParams &p, int y_type, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick<float>(p, stream);
        case TSB_TYPE_F16: return pick<__half>(p, stream);
        default: return pick<__nv_bfloat16>(p, stream);
    }
}

// The device's status word: waits for the stream, reads and clears it.
int inner_prod_status(cudaStream_t stream) {
    int word = 0, zero = 0;
    void *at = nullptr;
    TSB_CUDA(cudaGetSymbolAddress(&at, g_status));
    TSB_CUDA(cudaMemcpyAsync(&word, at, sizeof(word), cudaMemcpyDeviceToHost, stream));
    TSB_CUDA(cudaStreamSynchronize(stream));
    if (word == 0) return TSB_OK;
    TSB_CUDA(cudaMemcpyAsync(at, &zero, sizeof(zero), cudaMemcpyHostToDevice, stream));
    TSB_CUDA(cudaStreamSynchronize(stream));
    static const char *const kWaits[] = {"a stage to be free", "a stage to be loaded", "sums to be read", "sums to be complete"};
    return fail(TSB_ERR_DEVICE_TIMEOUT, "inner_prod_i8: the wait for %s ran out; results since the last check are not to be used",
                word >= 1 && word <= 4 ? kWaits[word - 1] : "an unknown event");
}

}  // namespace tc
}  // namespace tsb
