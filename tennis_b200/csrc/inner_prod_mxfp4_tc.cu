// The 4-bit inner product on the sm_100a tensor cores: y [m, n] = x [m, k] . w [n, k], both operands K-major as they lie in memory.
//
//   tile       128 tokens x BN output channels, or 256 x 256 of two CTAs, each with its half of both operands; 256 values of K a stage (128 bytes of a
//              row): boxes of both operands (128-byte swizzle; rows and columns behind the matrices' ends arrive as zeros) and of their tiles of scales
//              feed tcgen05.mma kind::mxf4, which applies the scales; scales go to tensor memory by copies that the MMAs' own thread issues in front of
//              them.  fp32 sums in tensor memory, two buffers of them
//   pairs      256 columns of sums twice are all of tensor memory, and the scales need 24 of them: the buffers share 32 columns.  The warps that read those
//              columns do so first, and the next tile's MMAs wait for that
//   roles      warp 0 loads, warp 1 issues the MMAs, sixteen warps (eight of narrow tiles) turn finished sums into outputs while the next tile is
//              computed
//   split      of few tiles, two or four CTAs of a cluster share one: each multiplies a part of K, hands its sums of the others' 32 channels over through
//              distributed shared memory and writes its own 32; the parts are added in a fixed order
//   grid       persistent, one CTA per multiprocessor; neighbouring CTAs work on a block of token tiles, whose operands the L2 then serves
//
// Measured, bf16 out: 8192^3 184 us (6.0 PFLOP/s; for seconds, at the power limit, 223), 4096^3 29.7 us (with a residual 39.3), 2048 x 4096 x 4096 16.7 us, 128 x 4096 x 4096
// 5.3 us, 1000^3 3.6 us; 100352 x 256 x 64 14.1 us, half of them stores (silu 19.2, gelu 22.0, where their instructions and the special-function unit bound it).  Of 8192^3 loads and shared memory
// alone take 132 us, the scales' copies nothing.
//
// Every wait on a barrier is bounded; one that runs out records a code in the status word, raises the CTA's abort flag, and all roles go to the common exit.
#include "inner_prod_mxfp4.h"
#include "inner_prod_tiles.cuh"

namespace tsb {
namespace tc {
namespace {

using Params = InnerProdMxfp4Params;

// code of the wait that ran out: 1 stage free, 2 stage full, 3 sums free, 4 sums complete, 5 shared columns free, 6 (few tokens) tokens quantized
__device__ int g_mxfp4_status;

struct Mxfp4Params : Walk {
    Params p;
};

// PAIR: tiles of two CTAs, each with 128 of 256 tokens and half of the channels' rows of w in its shared memory, and all channels' scales
template <typename T, int BN, bool RES, bool PAIR, int SPLIT>
struct Layout {
    // A step of the epilogue is 2 KB of y in rows of 128 bytes: a copy costs the engine that moves it 4.5 clocks a row of up to 128 bytes (100352 x 256 x 64, which
    // that engine bound, 20.5 -> 15.6 us).  Pairs, whose columns of sums are handed on 32 at a time, and splits take rows of 32 channels.
    static constexpr int kChannels = PAIR || SPLIT > 1 ? kCh : 128 / (int)sizeof(T);
    using Step = Staged<T, kChannels>;
    static constexpr bool kAhead = RES && SPLIT == 1;                             // residuals of a step come while the one in front of it is worked on
    static constexpr uint32_t kOutWarp = kAhead ? 2 * kOutRows : kOutRows;        // a warp's staged outputs (and the next step's residuals)
    static constexpr int kEpiWarps = BN >= 128 ? 16 : 8;                          // four (or two) for each quarter of the tokens
    static constexpr int kThreads = 32 * (2 + kEpiWarps);
    // those four share the channels, and where there are fewer steps' channels than that, the rows of the quarter
    static constexpr int kShares = kEpiWarps / 4 < BN / kChannels ? kEpiWarps / 4 : BN / kChannels, kRowShares = kEpiWarps / 4 / kShares;
    static constexpr int kBRows = PAIR ? BN / 2 : BN;
    static constexpr uint32_t kBBytes = kBRows * kKBytes;
    static constexpr int kScaleTiles = (BN + 127) / 128;                          // of 128 channels
    static constexpr uint32_t kScalesAt = kABytes + kBBytes;
    static constexpr uint32_t kWeights = kBBytes + kScaleTiles * kScales;         // of a stage
    static constexpr uint32_t kStage = kScalesAt + (1 + kScaleTiles) * kScales;
    static constexpr uint32_t kOut = kEpiWarps * kOutWarp;
    static constexpr uint32_t kParts = (SPLIT - 1) * kBM * kCh * 4;               // the other CTAs' sums of this CTA's channels
    static constexpr uint32_t kFixed = 1024 + 1024 + kOut + kParts;               // barriers, and what the alignment of the ring takes
    static constexpr int kStages = (int)((kSmem - kFixed) / kStage) < kMaxStages ? (int)((kSmem - kFixed) / kStage) : kMaxStages;      // at most
    // columns of tensor memory: the sums' buffers, x's scales (of a stage: twice four), w's (twice four for every 128 channels).  Where every CTA has one tile, one buffer.
    static constexpr bool kShared = BN == 256;
    static constexpr uint32_t kSecond = kShared ? 224 : BN;
    __host__ __device__ static constexpr uint32_t scale_columns(bool one) { return kShared ? 480 : one ? BN : 2 * BN; }
    __host__ __device__ static constexpr uint32_t columns(bool one) { return BN == 64 ? (one ? 128 : 256) : BN == 128 && one ? 256 : 512; }
};

// A lane's channels' biases of a step: channels 8 j + 2 (lane % 4) and the next one, for every j; zeros for channels that do not exist.
template <int J>
__device__ __forceinline__ void load_bias(const Params &p, int c0, float2 (&bias)[J]) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int c = c0 + 8 * j + 2 * (threadIdx.x & 3);
        bias[j] = make_float2(p.bias && c < p.n ? p.bias[c] : 0.0f, p.bias && c + 1 < p.n ? p.bias[c + 1] : 0.0f);
    }
}

// CH channels of Staged<T, CH>::kRows tokens, of which `live` exist: sums in tensor memory at `taddr` -> y, by way of `rows` in shared memory.
// m0, c0: the first token and channel; to: where in a staged row of eight the lane's pairs of channels 8 j lie; tile_store: y is written by a copy of
// its own accord that is under way when this returns, else by the lanes.  fetched: the residual is in `rows` already.  loaded(): called once
// the sums are in registers.  GIVEN: the sums are in `given` already.
template <typename T, int CH, bool RES, bool GIVEN = false, typename Loaded>
__device__ __forceinline__ void epilogue_rows(const Params &p, const CUtensorMap *map_y, uint32_t taddr, const float *given, int64_t m0, int live, int c0, const float2 (&bias)[CH / 8],
                                              uint8_t *rows, const uint32_t (&to)[CH / 8], bool tile_store, bool res_vec, bool fetched, const Loaded &loaded) {
    using S = Staged<T, CH>;
    constexpr int kN = Vec16<T>::kN, kHalves = S::kRows / 16, kPieces = CH / 32, kValues = kHalves * CH / 2;     // values of a unit; runs of 16 rows, of 32 channels; values of a lane
    const int lane = threadIdx.x & 31;
    // value i of a lane: channels 8 j + 2 (lane % 4) + i % 2 of j = i / 4 % (CH / 8), of the row lane / 4, plus 8 for i & 2, plus 16 a half
    float v[kValues];
    if constexpr (GIVEN) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) v[i] = given[i];
        if (RES && !fetched) fetch_residual<T, CH>(p, m0, live, c0, rows, res_vec);
    } else {
        int acc[kValues];
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int c = 0; c < kPieces; ++c)
                tmem_ld_rows16(taddr + ((uint32_t)(h * 16) << 16) + 32 * c, *reinterpret_cast<int (*)[16]>(&acc[(h * kPieces + c) * 16]));
        if (RES && !fetched) fetch_residual<T, CH>(p, m0, live, c0, rows, res_vec);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kValues; ++i) v[i] = __int_as_float(acc[i]);
        loaded();
    }
    auto at = [&](int i) { return rows + to[i / 4 % (CH / 8)] + ((i & 2) * 4 + i / (CH / 2) * 16) * S::kRowBytes; };
    finish_values<T, RES>(p, [&](int i) { return i & 1 ? bias[i / 4 % (CH / 8)].y : bias[i / 4 % (CH / 8)].x; },
                          [&](int i) { return to_f32(reinterpret_cast<const T *>(at(i))[i & 1]); }, v);      // (a lane's outputs go where its residuals were)
    if (!RES && lane == 0) bulk_wait_read();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kValues; i += 2) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float2 *>(at(i)) = make_float2(v[i], v[i + 1]);
        } else {
            const T pair[2] = {from_f32<T>(v[i]), from_f32<T>(v[i + 1])};
            *reinterpret_cast<uint32_t *>(at(i)) = *reinterpret_cast<const uint32_t *>(pair);
        }
    }
    if (tile_store && (c0 + CH <= p.n || p.n % kN == 0)) {      // (such a copy stops at 16 bytes, not at the value, where y ends)
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(map_y, smem_u32(rows), c0, (int)m0);    // (what lies outside y is not written)
            bulk_commit();
        }
    } else {
        __syncwarp();
        T *y = static_cast<T *>(p.y) + m0 * p.y_pitch + c0 + lane;
#pragma unroll 4
        for (int r = 0; r < live; ++r, y += p.y_pitch)
#pragma unroll
            for (int c = 0; c < CH; c += 32)
                if (c0 + c + lane < p.n) y[c] = *reinterpret_cast<const T *>(rows + S::value(r, c + lane));
        __syncwarp();
    }
}

template <typename T, int BN, bool RES, bool PAIR, int SPLIT>
__global__ void __launch_bounds__(Layout<T, BN, RES, PAIR, SPLIT>::kThreads, 1)
inner_prod_mxfp4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_xs,
                           const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_y, const __grid_constant__ Mxfp4Params t, int stages, int one, int keep, int tile_store, int res_vec) {
    static_assert(SPLIT == 1 || (!PAIR && BN == kCh * SPLIT), "split: kCh channels of the tile for each CTA");
    static_assert(PAIR == (BN == 256), "the widest tiles are pairs'");
    static_assert(Layout<T, BN, RES, PAIR, SPLIT>::scale_columns(true) + 8 + 8 * Layout<T, BN, RES, PAIR, SPLIT>::kScaleTiles <= Layout<T, BN, RES, PAIR, SPLIT>::columns(true) &&
                      Layout<T, BN, RES, PAIR, SPLIT>::scale_columns(false) + 8 + 8 * Layout<T, BN, RES, PAIR, SPLIT>::kScaleTiles <= Layout<T, BN, RES, PAIR, SPLIT>::columns(false),
                  "sums and scales fit tensor memory");
    using L = Layout<T, BN, RES, PAIR, SPLIT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), lowest = (raw + 1023u) & ~1023u;
    uint8_t *const bars_ptr = smem_raw + (lowest - raw), *const out_rows = bars_ptr + 1024, *const parts = out_rows + L::kOut;
    const uint32_t base = smem_u32(parts + L::kParts);       // of the ring
    const uint32_t bar_full = smem_u32(bars_ptr), bar_empty = bar_full + 8 * kMaxStages, bar_tfull = bar_empty + 8 * kMaxStages, bar_tempty = bar_tfull + 16, bar_shared = bar_tempty + 16;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars_ptr + 8 * (2 * kMaxStages + 6));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars_ptr + 8 * (2 * kMaxStages + 6) + 4);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int tiles = t.tiles_m * t.tiles_n;
    constexpr int kCluster = PAIR ? 2 : SPLIT;
    const int rank = kCluster > 1 ? (int)cluster_rank() : 0, first = (int)blockIdx.x / kCluster, step = (int)gridDim.x / kCluster;
    // the blocks of K that this CTA multiplies (split: a part of its tile's)
    const int kb0 = SPLIT > 1 ? t.kblocks * rank / SPLIT : 0, kb1 = SPLIT > 1 ? t.kblocks * (rank + 1) / SPLIT : t.kblocks;
    auto rows_of = [&](int m_tile) { return PAIR ? 2 * m_tile + rank : m_tile; };      // this CTA's 128 tokens of a tile

    if (warp == 0) {
        if (lane < stages) {
            mbar_init(bar_full + 8 * lane, 1);
            mbar_init(bar_empty + 8 * lane, 1);
        }
        if (lane < 2) {
            mbar_init(bar_tfull + 8 * lane, 1);
            mbar_init(bar_tempty + 8 * lane, PAIR ? 2 * L::kEpiWarps : L::kEpiWarps);
            mbar_init(bar_shared + 8 * lane, 8);         // (four warps of each CTA)
        }
        if (lane == 0) {
            *abort_flag = 0;
            prefetch_tensormap(&map_x);
            prefetch_tensormap(&map_w);
            prefetch_tensormap(&map_xs);
            prefetch_tensormap(&map_ws);
            prefetch_tensormap(&map_y);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        const uint32_t slot = smem_u32(const_cast<uint32_t *>(tmem_slot));
        if constexpr (PAIR) {
            pair_tmem_alloc(slot, L::columns(one));
            pair_tmem_relinquish();
        } else {
            tmem_alloc(slot, L::columns(one));
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kCluster > 1) {              // the other CTAs' shared and tensor memory are there too
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool met = false;                          // split: this warp has been at the cluster's meeting
    pdl_sync();
    auto give_up = [&](int code) {
        if (!*abort_flag) { *abort_flag = 1; atomicExch(&g_mxfp4_status, code); }
    };

    if (warp == 0) {
        // Both CTAs of a pair load their halves; the bytes of both count at the even one's barrier.  Neither can be a round ahead: its
        // own stage is free only when the MMAs that read both have completed.
        // `keep`: K's blocks divide the ring, and the CTA stays with its channels: the weights of its first tile serve the others too.
        uint32_t stage = 0, round = 1, at = base;
        int loads = 0;
        const uint32_t lead_full = PAIR ? map_to_rank(bar_full, 0) : bar_full;
        for (int i = first; i < tiles; i += step) {
            int mt, nt;
            tile_of(t, i, mt, nt);
            for (int kb = kb0; kb < kb1; ++kb, ++loads) {
                if (!mbar_wait_warp(bar_empty + 8 * stage, round, abort_flag)) { give_up(1); goto done; }
                const bool weights = !keep || loads < stages;
                if (elect_one()) {
                    if (!PAIR || rank == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, PAIR ? 2 * L::kStage : weights ? L::kStage : L::kStage - L::kWeights);
                    const uint32_t full = lead_full + 8 * stage;
                    // (scales: words of four, a tile's 128 after each other, two tiles a block of K)
                    if constexpr (PAIR) {
                        pair_tma_load_2d(at, &map_x, full, kb * kKBytes, rows_of(mt) * kBM);
                        pair_tma_load_2d(at + kABytes, &map_w, full, kb * kKBytes, nt * BN + rank * L::kBRows);
                        pair_tma_load_2d(at + L::kScalesAt, &map_xs, full, kb * 256, rows_of(mt));
                        pair_tma_load_2d(at + L::kScalesAt + kScales, &map_ws, full, kb * 256, nt * L::kScaleTiles);
                    } else {
                        tma_load_2d(at, &map_x, full, kb * kKBytes, rows_of(mt) * kBM);
                        tma_load_2d(at + L::kScalesAt, &map_xs, full, kb * 256, rows_of(mt));
                        if (weights) {
                            tma_load_2d(at + kABytes, &map_w, full, kb * kKBytes, nt * BN);
                            tma_load_2d(at + L::kScalesAt + kScales, &map_ws, full, kb * 256, BN < 128 ? nt * BN / 128 : nt);
                        }
                    }
                }
                __syncwarp();
                at += L::kStage;
                if (++stage == (uint32_t)stages) {
                    stage = 0;
                    at = base;
                    round ^= 1;
                }
            }
        }
        if constexpr (PAIR) {
            // no arrival from the other CTA is to come when this one leaves: the last rounds' stages, from the one that is loaded longest ago
            for (int back = min(loads, stages); back > 0; --back) {
                const uint32_t behind = (uint32_t)(loads - back) % (uint32_t)stages;
                if (!mbar_wait_warp(bar_empty + 8 * behind, (uint32_t)(loads - back) / (uint32_t)stages & 1, abort_flag)) { give_up(1); goto done; }
            }
        }
    } else if (warp == 1) {
        uint32_t stage = 0, round = 0, at = base, n = 0;
        constexpr uint64_t kDescHi = smem_desc_hi<kKBytes>(8 * kKBytes);
        constexpr uint32_t kInstr[2] = {instr_desc_mxf4<BN>(PAIR ? 2 * kBM : kBM, 0), instr_desc_mxf4<BN>(PAIR ? 2 * kBM : kBM, 1)};
        const uint32_t sfa = tmem + L::scale_columns(one), sfb = sfa + 8;
        if (!PAIR || rank == 0)
            for (int i = first; i < tiles; i += step, ++n) {
                const uint32_t acc = n & 1;
                auto wait_free = [&](uint32_t bar, uint32_t parity) {
                    return PAIR ? (bool)__all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, abort_flag)) : mbar_wait_warp(bar, parity, abort_flag);
                };
                if (!wait_free(bar_tempty + 8 * acc, ((n >> 1) & 1) ^ 1)) { give_up(3); goto done; }
                if (L::kShared && n > 0 && !wait_free(bar_shared + 8 * (acc ^ 1), ((n - 1) >> 1) & 1)) { give_up(5); goto done; }
                tc_fence_after();
                uint32_t odd = 0;                        // of a tile of 64 channels: the upper half of its 128 scales
                if constexpr (BN < 128) {
                    int mt, nt;
                    tile_of(t, i, mt, nt);
                    odd = nt * BN % 128 / 32;
                }
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait_warp(bar_full + 8 * stage, round, abort_flag)) { give_up(2); goto done; }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t a = kDescHi | (at >> 4), b = kDescHi | ((at + kABytes) >> 4);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {                // 128 values of K, the half of a stage
                            if constexpr (PAIR) pair_copy_scales(sfa + 4 * h, smem_desc_sliding(at + L::kScalesAt + 512 * h));
                            else copy_scales(sfa + 4 * h, smem_desc_sliding(at + L::kScalesAt + 512 * h));
#pragma unroll
                            for (int j = 0; j < L::kScaleTiles; ++j) {
                                const uint32_t to = sfb + 4 * (h * L::kScaleTiles + j);
                                const uint64_t from = smem_desc_sliding(at + L::kScalesAt + (1 + j) * kScales + 512 * h);
                                if constexpr (PAIR) pair_copy_scales(to, from);
                                else copy_scales(to, from);
                            }
                        }
#pragma unroll
                        for (int q = 0; q < kKBytes / 32; ++q) {
                            const uint32_t to = tmem + acc * L::kSecond, xs = sfa + 4 * (q / 2), ws = sfb + 4 * L::kScaleTiles * (q / 2) + odd;
                            if constexpr (PAIR) pair_mma_mxf4(to, a + 2 * q, b + 2 * q, kInstr[q & 1], xs, ws, kb > kb0 || q > 0);
                            else mma_mxf4(to, a + 2 * q, b + 2 * q, kInstr[q & 1], xs, ws, kb > kb0 || q > 0);
                        }
                        if constexpr (PAIR) {
                            pair_commit(bar_empty + 8 * stage);
                            if (kb == kb1 - 1) pair_commit(bar_tfull + 8 * acc);
                        } else {
                            tc_commit(bar_empty + 8 * stage);
                            if (kb == kb1 - 1) tc_commit(bar_tfull + 8 * acc);
                        }
                    }
                    __syncwarp();
                    at += L::kStage;
                    if (++stage == (uint32_t)stages) {
                        stage = 0;
                        at = base;
                        round ^= 1;
                    }
                }
            }
    } else {
        const int e = warp - 2, quarter = warp & 3;      // tensor memory lanes of this warp: 32 * (warp % 4)
        using S = typename L::Step;
        constexpr int kChannels = L::kChannels, kShare = BN / L::kShares, kSteps = kShare / kChannels, kRows = S::kRows, kQuarter = 32 / L::kRowShares;
        static_assert(kRows <= kQuarter, "a step's rows are a warp's");
        const int share = e / 4 % L::kShares * kShare;   // its channels of the tile, and from which of the quarter's rows on it has kQuarter of them
        const int row0 = quarter * 32 + e / 4 / L::kShares * kQuarter;
        // Its steps' channels from there.  (The columns that the buffers share are the last ones of the first buffer and the first ones of the second: the
        // warps of either take them in their first step.)
        const int turned = L::kShared && e / 4 == L::kShares - 1 ? kSteps - 1 : 0;
        auto channel_of = [&](int c) { return share + (c ^ turned) * kChannels; };
        uint8_t *rows = out_rows + e * L::kOutWarp;
        uint32_t n = 0, to[kChannels / 8];
#pragma unroll
        for (int j = 0; j < kChannels / 8; ++j) to[j] = S::value(lane >> 2, 8 * j + 2 * (lane & 3));
        int mt, nt, channels_of = -1;
        float2 bias[kSteps][kChannels / 8];
        tile_of(t, first, mt, nt);
        uint32_t turn = 0;                               // which half of its staging a step takes
        if constexpr (L::kAhead) {
            const int64_t m0 = (int64_t)rows_of(mt) * kBM + row0;
            start_residual<T, kChannels>(t.p, m0, (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0)), nt * BN + channel_of(0), rows, res_vec != 0);
        }
        const uint32_t lead_tempty = PAIR ? map_to_rank(bar_tempty, 0) : bar_tempty, lead_shared = PAIR ? map_to_rank(bar_shared, 0) : bar_shared;
        for (int i = first; i < tiles; i += step, ++n) {
            const uint32_t acc = n & 1;
            if (nt != channels_of) {
#pragma unroll
                for (int c = 0; c < kSteps; ++c) load_bias(t.p, nt * BN + channel_of(c), bias[c]);
            }
            channels_of = nt;
            int next_mt = mt, next_nt = nt;
            if (i + step < tiles) tile_of(t, i + step, next_mt, next_nt);
            if constexpr (RES) {                       // (the first step's, while the sums are not there yet)
                const int64_t m0 = (int64_t)rows_of(mt) * kBM + row0;
                const int live = (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0)), c0 = nt * BN + channel_of(0);
                if (live > 0 && c0 < t.p.n && (SPLIT == 1 || e / 4 == rank) && !(L::kAhead && whole_residual<kChannels>(t.p, c0, res_vec != 0)))
                    fetch_residual<T, kChannels>(t.p, m0, live, c0, rows + (L::kAhead ? kOutRows * (turn & 1) : 0), res_vec != 0);
            }
            if (!mbar_wait_warp(bar_tfull + 8 * acc, (n >> 1) & 1, abort_flag)) { give_up(4); goto done; }
            tc_fence_after();
            if constexpr (SPLIT > 1) {
                // The tile's channels kCh j are CTA j's: its sums come from the CTAs of the cluster, each with a part of K.  A lane's sums of a
                // fragment travel as they are, to the same lane of the same quarter: parts[sender, in the order of ranks][quarter][16 bytes i][lane]
                constexpr int kLane = kCh;                        // sums of a lane
                const int owner = e / 4;
                const bool any = (int64_t)mt * kBM + quarter * 32 < t.p.m;
                float sum[kLane];
                if (any) {
                    int part[kLane];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        tmem_ld_rows16(tmem + acc * L::kSecond + ((uint32_t)(quarter * 32 + h * 16) << 16) + share, *reinterpret_cast<int (*)[kLane / 2]>(&part[h * kLane / 2]));
                    tmem_ld_wait();
                    if (owner != rank) {
                        const int slot = rank < owner ? rank : rank - 1;
                        const uint32_t to_rank = map_to_rank(smem_u32(parts) + (slot * 4 + quarter) * (kLane * 32 * 4) + lane * 16, owner);
#pragma unroll
                        for (int i = 0; i < kLane / 4; ++i) sts128_cluster(to_rank + i * 512, part[4 * i], part[4 * i + 1], part[4 * i + 2], part[4 * i + 3]);
                    }
#pragma unroll
                    for (int i = 0; i < kLane; ++i) sum[i] = __int_as_float(part[i]);
                }
                cluster_arrive();
                cluster_wait();
                met = true;
                if (any && owner == rank) {
#pragma unroll
                    for (int from = 0; from < SPLIT - 1; ++from)
#pragma unroll
                        for (int i = 0; i < kLane / 4; ++i) {
                            const float4 v = *reinterpret_cast<const float4 *>(parts + (from * 4 + quarter) * (kLane * 32 * 4) + i * 512 + lane * 16);
                            sum[4 * i] = __fadd_rn(sum[4 * i], v.x);
                            sum[4 * i + 1] = __fadd_rn(sum[4 * i + 1], v.y);
                            sum[4 * i + 2] = __fadd_rn(sum[4 * i + 2], v.z);
                            sum[4 * i + 3] = __fadd_rn(sum[4 * i + 3], v.w);
                        }
#pragma unroll
                    for (int r = 0; r < 32; r += kRows) {
                        const int64_t m0 = (int64_t)mt * kBM + quarter * 32 + r;
                        const int live = (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0)), c0 = nt * BN + share;
                        if (live > 0 && c0 < t.p.n)
                            epilogue_rows<T, kChannels, RES, true>(t.p, &map_y, 0, sum + r / 16 * (kLane / 2), m0, live, c0, bias[0], rows, to, tile_store != 0, res_vec != 0, RES && r == 0, [] {});
                    }
                }
                goto done;
            }
#pragma unroll
            for (int c = 0; c < (SPLIT > 1 ? 0 : kSteps); ++c)
#pragma unroll
                for (int r = 0; r < kQuarter; r += kRows) {
                    const int64_t m0 = (int64_t)rows_of(mt) * kBM + row0 + r;
                    const int live = (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0)), c0 = nt * BN + channel_of(c);
                    bool fetched = RES && c == 0 && r == 0;
                    uint8_t *staged = rows;
                    if constexpr (L::kAhead) {
                        staged = rows + kOutRows * (turn++ & 1);
                        const bool last = c == kSteps - 1 && r + kRows == kQuarter;      // of the tile: the next step is the next tile's first
                        const int next_r = last ? 0 : (r + kRows) % kQuarter, next_c = last ? 0 : c + (r + kRows) / kQuarter;
                        const int64_t next_m0 = (int64_t)rows_of(last ? next_mt : mt) * kBM + row0 + next_r;
                        const int next_live = last && i + step >= tiles ? 0 : (int)max((int64_t)0, min((int64_t)kRows, t.p.m - next_m0));
                        start_residual<T, kChannels>(t.p, next_m0, next_live, (last ? next_nt : nt) * BN + channel_of(next_c), rows + kOutRows * (turn & 1), res_vec != 0);
                        asm volatile("cp.async.wait_group 1;" ::: "memory");              // this step's
                        __syncwarp();
                        fetched = fetched || whole_residual<kChannels>(t.p, c0, res_vec != 0);
                    }
                    // the shared columns: the last share's of the first buffer, the first share's of the second
                    const bool tells = L::kShared && c == 0 && r + kRows == kQuarter && e / 4 == (acc ? 0 : L::kShares - 1);
                    auto tell = [&] {
                        if (tells) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_cluster(lead_shared + 8 * acc);
                        }
                    };
                    if (live > 0 && c0 < t.p.n)
                        epilogue_rows<T, kChannels, RES>(t.p, &map_y, tmem + acc * L::kSecond + ((uint32_t)(row0 + r) << 16) + channel_of(c), nullptr, m0, live, c0, bias[c], staged, to, tile_store != 0,
                                              res_vec != 0, fetched, tell);
                    else tell();
                }
            mt = next_mt;
            nt = next_nt;
            tc_fence_before();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(lead_tempty + 8 * acc);
                else mbar_arrive(bar_tempty + 8 * acc);
            }
            __syncwarp();
        }
    }
done:
    // Every role of every CTA comes here, whether its work is done or a wait ran out, and meets the others once:
    //   one CTA   the block's barrier; then warp 1 frees the tensor memory
    //   pair      the block's barrier, then a phase of the cluster's in which all threads of both CTAs arrive and wait: what one CTA's MMAs, copies and
    //             arrivals reach in the other is there until both are through.  A wait that runs out in one CTA is not told to the other, whose own waits for
    //             it run out by themselves
    //   split     one phase of the cluster's behind the one at the start, in which each thread arrives once: the epilogue warps in their one tile (a
    //             cluster has one tile, so its loop is entered once and left for here: met), all other warps, and epilogue warps that
    //             gave up in front of that, below.  Warps that have not met arrive ahead of the block's barrier and wait for the phase behind it; those that have met are
    //             through it when they come here.  Either way each thread arrives once and waits once, and sums are written to another CTA ahead of the arrival only
    if (L::kAhead) asm volatile("cp.async.wait_all;" ::: "memory");
    if (warp >= 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");      // this warp's outputs are written
    if (*abort_flag) {
        // copies that may still be in flight get time to land before shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    }
    __syncwarp();
    if constexpr (SPLIT > 1) {
        if (!met) cluster_arrive();
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) {                      // nobody leaves while the other CTA may reach into its shared or tensor memory
        cluster_arrive();
        cluster_wait();
    }
    if constexpr (SPLIT > 1) {
        if (!met) cluster_wait();
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) pair_tmem_dealloc(tmem, L::columns(one));
        else tmem_dealloc(tmem, L::columns(one));
    }
}

template <typename T, int BN, bool RES, bool PAIR = false, int SPLIT = 1>
int launch(const Params &p, cudaStream_t stream) {
    using L = Layout<T, BN, RES, PAIR, SPLIT>;
    CUtensorMap mx, mw, mxs, mws, my;
    const int bytes = p.groups * (mx::kGroup / 2), tiles = ceil_div(p.groups, mx::kTileGroups);
    int st = encode(&mx, p.x, p.m, bytes, p.x_pitch, kBM);
    if (st == TSB_OK) st = encode(&mw, p.w, p.n, bytes, p.w_pitch, L::kBRows);
    if (st == TSB_OK) st = encode_scales(&mxs, p.x_scales, p.m, tiles, 1);
    if (st == TSB_OK) st = encode_scales(&mws, p.w_scales, p.n, tiles, L::kScaleTiles);
    if (st != TSB_OK) return st;
    const int type = sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16;
    const bool tile_store = aligned16(p.y, p.y_pitch, type) && p.y_pitch < (int64_t)1 << 37, res_vec = p.residual && aligned16(p.residual, p.residual_pitch, type);
    if (!tile_store) my = mx;
    else if ((st = encode_output<T, L::kChannels>(&my, p)) != TSB_OK) return st;
    auto kernel = inner_prod_mxfp4_tc_kernel<T, BN, RES, PAIR, SPLIT>;
    static DeviceOnce raised;
    if (raised.first()) {
        TSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        raised.done();
    }
    constexpr int kCluster = PAIR ? 2 : SPLIT;
    const Mxfp4Params t = {walk_of((int)ceil_div64(p.m, PAIR ? 2 * kBM : kBM), ceil_div(p.n, BN), ceil_div(bytes, kKBytes)), p};
    const int64_t tiles_all = (int64_t)t.tiles_m * t.tiles_n;
    int clusters = (int)std::min<int64_t>(tiles_all, SPLIT > 1 ? INT32_MAX : 148 / kCluster);      // (split: a tile a cluster)
    const int one = clusters == tiles_all;
    // Of few output channels, tiles of the same tokens follow each other: on a grid that is a multiple of them a CTA stays with its channels.
    if (!one && !PAIR && t.group_m == 1) clusters -= clusters % t.tiles_n;
    // No more stages than a CTA has blocks of K: what fits beside another kernel's CTAs starts while those run.  CTAs of a cluster hold tensor memory while they wait for each
    // other, so what fits a multiprocessor by its shared memory has to fit by its tensor memory too: a pair, which needs all of that, takes the shared memory as well, and
    // splits (119 KB for 256 columns, 61 KB for 128) and clusters of few tokens (47 KB or more for 128) never come to more than 512 columns.  (The clusters of the int8 product and
    // of the convolution take all of them, and 208 KB or more of shared memory, beside which none of these fits.)
    const int64_t loads = ceil_div64(tiles_all, clusters) * (SPLIT > 1 ? ceil_div(t.kblocks, SPLIT) : t.kblocks);
    int stages = PAIR ? L::kStages : (int)std::min<int64_t>(L::kStages, loads);
    static_assert(!PAIR || L::kFixed + L::kStages * L::kStage > 180 * 1024, "nothing that waits for a cluster fits beside a pair's CTA");
    static_assert(SPLIT != 4 || L::kFixed + L::kStage > 76 * 1024, "two splits of 256 columns a multiprocessor at most");
    static_assert(SPLIT != 2 || L::kFixed + L::kStage > 46 * 1024, "four splits of 128 columns a multiprocessor at most");
    const int keep = !PAIR && SPLIT == 1 && !one && t.group_m == 1 && t.kblocks <= stages;
    if (keep) stages -= stages % t.kblocks;
    TSB_CUDA(launch_pdl_cluster(kCluster, kernel, dim3(kCluster * clusters), dim3(L::kThreads), L::kFixed + stages * L::kStage, stream, mx, mw, mxs, mws, my, t, stages, one, keep,
                                (int)tile_store, (int)res_vec));
    TSB_LAUNCHED("inner_prod_mxfp4_tc_kernel");
    return TSB_OK;
}

template <typename T, bool RES>
int pick(const Params &p, cudaStream_t stream) {
    // The tile by the clocks that its rounds take: a multiprocessor gets 64 bytes a clock, so a stage of 128 + BN rows of 128 bytes takes
    // 2 (128 + BN); the epilogue some 9 BN; a pair's tile, of half the rows of w for each, 3500 more for what its CTAs wait for each other.
    const int kblocks = ceil_div(p.groups * (mx::kGroup / 2), kKBytes);
    auto clocks = [&](int bn, int ctas) {
        const int64_t rounds = ceil_div64(ceil_div64(p.m, kBM * ctas) * ceil_div(p.n, bn), 148 / ctas);
        return rounds * (kblocks * 2 * (int64_t)(128 + bn / ctas) + 9 * bn + (ctas - 1) * 3500);
    };
    const int64_t c64 = clocks(64, 1), c128 = clocks(128, 1), pair = clocks(256, 2);
    // Few tiles: two or four CTAs a tile, each with a part of K, and 1000 clocks a CTA for handing sums over.
    auto split_clocks = [&](int ctas) {
        const int64_t tiles = ceil_div64(p.m, kBM) * ceil_div(p.n, kCh * ctas);
        return tiles * ctas > 148 || kblocks < ctas ? INT64_MAX : ceil_div64(kblocks, ctas) * 2 * (128 + kCh * ctas) + 9 * kCh * ctas + 1000 * ctas;
    };
    const int64_t split2 = split_clocks(2), split4 = split_clocks(4), whole = std::min({c64, c128, pair});
    if (std::min(split2, split4) < whole) return split4 <= split2 ? launch<T, 128, RES, false, 4>(p, stream) : launch<T, 64, RES, false, 2>(p, stream);
    if (pair < std::min(c64, c128)) return launch<T, 256, RES, true>(p, stream);
    return c64 <= c128 ? launch<T, 64, RES>(p, stream) : launch<T, 128, RES>(p, stream);
}

// The status word's address on the current device
int status_word(int **at) {
    static std::atomic<int *> known[64];
    int device = 0;
    TSB_CUDA(cudaGetDevice(&device));
    std::atomic<int *> *slot = device >= 0 && device < 64 ? &known[device] : nullptr;
    *at = slot ? slot->load(std::memory_order_acquire) : nullptr;
    if (*at) return TSB_OK;
    void *found = nullptr;
    TSB_CUDA(cudaGetSymbolAddress(&found, g_mxfp4_status));
    *at = static_cast<int *>(found);
    if (slot) slot->store(*at, std::memory_order_release);
    return TSB_OK;
}

bool operand_fits(const uint8_t *at, const uint8_t *scales, int64_t rows, int64_t pitch, int groups) {
    return (reinterpret_cast<uintptr_t>(at) | reinterpret_cast<uintptr_t>(scales)) % 16 == 0 &&
           (rows == 1 || (pitch % 16 == 0 && pitch >= (int64_t)groups * (mx::kGroup / 2) && pitch < (int64_t)1 << 40));
}

}  // namespace

bool weights_fit(const Params &p) { return operand_fits(p.w, p.w_scales, p.n, p.w_pitch, p.groups); }

bool inner_prod_can(const Params &p, const char **why) {
    if (!operand_fits(p.x, p.x_scales, p.m, p.x_pitch, p.groups) || !weights_fit(p)) {
        *why = "an operand's address or pitch is no multiple of 16 bytes, or its rows overlap";
        return false;
    }
    if (p.m > INT32_MAX - 2 * kBM || ceil_div64(p.m, kBM) * ceil_div(p.n, 64) > INT32_MAX / 2) { *why = "too many rows or tiles"; return false; }
    return true;
}

int inner_prod(const Params &p, int y_type, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return p.residual ? pick<float, true>(p, stream) : pick<float, false>(p, stream);
        case TSB_TYPE_F16: return p.residual ? pick<__half, true>(p, stream) : pick<__half, false>(p, stream);
        default: return p.residual ? pick<__nv_bfloat16, true>(p, stream) : pick<__nv_bfloat16, false>(p, stream);
    }
}

int mxfp4_status_word(int **at) { return status_word(at); }

// What a status word stands for.
int inner_prod_mxfp4_status_decode(int word) {
    if (word == 0) return TSB_OK;
    static const char *const kWaits[] = {"a stage to be free", "a stage to be loaded", "sums to be read", "sums to be complete", "shared columns to be read", "tokens to be quantized"};
    return fail(TSB_ERR_DEVICE_TIMEOUT, "inner_prod_mxfp4: the wait for %s ran out; results since the last check are not to be used",
                word >= 1 && word <= 6 ? kWaits[word - 1] : "an unknown event");
}

// The device's status word: waits for the stream, reads and clears it.
int inner_prod_mxfp4_status(cudaStream_t stream) {
    int word = 0, zero = 0, *at = nullptr;
    const int st = mxfp4_status_word(&at);
    if (st != TSB_OK) return st;
    TSB_CUDA(cudaMemcpyAsync(&word, at, sizeof(word), cudaMemcpyDeviceToHost, stream));
    TSB_CUDA(cudaStreamSynchronize(stream));
    if (word == 0) return TSB_OK;
    TSB_CUDA(cudaMemcpyAsync(at, &zero, sizeof(zero), cudaMemcpyHostToDevice, stream));
    TSB_CUDA(cudaStreamSynchronize(stream));
    return inner_prod_mxfp4_status_decode(word);
}

}  // namespace tc
}  // namespace tsb
