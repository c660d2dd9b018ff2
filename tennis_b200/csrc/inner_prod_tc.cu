// The int8 inner product on the sm_100a tensor cores: y [m, n] = x [m, k] . w [n, k], both operands K-major as they lie in memory.
//
//   tile       128 tokens x BN output channels (or 256 x 256 of two CTAs, each with its half of both operands: a multiprocessor then reads
//              32 instead of 48 KB for the same arithmetic, and its 64 bytes a clock no longer bound the MMAs), 128 bytes of K a stage: two
//              TMA boxes (128-byte swizzle; rows and columns behind the matrices' ends arrive as zeros) feed tcgen05.mma kind::i8, int32 sums
//              in tensor memory, two buffers of them
//   roles      warp 0 loads, warp 1 issues the MMAs, sixteen warps (eight of narrow tiles) turn finished sums into outputs while the next
//              tile is computed
//   epilogue   sums come in fragments, so that a lane has the same few channels of many tokens and keeps their scales in registers (a lane
//              that has one token and all channels reads every channel's scales from shared memory, which then bounds the epilogue);
//              2 KB of a warp's at a time go through shared memory: residuals come by asynchronous copies while the step in front is worked on
//              (100352 x 256 x 64 with a residual 46 -> 27 us, 4096^3 62 -> 54), outputs are written by tensor-map copies (both value by value
//              where they do not lie on 16 bytes)
//   split      of few tiles, two or four CTAs of a cluster share one: each multiplies a part of K, hands its sums of the others' 32 channels
//              over through distributed shared memory (int32 sums are the same in any order) and writes its own 32
//   grid       persistent, one CTA per multiprocessor; neighbouring CTAs work on a block of kGroupM token tiles, whose operands
//              the L2 then serves
//
// Measured, bf16 out: 8192^3 331 us (3.3 POPS, tensor pipe 90 % active; with a residual 353), 4096^3 49 us (54), 64 x 4096 x 4096 8.1 us;
// 100352 x 256 x 64 19.4 us (27), where the epilogue bounds it (silu: 27.1).
//
// Every wait on a barrier is bounded; one that runs out records a code in the status word, raises the CTA's abort flag, and
// all roles go to the common exit.
#include "inner_prod_i8.h"
#include "inner_prod_tiles.cuh"

namespace tsb {
namespace tc {
namespace {

// code of the wait that ran out: 1 stage free, 2 stage full, 3 sums free, 4 sums complete
__device__ int g_status;

struct TcParams : Walk {
    InnerProdParams p;
};

// PAIR: tiles of two CTAs, each with 128 of 256 tokens and half of the channels' rows of w in its shared memory
template <typename T, int BN, bool RES, bool PAIR, int SPLIT = 1>
struct Layout {
    static constexpr bool kAhead = RES && SPLIT == 1;                        // residuals of a step come while the one in front of it is worked on
    static constexpr uint32_t kOutWarp = kAhead ? 2 * kOutRows : kOutRows;        // a warp's staged outputs (and the next step's residuals)
    static constexpr int kEpiWarps = BN >= 128 ? 16 : 8;                          // four (or two) share the channels of a tile
    static constexpr int kThreads = 32 * (2 + kEpiWarps);
    static constexpr int kBRows = PAIR ? BN / 2 : BN;
    static constexpr uint32_t kBBytes = kBRows * kKBytes;
    static constexpr uint32_t kStage = kABytes + kBBytes;
    static constexpr uint32_t kOut = kEpiWarps * kOutWarp;
    static constexpr uint32_t kParts = (SPLIT - 1) * kBM * kCh * 4;               // the other CTAs' sums of this CTA's channels
    static constexpr uint32_t kBars = 256;
    static constexpr int kStages = (int)((kSmem - 1024 - kOut - kParts - kBars) / kStage) < kMaxStages
                                       ? (int)((kSmem - 1024 - kOut - kParts - kBars) / kStage) : kMaxStages;
    static constexpr uint32_t kBytes = 1024 + kStages * kStage + kOut + kParts + kBars;
};

// A lane's channels of a tile: 8 j + 2 (lane % 4) and the next one, for every j; zeros for channels that do not exist.
template <int CH>
struct Channels {
    float2 ws[CH / 8], bias[CH / 8];
    __device__ __forceinline__ void load(const InnerProdParams &p, int c0) {
        if (c0 + CH <= p.n) {
            const float *w = p.w_scales + c0 + 2 * (threadIdx.x & 3), *b = p.bias + c0 + 2 * (threadIdx.x & 3);
#pragma unroll
            for (int j = 0; j < CH / 8; ++j) {
                ws[j] = make_float2(__ldg(w + 8 * j), __ldg(w + 8 * j + 1));
                bias[j] = p.bias ? make_float2(__ldg(b + 8 * j), __ldg(b + 8 * j + 1)) : make_float2(0.0f, 0.0f);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < CH / 8; ++j) {
            const int c = c0 + 8 * j + 2 * (threadIdx.x & 3);
            ws[j] = make_float2(c < p.n ? __ldg(p.w_scales + c) : 0.0f, c + 1 < p.n ? __ldg(p.w_scales + c + 1) : 0.0f);
            bias[j] = make_float2(p.bias && c < p.n ? __ldg(p.bias + c) : 0.0f, p.bias && c + 1 < p.n ? __ldg(p.bias + c + 1) : 0.0f);
        }
    }
};

// kCh channels of Staged<T>::kRows tokens, of which `live` exist: sums in tensor memory at `taddr` -> y, by way of `rows` in shared memory.
// m0, c0: the first token and channel; xs: the scales of tokens m0 + lane / 4 and every eighth behind it; to: where in a staged row of eight
// the lane's pairs of channels 8 j lie; tile_store: y is written by a copy of its own accord that is under way when this returns, else by the lanes.
// fetched: the residual is in `rows` already.  GIVEN: the sums are in `given` already.
template <typename T, bool RES, bool GIVEN = false>
__device__ __forceinline__ void epilogue_rows(const InnerProdParams &p, const CUtensorMap *map_y, uint32_t taddr, const int *given, int64_t m0, int live, int c0, const Channels<kCh> &ch, const float *xs,
                                              uint8_t *rows, const uint32_t (&to)[kCh / 8], bool tile_store, bool res_vec, bool fetched) {
    using S = Staged<T>;
    constexpr int kN = Vec16<T>::kN, kHalves = S::kRows / 16, kValues = kHalves * kCh / 2;     // values of a unit; runs of 16 rows; values of a lane
    const int lane = threadIdx.x & 31;
    // value i of a lane: channels 8 j + 2 (lane % 4) + i % 2 of j = i / 4 % 4, of the row lane / 4, plus 8 for i & 2, plus 16 a half
    int acc[kValues];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
        if (!GIVEN) tmem_ld_rows16(taddr + ((uint32_t)(h * 16) << 16), *reinterpret_cast<int (*)[kCh / 2]>(&acc[h * kCh / 2]));
    if (GIVEN) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) acc[i] = given[i];
    }
    auto at = [&](int i) { return rows + to[i / 4 % (kCh / 8)] + ((i & 2) * 4 + i / (kCh / 2) * 16) * S::kRowBytes; };
    float v[kValues];
    if (RES && !fetched) fetch_residual<T>(p, m0, live, c0, rows, res_vec);
    if (!GIVEN) tmem_ld_wait();
    inner_prod_values<T, RES>(p, acc, [&](int i) { return PairScales{ch.ws[i / 4 % (kCh / 8)], xs[i / (kCh / 2) * 2 + (i >> 1 & 1)], ch.bias[i / 4 % (kCh / 8)]}; },
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
    if (tile_store && (c0 + kCh <= p.n || p.n % kN == 0)) {      // (such a copy stops at 16 bytes, not at the value, where y ends)
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
            if (c0 + lane < p.n) *y = *reinterpret_cast<const T *>(rows + S::value(r, lane));
        __syncwarp();
    }
}

template <typename T, int BN, bool RES, bool PAIR, int SPLIT>
__global__ void __launch_bounds__(Layout<T, BN, RES, PAIR, SPLIT>::kThreads, 1)
inner_prod_i8_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_y,
                        const __grid_constant__ TcParams t, int tile_store, int res_vec) {
    static_assert(SPLIT == 1 || (!PAIR && BN == kCh * SPLIT), "split: kCh channels of the tile for each CTA");
    using L = Layout<T, BN, RES, PAIR, SPLIT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *out_rows = smem_raw + (base - raw) + L::kStages * L::kStage;
    uint8_t *parts = out_rows + L::kOut, *bars_ptr = parts + L::kParts;
    const uint32_t bar_full = smem_u32(bars_ptr), bar_empty = bar_full + 8 * kMaxStages, bar_tfull = bar_empty + 8 * kMaxStages, bar_tempty = bar_tfull + 16;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars_ptr + 8 * (2 * kMaxStages + 4));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars_ptr + 8 * (2 * kMaxStages + 4) + 4);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int tiles = t.tiles_m * t.tiles_n;
    constexpr int kCluster = PAIR ? 2 : SPLIT;
    const int rank = kCluster > 1 ? (int)cluster_rank() : 0, first = (int)blockIdx.x / kCluster, step = (int)gridDim.x / kCluster;
    // the blocks of K that this CTA multiplies (split: a part of its tile's)
    const int kb0 = SPLIT > 1 ? t.kblocks * rank / SPLIT : 0, kb1 = SPLIT > 1 ? t.kblocks * (rank + 1) / SPLIT : t.kblocks;
    auto rows_of = [&](int m_tile) { return PAIR ? 2 * m_tile + rank : m_tile; };      // this CTA's 128 tokens of a tile

    if (warp == 0) {
        if (lane < L::kStages) {
            mbar_init(bar_full + 8 * lane, 1);
            mbar_init(bar_empty + 8 * lane, 1);
        }
        if (lane < 2) {
            mbar_init(bar_tfull + 8 * lane, 1);
            mbar_init(bar_tempty + 8 * lane, PAIR ? 2 * L::kEpiWarps : L::kEpiWarps);
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
        const uint32_t slot = smem_u32(const_cast<uint32_t *>(tmem_slot));
        if constexpr (PAIR) {
            pair_tmem_alloc(slot, 512);
            pair_tmem_relinquish();
        } else {
            tmem_alloc(slot, 512);
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
        if (!*abort_flag) { *abort_flag = 1; atomicExch(&g_status, code); }
    };

    if (warp == 0) {
        // Both CTAs of a pair load their halves; the bytes of both count at the even one's barrier.  Neither can be a round ahead: its
        // own stage is free only when the MMAs that read both have completed.
        uint32_t s = 0;
        const uint32_t lead_full = PAIR ? map_to_rank(bar_full, 0) : bar_full;
        for (int i = first; i < tiles; i += step) {
            int mt, nt;
            tile_of(t, i, mt, nt);
            for (int kb = kb0; kb < kb1; ++kb, ++s) {
                const uint32_t stage = s % L::kStages, round = s / L::kStages, at = base + stage * L::kStage;
                if (!mbar_wait_warp(bar_empty + 8 * stage, (round & 1) ^ 1, abort_flag)) { give_up(1); goto done; }
                if (elect_one()) {
                    if (!PAIR || rank == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, PAIR ? 2 * L::kStage : L::kStage);
                    if constexpr (PAIR) {
                        pair_tma_load_2d(at, &map_x, lead_full + 8 * stage, kb * kKBytes, rows_of(mt) * kBM);
                        pair_tma_load_2d(at + kABytes, &map_w, lead_full + 8 * stage, kb * kKBytes, nt * BN + rank * L::kBRows);
                    } else {
                        tma_load_2d(at, &map_x, bar_full + 8 * stage, kb * kKBytes, rows_of(mt) * kBM);
                        tma_load_2d(at + kABytes, &map_w, bar_full + 8 * stage, kb * kKBytes, nt * BN);
                    }
                }
                __syncwarp();
            }
        }
        if constexpr (PAIR) {
            // no arrival from the other CTA is to come when this one leaves
            for (uint32_t back = min(s, (uint32_t)L::kStages); back > 0; --back)
                if (!mbar_wait_warp(bar_empty + 8 * ((s - back) % L::kStages), (s - back) / L::kStages & 1, abort_flag)) { give_up(1); goto done; }
        }
    } else if (warp == 1) {
        uint32_t s = 0, n = 0;
        constexpr uint64_t kDescHi = smem_desc_hi<kKBytes>(8 * kKBytes);
        constexpr uint32_t kInstr = instr_desc<BN>() + (PAIR ? (uint32_t)(kBM >> 4) << 24 : 0);      // (M = 256)
        if (!PAIR || rank == 0)
            for (int i = first; i < tiles; i += step, ++n) {
                const uint32_t acc = n & 1;
                if (!(PAIR ? __all_sync(0xffffffffu, mbar_wait_cluster(bar_tempty + 8 * acc, ((n >> 1) & 1) ^ 1, abort_flag))
                           : mbar_wait_warp(bar_tempty + 8 * acc, ((n >> 1) & 1) ^ 1, abort_flag))) { give_up(3); goto done; }
                tc_fence_after();
                for (int kb = kb0; kb < kb1; ++kb, ++s) {
                    const uint32_t stage = s % L::kStages, round = s / L::kStages;
                    if (!mbar_wait_warp(bar_full + 8 * stage, round & 1, abort_flag)) { give_up(2); goto done; }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t a = kDescHi | ((base + stage * L::kStage) >> 4), b = kDescHi | ((base + stage * L::kStage + kABytes) >> 4);
#pragma unroll
                        for (int q = 0; q < kKBytes / 32; ++q) {
                            if constexpr (PAIR) pair_mma_i8(tmem + acc * BN, a + 2 * q, b + 2 * q, kInstr, kb > kb0 || q > 0);
                            else mma_i8(tmem + acc * BN, a + 2 * q, b + 2 * q, kInstr, kb > kb0 || q > 0);
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
                }
            }
    } else {
        const int e = warp - 2, quarter = warp & 3;      // tensor memory lanes of this warp: 32 * (warp % 4)
        constexpr int kShare = BN / (L::kEpiWarps / 4);
        const int share = e / 4 * kShare;                // its channels of the tile
        uint8_t *rows = out_rows + e * L::kOutWarp;
        uint32_t n = 0, to[kCh / 8];
#pragma unroll
        for (int j = 0; j < kCh / 8; ++j) to[j] = Staged<T>::value(lane >> 2, 8 * j + 2 * (lane & 3));
        int mt, nt, channels_of = -1;
        Channels<kCh> channels[kShare / kCh];
        // the scales of this lane's tokens: lane / 4 and every eighth behind it
        auto scales_of = [&](int m_tile, float (&s)[4]) {
            const int m = rows_of(m_tile) * kBM + quarter * 32 + (lane >> 2), left = (int)t.p.m - m, every = 8 * (int)t.p.xs_stride;
            const float *from = t.p.x_scales + (t.p.xs_stride ? m : 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = left > 8 * i ? from[i * every] : 0.0f;
        };
        tile_of(t, first, mt, nt);
        float xs[4], next_xs[4];
        scales_of(mt, xs);
        uint32_t turn = 0;                               // which half of its staging a step takes
        if constexpr (L::kAhead) {
            const int64_t m0 = (int64_t)rows_of(mt) * kBM + quarter * 32;
            start_residual<T>(t.p, m0, (int)max((int64_t)0, min((int64_t)Staged<T>::kRows, t.p.m - m0)), nt * BN + share, rows, res_vec != 0);
        }
        const uint32_t lead_tempty = PAIR ? map_to_rank(bar_tempty, 0) : bar_tempty;
        for (int i = first; i < tiles; i += step, ++n) {
            const uint32_t acc = n & 1;
            if (nt != channels_of) {
#pragma unroll
                for (int c = 0; c < kShare / kCh; ++c) channels[c].load(t.p, nt * BN + share + c * kCh);
            }
            channels_of = nt;
            // the next tile, and its tokens' scales, while this one is worked on
            int next_mt = mt, next_nt = nt;
            if (i + step < tiles) tile_of(t, i + step, next_mt, next_nt);
            scales_of(next_mt, next_xs);
            constexpr int kRows = Staged<T>::kRows;
            if constexpr (RES) {                       // (the first step's, while the sums are not there yet)
                const int64_t m0 = (int64_t)rows_of(mt) * kBM + quarter * 32;
                const int live = (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0));
                if (live > 0 && nt * BN + share < t.p.n && (SPLIT == 1 || e / 4 == rank) && !(L::kAhead && whole_residual(t.p, nt * BN + share, res_vec != 0)))
                    fetch_residual<T>(t.p, m0, live, nt * BN + share, rows + (L::kAhead ? kOutRows * (turn & 1) : 0), res_vec != 0);
            }
            if (!mbar_wait_warp(bar_tfull + 8 * acc, (n >> 1) & 1, abort_flag)) { give_up(4); goto done; }
            tc_fence_after();
            if constexpr (SPLIT > 1) {
                // The tile's channels kCh j are CTA j's: its sums come from the CTAs of the cluster, each with a part of K.  A lane's sums of a
                // fragment travel as they are, to the same lane of the same quarter: parts[sender, in the order of ranks][quarter][16 bytes i][lane]
                constexpr int kLane = kCh;                        // sums of a lane
                const int owner = e / 4;
                const bool any = (int64_t)mt * kBM + quarter * 32 < t.p.m;
                int sum[kLane];
                if (any) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        tmem_ld_rows16(tmem + acc * BN + ((uint32_t)(quarter * 32 + h * 16) << 16) + share, *reinterpret_cast<int (*)[kLane / 2]>(&sum[h * kLane / 2]));
                    tmem_ld_wait();
                    if (owner != rank) {
                        const int slot = rank < owner ? rank : rank - 1;
                        const uint32_t to_rank = map_to_rank(smem_u32(parts) + (slot * 4 + quarter) * (kLane * 32 * 4) + lane * 16, owner);
#pragma unroll
                        for (int i = 0; i < kLane / 4; ++i) sts128_cluster(to_rank + i * 512, sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
                    }
                }
                cluster_arrive();
                cluster_wait();
                met = true;
                if (any && owner == rank) {
#pragma unroll
                    for (int from = 0; from < SPLIT - 1; ++from)
#pragma unroll
                        for (int i = 0; i < kLane / 4; ++i) {
                            const int4 v = *reinterpret_cast<const int4 *>(parts + (from * 4 + quarter) * (kLane * 32 * 4) + i * 512 + lane * 16);
                            sum[4 * i] += v.x;
                            sum[4 * i + 1] += v.y;
                            sum[4 * i + 2] += v.z;
                            sum[4 * i + 3] += v.w;
                        }
#pragma unroll
                    for (int r = 0; r < 32; r += kRows) {
                        const int64_t m0 = (int64_t)mt * kBM + quarter * 32 + r;
                        const int live = (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0)), c0 = nt * BN + share;
                        if (live > 0 && c0 < t.p.n)
                            epilogue_rows<T, RES, true>(t.p, &map_y, 0, sum + r / 16 * (kLane / 2), m0, live, c0, channels[0], xs + r / 8, rows, to, tile_store != 0, res_vec != 0, RES && r == 0);
                    }
                }
                goto done;
            }
#pragma unroll
            for (int c = 0; c < (SPLIT > 1 ? 0 : kShare / kCh); ++c)
#pragma unroll
                for (int r = 0; r < 32; r += kRows) {
                    const int64_t m0 = (int64_t)rows_of(mt) * kBM + quarter * 32 + r;
                    const int live = (int)max((int64_t)0, min((int64_t)kRows, t.p.m - m0)), c0 = nt * BN + share + c * kCh;
                    bool fetched = RES && c == 0 && r == 0;
                    uint8_t *staged = rows;
                    if constexpr (L::kAhead) {
                        staged = rows + kOutRows * (turn++ & 1);
                        const bool last = c == kShare / kCh - 1 && r + kRows == 32;       // of the tile: the next step is the next tile's first
                        const int next_r = last ? 0 : (r + kRows) % 32, next_c = last ? 0 : c + (r + kRows) / 32;
                        const int64_t next_m0 = (int64_t)rows_of(last ? next_mt : mt) * kBM + quarter * 32 + next_r;
                        const int next_live = last && i + step >= tiles ? 0 : (int)max((int64_t)0, min((int64_t)kRows, t.p.m - next_m0));
                        start_residual<T>(t.p, next_m0, next_live, (last ? next_nt : nt) * BN + share + next_c * kCh, rows + kOutRows * (turn & 1), res_vec != 0);
                        asm volatile("cp.async.wait_group 1;" ::: "memory");              // this step's
                        __syncwarp();
                        fetched = fetched || whole_residual(t.p, c0, res_vec != 0);
                    }
                    if (live > 0 && c0 < t.p.n)
                        epilogue_rows<T, RES>(t.p, &map_y, tmem + acc * BN + ((uint32_t)(quarter * 32 + r) << 16) + share + c * kCh, nullptr, m0, live, c0, channels[c], xs + r / 8, staged, to,
                                         tile_store != 0, res_vec != 0, fetched);
                }
            mt = next_mt;
            nt = next_nt;
#pragma unroll
            for (int j = 0; j < 4; ++j) xs[j] = next_xs[j];
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
        // The epilogue warps have met those of the other CTAs above, for which every thread of the cluster has to arrive: the other warps, and
        // one that gave up in front of that, do so here -- ahead of the block's own barrier, where the waiting warps are still missing.
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
        if constexpr (PAIR) pair_tmem_dealloc(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

template <typename T, int BN, bool RES, bool PAIR = false, int SPLIT = 1>
int launch(const InnerProdParams &p, cudaStream_t stream) {
    using L = Layout<T, BN, RES, PAIR, SPLIT>;
    CUtensorMap mx, mw, my;
    int st = encode(&mx, p.x, p.m, p.k, p.x_pitch, kBM);
    if (st == TSB_OK) st = encode(&mw, p.w, p.n, p.k, p.w_pitch, L::kBRows);
    if (st != TSB_OK) return st;
    const int type = sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16;
    const bool tile_store = aligned16(p.y, p.y_pitch, type) && p.y_pitch < (int64_t)1 << 37, res_vec = p.residual && aligned16(p.residual, p.residual_pitch, type);
    if (!tile_store) my = mx;
    else if ((st = encode_output<T>(&my, p)) != TSB_OK) return st;
    auto kernel = inner_prod_i8_tc_kernel<T, BN, RES, PAIR, SPLIT>;
    static DeviceOnce raised;
    if (raised.first()) {
        TSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes));
        raised.done();
    }
    constexpr int kCluster = PAIR ? 2 : SPLIT;
    const TcParams t = {walk_of((int)ceil_div64(p.m, PAIR ? 2 * kBM : kBM), ceil_div(p.n, BN), ceil_div(p.k, kKBytes)), p};
    const int grid = kCluster * (int)std::min<int64_t>((int64_t)t.tiles_m * t.tiles_n, SPLIT > 1 ? INT32_MAX : 148 / kCluster);      // (split: a tile a cluster)
    TSB_CUDA(launch_pdl_cluster(kCluster, kernel, dim3(grid), dim3(L::kThreads), L::kBytes, stream, mx, mw, my, t, (int)tile_store, (int)res_vec));
    TSB_LAUNCHED("inner_prod_i8_tc_kernel");
    return TSB_OK;
}

template <typename T, bool RES>
int pick(const InnerProdParams &p, cudaStream_t stream) {
    // The tile by the clocks that its rounds take: a multiprocessor gets 64 bytes a clock, so a stage of 128 + BN rows of 128 bytes takes
    // 2 (128 + BN); the epilogue some 9 BN; a pair's tile, of half the rows of w for each, 3500 more for what its CTAs wait for each other.
    // (Measured, 64, 128, 256 wide and by pairs: 64 x 4096 x 4096 9.7, 11.0, 16.2 us; 2048 x 1000 x 2048 9.9, 8.1, 11.0, 11.4;
    // 2048 x 4096 x 4096 48.6, 35.4, 29.1, 26.3; 8192^3 - , - , 359, 331; but 16384 x 8192 x 512 80 us 256 wide, 103 by pairs.
    // With a residual the 64 channels of a warp of the widest tiles do not fit its registers, and they take 16 BN: 16384 x 8192 x 512 143 us 256
    // wide, 123 in tiles of 128; 25088 x 1024 x 256 34.7 and 23.9.)
    auto clocks = [&](int bn, int ctas) {
        const int64_t rounds = ceil_div64(ceil_div64(p.m, kBM * ctas) * ceil_div(p.n, bn), 148 / ctas);
        return rounds * (ceil_div(p.k, kKBytes) * 2 * (int64_t)(128 + bn / ctas) + (RES && bn == 256 ? 16 : 9) * bn + (ctas - 1) * 3500);
    };
    const int64_t c64 = clocks(64, 1), c128 = clocks(128, 1), c256 = clocks(256, 1), pair = clocks(256, 2);
    // Few tiles: two or four CTAs a tile, each with a part of K, and 2000 clocks for handing sums over.  (64 x 2048 x 8192 15.4 -> 9.6 us,
    // 64 x 4096 x 4096 9.6 -> 8.1, 64 x 1000 x 2048 5.8 -> 4.9.)
    auto split_clocks = [&](int ctas) {
        const int64_t tiles = ceil_div64(p.m, kBM) * ceil_div(p.n, kCh * ctas), blocks = ceil_div(p.k, kKBytes);
        return tiles * ctas > 148 || blocks < ctas ? INT64_MAX : ceil_div64(blocks, ctas) * 2 * (128 + kCh * ctas) + 9 * kCh * ctas + 2000;
    };
    const int64_t split2 = split_clocks(2), split4 = split_clocks(4), whole = std::min({c64, c128, c256, pair});
    if (std::min(split2, split4) < whole) return split4 <= split2 ? launch<T, 128, RES, false, 4>(p, stream) : launch<T, 64, RES, false, 2>(p, stream);
    if (pair < std::min({c64, c128, c256})) return launch<T, 256, RES, true>(p, stream);
    if (c64 <= c128 && c64 <= c256) return launch<T, 64, RES>(p, stream);
    return c128 <= c256 ? launch<T, 128, RES>(p, stream) : launch<T, 256, RES>(p, stream);
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
    if (p.m > INT32_MAX - 2 * kBM || ceil_div64(p.m, kBM) * ceil_div(p.n, 64) > INT32_MAX / 2) { *why = "too many rows or tiles"; return false; }
    return true;
}

int inner_prod(const InnerProdParams &p, int y_type, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return p.residual ? pick<float, true>(p, stream) : pick<float, false>(p, stream);
        case TSB_TYPE_F16: return p.residual ? pick<__half, true>(p, stream) : pick<__half, false>(p, stream);
        default: return p.residual ? pick<__nv_bfloat16, true>(p, stream) : pick<__nv_bfloat16, false>(p, stream);
    }
}

// What a status word stands for.
int inner_prod_status_decode(int word) {
    if (word == 0) return TSB_OK;
    static const char *const kWaits[] = {"a stage to be free", "a stage to be loaded", "sums to be read", "sums to be complete"};
    return fail(TSB_ERR_DEVICE_TIMEOUT, "inner_prod_i8: the wait for %s ran out; results since the last check are not to be used",
                word >= 1 && word <= 4 ? kWaits[word - 1] : "an unknown event");
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
    return inner_prod_status_decode(word);
}

}  // namespace tc
}  // namespace tsb
