// The 4-bit inner product of few tokens on the sm_100a tensor cores: the weights' bytes are the work, each is read once.
//
//   tile       128 output channels on the rows of an MMA, up to 64 tokens on its columns: what the tensor cores multiply for tokens that do not exist costs
//              less than the weights' way from memory
//   split      the CTAs of a cluster share a tile's K, so that a layer of few channels reads from all multiprocessors; their sums meet in the
//              shared memory of the CTA that finishes a token (each has neighbouring ones, all that fit an MMA in equal parts), added in the order of ranks
//   loads      weights and their scales through a ring of TMA boxes, 256 values of K of 128 rows each
//   tokens     4-bit rows, by TMA through the same ring; or floating rows, which the CTA quantizes into shared memory, its part of K alone, while
//              its weights are on their way
//   roles      warp 0 loads, warp 1 multiplies, warps 2 to 5 (of more than 16 tokens 2 to 9) finish: a lane has a channel of all tokens, so rows of y are
//              written 32 channels at a time; warps 2 to 9 quantize
//
// Bound by the weights' bytes on large layers (one token through 16384 x 8192 14.3 us, 5.0 TB/s; 32 tokens through 8192 x 8192 9.0), by the chain of launch, load, product and meeting on
// small ones (through 4096 x 4096 4.1 us, quantized inside as much; 16 tokens through 2048 x 8192 4.8; 1000 x 1000 2.4).
//
// Every wait on a barrier is bounded; one that runs out records a code in the status word, raises the CTA's abort flag, and all roles go to the common exit.
#include "inner_prod_mxfp4.h"
#include "inner_prod_tiles.cuh"

#include <type_traits>

namespace tsb {
namespace few {
namespace {

using namespace tc;
using Params = InnerProdMxfp4Params;

constexpr int kMaxCluster = 4;
constexpr int kQuantizers = 8;                    // warps
constexpr uint32_t kMaxResident = 48 * 1024;      // bytes of quantized tokens that a CTA keeps

// NT: tokens of an MMA; X: uint8_t (4-bit rows), or the type of floating rows; CL: CTAs that share a tile
template <typename X, int NT, int CL>
struct Shape {
    static constexpr bool kQuantize = sizeof(X) > 1;
    static constexpr uint32_t kTokens = NT * kKBytes + kScales;                       // of a block of K: rows and scales
    static constexpr uint32_t kScalesAt = kABytes, kTokensAt = kABytes + kScales;     // within a stage
    static constexpr uint32_t kStage = kTokensAt + (kQuantize ? 0 : kTokens);
    static constexpr int kMost = 10;                                                  // stages
    static constexpr int kFinishers = NT > 16 ? 8 : 4;                                // warps; eight: two a quarter of the channels, which take turns
    static constexpr int kThreads = 32 * (2 + (kQuantize && kQuantizers > kFinishers ? kQuantizers : kFinishers));
    static constexpr int kMine = NT / CL;                                             // tokens that a CTA finishes
    static constexpr uint32_t kParts = CL > 1 ? NT * kBM * 4 : 0;                     // all CTAs' sums of those
    static constexpr uint32_t kBars = 1024;                                           // (what follows lies on 1024 bytes)
    // columns of tensor memory: sums, weights' scales, tokens' scales
    static constexpr uint32_t kScaleColumns = 64, kColumns = 128;
    static uint32_t fixed(int blocks) { return 1024 + kBars + kParts + (kQuantize ? blocks * kTokens : 0); }      // bytes beside the ring, and what its alignment takes
};

struct FewParams {
    Params p;
    int kblocks, stages;
    int cols;                      // values of a floating row
    int64_t x_pitch;               // elements between floating rows
    int x_aligned;
    int early;                     // the weights may be read before the kernel in front has completed
    int *status;
};

// Floating rows' part of K, 128 values of a token at a time, as the MMA reads them: rows of 128 bytes in 128-byte swizzle, scales in tiles.
template <typename X, int NT, int CL>
__device__ __forceinline__ void quantize_tokens(const FewParams &t, int kb0, int blocks, uint8_t *to) {
    using S = Shape<X, NT, CL>;
    constexpr int kN = Vec16<X>::kN, kLanes = 128 / kN, kAtOnce = 32 / kLanes, kTurns = 8;
    const int lane = threadIdx.x & 31, in = lane % kLanes, tiles = 2 * blocks, m = (int)t.p.m;
    const X *x = reinterpret_cast<const X *>(t.p.x);
    // a warp's tiles: kAtOnce neighbouring ones, then those kQuantizers * kAtOnce further, through the tokens one after the other
    const uint32_t units = (uint32_t)(m * tiles), inverse = 0xffffffffu / (uint32_t)tiles + 1;      // (units times tiles is far below 2^32)
    for (uint32_t first = ((threadIdx.x >> 5) - 2) * kAtOnce; first < units; first += kTurns * kQuantizers * kAtOnce) {
        uint4 held[kTurns];
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const uint32_t u = first + i * kQuantizers * kAtOnce + lane / kLanes, token = __umulhi(u, inverse), tile = u - token * tiles;
            held[i] = make_uint4(0, 0, 0, 0);
            if (u < units) held[i] = mx::load_values(x + token * t.x_pitch, (int64_t)kb0 * 256 + tile * 128 + in * kN, t.cols, t.x_aligned);
        }
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            if (first + i * kQuantizers * kAtOnce >= units) break;
            const uint32_t u = first + i * kQuantizers * kAtOnce + lane / kLanes, token = __umulhi(u, inverse), tile = u - token * tiles;
            uint32_t word;
            const uint32_t codes = mx::quantize_vector<X>(held[i], &word);
            if (u < units) {
                uint8_t *block = to + (tile >> 1) * S::kTokens;
                const uint32_t b = (tile & 1) * 64 + in * (kN / 2);
                mx::store_codes<kN>(block + token * kKBytes + (((b >> 4) ^ (token & 7)) << 4) + (b & 15), codes, true);
                if (in == 0) *reinterpret_cast<uint32_t *>(block + NT * kKBytes + (tile & 1) * 512 + token % 32 * 16 + token / 32 * 4) = word;
            }
        }
    }
}

// N tokens from m0 on, of a lane's channel c: sums -> y
template <typename T, int N>
__device__ __forceinline__ void finish_tokens(const Params &p, float (&v)[N], int m0, int c, float bias) {
    const bool live = c < p.n;
    const int left = (int)p.m - m0;
    const T *r = static_cast<const T *>(p.residual) + (p.residual ? m0 * p.residual_pitch + c : 0);
    finish_values<T>(p, [&](int) { return bias; }, [&](int i) { return live && i < left ? to_f32(r[i * p.residual_pitch]) : 0.0f; }, v);
    T *y = static_cast<T *>(p.y) + m0 * p.y_pitch + c;
#pragma unroll
    for (int i = 0; i < N; ++i, y += p.y_pitch)
        if (live && i < left) *y = from_f32<T>(v[i]);
}

template <typename T, typename X, int NT, int CL>
__global__ void __launch_bounds__(Shape<X, NT, CL>::kThreads)
inner_prod_mxfp4_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_x,
                            const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ FewParams t) {
    using S = Shape<X, NT, CL>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const bars = smem_raw + (base - smem_u32(smem_raw)), *const parts = bars + S::kBars, *const ring = parts + S::kParts;
    uint8_t *const tokens = ring + t.stages * S::kStage;
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::kMost, bar_sums = bar_empty + 8 * S::kMost, bar_tokens = bar_sums + 8;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars + 8 * (2 * S::kMost + 2));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 8 * (2 * S::kMost + 2) + 4);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = CL > 1 ? (int)cluster_rank() : 0, tile = (int)blockIdx.x / CL;
    const int kb0 = (int)((int64_t)t.kblocks * rank / CL), blocks = (int)((int64_t)t.kblocks * (rank + 1) / CL) - kb0;

    if (warp == 0) {
        if (lane < t.stages) {
            mbar_init(bar_full + 8 * lane, 1);
            mbar_init(bar_empty + 8 * lane, 1);
        }
        if (lane == 0) {
            mbar_init(bar_sums, 1);
            mbar_init(bar_tokens, kQuantizers);
            *abort_flag = 0;
            prefetch_tensormap(&map_w);
            prefetch_tensormap(&map_ws);
            if (!S::kQuantize) {
                prefetch_tensormap(&map_x);
                prefetch_tensormap(&map_xs);
            }
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), S::kColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    if (CL > 1) cluster_arrive();              // (waited for ahead of the first write to another CTA's shared memory)
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int c = tile * kBM + (warp & 3) * 32 + lane;       // a finishing lane's channel
    const bool finishes = warp >= 2 && warp < 2 + S::kFinishers;
    const int turn = (warp - 2) / 4 % 2, turns = S::kFinishers / 4;
    auto give_up = [&](int code) {
        if (!*abort_flag) { *abort_flag = 1; atomicExch(t.status, code); }
    };
    float bias = 0.0f;

    if (warp == 0) {
        uint32_t at = smem_u32(ring), stage = 0, round = 1;
        auto advance = [&] {
            at += S::kStage;
            if (++stage == (uint32_t)t.stages) {
                stage = 0;
                at = smem_u32(ring);
                round ^= 1;
            }
        };
        auto weights = [&](int kb) {
            mbar_arrive_expect_tx(bar_full + 8 * stage, S::kStage);
            tma_load_2d(at, &map_w, bar_full + 8 * stage, kb * kKBytes, tile * kBM);
            tma_load_2d(at + S::kScalesAt, &map_ws, bar_full + 8 * stage, kb * 256, tile);
        };
        int ahead = 0;
        if (t.early) {
            ahead = min(blocks, t.stages);
            for (int i = 0; i < ahead; ++i) {
                if (elect_one()) weights(kb0 + i);
                __syncwarp();
                advance();
            }
            at = smem_u32(ring);
            stage = 0;
            round = 1;
        }
        pdl_sync();
        for (int i = 0; i < blocks; ++i) {
            if (!mbar_wait_warp(bar_empty + 8 * stage, round, abort_flag)) { give_up(1); goto done; }
            if (elect_one()) {
                if (i >= ahead) weights(kb0 + i);
                if constexpr (!S::kQuantize) {
                    tma_load_2d(at + S::kTokensAt, &map_x, bar_full + 8 * stage, (kb0 + i) * kKBytes, 0);
                    tma_load_2d(at + S::kTokensAt + NT * kKBytes, &map_xs, bar_full + 8 * stage, (kb0 + i) * 256, 0);
                }
            }
            __syncwarp();
            advance();
        }
    } else if (warp == 1) {
        constexpr uint64_t kDescHi = smem_desc_hi<kKBytes>(8 * kKBytes);
        constexpr uint32_t kInstr[2] = {instr_desc_mxf4<NT>(kBM, 0), instr_desc_mxf4<NT>(kBM, 1)};
        const uint32_t sfa = tmem + S::kScaleColumns, sfb = sfa + 8;
        uint32_t at = smem_u32(ring), x = smem_u32(tokens), stage = 0, round = 0;
        pdl_sync();
        if (S::kQuantize && !mbar_wait_warp(bar_tokens, 0, abort_flag)) { give_up(6); goto done; }
        for (int i = 0; i < blocks; ++i) {
            if (!mbar_wait_warp(bar_full + 8 * stage, round, abort_flag)) { give_up(2); goto done; }
            tc_fence_after();
            if (elect_one()) {
                if (!S::kQuantize) x = at + S::kTokensAt;
                const uint64_t a = kDescHi | (at >> 4), b = kDescHi | (x >> 4);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    copy_scales(sfa + 4 * h, smem_desc_sliding(at + S::kScalesAt + 512 * h));
                    copy_scales(sfb + 4 * h, smem_desc_sliding(x + NT * kKBytes + 512 * h));
                }
#pragma unroll
                for (int q = 0; q < kKBytes / 32; ++q) mma_mxf4(tmem, a + 2 * q, b + 2 * q, kInstr[q & 1], sfa + 4 * (q / 2), sfb + 4 * (q / 2), i > 0 || q > 0);
                tc_commit(bar_empty + 8 * stage);
                if (i == blocks - 1) tc_commit(bar_sums);
            }
            __syncwarp();
            if (S::kQuantize) x += S::kTokens;
            at += S::kStage;
            if (++stage == (uint32_t)t.stages) {
                stage = 0;
                at = smem_u32(ring);
                round ^= 1;
            }
        }
    } else {
        pdl_sync();
        if constexpr (S::kQuantize) {
            quantize_tokens<X, NT, CL>(t, kb0, blocks, tokens);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_tokens);
        }
        if (finishes && t.p.bias && c < t.p.n) bias = t.p.bias[c];
    }
done:
    {
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const int m = (int)t.p.m, channel = (warp & 3) * 32 + lane;
        bool there = __all_sync(0xffffffffu, !*abort_flag) && finishes;
        if (there) {
            if (!mbar_wait_warp(bar_sums, 0, abort_flag)) { give_up(4); there = false; }
            tc_fence_after();
        }
        if constexpr (CL == 1) {
            if (there) {
#pragma unroll
                for (int m0 = 0; m0 < NT; m0 += 16) {
                    if (m0 >= m) break;
                    if (turns == 2 && m0 / 16 % 2 != turn) continue;
                    int part[16];
                    tmem_ld16(lanes + m0, part);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        if (m0 + i >= m) break;
                        float v[4] = {__int_as_float(part[i]), __int_as_float(part[i + 1]), __int_as_float(part[i + 2]), __int_as_float(part[i + 3])};
                        finish_tokens<T>(t.p, v, m0 + i, c, bias);
                    }
                }
            }
        } else {
            // Neighbouring tokens to one CTA, kMine each: parts[rank][four tokens][channel] there, 16 bytes each
            cluster_wait();
            if (there) {
                uint32_t to[CL];
#pragma unroll
                for (int r = 0; r < CL; ++r) to[r] = map_to_rank(smem_u32(parts) + (rank * (S::kMine / 4) * kBM + channel) * 16, r);
#pragma unroll
                for (int m0 = 0; m0 < NT; m0 += 16) {
                    if (m0 >= m) break;
                    if (turns == 2 && m0 / 16 % 2 != turn) continue;
                    int part[16];
                    tmem_ld16(lanes + m0, part);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        if (m0 + i < m) sts128_cluster(to[(m0 + i) / S::kMine] + (m0 + i) % S::kMine / 4 * (kBM * 16), part[i], part[i + 1], part[i + 2], part[i + 3]);
                }
            }
            cluster_arrive();
            cluster_wait();
            if (there) {
                const float4 *from = reinterpret_cast<const float4 *>(parts) + channel;
#pragma unroll
                for (int i = 0; i < S::kMine; i += 4) {
                    const int m0 = rank * S::kMine + i;
                    if (m0 >= m) break;
                    if (turns == 2 && i / 4 % 2 != turn) continue;
                    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int r = 0; r < CL; ++r) {
                        const float4 s = from[(r * (S::kMine / 4) + i / 4) * kBM];
                        v[0] = __fadd_rn(v[0], s.x);
                        v[1] = __fadd_rn(v[1], s.y);
                        v[2] = __fadd_rn(v[2], s.z);
                        v[3] = __fadd_rn(v[3], s.w);
                    }
                    finish_tokens<T>(t.p, v, m0, c, bias);
                }
            }
        }
    }
    // All roles meet here, whether their work is done or a wait ran out.  What other CTAs write to this one's shared memory is there: every thread of a cluster has
    // been at both of its meetings.
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
        tmem_dealloc(tmem, S::kColumns);
    }
}

template <typename T, typename X, int NT, int CL>
int launch(const Params &p, int64_t x_pitch, int cols, int early, cudaStream_t stream) {
    using S = Shape<X, NT, CL>;
    CUtensorMap mw, mws, mx, mxs;
    const int bytes = p.groups * (mx::kGroup / 2), tiles = ceil_div(p.groups, mx::kTileGroups);
    int st = encode(&mw, p.w, p.n, bytes, p.w_pitch, kBM);
    if (st == TSB_OK) st = encode_scales(&mws, p.w_scales, p.n, tiles, 1);
    if (S::kQuantize) {
        mx = mw;
        mxs = mws;
    } else {
        if (st == TSB_OK) st = encode(&mx, p.x, p.m, bytes, p.x_pitch, NT);
        if (st == TSB_OK) st = encode_scales(&mxs, p.x_scales, p.m, tiles, 1);
    }
    if (st != TSB_OK) return st;
    FewParams t = {};
    t.p = p;
    t.kblocks = ceil_div(bytes, kKBytes);
    t.cols = cols;
    t.x_pitch = x_pitch;
    t.x_aligned = aligned16(p.x, x_pitch, sizeof(X) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16);
    t.early = early;
    if ((st = mxfp4_status_word(&t.status)) != TSB_OK) return st;
    auto kernel = inner_prod_mxfp4_few_kernel<T, X, NT, CL>;
    static DeviceOnce raised;
    if (raised.first()) {
        TSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        raised.done();
    }
    const int ctas = ceil_div(p.n, kBM) * CL, blocks = ceil_div(t.kblocks, CL);
    const int room = (int)(ctas <= 148 ? kSmem : kSmem / 2 - 1024) - (int)S::fixed(blocks);
    // (two stages or more: a cluster's CTA so takes 46 KB or more, four a multiprocessor fit its tensor memory, and none waits for columns that one of another cluster holds)
    t.stages = std::max(2, std::min({blocks, S::kMost + 0, room / (int)S::kStage}));
    static_assert(CL == 1 || 1024 + S::kBars + S::kParts + (S::kQuantize ? S::kTokens : 0) + 2 * S::kStage > 46 * 1024, "four CTAs a multiprocessor at most");
    TSB_CUDA(launch_pdl_cluster(CL, kernel, dim3(ctas), dim3(S::kThreads), S::fixed(blocks) + t.stages * S::kStage, stream, mw, mws, mx, mxs, t));
    TSB_LAUNCHED("inner_prod_mxfp4_few_kernel");
    return TSB_OK;
}

// CTAs that share a tile: as many as two on every multiprocessor leave, and no more than there are blocks of K.  (32 tokens through 8192 x 8192, by one, two and four CTAs a
// tile 11.4, 9.3 and 9.2 us; one token through 4096 x 4096 6.8, 5.2 and 4.4, through 16384 x 8192 16.5, 14.6 and 16.2.)
int cluster_of(const Params &p) {
    const int tiles = ceil_div(p.n, kBM), kblocks = ceil_div(p.groups * (mx::kGroup / 2), kKBytes);
    int cluster = 1;
    while (cluster < kMaxCluster && 2 * cluster <= kblocks && (int64_t)tiles * cluster * 2 <= 2 * 148) cluster *= 2;
    return cluster;
}

template <typename T, typename X, int NT>
int pick(const Params &p, int64_t x_pitch, int cols, int early, cudaStream_t stream) {
    switch (cluster_of(p)) {
        case 1: return launch<T, X, NT, 1>(p, x_pitch, cols, early, stream);
        case 2: return launch<T, X, NT, 2>(p, x_pitch, cols, early, stream);
        default: return launch<T, X, NT, 4>(p, x_pitch, cols, early, stream);
    }
}

template <typename T>
int pick(const Params &p, int early, cudaStream_t stream) {
    if (p.m <= 16) return pick<T, uint8_t, 16>(p, 0, 0, early, stream);
    if (p.m <= 32) return pick<T, uint8_t, 32>(p, 0, 0, early, stream);
    return pick<T, uint8_t, 64>(p, 0, 0, early, stream);
}

}  // namespace

// Up to 64 tokens in 4 bits.
int inner_prod(const Params &p, int y_type, int early, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick<float>(p, early, stream);
        case TSB_TYPE_F16: return pick<__half>(p, early, stream);
        default: return pick<__nv_bfloat16>(p, early, stream);
    }
}

// Rows that the kernel quantizes itself: what a CTA's part takes it is less than a launch of quantize_rows_mxfp4 in front (2.2 us) up to some 16 Ki values (4096 x 4096, by the
// kernel and by a launch: 1 token 4.1 and 6.5 us, 8 tokens 4.9 and 6.7, 16 tokens 6.2 and 6.9).
bool can_quantize(const Params &p, int x_type, int y_type) {
    const int64_t blocks = ceil_div(ceil_div(p.groups * (mx::kGroup / 2), kKBytes), cluster_of(p));
    return x_type == y_type && p.m <= 16 && p.m * blocks <= 64 && blocks * (16 * kKBytes + kScales) <= kMaxResident;
}

// Up to 16 floating rows of y's type.
int inner_prod_quantize(const Params &p, int y_type, int64_t x_pitch, int cols, cudaStream_t stream) {
    switch (y_type) {
        case TSB_TYPE_F32: return pick<float, float, 16>(p, x_pitch, cols, 0, stream);
        case TSB_TYPE_F16: return pick<__half, __half, 16>(p, x_pitch, cols, 0, stream);
        default: return pick<__nv_bfloat16, __nv_bfloat16, 16>(p, x_pitch, cols, 0, stream);
    }
}

}  // namespace few
}  // namespace tsb
