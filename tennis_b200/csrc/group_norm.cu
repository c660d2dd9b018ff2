// Group norm with an activation on channels-last tensors (no counterpart in the reference).
//
// Bound by memory: each value is read once and written once, if what lies between -- the statistics of its whole group -- is had
// without reading it again from HBM.
//
//   sums       in 64 bits: with 53 bits the difference of the mean square and the squared mean keeps 32-bit accuracy for means up to
//              10^4 deviations, in one pass over the data, and the order of summation shows in the rounded mean and deviation next to never
//   threads    a thread owns one 16-byte vector of channels (or one channel, where vectors do not fit) and walks over pixels: loads of
//              neighbouring threads are neighbours, its channels' gamma, beta and statistics stay in registers
//   resident   an image's run of groups is held in the shared memory of a cluster of up to eight blocks: loaded once, summed on the
//              way, the blocks' sums exchanged through distributed shared memory, normalized from shared memory.  One launch
//   swept      larger images: one launch sums, a small one makes the statistics, the third reads again and normalizes, in the reverse
//              order, so that it finds in the L2 what the first read last.  (Batch by batch, each small enough for the L2, the
//              launches' beginnings and ends cost more than the reads of HBM that they save: 8 x 256 x 256 x 256 bf16 152 us in one
//              batch when that was tried, 176 in batches of two images, 266 image by image)
// Measured: 16 x 56 x 56 x 256 bf16 to int8 20 us (resident; load, meeting and writing follow each other in its one round of blocks), 8 x 256 x 256 x 256
// bf16 with silu 147 us (swept: 805 MB at 5.5 TB/s, near the rate of a copy), 16 x 16 x 128 fp32 3.5 us.
#include "typed.cuh"

#include <algorithm>
#include <cmath>

namespace tsb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;                  // the portable limit
constexpr int kMaxGroups = 256;                 // groups of a run of channels
constexpr int kResidentBlocks = 4;               // resident blocks a multiprocessor, by their registers (2000 x 14 x 14 x 256 bf16 with silu 128 us; with three 131, against 122 at the time)
constexpr int64_t kLargeTile = 200 * 1024;      // shared memory of a resident block, at most

struct GroupNormParams {
    const void *x;
    void *y;
    int64_t x_pixel, x_image, y_pixel, y_image;   // elements
    const float *gamma, *beta;                    // or NULL
    int n, channels, groups, per;                 // per = channels of a group
    int64_t pixels;
    int run_groups, runs;                         // groups of a run of channels, runs of an image
    int cols;                                     // vectors of a run that the block's threads own at a time
    int64_t tile;                                 // pixels of a block's tile
    int tiles;                                    // ... and tiles of an image
    int let_go;                                   // swept: tiles whose values are not kept in the L2 for the second reading, which starts with the last
    double eps, one_over_count;                   // of a group's values: a product with it is off by half a step of 64 bits more than a quotient
    int activation;
    float leaky;
    int out_channels;                             // channels written: int8 outputs are padded with zeros
    int64_t rne_limit;                            // int8: values below this (in channel-major order) round half to even
    int tail;                                     // ... and there are values at or above it that do not
    int nscales;
    float scales[TSB_MAX_REQUANT_SCALES];
};

// A block's part of the work: channels [c0, c0 + width) of an image, pixels [p0, p1)
struct Part {
    int image, c0, width, g0, groups;
    int64_t p0, p1;
};
__device__ __forceinline__ Part part_of(const GroupNormParams &p, int image, int run, int tile) {
    Part t;
    t.image = image;
    t.g0 = run * p.run_groups;
    t.groups = min(p.run_groups, p.groups - t.g0);
    t.c0 = t.g0 * p.per;
    t.width = t.groups * p.per;
    t.p0 = min((int64_t)tile * p.tile, p.pixels);
    t.p1 = min(t.p0 + p.tile, p.pixels);
    return t;
}

// q8_half_even without a conversion (of which a multiprocessor does 16 a clock, the norm's sums take one a value): a sum with 1.5 * 2^23
// rounds to a whole number, half to even, that its low bits hold.
__device__ __forceinline__ int round_even(float v) {
    const float in = fminf(fmaxf(v, -128.0f), 127.0f);
    return fabsf(v) < 2147483648.0f ? __float_as_int(__fadd_rn(in, 12582912.0f)) : -128;      // (the caller keeps the low byte)
}

// VEC values of a type, as they lie in memory
template <typename T, int VEC> struct Raw { using type = uint4; };
template <typename T> struct Raw<T, 1> { using type = T; };
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const typename Raw<T, VEC>::type &q, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = to_f32(q);
    else Vec16<T>::get(q, v);
}

// Sums of a thread's channels; ONE: all channels of a vector belong to one group, and one pair of sums serves them.
// Every value and square goes into the 64-bit sums as it is.
template <int VEC, bool ONE>
struct Sums {
    static constexpr int kN = ONE ? 1 : VEC;
    double s[kN], ss[kN];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kN; ++i) s[i] = ss[i] = 0.0;
    }
    __device__ __forceinline__ void add(const float (&v)[VEC]) {
        double d[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] = (double)v[i];
        if constexpr (ONE && VEC > 1) {
            // (two chains each, and sums of pairs: an addition takes longer than to issue the eight)
            double a = d[0] + d[1], b = d[2] + d[3], e = d[0] * d[0], f = d[1] * d[1];
#pragma unroll
            for (int i = 4; i < VEC; i += 4) {
                a += d[i] + d[i + 1];
                b += d[i + 2] + d[i + 3];
            }
#pragma unroll
            for (int i = 2; i < VEC; i += 2) {
                e = fma(d[i], d[i], e);
                f = fma(d[i + 1], d[i + 1], f);
            }
            s[0] += a + b;
            ss[0] += e + f;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                s[i] += d[i];
                ss[i] = fma(d[i], d[i], ss[i]);
            }
        }
    }
};

// Adds the threads' sums of channels [b0, b1) of the run to the groups' sums in shared memory, in a fixed order: a few lanes take a
// group, each its entries of some rows.  Thread (row, col) of `rows` x `cols` owns vector b0 / VEC + col.
template <int VEC, bool ONE>
__device__ __forceinline__ void collect(const Sums<VEC, ONE> &sums, double2 *scratch, double2 *group_sums, int b0, int b1, int per, int groups, int rows, int cols) {
    constexpr int kN = ONE ? 1 : VEC, kStep = VEC / kN;     // entries of a vector, channels of an entry
#pragma unroll
    for (int i = 0; i < kN; ++i) scratch[i * kThreads + threadIdx.x] = make_double2(sums.s[i], sums.ss[i]);
    __syncthreads();
    // as many lanes a group (a power of two) as give every thread one
    const int g0 = b0 / per, g1 = min(groups, (b1 + per - 1) / per);
    const int lanes = g1 - g0 >= kThreads ? 1 : min(32, 1 << (31 - __clz(kThreads / (g1 - g0)))), lane = threadIdx.x & (lanes - 1);
    for (int first_g = g0; first_g < g1; first_g += kThreads / lanes) {       // (all threads: shuffles)
        const int g = first_g + threadIdx.x / lanes;
        double s = 0.0, ss = 0.0;
        if (g < g1) {
            const int a = (max(g * per, b0) - b0) / kStep, b = (min((g + 1) * per, b1) - b0) / kStep;      // the group's entries of a row
            for (int entry = a; entry < b; ++entry) {
                const double2 *from = scratch + (kN == 1 ? 0 : entry % kN) * kThreads + entry / kN;
                for (int row = lane; row < rows; row += lanes) {
                    const double2 t = from[row * cols];
                    s += t.x;
                    ss += t.y;
                }
            }
        }
        for (int o = lanes / 2; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if (g < g1 && lane == 0) {
            group_sums[g].x += s;
            group_sums[g].y += ss;
        }
    }
    __syncthreads();
}

// ---- a thread's vectors of a tile, one every `step` elements from x on, in turn to use(i, vector)
// By asynchronous copies into slots of the thread's own, kDepth ahead of their use: a thread reads back what it loaded itself, so
// neither registers nor barriers hold loads up.  slot: its first slot, in shared memory; slot_step: bytes to the next one; KEEP: every
// vector has a slot of its own and stays there, otherwise the kDepth slots go round.
constexpr int kDepth = 8;
static_assert(kDepth >= 8, "the sums' scratch, up to eight pairs a thread, lies where the slots were");
// (policy: which values the L2 lets go of first)
__device__ __forceinline__ void copy16(uint32_t to, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t to, const void *from, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t l2_policy(bool first_out) {
    uint64_t p;
    if (first_out) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint4 read16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
template <typename T, int VEC, bool KEEP, typename Use>
__device__ __forceinline__ void stream(const T *x, int64_t step, int n, uint32_t slot, uint32_t slot_step, uint64_t policy, const Use &use) {
    if constexpr (VEC > 1) {
        constexpr int kAhead = KEEP ? 4 * kDepth : kDepth;
        const T *next = x;
        uint32_t to = slot, at = slot;
        const uint32_t end = slot + kAhead * slot_step;
#pragma unroll 4
        for (int i = 0; i < kAhead; ++i, next += step, to += slot_step) {
            if (i < n) KEEP ? copy16(to, next) : copy16(to, next, policy);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        if (!KEEP) to = slot;
#pragma unroll 2
        for (int i = 0; i < n; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
            use(i, read16(at));
            if (i + kAhead < n) KEEP ? copy16(to, next) : copy16(to, next, policy);
            asm volatile("cp.async.commit_group;" ::: "memory");
            next += step;
            to += slot_step;
            at += slot_step;
            if (!KEEP && at == end) to = at = slot;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        constexpr int kAhead = 8;
        for (int i0 = 0; i0 < n; i0 += kAhead, x += kAhead * step) {
            T v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (i0 + i < n) v[i] = x[i * step];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (i0 + i < n) use(i0 + i, v[i]);
        }
    }
}

// {mean, 1 / sqrt(variance + eps)} of a group, each rounded once
__device__ __forceinline__ float2 statistics(const GroupNormParams &p, double s, double ss) {
    const double mean = s * p.one_over_count;
    const double raw = fma(-mean, mean, ss * p.one_over_count);
    const double var = raw < 0.0 ? 0.0 : raw;            // (a NaN stays one)
    return make_float2((float)mean, (float)(1.0 / sqrt(var + p.eps)));
}

// What a thread applies to its channels: statistics, gamma, beta, activation, rounding.  (Results of 16 bits could take gamma into the reciprocal
// deviation and the sum with beta into the product; but that product may lie beyond fp32 where what it is multiplied with brings it back.)
template <typename T, typename Y, int VEC, bool ONE>
struct Apply {
    static constexpr int kG = ONE ? 1 : VEC;
    float mean[kG], rstd[kG], gamma[VEC], beta[VEC];
    // c: the thread's first channel within the run
    __device__ __forceinline__ void init(const GroupNormParams &p, const Part &t, const float2 *stats, int c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float2 st = stats[(c + (ONE ? 0 : i)) / p.per];
            if (i < kG) {
                mean[i] = st.x;
                rstd[i] = st.y;
            }
            gamma[i] = p.gamma ? __ldg(p.gamma + t.c0 + c + i) : 1.0f;      // (a product with 1 and a sum with -0 change nothing)
            beta[i] = p.beta ? __ldg(p.beta + t.c0 + c + i) : -0.0f;
        }
    }
    // y: where the thread's channels of `pixel` go; first_out: they are the first that the L2 lets go of
    template <int ACT>
    __device__ __forceinline__ void run(const GroupNormParams &p, const Part &t, const typename Raw<T, VEC>::type &q, int64_t pixel, int c, Y *y, bool first_out) const {
        float v[VEC];
        unpack<T, VEC>(q, v);
        if constexpr (VEC > 1) {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float2 d = add2(make_float2(v[i], v[i + 1]), make_float2(-mean[ONE ? 0 : i], -mean[ONE ? 0 : i + 1]));
                // (products by twos, the sum one by one: the assembler makes fused operations of a packed product and a packed sum)
                const float2 r = mul2(mul2(d, make_float2(rstd[ONE ? 0 : i], rstd[ONE ? 0 : i + 1])), make_float2(gamma[i], gamma[i + 1]));
                v[i] = __fadd_rn(r.x, beta[i]);
                v[i + 1] = __fadd_rn(r.y, beta[i + 1]);
            }
        } else {
            v[0] = __fadd_rn(__fmul_rn(__fmul_rn(__fsub_rn(v[0], mean[0]), rstd[0]), gamma[0]), beta[0]);
        }
        activate<ACT, Y>(v, p.leaky);
        if constexpr (sizeof(Y) > 1) {
            if constexpr (VEC == 1) *y = from_f32<Y>(v[0]);
            else if (first_out) __stcs(reinterpret_cast<uint4 *>(y), Vec16<Y>::put(v));
            else *reinterpret_cast<uint4 *>(y) = Vec16<Y>::put(v);
        } else {
            const float scale = p.scales[p.nscales == 1 ? 0 : t.image];
            int r[VEC];
            if (p.nscales == 1 && !p.tail) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) r[i] = round_even(__fmul_rn(v[i], scale));
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) r[i] = q8(v[i], scale, ((int64_t)t.image * p.channels + t.c0 + c + i) * p.pixels + pixel < p.rne_limit);
            }
            if constexpr (VEC == 1) {
                *y = (int8_t)r[0];
            } else {
                uint32_t w[VEC / 4];
#pragma unroll
                for (int i = 0; i < VEC / 4; ++i)
                    w[i] = (uint32_t)(uint8_t)r[4 * i] | (uint32_t)(uint8_t)r[4 * i + 1] << 8 | (uint32_t)(uint8_t)r[4 * i + 2] << 16 | (uint32_t)(uint8_t)r[4 * i + 3] << 24;
                if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(y) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t *>(y) = w[0];
            }
        }
    }
};

// The zeros behind the last channel of an int8 output
template <typename Y>
__device__ __forceinline__ void pad_channels(const GroupNormParams &p, const Part &t) {
    if (sizeof(Y) > 1 || t.g0 + t.groups < p.groups) return;
    const int extra = p.out_channels - p.channels;
    for (int64_t i = threadIdx.x; i < (t.p1 - t.p0) * extra; i += kThreads)
        static_cast<int8_t *>(p.y)[t.image * p.y_image + (t.p0 + i / extra) * p.y_pixel + p.channels + i % extra] = 0;
}

// (not the aligned forms, for which all threads of a warp have to come at once: here they come from loops of different lengths)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ double2 load_of_rank(const double2 *mine, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    double2 v;
    asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(v.x), "=d"(v.y) : "r"(at) : "memory");
    return v;
}

// ---- resident: a cluster of p.tiles blocks holds a run of an image's groups
template <typename T, typename Y, int VEC, bool ONE>
__global__ void __launch_bounds__(kThreads, kResidentBlocks)
group_norm_resident_kernel(const __grid_constant__ GroupNormParams p) {
    using R = typename Raw<T, VEC>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    double2 *group_sums = reinterpret_cast<double2 *>(smem);
    double2 *scratch = group_sums + p.run_groups;
    float2 *stats = reinterpret_cast<float2 *>(scratch + (ONE ? 1 : VEC) * kThreads);
    R *held = reinterpret_cast<R *>(stats + (p.run_groups + 1) / 2 * 2);
    const int tile = blockIdx.x % p.tiles, unit = blockIdx.x / p.tiles;
    const Part t = part_of(p, unit / p.runs, unit % p.runs, tile);
    const int cols = t.width / VEC, rows = kThreads / cols, row = threadIdx.x / cols, col = threadIdx.x % cols;
    for (int g = threadIdx.x; g < t.groups; g += kThreads) group_sums[g] = make_double2(0.0, 0.0);
    pdl_sync();

    Sums<VEC, ONE> sums;
    sums.clear();
    const int count = (int)(t.p1 - t.p0);
    const int mine = row < rows && row < count ? (count - row + rows - 1) / rows : 0;      // this thread's pixels: row, row + rows, ...
    R *slots = held + row * cols + col;
    stream<T, VEC, true>(static_cast<const T *>(p.x) + t.image * p.x_image + (t.p0 + row) * p.x_pixel + t.c0 + col * VEC, rows * p.x_pixel, mine,
                         (uint32_t)__cvta_generic_to_shared(slots), rows * cols * sizeof(R), 0, [&](int i, const R &raw) {
                             float v[VEC];
                             unpack<T, VEC>(raw, v);
                             sums.add(v);
                             if (VEC == 1) slots[i * rows * cols] = raw;
                         });
    __syncthreads();
    collect(sums, scratch, group_sums, 0, t.width, p.per, t.groups, rows, cols);
    if (p.tiles > 1) {
        cluster_arrive();
        cluster_wait();
    }
    for (int g = threadIdx.x; g < t.groups; g += kThreads) {
        double2 v[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r) v[r] = r >= p.tiles ? make_double2(0.0, 0.0) : p.tiles > 1 ? load_of_rank(group_sums + g, r) : group_sums[g];
#pragma unroll
        for (int o = 1; o < kMaxCluster; o *= 2)
#pragma unroll
            for (int r = 0; r + o < kMaxCluster; r += 2 * o) {
                v[r].x += v[r + o].x;
                v[r].y += v[r + o].y;
            }
        stats[g] = statistics(p, v[0].x, v[0].y);
    }
    if (p.tiles > 1) cluster_arrive();       // this block has read the others' sums (they stay until all have: the wait at the end)
    __syncthreads();
    if (mine > 0) {
        Apply<T, Y, VEC, ONE> apply;
        apply.init(p, t, stats, col * VEC);
        Y *y = static_cast<Y *>(p.y) + t.image * p.y_image + (t.p0 + row) * p.y_pixel + t.c0 + col * VEC;
        const R *from = slots;
        by_activation(p.activation, [&](auto act) {
#pragma unroll 4
            for (int i = 0; i < mine; ++i, from += rows * cols, y += rows * p.y_pixel)
                apply.template run<decltype(act)::value>(p, t, *from, t.p0 + row + i * rows, col * VEC, y, false);
        });
    }
    pad_channels<Y>(p, t);
    if (p.tiles > 1) cluster_wait();
}

// ---- swept: the sums, a block a tile, to sums[image][run][tile][group of the run]
template <typename T, int VEC, bool ONE>
__global__ void __launch_bounds__(kThreads, 4)
group_norm_sums_kernel(const __grid_constant__ GroupNormParams p, double2 *all_sums) {
    using R = typename Raw<T, VEC>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    double2 *group_sums = reinterpret_cast<double2 *>(smem);
    double2 *scratch = group_sums + p.run_groups;
    const int tile = blockIdx.x % p.tiles, unit0 = blockIdx.x / p.tiles, run = unit0 % p.runs, image = unit0 / p.runs;
    const Part t = part_of(p, image, run, tile);
    const int count = (int)(t.p1 - t.p0);
    const int rows = kThreads / p.cols, row = threadIdx.x / p.cols, col = threadIdx.x % p.cols;
    for (int g = threadIdx.x; g < t.groups; g += kThreads) group_sums[g] = make_double2(0.0, 0.0);
    pdl_sync();
    for (int b0 = 0; b0 < t.width; b0 += p.cols * VEC) {
        const int b1 = min(b0 + p.cols * VEC, t.width), c = b0 + col * VEC;
        Sums<VEC, ONE> sums;
        sums.clear();
        if (row < rows && row < count && c < b1)
            stream<T, VEC, false>(static_cast<const T *>(p.x) + t.image * p.x_image + (t.p0 + row) * p.x_pixel + t.c0 + c, rows * p.x_pixel, (count - row + rows - 1) / rows,
                                  (uint32_t)__cvta_generic_to_shared(scratch) + threadIdx.x * 16, kThreads * 16, l2_policy((int)blockIdx.x < p.let_go), [&](int, const R &raw) {
                                      float v[VEC];
                                      unpack<T, VEC>(raw, v);
                                      sums.add(v);
                                  });
        __syncthreads();
        collect(sums, scratch, group_sums, b0, b1, p.per, t.groups, rows, p.cols);
    }
    double2 *mine = all_sums + (((int64_t)image * p.runs + run) * p.tiles + tile) * p.run_groups;
    for (int g = threadIdx.x; g < t.groups; g += kThreads) mine[g] = group_sums[g];
}

// ---- swept: the statistics, a warp a group; its tiles' sums in a fixed order
__global__ void __launch_bounds__(kThreads)
group_norm_stats_kernel(const __grid_constant__ GroupNormParams p, const double2 *all_sums, float2 *all_stats) {
    pdl_sync();
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (i >= (int64_t)p.n * p.groups) return;
    const int64_t image = i / p.groups;
    const int group = (int)(i - image * p.groups), run = group / p.run_groups;
    const double2 *from = all_sums + (image * p.runs + run) * p.tiles * p.run_groups + (group - run * p.run_groups);
    double s = 0.0, ss = 0.0;
#pragma unroll 4
    for (int k = lane; k < p.tiles; k += 32) {
        const double2 v = from[(int64_t)k * p.run_groups];
        s += v.x;
        ss += v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (lane == 0) all_stats[i] = statistics(p, s, ss);
}

// ---- swept: the outputs, last tile first (what the sums read last is in the L2 for certain)
template <typename T, typename Y, int VEC, bool ONE>
__global__ void __launch_bounds__(kThreads, 4)
group_norm_apply_kernel(const __grid_constant__ GroupNormParams p, const float2 *all_stats) {
    using R = typename Raw<T, VEC>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    const int item = gridDim.x - 1 - blockIdx.x, tile = item % p.tiles, unit0 = item / p.tiles, run = unit0 % p.runs, image = unit0 / p.runs;
    const Part t = part_of(p, image, run, tile);
    const int count = (int)(t.p1 - t.p0);
    const int rows = kThreads / p.cols, row = threadIdx.x / p.cols, col = threadIdx.x % p.cols;
    pdl_sync();
    const float2 *stats = all_stats + (int64_t)image * p.groups + t.g0;
    for (int c = col * VEC; c < t.width; c += p.cols * VEC) {
        if (row >= rows || row >= count) break;
        Apply<T, Y, VEC, ONE> apply;
        apply.init(p, t, stats, c);
        Y *y = static_cast<Y *>(p.y) + t.image * p.y_image + (t.p0 + row) * p.y_pixel + t.c0 + c;
        by_activation(p.activation, [&](auto act) {
            stream<T, VEC, false>(static_cast<const T *>(p.x) + t.image * p.x_image + (t.p0 + row) * p.x_pixel + t.c0 + c, rows * p.x_pixel, (count - row + rows - 1) / rows,
                                  (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16, kThreads * 16, l2_policy(p.let_go > 0), [&](int i, const R &raw) {
                                      apply.template run<decltype(act)::value>(p, t, raw, t.p0 + row + i * rows, c, y, p.let_go > 0);
                                      y += rows * p.y_pixel;
                                  });
        });
    }
    pad_channels<Y>(p, t);
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

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// How a call runs: by 16-byte vectors or value by value, resident or swept, in which runs of channels and tiles of pixels.
struct Plan {
    int vec;
    bool one, resident;
    int run_groups, runs, cols, tiles;
    int64_t tile;
    int let_go;
    size_t smem, off_stats, bytes;    // of shared memory; of the workspace
};

size_t scratch_bytes(int vec, bool one, int run_groups) { return (size_t)run_groups * 16 + (size_t)(one ? 1 : vec) * kThreads * 16 + (size_t)(run_groups + 1) / 2 * 16; }

Plan make_plan(const tsb_group_norm_desc *d) {
    const int size = (int)type_bytes(d->x_type), per = (int)(d->channels / d->groups), groups = (int)d->groups, vectors = 16 / size;
    auto fits = [&](const void *at, int64_t pixel, int64_t image) {
        return reinterpret_cast<uintptr_t>(at) % 16 == 0 && (d->pixels == 1 || pixel * size % 16 == 0) && (d->n == 1 || image * size % 16 == 0);
    };
    Plan q = {};
    const bool wide = d->channels % vectors == 0 && fits(d->x, d->x_pixel_stride, d->x_image_stride) &&
                      (d->y_type == TSB_TYPE_I8 || fits(d->y, d->y_pixel_stride, d->y_image_stride));
    q.vec = wide ? vectors : 1;
    q.one = per % q.vec == 0;
    // groups that make whole vectors
    int step = 1;
    while (step * per % q.vec) ++step;
    // Resident: as many blocks as run at the same time (a second round of them waits for the first to be through all of its steps:
    // 16 x 56 x 56 x 256 bf16 in 512 blocks of 50 KB, four a multiprocessor, 20 us; three, which makes two rounds, 25), of as many the smaller cluster; rows of 64
    // bytes or more, tiles of 16 KB or more where there is a choice.  Images that do not fit so are swept (4 x 128 x 128 x 128 fp32: 22 us,
    // resident in two rounds 33).
    int64_t best = 0;
    for (int rg = (groups + step - 1) / step * step; rg >= step; rg = rg > step ? std::max(step, rg / 2 / step * step) : 0) {
        const int run = std::min(rg, groups), width = run * per;
        if (run > kMaxGroups || width / q.vec > kThreads) continue;
        if (width * size < 64 && run < groups) break;
        const int runs = ceil_div(groups, run);
        for (int s = 1; s <= kMaxCluster; s *= 2) {
            const int64_t tile = ceil_div64(d->pixels, s), bytes = tile * width * size, smem = bytes + (int64_t)scratch_bytes(q.vec, q.one, run);
            if (smem > kLargeTile) continue;
            if (best && bytes < 16 * 1024) break;
            const int64_t blocks = d->n * runs * s, at_once = 148 * std::min<int64_t>(kResidentBlocks, (227 * 1024) / (smem + 1024));
            if (blocks > at_once && !(s == 1 && smem <= 113 * 1024)) continue;      // (blocks that meet no others may take turns, two a multiprocessor or more)
            if (blocks < best || (blocks == best && s >= q.tiles) || blocks > INT32_MAX) continue;
            best = blocks;
            q.resident = true;
            q.run_groups = run; q.runs = runs; q.tiles = s; q.tile = tile; q.cols = width / q.vec;
            q.smem = (size_t)smem;
        }
    }
    if (q.resident) return q;
    // Swept: runs of as many channels as the block's threads own vectors, of 16 KB or more
    q.run_groups = std::max(step, std::min({groups, kMaxGroups, kThreads * q.vec / per}) / step * step);
    q.run_groups = std::min(q.run_groups, groups);
    q.runs = ceil_div(groups, q.run_groups);
    const int width = q.run_groups * per;
    q.cols = std::min(width / q.vec, kThreads);
    const int64_t blocks = std::max<int64_t>(1, 148 * 4 / (d->n * q.runs));      // four blocks a multiprocessor, all at once
    q.tile = std::max(ceil_div64(d->pixels, blocks), std::max<int64_t>(1, 16384 / ((int64_t)width * size)));
    q.tiles = (int)ceil_div64(d->pixels, q.tile);
    q.smem = (size_t)q.run_groups * 16 + (size_t)kDepth * kThreads * 16;      // (at least collect's scratch: a vector has at most eight pairs of sums)
    // Of a tensor beyond 80 MB the L2 is to keep that much, the end of it, for the second reading: what comes before, and the outputs, goes
    // first (8 x 256 x 256 x 256 bf16 154 -> 151 us, 16 x 128 x 128 x 256 79 -> 73 when it came; 147 and 76 now)
    q.let_go = (int)std::max<int64_t>(0, std::min<int64_t>(INT32_MAX, d->n * q.runs * q.tiles - (80 << 20) / std::max<int64_t>(1, q.tile * width * size)));
    q.off_stats = align256((size_t)d->n * q.runs * q.tiles * q.run_groups * sizeof(double2));
    q.bytes = q.off_stats + align256((size_t)d->n * groups * sizeof(float2));
    return q;
}

template <typename T, typename Y, int VEC, bool ONE>
int launch(const GroupNormParams &p, const Plan &q, char *workspace, cudaStream_t stream) {
    if (q.resident) {
        auto kernel = group_norm_resident_kernel<T, Y, VEC, ONE>;
        static DeviceOnce raised;
        if (raised.first()) {
            TSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLargeTile));
            raised.done();
        }
        TSB_CUDA(launch_pdl_cluster(p.tiles, kernel, dim3(p.n * p.runs * p.tiles), dim3(kThreads), q.smem, stream, p));
        TSB_LAUNCHED("group_norm_resident_kernel");
        return TSB_OK;
    }
    double2 *sums = reinterpret_cast<double2 *>(workspace);
    float2 *stats = reinterpret_cast<float2 *>(workspace + q.off_stats);
    const int64_t blocks = (int64_t)p.n * p.runs * p.tiles, groups = (int64_t)p.n * p.groups;
    if (blocks > INT32_MAX) return fail(TSB_ERR_UNSUPPORTED, "group_norm: more than 2^31 tiles");
    TSB_CUDA(launch_pdl(group_norm_sums_kernel<T, VEC, ONE>, dim3((unsigned)blocks), dim3(kThreads), q.smem, stream, p, sums));
    TSB_LAUNCHED("group_norm_sums_kernel");
    TSB_CUDA(launch_pdl(group_norm_stats_kernel, dim3((unsigned)ceil_div64(groups, kWarps)), dim3(kThreads), 0, stream, p, sums, stats));
    TSB_LAUNCHED("group_norm_stats_kernel");
    TSB_CUDA(launch_pdl(group_norm_apply_kernel<T, Y, VEC, ONE>, dim3((unsigned)blocks), dim3(kThreads), (size_t)kDepth * kThreads * 16, stream, p, stats));
    TSB_LAUNCHED("group_norm_apply_kernel");
    return TSB_OK;
}

template <typename T, typename Y>
int pick(const GroupNormParams &p, const Plan &q, char *workspace, cudaStream_t stream) {
    if (q.vec == 1) return launch<T, Y, 1, true>(p, q, workspace, stream);
    return q.one ? launch<T, Y, Vec16<T>::kN, true>(p, q, workspace, stream) : launch<T, Y, Vec16<T>::kN, false>(p, q, workspace, stream);
}

}  // namespace

size_t group_norm_workspace_bytes(const tsb_group_norm_desc *d) {
    return check_desc(d) != TSB_OK || d->n == 0 || d->pixels == 0 ? 0 : make_plan(d).bytes;
}

int group_norm_nhwc(const tsb_group_norm_desc *d, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    int st = check_desc(d);
    if (st != TSB_OK || d->n == 0 || d->pixels == 0) return st;
    const Plan q = make_plan(d);
    if (q.bytes) {
        if (!workspace || workspace_bytes < q.bytes) return fail(TSB_ERR_WORKSPACE_TOO_SMALL, "group_norm: %zu bytes of workspace, %zu needed", workspace ? workspace_bytes : (size_t)0, q.bytes);
        if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(TSB_ERR_INVALID_ARGUMENT, "group_norm: the workspace must be 256-byte aligned");
    }
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
    p.run_groups = q.run_groups;
    p.runs = q.runs;
    p.cols = q.cols;
    p.tile = q.tile;
    p.tiles = q.tiles;
    p.let_go = q.let_go;
    p.eps = d->eps;
    p.one_over_count = 1.0 / ((double)d->pixels * p.per);
    p.activation = d->activation;
    p.leaky = d->leaky_scale;
    p.out_channels = i8 ? tsb_padded_channels(p.channels) : p.channels;
    p.y_pixel = i8 ? p.out_channels : d->y_pixel_stride;
    p.y_image = i8 ? p.out_channels * d->pixels : d->y_image_stride;
    if (i8) {
        p.nscales = d->n_requant_scales;
        p.rne_limit = p.nscales == 1 ? d->n * d->pixels * d->channels / 8 * 8 : 0;
        p.tail = p.nscales == 1 && p.rne_limit < d->n * d->pixels * d->channels;
        for (int i = 0; i < p.nscales; ++i) p.scales[i] = d->requant_scales_host[i];
    }
    char *room = static_cast<char *>(workspace);
    switch (d->x_type) {
        case TSB_TYPE_F32: return i8 ? pick<float, int8_t>(p, q, room, stream) : pick<float, float>(p, q, room, stream);
        case TSB_TYPE_F16: return i8 ? pick<__half, int8_t>(p, q, room, stream) : pick<__half, __half>(p, q, room, stream);
        default: return i8 ? pick<__nv_bfloat16, int8_t>(p, q, room, stream) : pick<__nv_bfloat16, __nv_bfloat16>(p, q, room, stream);
    }
}

}  // namespace tsb
