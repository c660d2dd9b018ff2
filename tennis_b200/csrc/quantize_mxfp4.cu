// Rows in microscaled 4-bit floating point, and back.
//
// Bound by memory.  A warp takes neighbouring values of a row: the largest magnitude of a group is found among the lanes that hold it, so nothing goes
// through shared memory.  Instructions are what it takes to get there (at 19 a value, with 64-bit indexes and checks for every 16 bytes, 8192 x 16384
// bf16 took 91 us): rows of more than a run go by runs whose ends are checked once.
// Measured: 8192 x 16384 bf16 49 us (7.0 TB/s), back 52 us (6.5 TB/s); 16384 x 8192 fp32 85 and 93 us; 200000 x 64 bf16 7.1 and 15 us; 16 x 4096 bf16 1.5 and 1.6 us; rows off 16 bytes,
// value by value, 32768 x 1111 bf16 48 and 80 us.
#include "mxfp4.cuh"

#include <algorithm>

namespace tsb {
namespace {

constexpr int kThreads = 256;

// 32 neighbouring bytes
struct Bytes32 {
    uint4 v[2];
    __device__ __forceinline__ void load(const void *from) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w) : "l"(from) : "memory");
    }
};

// A warp's tiles of 128 values in rows of few of them: kLanes lanes a tile, kAtOnce neighbouring tiles in each of kTurns turns, one row behind the other (at most 2^31
// tiles in all).
template <int kN>
struct Tiles {
    static constexpr int kLanes = 128 / kN, kAtOnce = 32 / kLanes, kTurns = 4, kRun = kAtOnce * kTurns;
    uint32_t first, inverse, tiles;
    __device__ __forceinline__ Tiles(int tiles_of_row, uint32_t inverse_of_tiles) : inverse(inverse_of_tiles), tiles(tiles_of_row) {
        first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kRun + (threadIdx.x & 31) / kLanes;
    }
    // the tile of turn i
    __device__ __forceinline__ void at(int i, int64_t &r, int &t) const {
        const uint32_t u = first + i * kAtOnce;
        uint32_t q = tiles == 1 ? u : __umulhi(u, inverse);      // the quotient or one less (inverse: 2^32 / tiles, rounded down)
        if (u - q * tiles >= tiles) ++q;
        r = q;
        t = (int)(u - q * tiles);
    }
    static bool narrow(int64_t rows, int64_t tiles) { return tiles < kRun && rows * tiles < ((int64_t)1 << 31) - 65536; }
    static int64_t blocks(int64_t rows, int64_t tiles) { return ceil_div64(rows * tiles, (int64_t)kRun * (kThreads / 32)); }
    static uint32_t inverse_of(int64_t tiles) { return (uint32_t)std::min<uint64_t>(UINT32_MAX, ((uint64_t)1 << 32) / (uint64_t)tiles); }
};

// Other rows: a run of 2 KB of a row a warp, 32 neighbouring bytes a lane and turn, two (four) lanes a group.  `whole`: all rows start on 32 bytes, their
// codes on 8 and the scales on 4, so that runs within a row need no check.
template <typename T>
struct Run {
    static constexpr int kN = 32 / sizeof(T), kLanes = 128 / kN, kTurns = 2, kTurn = 32 * kN, kValues = kTurns * kTurn;
};
template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_mxfp4_kernel(const T *x, int64_t x_pitch, uint8_t *q, int64_t q_pitch, uint8_t *scales, int64_t rows, int64_t room_rows, int cols, int tiles, int runs, int whole,
                           int x_aligned, int q_aligned, int s_aligned) {
    using R = Run<T>;
    pdl_sync();
    const int lane = threadIdx.x & 31, in = lane % R::kLanes;
    const int64_t run = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), r = runs == 1 ? run : run / runs;
    const int c0 = (int)(run - r * runs) * R::kValues + lane * R::kN;      // the lane's first value
    if (r >= room_rows) return;
    const T *from = x + r * x_pitch + c0;
    uint8_t *to = q + r * q_pitch + c0 / 2, *words = scales + mx::word_at(r, c0 / 128, tiles);
    if (whole && r < rows && c0 - lane * R::kN + R::kValues <= cols) {
        Bytes32 held[R::kTurns];
#pragma unroll
        for (int i = 0; i < R::kTurns; ++i) held[i].load(from + i * R::kTurn);
#pragma unroll
        for (int i = 0; i < R::kTurns; ++i) {
            uint32_t codes[R::kN / 8], word;
            mx::quantize_bytes<T>(held[i].v, codes, &word);
            if constexpr (R::kN == 16) *reinterpret_cast<uint2 *>(to + i * (R::kTurn / 2)) = make_uint2(codes[0], codes[1]);
            else *reinterpret_cast<uint32_t *>(to + i * (R::kTurn / 2)) = codes[0];
            if (in == 0) *reinterpret_cast<uint32_t *>(words + i * (R::kTurn / 128 * mx::kTileBytes)) = word;
        }
        return;
    }
    const int used = (cols + mx::kGroup - 1) / mx::kGroup * mx::kGroup;      // values of a row with those that fill up its last group
#pragma unroll 1
    for (int i = 0; i < R::kTurns; ++i) {
        const int c = c0 + i * R::kTurn;
        Bytes32 held;
        held.v[0] = held.v[1] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            held.v[0] = mx::load_values(from, 0, cols - c, x_aligned);
            held.v[1] = mx::load_values(from, R::kN / 2, cols - c, x_aligned);
        }
        uint32_t codes[R::kN / 8], word;
        mx::quantize_bytes<T>(held.v, codes, &word);
        if (r < rows && c < used) {
#pragma unroll
            for (int h = 0; h < R::kN / 8; ++h) mx::store_codes<8>(to + 4 * h, codes[h], q_aligned);
        }
        if (in == 0 && c / 128 < tiles) mx::store_scales(words, word, s_aligned);
        from += R::kTurn;
        to += R::kTurn / 2;
        words += R::kTurn / 128 * mx::kTileBytes;
    }
}

// Rows of few tiles: a group a lane, which reads 64 (fp32: 128) bytes of it; four lanes a tile, one row behind the other.  (With a group among lanes, as above, and where it lies
// worked out for every 16 bytes, 200000 x 64 bf16 took 24 us, so 7.)
template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_mxfp4_narrow_kernel(const T *x, int64_t x_pitch, uint8_t *q, int64_t q_pitch, uint8_t *scales, int64_t rows, int64_t room_rows, int cols, int tiles, uint32_t inverse,
                                  int x_aligned, int q_aligned, int s_aligned) {
    constexpr int kN = Vec16<T>::kN, kVectors = mx::kGroup / kN;
    pdl_sync();
    const uint32_t u = blockIdx.x * kThreads + threadIdx.x, groups = 4 * (uint32_t)tiles;
    uint32_t row = __umulhi(u, inverse);                     // the quotient or one less (inverse: 2^32 / groups, rounded down)
    if (u - row * groups >= groups) ++row;
    const int64_t r = row;
    const int c = (int)(u - row * groups) * mx::kGroup;
    const bool live = r < rows && c < cols;
    uint4 held[kVectors];
    const T *from = x + r * x_pitch + c;
    if (live && x_aligned && c + mx::kGroup <= cols) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) held[i] = reinterpret_cast<const uint4 *>(from)[i];
    } else {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            held[i] = make_uint4(0, 0, 0, 0);
            if (live) held[i] = mx::load_values(from, i * kN, cols - c, x_aligned);
        }
    }
    Largest<T> largest;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) largest.add(held[i]);
    const uint32_t byte = mx::scale_byte(largest.bits());
    uint32_t word = byte << (8 * (threadIdx.x % 4));
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    if (live) {
        const float by = mx::inverse_scale(byte);
        float v[mx::kGroup];
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            float some[kN];
            Vec16<T>::get(held[i], some);
#pragma unroll
            for (int j = 0; j < kN; j += 2) {
                const float2 t = mul2(make_float2(some[j], some[j + 1]), make_float2(by, by));
                v[i * kN + j] = t.x;
                v[i * kN + j + 1] = t.y;
            }
        }
        uint32_t codes[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float some[8] = {v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]};
            codes[i] = mx::codes8(some);
        }
        uint8_t *to = q + r * q_pitch + c / 2;
        if (q_aligned) *reinterpret_cast<uint4 *>(to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) mx::store_codes<8>(to + 4 * i, codes[i], false);
    }
    if (threadIdx.x % 4 == 0 && r < room_rows) mx::store_scales(scales + mx::word_at(r, c / 128, tiles), word, s_aligned);
}

// Runs of other rows' values to y: 16 bytes of y a lane and turn.  `whole`: rows of codes start on their lanes' bytes and rows of y on 16 bytes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
dequantize_rows_mxfp4_kernel(const uint8_t *q, int64_t q_pitch, const uint8_t *scales, T *y, int64_t y_pitch, int64_t rows, int cols, int tiles, int runs, int whole, int q_aligned, int y_aligned) {
    constexpr int kN = Vec16<T>::kN, kTurns = 4, kTurn = 32 * kN;
    pdl_sync();
    const int lane = threadIdx.x & 31;
    const int64_t run = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), r = runs == 1 ? run : run / runs;
    const int c0 = (int)(run - r * runs) * (kTurns * kTurn) + lane * kN;
    if (r >= rows) return;
    const uint8_t *from = q + r * q_pitch + c0 / 2, *bytes = scales + mx::word_at(r, c0 / 128, tiles) + lane * kN % 128 / mx::kGroup;
    T *to = y + r * y_pitch + c0;
    const bool all = whole && c0 - lane * kN + kTurns * kTurn <= cols;
    uint32_t codes[kTurns], byte[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        codes[i] = byte[i] = 0;
        if (all || c0 + i * kTurn < cols) {
            const uint8_t *at = from + i * (kTurn / 2);
            if (all || q_aligned) {
                if constexpr (kN == 8) codes[i] = *reinterpret_cast<const uint32_t *>(at);
                else codes[i] = *reinterpret_cast<const uint16_t *>(at);
            } else {
#pragma unroll
                for (int b = 0; b < kN / 2; ++b) codes[i] |= (uint32_t)at[b] << (8 * b);
            }
            byte[i] = bytes[i * (kTurn / 128 * mx::kTileBytes)];
        }
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const uint4 out = mx::values_vector<T>(codes[i], byte[i]);
        if (all || (y_aligned && c0 + i * kTurn + kN <= cols)) {
            *reinterpret_cast<uint4 *>(to + i * kTurn) = out;
        } else {
            const T *o = reinterpret_cast<const T *>(&out);
#pragma unroll
            for (int j = 0; j < kN; ++j)
                if (c0 + i * kTurn + j < cols) to[i * kTurn + j] = o[j];
        }
    }
}

// Rows of few tiles.
template <typename T>
__global__ void __launch_bounds__(kThreads)
dequantize_rows_mxfp4_narrow_kernel(const uint8_t *q, int64_t q_pitch, const uint8_t *scales, T *y, int64_t y_pitch, int64_t rows, int64_t cols, int tiles, uint32_t inverse, int q_aligned, int y_aligned) {
    constexpr int kN = Vec16<T>::kN;
    using W = Tiles<kN>;
    pdl_sync();
    const int in = (threadIdx.x & 31) % W::kLanes;
    const W walk(tiles, inverse);
    uint32_t codes[W::kTurns];
    uint8_t byte[W::kTurns];
#pragma unroll
    for (int i = 0; i < W::kTurns; ++i) {
        int64_t r;
        int t;
        walk.at(i, r, t);
        const int64_t c = (int64_t)t * 128 + in * kN;
        codes[i] = byte[i] = 0;
        if (r < rows && c < cols) {
            const uint8_t *from = q + r * q_pitch + c / 2;
            if (q_aligned) {
                if constexpr (kN == 8) codes[i] = *reinterpret_cast<const uint32_t *>(from);
                else codes[i] = *reinterpret_cast<const uint16_t *>(from);
            } else {
#pragma unroll
                for (int b = 0; b < kN / 2; ++b) codes[i] |= (uint32_t)from[b] << (8 * b);
            }
            byte[i] = scales[mx::word_at(r, t, tiles) + in * kN / mx::kGroup];
        }
    }
#pragma unroll
    for (int i = 0; i < W::kTurns; ++i) {
        int64_t r;
        int t;
        walk.at(i, r, t);
        const int64_t c = (int64_t)t * 128 + in * kN;
        if (r >= rows || c >= cols) continue;
        T *to = y + r * y_pitch + c;
        const uint4 out = mx::values_vector<T>(codes[i], byte[i]);
        if (y_aligned && c + kN <= cols) {
            *reinterpret_cast<uint4 *>(to) = out;
        } else {
            const T *o = reinterpret_cast<const T *>(&out);
#pragma unroll
            for (int j = 0; j < kN; ++j)
                if (c + j < cols) to[j] = o[j];
        }
    }
}

template <typename T>
int launch_quantize(const void *x, int64_t x_pitch, uint8_t *q, int64_t q_pitch, uint8_t *scales, int64_t rows, int64_t cols, cudaStream_t stream) {
    using W = Tiles<Vec16<T>::kN>;
    const int64_t tiles = mx::tiles_of(cols), room_rows = ceil_div64(rows, mx::kTileRows) * mx::kTileRows;
    const auto address = reinterpret_cast<uintptr_t>(x);
    const int x_aligned = aligned16(x, x_pitch, sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16);
    const int q_aligned = reinterpret_cast<uintptr_t>(q) % 4 == 0 && q_pitch % 4 == 0, s_aligned = reinterpret_cast<uintptr_t>(scales) % 4 == 0;
    if (W::narrow(4 * room_rows, tiles)) {
        const int q_wide = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_pitch % 16 == 0;
        TSB_CUDA(launch_pdl(quantize_rows_mxfp4_narrow_kernel<T>, dim3((int)ceil_div64(4 * room_rows * tiles, kThreads)), dim3(kThreads), 0, stream, static_cast<const T *>(x), x_pitch, q, q_pitch,
                            scales, rows, room_rows, (int)cols, (int)tiles, W::inverse_of(4 * tiles), x_aligned, q_wide, s_aligned));
        TSB_LAUNCHED("quantize_rows_mxfp4_narrow_kernel");
        return TSB_OK;
    }
    const int64_t runs = ceil_div64(tiles * 128, Run<T>::kValues), blocks = ceil_div64(room_rows * runs, kThreads / 32);
    if (blocks > INT32_MAX) return fail(TSB_ERR_INVALID_ARGUMENT, "quantize_rows_mxfp4: too many values");
    const int whole = address % 32 == 0 && x_pitch * (int64_t)sizeof(T) % 32 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && q_pitch % 8 == 0 && s_aligned;
    TSB_CUDA(launch_pdl(quantize_rows_mxfp4_kernel<T>, dim3((int)blocks), dim3(kThreads), 0, stream, static_cast<const T *>(x), x_pitch, q, q_pitch, scales, rows, room_rows, (int)cols,
                        (int)tiles, (int)runs, whole, x_aligned, q_aligned, s_aligned));
    TSB_LAUNCHED("quantize_rows_mxfp4_kernel");
    return TSB_OK;
}

template <typename T>
int launch_dequantize(const uint8_t *q, int64_t q_pitch, const uint8_t *scales, void *y, int64_t y_pitch, int64_t rows, int64_t cols, cudaStream_t stream) {
    constexpr int kN = Vec16<T>::kN;
    using W = Tiles<kN>;
    const int64_t tiles = mx::tiles_of(cols);
    const int q_aligned = reinterpret_cast<uintptr_t>(q) % 4 == 0 && q_pitch % 4 == 0, y_aligned = aligned16(y, y_pitch, sizeof(T) == 4 ? TSB_TYPE_F32 : TSB_TYPE_F16);
    if (W::narrow(rows, tiles)) {
        TSB_CUDA(launch_pdl(dequantize_rows_mxfp4_narrow_kernel<T>, dim3((int)W::blocks(rows, tiles)), dim3(kThreads), 0, stream, q, q_pitch, scales, static_cast<T *>(y), y_pitch, rows, cols,
                            (int)tiles, W::inverse_of(tiles), q_aligned, y_aligned));
        TSB_LAUNCHED("dequantize_rows_mxfp4_narrow_kernel");
        return TSB_OK;
    }
    const int64_t runs = ceil_div64(cols, 4 * 32 * kN), blocks = ceil_div64(rows * runs, kThreads / 32);
    if (blocks > INT32_MAX) return fail(TSB_ERR_INVALID_ARGUMENT, "dequantize_rows_mxfp4: too many values");
    TSB_CUDA(launch_pdl(dequantize_rows_mxfp4_kernel<T>, dim3((int)blocks), dim3(kThreads), 0, stream, q, q_pitch, scales, static_cast<T *>(y), y_pitch, rows, (int)cols, (int)tiles, (int)runs,
                        (int)(q_aligned && y_aligned), q_aligned, y_aligned));
    TSB_LAUNCHED("dequantize_rows_mxfp4_kernel");
    return TSB_OK;
}

// What both directions ask of a 4-bit matrix and the floating one beside it (f: that one)
int check(const char *name, const void *q, int64_t q_pitch, const void *scales, const void *f, int type, int64_t f_pitch, bool f_is_read, int64_t rows, int64_t cols) {
    if (!is_float_type(type)) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: type %d is no floating type", name, type);
    if (rows < 0 || cols < 1 || cols > INT32_MAX - 65536) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: bad shape [%lld, %lld]", name, (long long)rows, (long long)cols);
    if (rows == 0) return TSB_OK;
    if (!q || !scales || !f) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (reinterpret_cast<uintptr_t>(f) % type_bytes(type)) return fail(TSB_ERR_INVALID_ARGUMENT, "%s: tensors must be aligned to their element", name);
    if (rows > 1 && (f_pitch < (f_is_read ? 0 : cols) || q_pitch < (f_is_read ? mx::row_bytes(cols) : 0)))
        return fail(TSB_ERR_INVALID_ARGUMENT, "%s: rows overlap (pitch)", name);
    if (extent_bytes(rows, rows > 1 ? f_pitch : 0, cols, type) < 0 || extent_bytes(rows, rows > 1 ? q_pitch : 0, mx::row_bytes(cols), TSB_TYPE_I8) < 0 || rows > (int64_t)1 << 38)
        return fail(TSB_ERR_INVALID_ARGUMENT, "%s: extent beyond the address range", name);
    return TSB_OK;
}

}  // namespace

// Sizes that are none have no bytes.
int64_t mxfp4_row_bytes(int64_t cols) { return cols > 0 && cols <= INT32_MAX ? mx::row_bytes(cols) : 0; }
int64_t mxfp4_scale_bytes(int64_t rows, int64_t cols) { return rows > 0 && cols > 0 && rows <= (int64_t)1 << 38 && cols <= INT32_MAX ? mx::scale_bytes(rows, cols) : 0; }

int quantize_rows_mxfp4(const void *x, int x_type, int64_t x_pitch, void *q, int64_t q_pitch, void *scales, int64_t rows, int64_t cols, cudaStream_t stream) {
    const int st = check("quantize_rows_mxfp4", q, q_pitch, scales, x, x_type, x_pitch, true, rows, cols);
    if (st != TSB_OK || rows == 0) return st;
    if (rows == 1) x_pitch = q_pitch = 0;      // (never stepped by)
    uint8_t *to = static_cast<uint8_t *>(q), *s = static_cast<uint8_t *>(scales);
    switch (x_type) {
        case TSB_TYPE_F32: return launch_quantize<float>(x, x_pitch, to, q_pitch, s, rows, cols, stream);
        case TSB_TYPE_F16: return launch_quantize<__half>(x, x_pitch, to, q_pitch, s, rows, cols, stream);
        default: return launch_quantize<__nv_bfloat16>(x, x_pitch, to, q_pitch, s, rows, cols, stream);
    }
}

int dequantize_rows_mxfp4(const void *q, int64_t q_pitch, const void *scales, void *y, int y_type, int64_t y_pitch, int64_t rows, int64_t cols, cudaStream_t stream) {
    const int st = check("dequantize_rows_mxfp4", q, q_pitch, scales, y, y_type, y_pitch, false, rows, cols);
    if (st != TSB_OK || rows == 0) return st;
    if (rows == 1) y_pitch = q_pitch = 0;
    const uint8_t *from = static_cast<const uint8_t *>(q), *s = static_cast<const uint8_t *>(scales);
    switch (y_type) {
        case TSB_TYPE_F32: return launch_dequantize<float>(from, q_pitch, s, y, y_pitch, rows, cols, stream);
        case TSB_TYPE_F16: return launch_dequantize<__half>(from, q_pitch, s, y, y_pitch, rows, cols, stream);
        default: return launch_dequantize<__nv_bfloat16>(from, q_pitch, s, y, y_pitch, rows, cols, stream);
    }
}

}  // namespace tsb
