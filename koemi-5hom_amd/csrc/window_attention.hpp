// What the kernels of the windowed attention with sinks share (window_attention.hip,
// window_attention_grad.hip): the call's shape, tiles of rows staged through LDS, and the
// matrix products on them.
//
// Position i of the keys sees j if both are valid, j <= i, and i - j < window or j <
// sinks. Queries stand at the last `length` of `total` positions. The `shared` query heads
// of one key head are rows of one matrix: row m is position m / shared, head m % shared,
// so heads that share keys share every tile of them, whatever `shared` is.
//
// Products are v_mfma_f32_32x32x16 (16-bit types) and v_mfma_f32_32x32x2f32 (fp32, whole
// products): lane l holds column l % 32 of a result, rows 8 (r / 4) + 4 (l / 32) + r % 4
// in register r. A product over the columns of a staged tile reads its rows as they lie (16
// bytes a lane, mma_rows). A product over the tile's rows takes the other operand straight
// from a result's registers: the rows a lane holds there are the K values it brings,
// whatever their order, as long as the tile's operand is read in the same one
// (mma_acc; 16-bit through ds_read_b64_tr_b16, which hands each lane four rows of a column).
#pragma once

#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace koemi {
namespace window_attention {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kRows = 32 * kWaves;  // rows (or keys) of a workgroup, 32 a wave
constexpr float kLog2e = 1.44269504088896341f;

struct Strides {
    int64_t batch, position, head;
};

struct Shape {
    // rows are whole, aligned 16-byte pieces, less than 2^24 bytes apart
    const void* q;
    const void* k;
    const void* v;
    const uint8_t* valid;  // [batch, total] or null
    Strides qs, ks, vs;
    int batch, length, total, groups, shared, width;
    int window, sinks;  // at most total
    float scale;        // of the scores
    uint32_t magic;     // rows / shared = (rows * magic >> 32) >> shift, rows below 2^31
    int shift;
};

// The position of row m, and its head among those that share.
__device__ __forceinline__ int position_of(const Shape& a, int m) {
    return a.shared == 1 ? m : static_cast<int>(__umulhi(static_cast<uint32_t>(m), a.magic) >> a.shift);
}

// Probabilities of fp16 calls are kept times 2^8: what is below 2^-14 of the largest would lose bits.
template <typename T> inline constexpr float kLift = 0.0f;
template <> inline constexpr float kLift<f16> = 8.0f;

template <typename T> inline constexpr int kPer16 = 16 / static_cast<int>(sizeof(T));  // values in 16 bytes

// NB: blocks of 32 columns that a head's width fills. A staged row is a power of two of bytes.
template <typename T, int NB>
struct Tile {
    static constexpr int kBytes = NB * 32 * static_cast<int>(sizeof(T));
    static constexpr int kUnits = kBytes / 16;
    static constexpr int kStride = kBytes <= 64 ? 64 : kBytes <= 128 ? 128 : kBytes <= 256 ? 256 : kBytes <= 512 ? 512 : 1024;
    static constexpr int kFrags = kUnits / 2;  // 16-byte pieces of a row that a lane brings to mma_rows
    // 16-byte unit u of row r lies at unit u ^ turn(r): the sixteen rows that sixteen lanes
    // read at one unit, and the four rows by 64 bytes of a transposed read, fill all banks.
    static __device__ __forceinline__ int turn(int r) {
        return kStride >= 256 ? ((r & 3) << 2) | ((r >> 2) & 3) : kStride == 128 ? ((r & 2) << 1) | ((r >> 2) & 3) : (r >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int r, int unit) { return r * kStride + ((unit ^ turn(r)) << 4); }
};

// The lowest n bits, n of any sign.
__device__ __forceinline__ uint32_t low_bits32(int n) { return n >= 32 ? ~0u : (1u << (max(n, 0) & 31)) - 1u; }
__device__ __forceinline__ uint64_t low_bits(int n) {
    return static_cast<uint64_t>(low_bits32(n)) | static_cast<uint64_t>(low_bits32(n < 32 ? 0 : n - 32)) << 32;
}

// The largest sizes, by their bits, of values seen so far: an infinity or NaN among them?
template <typename T>
struct Largest {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    uint32_t bits = 0;
    __device__ __forceinline__ void add(const uint4& x) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4)
                bits = max(bits, w[i] & 0x7fffffffu);
            else
                bits = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, bits),
                                                                              __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
        }
    }
    __device__ __forceinline__ bool nonfinite() const {
        if constexpr (sizeof(T) == 4) return bits >= 0x7f800000u;
        constexpr uint32_t E = std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
        return (bits & 0xffffu) >= E || bits >> 16 >= E;
    }
};

// 16 bytes of a row from column 16 / sizeof(T) * unit on, zeros past the width.
template <typename T>
__device__ __forceinline__ uint4 load_unit(const T* row, int unit, int width) {
    const int c = unit * kPer16<T>;
    return c < width ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
}

// A tile's rows on their way from memory to LDS: each thread brings the same pieces of
// every tile. The loads are unconditional (rows past the last one read that one again, pieces
// past the width the row's first), so that nothing waits for them before store(), which
// puts zeros in those places.
template <typename T, int NB, int ROWS>
struct Staged {
    using L = Tile<T, NB>;
    static constexpr int kEach = ROWS * L::kUnits / kThreads;
    static_assert(ROWS * L::kUnits % kThreads == 0, "whole pieces a thread");
    uint4 piece[kEach];

    static __device__ __forceinline__ int row(int n) { return (static_cast<int>(threadIdx.x) + n * kThreads) / L::kUnits; }
    static __device__ __forceinline__ int unit(int n) { return (static_cast<int>(threadIdx.x) + n * kThreads) % L::kUnits; }
    // `first`: the tile's first row, a uniform address; `last`: the last row to read.
    __device__ __forceinline__ void load(const T* first, int64_t stride, int last, int width) {
        const uint32_t bytes = static_cast<uint32_t>(stride) * static_cast<uint32_t>(sizeof(T));
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const uint32_t at = __umul24(static_cast<uint32_t>(min(row(n), last)), bytes) + (unit(n) * kPer16<T> < width ? unit(n) * 16u : 0u);
            piece[n] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(first) + at);
        }
    }
    // Zeros for the rows without a bit; true if what is left holds an infinity or NaN.
    __device__ __forceinline__ bool keep(const uint64_t (&rows)[(ROWS + 63) / 64]) {
        Largest<T> largest;
        bool every = true;
#pragma unroll
        for (int w = 0; w < (ROWS + 63) / 64; ++w) every = every && rows[w] == low_bits(ROWS - 64 * w);
        if (!every) {
#pragma unroll
            for (int n = 0; n < kEach; ++n)
                if (!((rows[ROWS > 64 && row(n) >= 64 ? 1 : 0] >> (row(n) & 63)) & 1ull)) piece[n] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < kEach; ++n) largest.add(piece[n]);
        return largest.nonfinite();
    }
    __device__ __forceinline__ void store(char* tile, int width) {
        if (width < 32 * NB) {
#pragma unroll
            for (int n = 0; n < kEach; ++n)
                if (unit(n) * kPer16<T> >= width) piece[n] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < kEach; ++n) *reinterpret_cast<uint4*>(tile + L::at(row(n), unit(n))) = piece[n];
    }
};

template <typename T>
__device__ __forceinline__ f32x16 mfma16(const uint4& a, const uint4& b, f32x16 c) {
    if constexpr (std::is_same<T, bf16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// acc[tile row first + ...][column] += tile row . frag, frag being the lane's pieces of column l % 32's row.
template <typename T, int NB>
__device__ __forceinline__ void mma_rows(f32x16& acc, const char* tile, int first, const uint4 (&frag)[Tile<T, NB>::kFrags]) {
    using L = Tile<T, NB>;
    const int lane = lane_id(), r = first + (lane & 31);
    const char* base = tile + r * L::kStride;
    const int turned = ((lane >> 5) ^ L::turn(r)) << 4;
#pragma unroll
    for (int s = 0; s < L::kFrags; ++s) {
        const uint4 a = *reinterpret_cast<const uint4*>(base + (turned ^ (s << 5)));
        if constexpr (sizeof(T) == 4) {
            const float* x = reinterpret_cast<const float*>(&a);
            const float* y = reinterpret_cast<const float*>(&frag[s]);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[c], y[c], acc, 0, 0, 0);
        } else {
            acc = mfma16<T>(a, frag[s], acc);
        }
    }
}

// acc[n][32 n + ...][column] += sum over the tile's rows first .. first + 31 of row[32 n + ...] coef[row][column],
// coef (a probability, or its derivative) of 16-bit calls as two values of T that sum to it within 2^-17 or
// 2^-22. Rounded to T alone it would add an error as large as the result's own rounding (1.41 times the error; 1.5
// to 1.8 times where few keys are seen, whose output D takes in), whatever the call's size.
template <typename T, int NB>
__device__ __forceinline__ void mma_acc(f32x16 (&acc)[NB], const char* tile, int first, const f32x16& coef) {
    using L = Tile<T, NB>;
    const int lane = lane_id(), half = lane >> 5;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = first + 8 * (r / 4) + 4 * half + r % 4;
            const char* base = tile + row * L::kStride + (lane & 3) * 4;
            const int unit = ((lane & 31) >> 2) ^ L::turn(row);
#pragma unroll
            for (int n = 0; n < NB; ++n)
                acc[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float*>(base + ((unit ^ (8 * n)) << 4)),
                                                              coef[r], acc[n], 0, 0, 0);
        }
    } else {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const int j = (lane & 15) >> 2, unit = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            alignas(16) T e[8];
            alignas(16) T low[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = static_cast<T>(coef[8 * s + i]);
                low[i] = static_cast<T>(coef[8 * s + i] - to_f32(e[i]));
            }
            const uint4 b = *reinterpret_cast<const uint4*>(e);
            const char* base[2];
            int turned[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = first + 16 * s + 8 * i + 4 * half + j;
                base[i] = tile + row * L::kStride + (lane & 1) * 8;
                turned[i] = (unit ^ L::turn(row)) << 4;
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                union {
                    s16x4 part[2];
                    uint4 whole;
                } a;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    a.part[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base[i] + (turned[i] ^ (n << 6))));
                acc[n] = mfma16<T>(a.whole, b, acc[n]);
                acc[n] = mfma16<T>(a.whole, *reinterpret_cast<const uint4*>(low), acc[n]);
            }
        }
    }
}

// mma_acc for a block that holds an infinity or NaN and is masked in places: 0 times one of
// them is not 0, so only what a column sees is added, one row after another. `seen`: the
// lane's column's 32 rows. `scratch`: kScratch floats of this wave's own.
constexpr int kScratch = 16 * 32;
template <typename T, int NB>
__device__ __forceinline__ void seen_acc(f32x16 (&acc)[NB], const char* tile, int first, const f32x16& coef, uint32_t seen, float* scratch) {
    using L = Tile<T, NB>;
    const int lane = lane_id(), half = lane >> 5, col = lane & 31;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 8; ++r) scratch[(8 * (r / 4) + 4 * half + r % 4) * 32 + col] = coef[8 * h + r];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
            const float c = scratch[k * 32 + col];
            if (!((seen >> (16 * h + k)) & 1u)) continue;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int d = 32 * n + 8 * q + 4 * half;
                    const T* x = reinterpret_cast<const T*>(tile + L::at(first + 16 * h + k, d / kPer16<T>) + (d % kPer16<T>) * sizeof(T));
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][4 * q + i] = fmaf(c, to_f32(x[i]), acc[n][4 * q + i]);
                }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Both halves of the wave hold a part of a column's maximum or sum.
__device__ __forceinline__ float max_of_halves(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// Of the 64 keys from key0 on, those that a query at `place` sees by position. Keys from..to - 1 are sinks as well.
__device__ __forceinline__ uint64_t keys_seen(const Shape& a, int place, int key0, int from = 0, int to = 0) {
    const int rel = place - key0;
    return low_bits(rel + 1) & (~low_bits(rel - a.window + 1) | low_bits(a.sinks - key0) | (low_bits(to - key0) & ~low_bits(from - key0)));
}

// x where the lane's register r of a 32-row block is seen (seen_half: the block's mask from
// the lane's half on), else `other`.
__device__ __forceinline__ float where_seen(uint32_t seen_half, int r, float x, float other) {
    const uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(seen_half), 8 * (r / 4) + r % 4, 1));
    return __uint_as_float((all & __float_as_uint(x)) | (~all & __float_as_uint(other)));
}

// A workgroup's key head (of `heads` in all, batch rows times key heads) and its part of it.
// Consecutive workgroups go to the eight XCDs in turn, and parts of a head read the same
// keys: so each XCD takes whole heads, every eighth one (rows of a batch differ in
// length), and the heads left over are cut into eight runs of parts.
struct Place {
    int head, part;
    __device__ __forceinline__ Place(int id, int heads, int parts) {
        const int even = (heads & ~7) * parts;
        if (id < even) {
            head = (id >> 3) / parts * 8 + (id & 7);
            part = (id >> 3) % parts;
        } else {
            const int rest = heads * parts - even, whole = rest & ~7;
            id -= even;
            id = id < whole ? (id & 7) * (whole >> 3) + (id >> 3) : id;
            head = (heads & ~7) + id / parts;
            part = id % parts;
        }
    }
};

// Key tiles of KT that rows at places first .. last (of the keys' positions) see: the
// sinks' before the window, then the window's; between them those of keys from..to - 1, sinks as well.
template <int KT>
struct KeyTiles {
    int lead, middle, jump, skip, count;
    __device__ __forceinline__ KeyTiles(const Shape& a, int first, int last, int from = 0, int to = 0) {
        const int low = max(first - a.window + 1, 0) / KT;
        lead = min((a.sinks + KT - 1) / KT, low);
        const int end = min((to + KT - 1) / KT, low), begin = max(from / KT, lead);
        middle = to > from ? max(end - begin, 0) : 0;
        jump = begin - lead;
        skip = low - lead - middle;
        count = lead + middle + last / KT - low + 1;
    }
    __device__ __forceinline__ int operator[](int t) const { return t < lead ? t : t < lead + middle ? t + jump : t + skip; }
};

// Checks, and the shape as the kernels take it (window_attention.hip).
int shape_of(const char* what, const void* queries, const void* keys, const void* values, const uint8_t* valid,
             const int64_t* strides, int64_t batch, int64_t length, int64_t total, int64_t heads, int64_t groups,
             int64_t width, int64_t window, int64_t sinks, float scale, int dtype, Shape& s);

// Four consecutive values of a row of `width` (a multiple of four) from column d on.
template <typename T>
__device__ __forceinline__ void store_four(T* row, int d, int width, const float (&x)[4]) {
    alignas(16) T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(x[i]);
    if (d < width) __builtin_memcpy(__builtin_assume_aligned(row + d, 4 * sizeof(T)), e, 4 * sizeof(T));
}

}  // namespace window_attention
}  // namespace koemi
