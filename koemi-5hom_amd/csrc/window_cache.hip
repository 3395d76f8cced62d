// The 8-bit cache of the windowed attention: the first `sinks` entries of a row and a ring
// of the last `window` others, as codes of one byte with one fp32 scale for each entry and key
// head.
//
//   entry p lies at slot p < sinks ? p : sinks + (p - sinks) mod window
//   scale = max(max |x| (1 / limit), 2^-126), 1 / limit rounded to fp32, code = x / scale rounded (int8, limit 127) or
//   converted (e4m3, limit 448), both to nearest even; an entry that is not finite keeps
//   codes 0 and a NaN scale, so it stands for NaN
//
// Rows of codes are whole blocks of 32 bytes, zeros behind the head's width.
// All three are bound by bytes, the small ones by one pass of their workgroups: [8, 2048, 4, 64] bf16 written
// in 13 us, read back in 9; a step of 8 rows over up to 32784 entries of 8 key heads of 128 in e4m3 94 to 104 us a call
// (471 MB, 4.5 to 5.0 TB/s), of 64 rows over 1028 entries of 4 of 64 in int8 16 (36 MB).
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace koemi {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kInt8 = 0, kE4m3 = 1;
constexpr int64_t kMostThreads = int64_t(1) << 32;  // a launch has fewer

struct Cache {
    uint8_t* keys;          // [batch, groups, slots, stored]
    uint8_t* values;
    float* key_scales;      // [batch, groups, slots]
    float* value_scales;
    int window, sinks;      // together below 2^31
    int batch, groups, width, stored, kind;
    __host__ __device__ int slots() const { return window + sinks; }
    __device__ __forceinline__ int slot_of(int64_t entry) const {
        return entry < sinks ? static_cast<int>(entry) : sinks + static_cast<int>((entry - sinks) % window);
    }
};

// Eight values' codes in two words.
template <int KIND>
__device__ __forceinline__ uint2 encode(const float (&x)[8], float scale, bool fine) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fine ? x[i] / scale : 0.0f;
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (KIND == kE4m3) {
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
            w[h] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], v, true));
        } else {
            w[h] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = static_cast<int>(fminf(fmaxf(__builtin_rintf(y[4 * h + i]), -127.0f), 127.0f));
                w[h] |= (static_cast<uint32_t>(c) & 255u) << (8 * i);
            }
        }
    }
    return make_uint2(w[0], w[1]);
}

template <int KIND>
__device__ __forceinline__ void decode(const uint2& w, float (&x)[8]) {
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (KIND == kE4m3) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u[h]), false);
            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u[h]), true);
            x[4 * h] = lo[0], x[4 * h + 1] = lo[1], x[4 * h + 2] = hi[0], x[4 * h + 3] = hi[1];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * h + i] = static_cast<float>(static_cast<int8_t>(u[h] >> (8 * i)));
        }
    }
}

// Values 8 i .. 8 i + 7 of a row, zeros past the width.
template <typename T>
__device__ __forceinline__ void load_eight(const T* row, int i, int width, bool vector, float (&x)[8]) {
    alignas(16) T e[8];
    if (vector && 8 * i + 8 <= width) {
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
            reinterpret_cast<uint4*>(e)[h] = reinterpret_cast<const uint4*>(row + 8 * i)[h];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = 8 * i + j < width ? row[8 * i + j] : static_cast<T>(0.0f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = to_f32(e[j]);
}

// A row's scale from the largest of its lanes' values; `lanes` (a power of two) share a row.
template <int KIND>
__device__ __forceinline__ float scale_of(const float (&x)[8], int lanes, bool& fine) {
    float m = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    for (int off = 1; off < lanes; off <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, kWave)));
    fine = top < 0x7f800000u;
    m = __uint_as_float(top) * (KIND == kE4m3 ? 1.0f / 448.0f : 1.0f / 127.0f);
    return fmaxf(m, 1.17549435e-38f);
}

struct Write {
    Cache c;
    const void* keys;    // [batch, length, groups, width]
    const void* values;
    int64_t kb, kp, kh, vb, vp, vh;
    const int64_t* lengths;
    const int64_t* counts;  // or null: length
    int length, lanes, vector, per_batch;  // per_batch: workgroups of a batch row
};

// `lanes` lanes quantise a row of a key head. Of the rows that this call appends only
// those that stay are written, so no two go to one slot. Bound by memory; the batch row's
// ring position is a workgroup's own, so that a row needs no 64-bit division.
template <typename T, int KIND>
__global__ __launch_bounds__(kThreads) void window_cache_write_kernel(Write f) {
    const Cache& c = f.c;
    const int per = kThreads / f.lanes, i = static_cast<int>(threadIdx.x) % f.lanes;
    const int b = static_cast<int>(blockIdx.x) / f.per_batch;
    const int row = (static_cast<int>(blockIdx.x) - b * f.per_batch) * per + static_cast<int>(threadIdx.x) / f.lanes;
    const int t = row / c.groups, g = row - t * c.groups;
    const int64_t before = f.lengths[b], count = f.counts ? min(f.counts[b], static_cast<int64_t>(f.length)) : f.length;
    const int64_t entry = before + t;
    // a whole row's lanes at once
    if (before < 0 || t >= count || !(entry < c.sinks || entry >= before + count - c.window)) return;
    const uint32_t turn = before >= c.sinks ? static_cast<uint32_t>((before - c.sinks) % c.window) : 0u;
    const uint32_t along = static_cast<uint32_t>(before >= c.sinks ? t : entry - c.sinks);
    const int slot = entry < c.sinks ? static_cast<int>(entry) : c.sinks + static_cast<int>((turn + along) % static_cast<uint32_t>(c.window));
    const int64_t at = (static_cast<int64_t>(b) * c.groups + g) * c.slots() + slot;
    const T* x[2] = {static_cast<const T*>(f.keys) + b * f.kb + t * f.kp + g * f.kh,
                     static_cast<const T*>(f.values) + b * f.vb + t * f.vp + g * f.vh};
    float e[2][8];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) load_eight(x[kv], i, c.width, f.vector, e[kv]);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        bool fine;
        const float scale = scale_of<KIND>(e[kv], f.lanes, fine);
        const uint2 w = encode<KIND>(e[kv], scale, fine);
        if (8 * i < c.stored) *reinterpret_cast<uint2*>((kv ? c.values : c.keys) + at * c.stored + 8 * i) = w;
        if (i == 0) (kv ? c.value_scales : c.key_scales)[at] = fine ? scale : NAN;
    }
}

struct Entries {
    Cache c;
    const int64_t* lengths;
    void* keys;    // [batch, slots, groups, width]
    void* values;
    uint8_t* present;  // [batch, slots]
    int lanes, per_batch;
};

// The sinks, then the last `window` entries in their order, as the values they stand for.
template <typename T, int KIND>
__global__ __launch_bounds__(kThreads) void window_cache_entries_kernel(Entries f) {
    const Cache& c = f.c;
    const int per = kThreads / f.lanes, i = static_cast<int>(threadIdx.x) % f.lanes, slots = c.slots();
    const int b = static_cast<int>(blockIdx.x) / f.per_batch;
    const int row = (static_cast<int>(blockIdx.x) - b * f.per_batch) * per + static_cast<int>(threadIdx.x) / f.lanes;
    const int place = row / c.groups, g = row - place * c.groups;
    if (place >= slots) return;
    const int64_t held = f.lengths[b], entry = place < c.sinks ? place : held - slots + place;
    const bool here = entry < held && (place < c.sinks || entry >= c.sinks);
    // entry - sinks = (held - sinks) + (place - sinks) - window
    const uint32_t turn = held >= c.sinks ? static_cast<uint32_t>((held - c.sinks) % c.window) : 0u;
    uint32_t ring = turn + static_cast<uint32_t>(place - c.sinks);
    if (held >= c.sinks && ring >= static_cast<uint32_t>(c.window)) ring -= static_cast<uint32_t>(c.window);
    const int slot = !here ? 0 : place < c.sinks ? place : c.sinks + static_cast<int>(ring);
    const int64_t at = (static_cast<int64_t>(b) * c.groups + g) * slots + slot;
    if (g == 0 && i == 0) f.present[static_cast<int64_t>(b) * slots + place] = here;
    if (8 * i >= c.width) return;
    uint2 w[2];
    float scale[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        w[kv] = *reinterpret_cast<const uint2*>((kv ? c.values : c.keys) + at * c.stored + 8 * i);
        scale[kv] = (kv ? c.value_scales : c.key_scales)[at];
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        float x[8];
        decode<KIND>(w[kv], x);
        T* o = static_cast<T*>(kv ? f.values : f.keys) + (static_cast<int64_t>(b) * slots * c.groups + row) * c.width + 8 * i;
        alignas(16) T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = here ? from_f32<T>(x[j] * scale[kv]) : static_cast<T>(0.0f);
        if (c.width % 8 == 0) {
#pragma unroll
            for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h) reinterpret_cast<uint4*>(o)[h] = reinterpret_cast<const uint4*>(e)[h];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * i + j < c.width) o[j] = e[j];
        }
    }
}

// ------------------------------------------------------------------- one position ---
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Step {
    Cache c;
    const void* queries;   // [batch, heads, width]
    const void* new_keys;  // [batch, groups, width], null: nothing is written
    const void* new_values;
    int64_t qb, qh, kb, kh, vb, vh;
    const int64_t* lengths;
    const uint8_t* active;  // or null: all
    void* out;              // [batch, heads, width]
    float* parts;           // [splits, batch, heads, width] and
    float* part_lse;        // [splits, batch, heads], where splits > 1
    float scale;
    int shared, blocks16, splits, vector;  // blocks16: of sixteen query heads
};

// Two bytes of a word (or one of each of two words) as fp16, exactly. int8: byte + 128 as
// the last bits of 1024, minus 1152.
template <int KIND>
__device__ __forceinline__ f16x2 widen(uint32_t pair) {  // bytes 0 and 2 (int8, biased) or 0 and 1 (e4m3)
    if (KIND == kE4m3) return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(pair), 1.0f, false);
    return __builtin_bit_cast(f16x2, pair | 0x64006400u) - f16x2{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
}
template <int KIND>
__device__ __forceinline__ f16x8 widen8(uint32_t lo, uint32_t hi) {  // eight bytes in their order
    f16x2 p[4];
    const uint32_t w[2] = {KIND == kE4m3 ? lo : lo ^ 0x80808080u, KIND == kE4m3 ? hi : hi ^ 0x80808080u};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (KIND == kE4m3) {
            p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w[h]), 1.0f, false);
            p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w[h]), 1.0f, true);
        } else {
            p[2 * h] = widen<KIND>(__builtin_amdgcn_perm(0u, w[h], 0x0c010c00u));
            p[2 * h + 1] = widen<KIND>(__builtin_amdgcn_perm(0u, w[h], 0x0c030c02u));
        }
    }
    return f16x8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

// Over the four lane groups (of sixteen) that hold a query.
template <typename Op>
__device__ __forceinline__ float over_groups(float x, Op op) {
    const auto odd = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(odd[0]), __uint_as_float(odd[1]));
    const auto high = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(high[0]), __uint_as_float(high[1]));
}
__device__ __forceinline__ float max_of_groups(float x) {
    return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_of_groups(float x) {
    return over_groups(x, [](float a, float b) { return a + b; });
}

template <int NB>
struct alignas(2) Bytes {
    uint16_t w[NB];
};

// A wave's sums for sixteen queries (lane % 16) over chunks of 32 entries. Results of the
// 16 x 16 products: register r of lane group m = lane / 16 is entry 4 m + r of its half of
// the chunk; so the group brings those entries' rows of values, and its eight probabilities
// are the product's other operand as they are. Columns: a lane of the keys holds the bytes
// from 8 NB m on, of the values the 2 NB from 2 NB (lane % 16) on, one for each product.
//
// Products are fp16 x fp16 with fp32 sums: codes are exact, queries and probabilities times
// the values' scale are two planes each, which sum to them within 2^-22.
template <int NB, int KIND>
struct Walk {
    f32x4 acc[2 * NB];
    float top = -INFINITY, sum = 0.0f;
    float peak = 0.0f;  // the largest probability times its value's scale, in units of the top as `acc`
    int power = 0;      // acc is held times 2^power
    f16x8 q[2][NB];
    // of a product of codes and planes, and of a key's scale, to a score in powers of two: half of the queries' power each, so
    // that neither large keys under small queries nor the reverse pass the range on the way
    float factor, key_factor;

    template <typename T>
    __device__ __forceinline__ void begin(const T* row, int width, bool ok, bool vector, float scale) {
        const int m = lane_id() >> 4;
        float x[NB][8], high = 0.0f;
#pragma unroll
        for (int s = 0; s < NB; ++s) {
            if (ok) load_eight(row, m * NB + s, width, vector, x[s]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (!ok) x[s][j] = 0.0f;
                high = fmaxf(high, fabsf(x[s][j]));
            }
        }
        high = max_of_groups(high);
        // the largest comes to 2^14 .. 2^15, so that what the second plane has no digits for is below 2^-39 of it
        const int e = min(max(static_cast<int>(__float_as_uint(high) >> 23), 16), 254);
        const int power = 141 - e;
        const float lift = __uint_as_float(static_cast<uint32_t>(127 + power) << 23);
        factor = scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - power / 2) << 23);
        key_factor = __uint_as_float(static_cast<uint32_t>(127 - (power - power / 2)) << 23);
#pragma unroll
        for (int s = 0; s < NB; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[s][j] * lift;
                const _Float16 h = static_cast<_Float16>(y);
                q[0][s][j] = h;
                q[1][s][j] = static_cast<_Float16>(y - static_cast<float>(h));
            }
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n) acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // keys: words of entries lane % 16 and 16 + lane % 16; values: of the group's eight entries;
    // scales, ok (a bit each) in the order of the group's eight.
    __device__ __forceinline__ void chunk(const uint32_t (&keys)[2][2 * NB], const Bytes<NB> (&values)[8], const float (&ks)[8],
                                          const float (&vs)[8], uint32_t ok) {
        float s[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const f16x8 a = widen8<KIND>(keys[h][2 * n], keys[h][2 * n + 1]);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[0][n], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[1][n], d, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * h + r] = (ok >> (4 * h + r)) & 1u ? (d[r] * factor) * (ks[4 * h + r] * key_factor) : -INFINITY;
        }
        float high = s[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) high = fmaxf(high, s[j]);
        high = fmaxf(top, max_of_groups(high));
        const bool higher = high > top;
        const float shrink = higher ? __builtin_amdgcn_exp2f(top - high) : 1.0f;
        const float base = high == -INFINITY ? 0.0f : high, was = top;
        top = high;
        sum *= shrink;
        float prob[8], v[8], most = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            prob[j] = __builtin_amdgcn_exp2f(s[j] - base);
            sum += prob[j];
            v[j] = (ok >> j) & 1u ? vs[j] : 0.0f;
            most = fmaxf(most, fabsf(prob[j] * v[j]));
        }
        // fp16 planes of p v: a power of two holds the largest so far at 2^13 to 2^15 (2^126 at most: scales from 2^-126 on
        // stay above 1). It falls with the probabilities when the top rises, so the sums' change stays under 2^2.
        peak = fmaxf(peak * shrink, max_of_groups(most));
        const int want = min(140 - static_cast<int>(__float_as_uint(peak) >> 23), 126);
        const bool move = peak > 0.0f && (want < power - 1 || want > power);
        if (__any(higher || move)) {
            const int next = move ? want : power;
            const float change = shrink > 0.0f ? __builtin_amdgcn_exp2f((higher ? was - high : 0.0f) + static_cast<float>(next - power)) : 0.0f;
            power = next;
#pragma unroll
            for (int n = 0; n < 2 * NB; ++n) acc[n] *= change;
        }
        // up to the scale before the value, down after it: neither passes the range on the way
        const float up = __uint_as_float(static_cast<uint32_t>(127 + max(power, 0)) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(127 + min(power, 0)) << 23);
        f16x8 p[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float y = prob[j] * up * v[j] * down;
            const _Float16 h = static_cast<_Float16>(y);
            p[0][j] = h;
            p[1][j] = static_cast<_Float16>(y - static_cast<float>(h));
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            // columns 2 n and 2 n + 1 of the lane: byte 0 and 1 of each entry's half word n
            f16x2 even[4], odd[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t flip = KIND == kE4m3 ? 0u : 0x80808080u;
                const uint32_t two = (static_cast<uint32_t>(values[2 * j].w[n]) | static_cast<uint32_t>(values[2 * j + 1].w[n]) << 16) ^ flip;
                if (KIND == kE4m3) {
                    even[j] = widen<KIND>(__builtin_amdgcn_perm(0u, two, 0x0c0c0200u));
                    odd[j] = widen<KIND>(__builtin_amdgcn_perm(0u, two, 0x0c0c0301u));
                } else {
                    even[j] = widen<KIND>(two & 0x00ff00ffu);
                    odd[j] = widen<KIND>((two >> 8) & 0x00ff00ffu);
                }
            }
            const f16x8 a0 = {even[0][0], even[0][1], even[1][0], even[1][1], even[2][0], even[2][1], even[3][0], even[3][1]};
            const f16x8 a1 = {odd[0][0], odd[0][1], odd[1][0], odd[1][1], odd[2][0], odd[2][1], odd[3][0], odd[3][1]};
            acc[2 * n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, p[0], acc[2 * n], 0, 0, 0);
            acc[2 * n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, p[1], acc[2 * n], 0, 0, 0);
            acc[2 * n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, p[0], acc[2 * n + 1], 0, 0, 0);
            acc[2 * n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, p[1], acc[2 * n + 1], 0, 0, 0);
        }
    }
};

// Waves of a workgroup: eight where two of them fit a SIMD's registers.
template <int NB> constexpr int kStepWaves = NB <= 4 ? 8 : 4;

// A workgroup answers sixteen query heads of one key head from one part of the slots, its
// waves 32 slots each in turn. The new entry is quantised by the first part's workgroups
// (of every sixteen heads), which read it from LDS; the others leave its slot out.
template <typename T, int NB, int KIND>
__global__ __launch_bounds__(kStepWaves<NB> * kWave) void window_cache_step_kernel(Step f) {
    constexpr int kWaves = kStepWaves<NB>, kThreads = kWaves * kWave;
    const Cache& c = f.c;
    __shared__ __attribute__((aligned(16))) uint8_t fresh[2][NB * 32];
    __shared__ float fresh_scale[2];
    __shared__ float sums[kWaves][16][NB * 32 + 1];
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, m = lane >> 4, col = lane & 15;
    int64_t id = blockIdx.x;
    const int split = static_cast<int>(id % f.splits);
    id /= f.splits;
    const int block = static_cast<int>(id % f.blocks16);
    id /= f.blocks16;
    const int g = static_cast<int>(id % c.groups);
    const int64_t b = id / c.groups, slots = c.slots(), heads = static_cast<int64_t>(c.groups) * f.shared;
    const int64_t before = f.lengths[b];
    const bool live = before >= 0 && (!f.active || f.active[b]);
    const bool writes = live && f.new_keys;
    const int64_t held = live ? min(before, slots) : 0, slot = writes ? c.slot_of(before) : -1;
    const int64_t base = (b * c.groups + g) * slots;
    const uint8_t* keys = c.keys + base * c.stored;
    const uint8_t* values = c.values + base * c.stored;
    const float* key_scales = c.key_scales + base;
    const float* value_scales = c.value_scales + base;

    const int64_t chunks = (held + 31) / 32;
    const int c0 = static_cast<int>(chunks * split / f.splits), c1 = static_cast<int>(chunks * (split + 1) / f.splits);
    uint32_t kw[2][2 * NB];
    Bytes<NB> vw[8];
    float ks[8], vs[8];
    // chunk n's loads; past the last entry that one again
    auto fetch = [&](int n) {
        const int s0 = n * 32, end = static_cast<int>(held) - 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t s = min(s0 + 16 * h + col, end);
            const uint32_t* p = reinterpret_cast<const uint32_t*>(keys + s * c.stored + m * 8 * NB);
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) kw[h][i] = p[i];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t s = min(s0 + 16 * (j / 4) + 4 * m + j % 4, end);
            vw[j] = *reinterpret_cast<const Bytes<NB>*>(values + s * c.stored + col * 2 * NB);
        }
        if (s0 + 32 <= static_cast<int>(held)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // four at once, at any place
                __builtin_memcpy(&ks[4 * h], key_scales + s0 + 16 * h + 4 * m, 16);
                __builtin_memcpy(&vs[4 * h], value_scales + s0 + 16 * h + 4 * m, 16);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int s = min(s0 + 16 * (j / 4) + 4 * m + j % 4, end);
                ks[j] = key_scales[s], vs[j] = value_scales[s];
            }
        }
    };
    if (c0 + wave < c1) fetch(c0 + wave);
    const int head = block * 16 + col;
    const bool head_ok = live && head < f.shared;
    Walk<NB, KIND> walk;
    walk.begin(static_cast<const T*>(f.queries) + b * f.qb + (static_cast<int64_t>(g) * f.shared + head) * f.qh, c.width, head_ok, f.vector, f.scale);

    if (writes && split == 0 && wave < 2) {  // wave 0 the key, wave 1 the value
        const T* x = wave ? static_cast<const T*>(f.new_values) + b * f.vb + g * f.vh : static_cast<const T*>(f.new_keys) + b * f.kb + g * f.kh;
        float e[8];
        load_eight(x, lane, c.width, f.vector, e);  // lanes past the width hold zeros
        bool fine;
        const float scale = scale_of<KIND>(e, kWave, fine);
        const uint2 w = encode<KIND>(e, scale, fine);
        if (lane < 4 * NB) {
            *reinterpret_cast<uint2*>(&fresh[wave][8 * lane]) = w;
            if (block == 0) *reinterpret_cast<uint2*>((wave ? c.values : c.keys) + (base + slot) * c.stored + 8 * lane) = w;
        }
        if (lane == 0) {
            fresh_scale[wave] = fine ? scale : NAN;
            if (block == 0) (wave ? c.value_scales : c.key_scales)[base + slot] = fine ? scale : NAN;
        }
    }
    for (int n = c0 + wave; n < c1; n += kWaves) {
        uint32_t kn[2][2 * NB], ok = 0;
        Bytes<NB> vn[8];
        float ksn[8], vsn[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) kn[h][i] = kw[h][i];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            vn[j] = vw[j], ksn[j] = ks[j], vsn[j] = vs[j];
            const int at = n * 32 + 16 * (j / 4) + 4 * m + j % 4;
            ok |= static_cast<uint32_t>(at < held && at != slot) << j;
        }
        fetch(min(n + kWaves, c1 - 1));
        walk.chunk(kn, vn, ksn, vsn, ok);
    }
    if (writes && split == 0) {
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i)
                    kw[h][i] = h == 0 && col == 0 ? *reinterpret_cast<const uint32_t*>(&fresh[0][m * 8 * NB + 4 * i]) : 0u;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ks[j] = fresh_scale[0], vs[j] = fresh_scale[1];
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    vw[j].w[i] = j == 0 && m == 0 ? *reinterpret_cast<const uint16_t*>(&fresh[1][col * 2 * NB + 2 * i]) : static_cast<uint16_t>(0);
            }
            walk.chunk(kw, vw, ks, vs, m == 0 ? 1u : 0u);
        }
    }
    // the waves' means joined in their order, by their shares of the whole: sums of large values would pass the range
    const float total = sum_of_groups(walk.sum), invert = total == 0.0f ? 0.0f : 1.0f / total;
    const float back = __uint_as_float(static_cast<uint32_t>(127 - walk.power) << 23);
    if (m == 0) tops[wave][col] = walk.top, totals[wave][col] = total;
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[wave][col][(4 * m + r) * 2 * NB + n] = walk.acc[n][r] * invert * back;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NB * 32; i += kThreads) {
        const int h = i / (NB * 32), d = i % (NB * 32), hd = block * 16 + h;
        if (hd >= f.shared || d >= c.width) continue;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = tops[w][h] > top || tops[w][h] != tops[w][h] ? tops[w][h] : top;
        float share[kWaves], all = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const bool empty = tops[w][h] == -INFINITY && totals[w][h] == 0.0f;
            share[w] = empty ? 0.0f : totals[w][h] * __builtin_amdgcn_exp2f(tops[w][h] - top);
            all += share[w];
        }
        const bool none = all == 0.0f;
        const float whole = 1.0f / all;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x = fmaf(share[w] * whole, sums[w][h][d], x);
        if (none) x = 0.0f;
        const int64_t cell = b * heads + static_cast<int64_t>(g) * f.shared + hd;
        if (f.splits == 1) {
            static_cast<T*>(f.out)[cell * c.width + d] = from_f32<T>(x);
        } else {
            const int64_t at = cell + static_cast<int64_t>(split) * c.batch * heads;
            f.parts[at * c.width + d] = x;
            if (d == 0) f.part_lse[at] = none ? INFINITY : top + __builtin_amdgcn_logf(all);
        }
    }
}

// The parts of a head joined in their order: each brings its mean and its log-sum.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_cache_join_kernel(Step f) {
    const int64_t cells = static_cast<int64_t>(f.c.batch) * f.c.groups * f.shared;
    const int64_t cell = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
    if (cell >= cells) return;
    const int lane = lane_id(), width = f.c.width;
    const float own = lane < f.splits ? f.part_lse[cell + lane * cells] : INFINITY;  // at most 64 parts
    const bool some = own != INFINITY;
    float top = some && own == own ? own : -INFINITY;
    top = wave_max_xor(top);
    float share = some ? __builtin_amdgcn_exp2f(own - top) : 0.0f;
    const float all = wave_sum_xor(share);
    share = all == 0.0f ? 0.0f : share / all;
    for (int d0 = 0; d0 < width; d0 += kWave) {  // all lanes in every round: each holds a part's share
        const int d = d0 + lane;
        float x = 0.0f;
#pragma unroll 8
        for (int p = 0; p < f.splits; ++p) {
            const float part = f.parts[(cell + p * cells) * width + min(d, width - 1)];
            x = fmaf(part, __shfl(share, p, kWave), x);
        }
        if (d < width) static_cast<T*>(f.out)[cell * width + d] = from_f32<T>(x);
    }
}

// Parts of the slots: one workgroup for each compute unit, none under 256 slots. A workgroup's start and end cost
// as much as a few chunks: [64] rows of 4 key heads, 1028 slots: 16.2 us in 256 workgroups, 19.8 (and 3.9 for the join) in
// 512, 29.4 in 1024; [8] of 8, 32784 slots: 93.8 + 5.5, 100.4 + 8.8, 111.6 + 12.0.
int splits_for(int64_t batch, int64_t heads, int64_t groups, int64_t slots) {
    const int64_t wide = batch * groups * ((heads / groups + 15) / 16);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({64, slots / 256, 256 / std::max<int64_t>(wide, 1)})));
}

template <typename T, int NB, int KIND>
int run_step(const Step& f, hipStream_t stream) {
    const int64_t grid = static_cast<int64_t>(f.c.batch) * f.c.groups * f.blocks16 * f.splits;
    hipLaunchKernelGGL((window_cache_step_kernel<T, NB, KIND>), dim3(static_cast<unsigned>(grid)), dim3(kStepWaves<NB> * kWave), 0, stream, f);
    const int rc = check_launch("koemi_window_cache_step");
    if (rc != KOEMI_OK || f.splits == 1) return rc;
    hipLaunchKernelGGL((window_cache_join_kernel<T>), dim3(grid_for(static_cast<int64_t>(f.c.batch) * f.c.groups * f.shared, kWaves)),
                       dim3(kThreads), 0, stream, f);
    return check_launch("koemi_window_cache_step(join)");
}
template <typename T, int KIND>
int step_by_width(const Step& f, hipStream_t stream) {
    switch (f.c.stored / 32) {
        case 1: return run_step<T, 1, KIND>(f, stream);
        case 2: return run_step<T, 2, KIND>(f, stream);
        case 3: return run_step<T, 3, KIND>(f, stream);
        case 4: return run_step<T, 4, KIND>(f, stream);
        case 5: return run_step<T, 5, KIND>(f, stream);
        case 6: return run_step<T, 6, KIND>(f, stream);
        case 7: return run_step<T, 7, KIND>(f, stream);
        default: return run_step<T, 8, KIND>(f, stream);
    }
}

int cache_of(const char* what, void* keys, float* key_scales, void* values, float* value_scales, int code, int64_t batch,
             int64_t groups, int64_t width, int64_t window, int64_t sinks, Cache& c) {
    if (batch < 0 || groups < 1 || width < 1 || window < 1 || sinks < 0)
        return fail(KOEMI_ERR_INVALID, "%s: sizes must be positive, batch and sinks not negative", what);
    if (width > 256) return fail(KOEMI_ERR_UNSUPPORTED, "%s: heads are at most 256 wide", what);
    if (code != kInt8 && code != kE4m3) return fail(KOEMI_ERR_UNSUPPORTED, "%s: codes are int8 (0) or e4m3 (1)", what);
    if (window >= (int64_t(1) << 31) || sinks >= (int64_t(1) << 31) || batch >= (1 << 24) || groups >= (1 << 20) ||
        (window + sinks) * groups >= (int64_t(1) << 31) - 256)
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^31 entries x key heads, 2^20 key heads and 2^24 rows", what);
    if (batch && (!keys || !key_scales || !values || !value_scales)) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    if (reinterpret_cast<uintptr_t>(keys) % 16 || reinterpret_cast<uintptr_t>(values) % 16)
        return fail(KOEMI_ERR_INVALID, "%s: the codes must be 16-byte aligned", what);
    c = Cache{static_cast<uint8_t*>(keys), static_cast<uint8_t*>(values), key_scales, value_scales, static_cast<int>(window),
              static_cast<int>(sinks), static_cast<int>(batch), static_cast<int>(groups), static_cast<int>(width), static_cast<int>((width + 31) / 32 * 32), code};
    return KOEMI_OK;
}

int lanes_of(int stored) {
    int n = 4;
    while (n * 8 < stored) n *= 2;
    return n;
}

bool aligned16(const void* p, int64_t size, std::initializer_list<int64_t> strides) {
    bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (const int64_t s : strides) ok = ok && s * size % 16 == 0;
    return ok;
}

int64_t size_of(int dtype) { return dtype == KOEMI_F32 ? 4 : 2; }

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" int koemi_window_cache_write(void* keys, float* key_scales, void* values, float* value_scales, int code,
                                        const void* new_keys, const void* new_values, const int64_t* strides,
                                        const int64_t* lengths, const int64_t* counts, int64_t batch, int64_t length,
                                        int64_t groups, int64_t width, int64_t window, int64_t sinks, int dtype,
                                        koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_window_cache_write";
    Write f{};
    const int rc = cache_of(what, keys, key_scales, values, value_scales, code, batch, groups, width, window, sinks, f.c);
    if (rc != KOEMI_OK) return rc;
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16, not %s", what, dtype_name(dtype));
    if (length < 0) return fail(KOEMI_ERR_INVALID, "%s: length must not be negative", what);
    if (batch == 0 || length == 0) return KOEMI_OK;
    if (!new_keys || !new_values || !strides || !lengths) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    f.keys = new_keys, f.values = new_values, f.lengths = lengths, f.counts = counts, f.length = static_cast<int>(length);
    f.kb = strides[0], f.kp = strides[1], f.kh = strides[2], f.vb = strides[3], f.vp = strides[4], f.vh = strides[5];
    f.lanes = lanes_of(f.c.stored);
    f.vector = aligned16(new_keys, size_of(dtype), {f.kb, f.kp, f.kh}) && aligned16(new_values, size_of(dtype), {f.vb, f.vp, f.vh});
    if (length >= (int64_t(1) << 31) / groups - 256) return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^31 new entries x key heads", what);
    const int64_t per_batch = (length * groups * f.lanes + kThreads - 1) / kThreads;
    if (batch * per_batch >= kMostThreads / kThreads) return fail(KOEMI_ERR_UNSUPPORTED, "%s: too many rows: a launch has fewer than 2^32 threads", what);
    f.per_batch = static_cast<int>(per_batch);
    const dim3 grid(static_cast<unsigned>(batch * per_batch));
    auto launch = [&](auto type, auto kind) {
        hipLaunchKernelGGL((window_cache_write_kernel<decltype(type), decltype(kind)::value>), grid, dim3(kThreads), 0, as_stream(stream), f);
    };
    auto by_type = [&](auto kind) {
        if (dtype == KOEMI_F32) launch(float{}, kind);
        else if (dtype == KOEMI_F16) launch(f16{}, kind);
        else launch(bf16{}, kind);
    };
    if (code == kInt8) by_type(std::integral_constant<int, kInt8>{});
    else by_type(std::integral_constant<int, kE4m3>{});
    return check_launch(what);
}

extern "C" int koemi_window_cache_entries(const void* keys, const float* key_scales, const void* values, const float* value_scales,
                                          int code, const int64_t* lengths, void* out_keys, void* out_values, uint8_t* present,
                                          int64_t batch, int64_t groups, int64_t width, int64_t window, int64_t sinks, int dtype,
                                          koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_window_cache_entries";
    Entries f{};
    const int rc = cache_of(what, const_cast<void*>(keys), const_cast<float*>(key_scales), const_cast<void*>(values),
                            const_cast<float*>(value_scales), code, batch, groups, width, window, sinks, f.c);
    if (rc != KOEMI_OK) return rc;
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16, not %s", what, dtype_name(dtype));
    if (batch == 0) return KOEMI_OK;
    if (!lengths || !out_keys || !out_values || !present) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    if (reinterpret_cast<uintptr_t>(out_keys) % 16 || reinterpret_cast<uintptr_t>(out_values) % 16)
        return fail(KOEMI_ERR_INVALID, "%s: the outputs must be 16-byte aligned", what);
    f.lengths = lengths, f.keys = out_keys, f.values = out_values, f.present = present;
    f.lanes = lanes_of(f.c.stored);
    const int64_t per_batch = ((window + sinks) * groups * f.lanes + kThreads - 1) / kThreads;
    if (batch * per_batch >= kMostThreads / kThreads) return fail(KOEMI_ERR_UNSUPPORTED, "%s: too many rows: a launch has fewer than 2^32 threads", what);
    f.per_batch = static_cast<int>(per_batch);
    const dim3 grid(static_cast<unsigned>(batch * per_batch));
    auto launch = [&](auto type, auto kind) {
        hipLaunchKernelGGL((window_cache_entries_kernel<decltype(type), decltype(kind)::value>), grid, dim3(kThreads), 0, as_stream(stream), f);
    };
    auto by_type = [&](auto kind) {
        if (dtype == KOEMI_F32) launch(float{}, kind);
        else if (dtype == KOEMI_F16) launch(f16{}, kind);
        else launch(bf16{}, kind);
    };
    if (code == kInt8) by_type(std::integral_constant<int, kInt8>{});
    else by_type(std::integral_constant<int, kE4m3>{});
    return check_launch(what);
}

extern "C" size_t koemi_window_cache_step_workspace_bytes(int64_t batch, int64_t heads, int64_t groups, int64_t width,
                                                          int64_t window, int64_t sinks) {
    if (batch < 1 || groups < 1 || heads < groups || width < 1 || window < 1 || sinks < 0) return 0;
    const int n = splits_for(batch, heads, groups, window + sinks);
    return n == 1 ? 0 : static_cast<size_t>(n) * batch * heads * (width + 1) * 4;
}

extern "C" int koemi_window_cache_step(void* keys, float* key_scales, void* values, float* value_scales, int code,
                                       const void* queries, const void* new_keys, const void* new_values, const int64_t* strides,
                                       const int64_t* lengths, const uint8_t* active, void* output, int64_t batch, int64_t heads,
                                       int64_t groups, int64_t width, int64_t window, int64_t sinks, float scale, int dtype,
                                       void* workspace, size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_window_cache_step";
    Step f{};
    const int rc = cache_of(what, keys, key_scales, values, value_scales, code, batch, groups, width, window, sinks, f.c);
    if (rc != KOEMI_OK) return rc;
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16, not %s", what, dtype_name(dtype));
    if (heads < 1 || heads % groups) return fail(KOEMI_ERR_INVALID, "%s: the key heads must divide the query heads", what);
    if (!(scale > 0.0f) || scale > 3.0e38f) return fail(KOEMI_ERR_INVALID, "%s: scale must be positive and finite", what);
    if (!new_keys != !new_values) return fail(KOEMI_ERR_INVALID, "%s: a key comes with its value", what);
    if (batch == 0) return KOEMI_OK;
    if (!queries || !strides || !lengths || !output) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    if (batch * heads >= (1 << 26)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^26 query heads", what);
    f.queries = queries, f.new_keys = new_keys, f.new_values = new_values, f.lengths = lengths, f.active = active, f.out = output;
    f.qb = strides[0], f.qh = strides[1], f.kb = strides[2], f.kh = strides[3], f.vb = strides[4], f.vh = strides[5];
    const int64_t size = size_of(dtype);
    f.vector = aligned16(queries, size, {f.qb, f.qh}) && aligned16(new_keys, size, {f.kb, f.kh}) && aligned16(new_values, size, {f.vb, f.vh});
    f.scale = scale;
    f.shared = static_cast<int>(heads / groups), f.blocks16 = (f.shared + 15) / 16;
    f.splits = splits_for(batch, heads, groups, window + sinks);
    if (batch * groups * f.blocks16 * f.splits >= kMostThreads / (f.c.stored <= 128 ? kStepWaves<4> * kWave : kStepWaves<8> * kWave))
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: too many rows of heads: a launch has fewer than 2^32 threads", what);
    if (f.splits > 1) {
        const size_t cells = static_cast<size_t>(f.splits) * batch * heads;
        if (!workspace || workspace_bytes < cells * (width + 1) * 4) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
        f.part_lse = static_cast<float*>(workspace);
        f.parts = f.part_lse + cells;
    }
    auto by_type = [&](auto kind) {
        constexpr int K = decltype(kind)::value;
        if (dtype == KOEMI_F32) return step_by_width<float, K>(f, as_stream(stream));
        if (dtype == KOEMI_F16) return step_by_width<f16, K>(f, as_stream(stream));
        return step_by_width<bf16, K>(f, as_stream(stream));
    };
    return code == kInt8 ? by_type(std::integral_constant<int, kInt8>{}) : by_type(std::integral_constant<int, kE4m3>{});
}
