// Attention over a window and the first positions (sinks), forward:
//
//   out_i = sum_j p_ij v_j,  p_ij = 2^(c s_ij - lse_i),  s_ij = q_i . k_j,  c = scale log2(e)
//   lse_i = log2 sum_j 2^(c s_ij) over the j that i sees
//
// in one pass over the keys with a running maximum and sum. A workgroup owns 128 rows
// (positions x the heads that share a key head) and walks the tiles of keys that any of
// them sees; a wave holds 32 rows as the columns of its products, so a row's maximum, sum
// and rescaling are a lane's own (two lanes a row).
// 128 rows and 64 keys: 16-bit heads of 64 leave registers for three waves a SIMD, of 128 for two; more
// rows a wave or a second tile in flight spilled. Bound by the products (three of a pair: the probabilities are two planes)
// and, beside them, an exponential for each 3 D multiply-adds: bf16, 16 heads on 4, [1, 16384] of 128, window 2048 behind 2052
// carried keys 434 us a call (0.63 PFLOP/s of the two products that count, 0.95 of the three; a large product 1.12),
// [8, 2048] of 64, window 512, 57 us. The smallest calls are a chain of latencies: [1, 16] 6.1 us.
#include "window_attention.hpp"

#include <algorithm>
#include <type_traits>

namespace koemi {
namespace window_attention {
namespace {

template <typename T> constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;  // of a tile

struct Forward {
    Shape s;
    void* out;
    void* rest;       // what 16-bit outputs are rounded off by, in their type, or null
    float* lse;       // [batch, heads, length] or null
    float* parts;     // one of several parts of the keys: [parts, batch, groups, rows, width] sums, null for one part
    float* part_lse;  // [parts, batch, groups, rows]
    const int64_t* held;  // [batch]: entries of the cache that the keys begin with, or null
    int row_tiles, splits;
};

// LATE: the keys begin with a cache's entries (as many as it has slots), and rows that held fewer than their sinks have
// the others among the first of the queries' own positions.
template <typename T, int NB, bool LATE>
__global__ __launch_bounds__(kThreads, NB == 1 ? 4 : NB == 2 ? 3 : NB <= 4 ? 2 : 1) void window_forward_kernel(Forward f) {
    using L = Tile<T, NB>;
    constexpr int KT = kKeys<T>, KB = KT / 32;
    __shared__ __attribute__((aligned(1024))) char k_tile[KT * L::kStride];
    __shared__ __attribute__((aligned(1024))) char v_tile[KT * L::kStride];
    __shared__ float scratch[kWaves][kScratch];
    __shared__ int bad_tile, any_row;
    const Shape& a = f.s;
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, half = lane >> 5, col = lane & 31;
    const Place at_work(static_cast<int>(blockIdx.x), a.batch * a.groups, f.row_tiles * f.splits);
    const int split = at_work.part % f.splits, tile = at_work.part / f.splits;
    const int g = at_work.head % a.groups, b = at_work.head / a.groups;
    const int rows = a.length * a.shared, before = a.total - a.length;
    const int row = tile * kRows + wave * 32 + col, last_row = min(tile * kRows + kRows, rows) - 1;
    const int position = position_of(a, min(row, rows - 1)), place = before + position;
    const int head = g * a.shared + min(row, rows - 1) - position * a.shared;
    const int first = before + position_of(a, tile * kRows), last = before + position_of(a, last_row);
    const uint8_t* valid = a.valid ? a.valid + static_cast<int64_t>(b) * a.total : nullptr;
    const bool row_ok = row < rows && (!valid || valid[place]);
    const uint8_t* shown_at = valid ? valid : static_cast<const uint8_t*>(a.k);  // any byte where all are valid
    const int late = LATE ? static_cast<int>(max(a.sinks - max(f.held[b], int64_t{0}), int64_t{0})) : 0;
    const int late_from = LATE ? before : 0, late_to = LATE ? before + min(late, a.length) : 0;
    if (threadIdx.x == 0) bad_tile = -1, any_row = 0;
    __syncthreads();
    if (__ballot(row_ok) && lane == 0) any_row = 1;
    __syncthreads();

    f32x16 acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x16(0.0f);
    float top = -INFINITY, sum = 0.0f;
    const float c = a.scale * kLog2e;
    if (any_row) {
        const T* q = static_cast<const T*>(a.q) + b * a.qs.batch + position * a.qs.position + head * a.qs.head;
        const T* k = static_cast<const T*>(a.k) + b * a.ks.batch + g * a.ks.head;
        const T* v = static_cast<const T*>(a.v) + b * a.vs.batch + g * a.vs.head;
        uint4 qf[L::kFrags];
#pragma unroll
        for (int s = 0; s < L::kFrags; ++s)
            qf[s] = row_ok ? load_unit<T>(q, 2 * s + half, a.width) : make_uint4(0, 0, 0, 0);
        const KeyTiles<KT> tiles(a, first, last, late_from, late_to);
        const int t0 = static_cast<int>(static_cast<int64_t>(tiles.count) * split / f.splits);
        const int t1 = static_cast<int>(static_cast<int64_t>(tiles.count) * (split + 1) / f.splits);
        // the wave's own rows
        const int wave_row = tile * kRows + wave * 32;
        const int wave_first = before + position_of(a, min(wave_row, rows - 1));
        const int wave_last = before + position_of(a, min(wave_row + 31, rows - 1));
        const bool wave_rows = __ballot(row_ok) != 0;
        Staged<T, NB, KT> next_k, next_v;
        uint8_t next_ok = 0;
        auto fetch = [&](int t) {
            const int key0 = tiles[t] * KT, last = a.total - 1 - key0;
            next_ok = shown_at[valid ? min(key0 + lane, a.total - 1) : 0];
            next_k.load(k + key0 * a.ks.position, a.ks.position, last, a.width);
            next_v.load(v + key0 * a.vs.position, a.vs.position, last, a.width);
        };
        if (t0 < t1) fetch(t0);
        for (int t = t0; t < t1; ++t) {
            const int key0 = tiles[t] * KT;
            const uint64_t shown = __ballot(lane < KT && key0 + lane < a.total && (!valid || next_ok)), every = low_bits(KT);
            auto whole = [&](int lo, int hi) {  // rows at places lo .. hi see all of the tile
                return shown == every && key0 + KT - 1 <= lo && (hi - key0 < a.window || key0 + KT <= a.sinks || (LATE && key0 >= late_from && key0 + KT <= late_to));
            };
            __syncthreads();
            if (!whole(first, last)) {
                next_k.keep({shown});
                if (next_v.keep({shown})) bad_tile = t;
            }
            next_k.store(k_tile, a.width);
            next_v.store(v_tile, a.width);
            __syncthreads();
            if (t + 1 < t1) fetch(t + 1);
            if (!shown || !wave_rows || key0 > wave_last || (key0 + KT <= wave_first - a.window + 1 && key0 >= a.sinks && !(LATE && key0 < late_to && key0 + KT > late_from)))
                continue;
            f32x16 s[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                s[kb] = f32x16(0.0f);
                mma_rows<T, NB>(s[kb], k_tile, kb * 32, qf);
            }
            const bool masked = !whole(wave_first, wave_last);
            uint64_t seen = every;
            if (masked) {
                seen = row_ok ? keys_seen(a, place, key0, late_from, late_to) & shown : 0ull;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const uint32_t mine = static_cast<uint32_t>(seen >> (32 * kb)) >> (4 * half);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = where_seen(mine, r, s[kb][r], -INFINITY);
                }
            }
            float high = s[0][0];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) high = fmaxf(high, s[kb][r]);
            high = fmaxf(top, max_of_halves(high));
            // The maximum only keeps the exponentials in range: while no row's grows by 2^6, all keep the one they have.
            if (__any(high * c > top * c + 6.0f || (top == -INFINITY && high > top))) {
                const float shrink = high > top ? __builtin_amdgcn_exp2f((top - high) * c) : 1.0f;
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[n] *= shrink;
                sum *= shrink;
                top = high;
            }
            const float base = (top == -INFINITY ? 0.0f : top * c) - kLift<T>;
            auto terms = [&](int kb) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[kb][r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], c, -base));
                    sum += s[kb][r];
                }
            };
            if (masked && bad_tile == t) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    terms(kb);
                    seen_acc<T, NB>(acc, v_tile, kb * 32, s[kb], static_cast<uint32_t>(seen >> (32 * kb)), scratch[wave]);
                }
            } else {  // one block's products run beside the next one's exponentials
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    terms(kb);
                    mma_acc<T, NB>(acc, v_tile, kb * 32, s[kb]);
                }
            }
        }
        if constexpr (sizeof(T) == 2) {
            // An infinite value times two planes may be NaN, by a second plane of 0 or of the other sign. Where such sums
            // are NaN and the probabilities are not, they are what the infinities and NaN among the values seen add up to.
            float any[4] = {};  // NaN if one of the sums is
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) any[r % 4] += acc[n][r];
            any[0] = (any[0] + any[1]) + (any[2] + any[3]);
            const float all = sum_of_halves(sum);
            const bool nan = row_ok && any[0] != any[0] && all == all;
            if (__builtin_expect(__any(nan), 0)) {
                uint32_t lost[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    lost[n] = 0;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (nan && acc[n][r] != acc[n][r]) acc[n][r] = 0.0f, lost[n] |= 1u << r;
                }
#pragma unroll 1
                for (int t = t0; t < t1; ++t)
#pragma unroll 1
                    for (int key = tiles[t] * KT; key < min(tiles[t] * KT + KT, a.total); ++key) {
                        if (!nan || key > place || (place - key >= a.window && key >= a.sinks && !(LATE && key >= late_from && key < late_to)) || (valid && !valid[key])) continue;
                        const T* x = v + key * a.vs.position;
#pragma unroll
                        for (int n = 0; n < NB; ++n)
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int d = 32 * n + 8 * q + 4 * half;
                                if (d >= a.width) continue;
                                alignas(8) T e[4];
                                *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(x + d);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float y = to_f32(e[i]);
                                    acc[n][4 * q + i] += fabsf(y) < INFINITY ? 0.0f : y;
                                }
                            }
                    }
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if ((lost[n] >> r & 1u) && acc[n][r] == 0.0f) acc[n][r] = NAN;
            }
        }
    }
    sum = sum_of_halves(sum);
    if (row >= rows) return;
    const bool none = sum == 0.0f || !row_ok;  // nothing seen: zeros (a masked row's sums are of a zero query)
    const float invert = none ? 0.0f : 1.0f / sum;
    const float lse = none ? INFINITY : top * c - kLift<T> + __builtin_amdgcn_logf(sum);
    const int64_t at = (static_cast<int64_t>(b) * a.groups * a.shared + head) * a.length + position;
    if (f.parts) {
        const int64_t cell = (static_cast<int64_t>(b) * a.groups + g) * rows + row + static_cast<int64_t>(split) * a.batch * a.groups * rows;
        if (half == 0) f.part_lse[cell] = lse;
        float* o = f.parts + cell * a.width;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * n + 8 * (r / 4) + 4 * half + r % 4;
                if (d < a.width) o[d] = none ? 0.0f : acc[n][r] * invert;
            }
        return;
    }
    if (f.lse && half == 0) f.lse[at] = lse;
    T* o = static_cast<T*>(f.out) + ((static_cast<int64_t>(b) * a.length + position) * a.groups * a.shared + head) * a.width;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = none ? 0.0f : acc[n][4 * q + i] * invert;
            const int d = 32 * n + 8 * q + 4 * half;
            store_four(o, d, a.width, x);
            if (f.rest) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = fabsf(x[i]) < INFINITY ? x[i] - to_f32(from_f32<T>(x[i])) : 0.0f;
                store_four(static_cast<T*>(f.rest) + (o - static_cast<T*>(f.out)), d, a.width, x);
            }
        }
}

// The parts of a row's keys joined, in their order: each part brings its own mean and log-sum.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_join_kernel(Forward f) {
    const Shape& a = f.s;
    const int64_t rows = static_cast<int64_t>(a.length) * a.shared, cells = rows * a.batch * a.groups;
    const int64_t cell = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
    if (cell >= cells) return;
    const int lane = lane_id();
    float top = -INFINITY;
    for (int p = 0; p < f.splits; ++p) {
        const float x = f.part_lse[cell + p * cells];
        if (x != INFINITY || x != x) top = x > top || x != x ? x : top;
    }
    float sum = 0.0f;
    for (int p = 0; p < f.splits; ++p) {
        const float x = f.part_lse[cell + p * cells];
        if (x != INFINITY) sum += __builtin_amdgcn_exp2f(x - top);
    }
    const float invert = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t row = cell % rows, g = cell / rows % a.groups, b = cell / rows / a.groups;
    const int64_t position = row / a.shared, head = g * a.shared + row % a.shared, heads = static_cast<int64_t>(a.groups) * a.shared;
    if (f.lse && lane == 0) f.lse[(b * heads + head) * a.length + position] = sum == 0.0f ? INFINITY : top + __builtin_amdgcn_logf(sum);
    T* o = static_cast<T*>(f.out) + ((b * a.length + position) * heads + head) * a.width;
    for (int d = lane; d < a.width; d += kWave) {
        float x = 0.0f;
        for (int p = 0; p < f.splits; ++p) {
            const float y = f.part_lse[cell + p * cells];
            if (y != INFINITY) x = fmaf(f.parts[(cell + p * cells) * a.width + d], __builtin_amdgcn_exp2f(y - top), x);
        }
        x *= invert;
        o[d] = from_f32<T>(x);
        if (f.rest)
            static_cast<T*>(f.rest)[o - static_cast<T*>(f.out) + d] = from_f32<T>(fabsf(x) < INFINITY ? x - to_f32(from_f32<T>(x)) : 0.0f);
    }
}

// Parts the keys are cut into where the rows alone leave compute units idle: so many that there are
// about 512 workgroups, at most 64, and no part under four tiles.
int splits_of(int64_t workgroups, int64_t tiles) {
    int64_t n = std::min<int64_t>(tiles / 4, 512 / std::max<int64_t>(workgroups, 1));
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(n, 64)));
}

int64_t workgroups_of(int64_t batch, int64_t groups, int64_t rows) { return batch * groups * ((rows + kRows - 1) / kRows); }

int splits_for(int64_t batch, int64_t length, int64_t total, int64_t heads, int64_t groups, int64_t window, int64_t sinks, int dtype) {
    const int64_t kt = dtype == KOEMI_F32 ? 32 : 64, shared = heads / groups;
    const int64_t span = std::min(total, std::min(window, total) + std::min(kRows / shared + 1, length) + std::min(sinks, total));
    return splits_of(workgroups_of(batch, groups, length * shared), (span + kt - 1) / kt);
}

template <typename T, int NB>
int run(const Forward& f, hipStream_t stream) {
    const int64_t grid = workgroups_of(f.s.batch, f.s.groups, static_cast<int64_t>(f.s.length) * f.s.shared) * f.splits;
    if (f.held)
        hipLaunchKernelGGL((window_forward_kernel<T, NB, true>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, f);
    else
        hipLaunchKernelGGL((window_forward_kernel<T, NB, false>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, f);
    int rc = check_launch("koemi_window_attention_forward");
    if (rc != KOEMI_OK || f.splits == 1) return rc;
    const int64_t cells = static_cast<int64_t>(f.s.length) * f.s.shared * f.s.batch * f.s.groups;
    hipLaunchKernelGGL((window_join_kernel<T>), dim3(grid_for(cells, kWaves)), dim3(kThreads), 0, stream, f);
    return check_launch("koemi_window_attention_forward(join)");
}

template <typename T>
int by_width(const Forward& f, hipStream_t stream) {
    const int nb = (f.s.width + 31) / 32;
    if (nb <= 1) return run<T, 1>(f, stream);
    if (nb <= 2) return run<T, 2>(f, stream);
    if (nb <= 3) return run<T, 3>(f, stream);
    if (nb <= 4) return run<T, 4>(f, stream);
    if (nb <= 6) return run<T, 6>(f, stream);
    return run<T, 8>(f, stream);
}

}  // namespace

int shape_of(const char* what, const void* queries, const void* keys, const void* values, const uint8_t* valid,
             const int64_t* strides, int64_t batch, int64_t length, int64_t total, int64_t heads, int64_t groups,
             int64_t width, int64_t window, int64_t sinks, float scale, int dtype, Shape& s) {
    if (batch < 0 || length < 0 || total < length || heads < 1 || groups < 1 || width < 1)
        return fail(KOEMI_ERR_INVALID, "%s: sizes must not be negative, and no fewer keys than queries", what);
    if (heads % groups) return fail(KOEMI_ERR_INVALID, "%s: the key heads must divide the query heads", what);
    if (window < 1 || sinks < 0) return fail(KOEMI_ERR_INVALID, "%s: window must be positive and sinks not negative", what);
    if (!(scale > 0.0f) || scale > 3.0e38f) return fail(KOEMI_ERR_INVALID, "%s: scale must be positive and finite", what);
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16, not %s", what, dtype_name(dtype));
    if (width > 256) return fail(KOEMI_ERR_UNSUPPORTED, "%s: heads are at most 256 wide", what);
    const int64_t shared = heads / groups;
    // rows and the places they reach stay below 2^30, workgroups below 2^30
    if (total >= (1 << 29) || shared > (1 << 20) || total * shared >= (1 << 29) || batch >= (1 << 24) || groups >= (1 << 24) ||
        batch * groups * ((std::max(length * shared, total) + kRows - 1) / kRows) >= (1 << 24))
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^29 positions x shared heads and 2^24 tiles of 128 of them", what);
    const int64_t size = dtype == KOEMI_F32 ? 4 : 2;
    if (batch && length && (!queries || !keys || !values || !strides)) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    s = Shape{};
    s.q = queries, s.k = keys, s.v = values, s.valid = valid;
    if (strides) {
        s.qs = {strides[0], strides[1], strides[2]};
        s.ks = {strides[3], strides[4], strides[5]};
        s.vs = {strides[6], strides[7], strides[8]};
        bool fits = width * size % 16 == 0 && heads * width * size < (1 << 24);
        for (int i = 0; i < 9; ++i) fits = fits && strides[i] * size % 16 == 0 && strides[i] >= 0;
        for (int i = 1; i < 9; i += 3) fits = fits && strides[i] * size < (1 << 24);
        for (const void* p : {queries, keys, values}) fits = fits && reinterpret_cast<uintptr_t>(p) % 16 == 0;
        if (!fits)
            return fail(KOEMI_ERR_UNSUPPORTED, "%s: rows must be whole 16-byte pieces, 16-byte aligned and less than 2^24 bytes apart", what);
    }
    s.batch = static_cast<int>(batch), s.length = static_cast<int>(length), s.total = static_cast<int>(total);
    s.groups = static_cast<int>(groups), s.shared = static_cast<int>(shared), s.width = static_cast<int>(width);
    s.window = static_cast<int>(std::min(window, std::max<int64_t>(total, 1)));
    s.sinks = static_cast<int>(std::min(sinks, total));
    s.scale = scale;
    if (shared > 1) {
        int bits = 0;
        while ((int64_t(1) << bits) < shared) ++bits;
        s.magic = static_cast<uint32_t>(((int64_t(1) << (31 + bits)) + shared - 1) / shared);
        s.shift = bits - 1;
    }
    return KOEMI_OK;
}

}  // namespace window_attention
}  // namespace koemi

using namespace koemi;
using namespace koemi::window_attention;

extern "C" size_t koemi_window_attention_workspace_bytes(int64_t batch, int64_t length, int64_t total, int64_t heads,
                                                         int64_t groups, int64_t width, int64_t window, int64_t sinks, int dtype) {
    Shape s;
    if (shape_of("koemi_window_attention_workspace_bytes", nullptr, nullptr, nullptr, nullptr, nullptr, 0, length, total, heads,
                 groups, width, window, sinks, 1.0f, dtype, s) != KOEMI_OK || batch < 1 || length < 1) {
        clear_error();
        return 0;
    }
    const int n = splits_for(batch, length, total, heads, groups, window, sinks, dtype);
    return n == 1 ? 0 : static_cast<size_t>(n) * batch * heads * length * (width + 1) * 4;
}

namespace {

int forward(const char* what, const void* queries, const void* keys, const void* values, const uint8_t* valid, const int64_t* strides,
            const int64_t* held, void* output, void* rest, float* lse, int64_t batch, int64_t length, int64_t total, int64_t heads,
            int64_t groups, int64_t width, int64_t window, int64_t sinks, float scale, int dtype, void* workspace,
            size_t workspace_bytes, koemi_stream_t stream) {
    Forward f{};
    const int rc = shape_of(what, queries, keys, values, valid, strides, batch, length, total, heads, groups, width, window, sinks,
                            scale, dtype, f.s);
    if (rc != KOEMI_OK || batch == 0 || length == 0) return rc;
    if (!output) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    f.out = output, f.rest = dtype == KOEMI_F32 ? nullptr : rest, f.lse = lse, f.held = held;
    f.row_tiles = static_cast<int>((length * f.s.shared + kRows - 1) / kRows);
    f.splits = splits_for(batch, length, total, heads, groups, window, sinks, dtype);
    if (f.splits > 1) {
        const size_t cells = static_cast<size_t>(f.splits) * batch * heads * length;
        if (!workspace || workspace_bytes < cells * (width + 1) * 4) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
        f.part_lse = static_cast<float*>(workspace);
        f.parts = f.part_lse + cells;
    }
    if (dtype == KOEMI_F32) return by_width<float>(f, as_stream(stream));
    if (dtype == KOEMI_F16) return by_width<f16>(f, as_stream(stream));
    return by_width<bf16>(f, as_stream(stream));
}

}  // namespace

extern "C" int koemi_window_attention_forward(const void* queries, const void* keys, const void* values, const uint8_t* valid,
                                              const int64_t* strides, void* output, void* rest, float* lse, int64_t batch, int64_t length,
                                              int64_t total, int64_t heads, int64_t groups, int64_t width, int64_t window,
                                              int64_t sinks, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                              koemi_stream_t stream) {
    clear_error();
    return forward("koemi_window_attention_forward", queries, keys, values, valid, strides, nullptr, output, rest, lse, batch, length, total,
                   heads, groups, width, window, sinks, scale, dtype, workspace, workspace_bytes, stream);
}

extern "C" int koemi_window_attention_chunk(const void* queries, const void* keys, const void* values, const uint8_t* valid,
                                            const int64_t* strides, const int64_t* held, void* output, int64_t batch, int64_t length,
                                            int64_t heads, int64_t groups, int64_t width, int64_t window, int64_t sinks, float scale,
                                            int dtype, void* workspace, size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_window_attention_chunk";
    if (length < 0 || window < 1 || sinks < 0) return fail(KOEMI_ERR_INVALID, "%s: window must be positive, length and sinks not negative", what);
    if (length >= (1 << 29) || window >= (1 << 29) || sinks >= (1 << 29))
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^29 positions", what);
    if (batch > 0 && length > 0 && (!valid || !held)) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    return forward(what, queries, keys, values, valid, strides, held, output, nullptr, nullptr, batch, length, window + sinks + length, heads,
                   groups, width, window, sinks, scale, dtype, workspace, workspace_bytes, stream);
}
