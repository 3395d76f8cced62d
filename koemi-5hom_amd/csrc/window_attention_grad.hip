// Gradients of the attention over a window and the first positions (sinks):
//
//   p_ij = 2^(c s_ij - lse_i) again from the kept lse,  D_i = sum_d dout_id out_id
//   dp_ij = dout_i . v_j,  ds_ij = p_ij (dp_ij - D_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//
// Two kernels, each owning what it sums, so that no sum depends on an order of arrival: one
// holds 128 rows (positions x shared heads) and walks the keys for dq and D, one holds 128
// keys and walks the rows for dk and dv, all heads that share the keys among them. That
// forms s and dp twice (seven products of a pair instead of five; in 16 bits, where p and ds are two planes, ten). The sinks are seen by every
// later row: what lies beyond their window is cut into chunks of rows that run beside the
// others, and the sinks' own workgroups add the chunks' sums in order.
//
// Bound by the products, the exponentials and, at heads of 128, by one wave a SIMD (dk, dv, p and
// ds take 467 registers). bf16, 16 heads on 4, [8, 2048] of 64, window 512: dq 65 us, dk and dv 149, the sinks'
// far rows 22, their sums 5. 8 heads on 2, [1, 16384] of 128, window 4096: 547, 939, 43, 11 (a large
// product's rate would take 750 for forward and gradients of seven products). fp32, 4 heads on 1, [2, 1500] of 48, window
// 256: 40 and 79.
#include "window_attention.hpp"

#include <algorithm>

namespace koemi {
namespace window_attention {
namespace {

struct Backward {
    Shape s;
    const void* out;
    const void* rest;   // what out was rounded off by, or null: D is a small difference of large terms
    const void* d_out;  // each [batch, length, heads, width]
    const float* lse;
    float* delta;       // D: [batch, heads, length], kAlone for a row that sees one key
    void* dq;
    void* dk;
    void* dv;
    float* far_parts;   // [chunks, batch, groups, 32 x far_tiles keys, 2, width]
    int row_tiles;
    int far_tiles, far_chunks, far_first;  // tiles of 32 sinks; the first position past the first one's window
};

template <typename T> constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;  // of a tile that dq walks

// D in place of a number: the row sees one key. A NaN that no sum is stored as: D may be infinite or NaN by
// itself, and has to reach the keys' gradients then.
constexpr uint32_t kAlone = 0x7fffffffu;
__device__ __forceinline__ float stored_delta(float delta, bool alone) {
    return __uint_as_float(alone ? kAlone : delta != delta ? 0x7fc00000u : __float_as_uint(delta));
}

__device__ __forceinline__ float largest(const f32x16& x) {
    float m = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(x[r]));
    return max_of_halves(m);
}

// fp16 products of ds: its size is the loss's, so each column's ds is brought to about 2^10
// by a power of two, which is lowered (the sums with it) where a later block exceeds 2^14.
template <typename T, int NB>
struct Range {
    float by = 0.0f;
    __device__ __forceinline__ void fit(f32x16& ds, f32x16 (&acc)[NB]) {
        if constexpr (std::is_same<T, f16>::value) {
            const float high = largest(ds);
            const bool over = high * by > 16384.0f || (by == 0.0f && high > 0.0f);
            if (__any(over)) {
                const int e = static_cast<int>(__float_as_uint(high) >> 23);
                const float to = over ? __uint_as_float(static_cast<uint32_t>(min(264 - e, 254)) << 23) : by;
                const float change = over && by != 0.0f ? to / by : 1.0f;
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[n] *= change;
                by = to;
            }
            ds *= by;
        }
    }
    __device__ __forceinline__ float back() const {
        if constexpr (std::is_same<T, f16>::value) return by == 0.0f ? 1.0f : 1.0f / by;
        return 1.0f;
    }
};

template <typename T, int NB>
__global__ __launch_bounds__(kThreads, NB == 1 ? 4 : NB == 2 && sizeof(T) == 2 ? 3 : NB <= 4 ? 2 : 1) void window_dq_kernel(Backward f) {
    using L = Tile<T, NB>;
    constexpr int KT = kKeys<T>, KB = KT / 32;
    __shared__ __attribute__((aligned(1024))) char k_tile[KT * L::kStride];
    __shared__ __attribute__((aligned(1024))) char v_tile[KT * L::kStride];
    __shared__ float scratch[kWaves][kScratch];
    __shared__ int bad_tile, any_row;
    const Shape& a = f.s;
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, half = lane >> 5, col = lane & 31;
    const Place at_work(static_cast<int>(blockIdx.x), a.batch * a.groups, f.row_tiles);
    const int tile = at_work.part, g = at_work.head % a.groups, b = at_work.head / a.groups;
    const int rows = a.length * a.shared, before = a.total - a.length;
    const int row = tile * kRows + wave * 32 + col, last_row = min(tile * kRows + kRows, rows) - 1;
    const int position = position_of(a, min(row, rows - 1)), place = before + position;
    const int head = g * a.shared + min(row, rows - 1) - position * a.shared;
    const int first = before + position_of(a, tile * kRows), last = before + position_of(a, last_row);
    const uint8_t* valid = a.valid ? a.valid + static_cast<int64_t>(b) * a.total : nullptr;
    const bool row_ok = row < rows && (!valid || valid[place]);
    const uint8_t* shown_at = valid ? valid : static_cast<const uint8_t*>(a.k);  // any byte where all are valid
    const int64_t at = (static_cast<int64_t>(b) * a.groups * a.shared + head) * a.length + position;
    const int64_t cell = ((static_cast<int64_t>(b) * a.length + position) * a.groups * a.shared + head) * a.width;
    if (threadIdx.x == 0) bad_tile = -1, any_row = 0;
    __syncthreads();
    if (__ballot(row_ok) && lane == 0) any_row = 1;
    __syncthreads();

    f32x16 acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x16(0.0f);
    Range<T, NB> range;
    float delta = 0.0f;
    int sees = 0;  // keys
    const float c = a.scale * kLog2e;
    if (any_row) {
        const T* q = static_cast<const T*>(a.q) + b * a.qs.batch + position * a.qs.position + head * a.qs.head;
        const T* k = static_cast<const T*>(a.k) + b * a.ks.batch + g * a.ks.head;
        const T* v = static_cast<const T*>(a.v) + b * a.vs.batch + g * a.vs.head;
        uint4 qf[L::kFrags], gf[L::kFrags];
#pragma unroll
        for (int s = 0; s < L::kFrags; ++s) {
            qf[s] = gf[s] = make_uint4(0, 0, 0, 0);
            if (row_ok) {
                qf[s] = load_unit<T>(q, 2 * s + half, a.width);
                gf[s] = load_unit<T>(static_cast<const T*>(f.d_out) + cell, 2 * s + half, a.width);
                const uint4 o = load_unit<T>(static_cast<const T*>(f.out) + cell, 2 * s + half, a.width);
                uint4 l = make_uint4(0, 0, 0, 0);
                if (f.rest) l = load_unit<T>(static_cast<const T*>(f.rest) + cell, 2 * s + half, a.width);
                const T* x = reinterpret_cast<const T*>(&gf[s]);
                const T* y = reinterpret_cast<const T*>(&o);
                const T* z = reinterpret_cast<const T*>(&l);
#pragma unroll
                for (int i = 0; i < kPer16<T>; ++i) delta = fmaf(to_f32(x[i]), to_f32(y[i]) + to_f32(z[i]), delta);
            }
        }
        delta = sum_of_halves(delta);
        const float lse = row_ok ? f.lse[at] : INFINITY;
        const KeyTiles<KT> tiles(a, first, last);
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
        fetch(0);
        for (int t = 0; t < tiles.count; ++t) {
            const int key0 = tiles[t] * KT;
            const uint64_t shown = __ballot(lane < KT && key0 + lane < a.total && (!valid || next_ok)), every = low_bits(KT);
            auto whole = [&](int lo, int hi) {  // rows at places lo .. hi see all of the tile
                return shown == every && key0 + KT - 1 <= lo && (hi - key0 < a.window || key0 + KT <= a.sinks);
            };
            __syncthreads();
            if (!whole(first, last)) {
                next_v.keep({shown});
                if (next_k.keep({shown})) bad_tile = t;
            }
            next_k.store(k_tile, a.width);
            next_v.store(v_tile, a.width);
            __syncthreads();
            if (t + 1 < tiles.count) fetch(t + 1);
            if (!shown || !wave_rows || key0 > wave_last || (key0 + KT <= wave_first - a.window + 1 && key0 >= a.sinks)) continue;
            const bool masked = !whole(wave_first, wave_last);
            const uint64_t seen = !masked ? every : row_ok ? keys_seen(a, place, key0) & shown : 0ull;
            sees += __popcll(seen);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                f32x16 s = f32x16(0.0f), d = f32x16(0.0f);
                mma_rows<T, NB>(s, k_tile, kb * 32, qf);
                mma_rows<T, NB>(d, v_tile, kb * 32, gf);
#pragma unroll
                for (int r = 0; r < 16; ++r) d[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (d[r] - delta);
                const uint32_t block = static_cast<uint32_t>(seen >> (32 * kb));
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) d[r] = where_seen(block >> (4 * half), r, d[r], 0.0f);
                }
                range.fit(d, acc);
                if (masked && bad_tile == t)
                    seen_acc<T, NB>(acc, k_tile, kb * 32, d, block, scratch[wave]);
                else
                    mma_acc<T, NB>(acc, k_tile, kb * 32, d);
            }
        }
    }
    if (row >= rows) return;
    // A row that sees one key has p = 1 whatever the score: no gradient, to the bit. Its D says so to the other kernel.
    const bool alone = sees <= 1;
    if (half == 0) f.delta[at] = stored_delta(delta, alone);
    if (!f.dq) return;
    const float by = a.scale * range.back();
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = row_ok && !alone ? acc[n][4 * q + i] * by : 0.0f;
            store_four(static_cast<T*>(f.dq) + cell, 32 * n + 8 * q + 4 * half, a.width, x);
        }
}

// Rows of a tile where the waves share their keys: 32 a wave, or what LDS holds.
template <typename T, int NB> constexpr int kShareRows = Tile<T, NB>::kStride > 512 ? 64 : 32 * kWaves;

// The rows of one head after another, in tiles. Each wave holds 32 keys of its own (SHARE
// false: 128 a workgroup), or all hold the same 32 and take blocks of 32 rows in turn, their
// sums added in their order: four times the workgroups, each with a quarter of the work, for
// calls of few keys, and (far) for the sinks against a chunk of the tiles past their window,
// whose sums go to far_parts. fp32 heads of 33 to 64 that share: with all registers of a SIMD to a wave
// 80 us at [2, 1500], with half of them and 153 spilled 108.
template <typename T, int NB, bool SHARE>
__global__ __launch_bounds__(kThreads, NB == 1 || (NB == 2 && !(SHARE && sizeof(T) == 4)) ? 2 : 1) void window_dkv_kernel(Backward f, int far) {
    using L = Tile<T, NB>;
    constexpr int RT = SHARE ? kShareRows<T, NB> : kKeys<T>, RB = RT / 32, RW = (RT + 63) / 64;
    constexpr int kOwn = SHARE ? 32 : kRows;  // keys of the workgroup
    __shared__ __attribute__((aligned(1024))) char tiles[2 * RT * L::kStride];
    char *const q_tile = tiles, *const g_tile = tiles + RT * L::kStride;
    __shared__ __attribute__((aligned(16))) float stats[2][RT];  // lse, D
    __shared__ float scratch[kWaves][kScratch];
    __shared__ int bad_tile;
    const Shape& a = f.s;
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave, half = lane >> 5, col = lane & 31;
    const int chunks = SHARE && far ? f.far_chunks : 1, own_tiles = SHARE && far ? f.far_tiles : (a.total + kOwn - 1) / kOwn;
    const Place at_work(static_cast<int>(blockIdx.x), a.batch * a.groups, own_tiles * chunks);
    const int chunk = at_work.part % chunks, tile = at_work.part / chunks;
    const int g = at_work.head % a.groups, b = at_work.head / a.groups;
    const int before = a.total - a.length;
    const int key0 = tile * kOwn, wave_key = SHARE ? key0 : key0 + wave * 32, key = wave_key + col;
    const uint8_t* valid = a.valid ? a.valid + static_cast<int64_t>(b) * a.total : nullptr;
    const bool key_ok = key < a.total && (!valid || valid[key]) && (!(SHARE && far) || key < a.sinks);
    const T* q = static_cast<const T*>(a.q) + b * a.qs.batch + g * a.shared * a.qs.head;
    const T* k = static_cast<const T*>(a.k) + b * a.ks.batch + key * a.ks.position + g * a.ks.head;
    const T* v = static_cast<const T*>(a.v) + b * a.vs.batch + key * a.vs.position + g * a.vs.head;
    const int64_t out_row = static_cast<int64_t>(a.groups) * a.shared * a.width;
    const T* d_out = static_cast<const T*>(f.d_out) + b * a.length * out_row + static_cast<int64_t>(g) * a.shared * a.width;
    const int64_t stat = (static_cast<int64_t>(b) * a.groups + g) * a.shared * a.length;
    if (threadIdx.x == 0) bad_tile = -1;

    uint4 kf[L::kFrags], vf[L::kFrags];
#pragma unroll
    for (int s = 0; s < L::kFrags; ++s) {
        kf[s] = key_ok ? load_unit<T>(k, 2 * s + half, a.width) : make_uint4(0, 0, 0, 0);
        vf[s] = key_ok ? load_unit<T>(v, 2 * s + half, a.width) : make_uint4(0, 0, 0, 0);
    }
    f32x16 dk[NB], dv[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) dk[n] = dv[n] = f32x16(0.0f);
    Range<T, NB> range;
    const float c = a.scale * kLog2e;
    // queries that see key j: from begins(j) on, up to ends(j)
    auto begins = [&](int j) { return max(j - before, 0); };
    auto ends = [&](int j) { return max(j - before + a.window, 0); };
    const int from = SHARE && far ? f.far_first : begins(key0);
    const int to = SHARE && far ? a.length : min(ends(min(key0 + kOwn, a.total) - 1), a.length);
    const bool wave_keys = __ballot(key_ok) != 0, wave_whole = __ballot(key_ok) == ~0ull;
    const int key_begin = begins(key), key_end = ends(key);
    const int wave_begin = begins(wave_key), wave_end = ends(wave_key);
    const int wave_last_begin = begins(wave_key + 31), wave_last_end = ends(wave_key + 31);
    const int first = from & ~(RT - 1), walk = to > from ? (to - first + RT - 1) / RT : 0;
    const int64_t whole = static_cast<int64_t>(walk) * a.shared;
    const int t0 = static_cast<int>(whole * chunk / chunks), t1 = static_cast<int>(whole * (chunk + 1) / chunks);

    Staged<T, NB, RT> next_q, next_g;
    const uint8_t* shown_at = valid ? valid + before : static_cast<const uint8_t*>(a.q);  // any byte where all are valid
    constexpr int SE = (2 * RT + kThreads - 1) / kThreads;  // statistics a thread brings
    uint8_t next_ok[RW] = {};
    float next_delta[RW] = {};
    float next_stat[SE] = {};
    int next_head = walk ? t0 / walk : 0, next_p = first + (walk ? t0 % walk : 0) * RT;  // of the tile to fetch
    auto fetch = [&]() {
        const int p0 = next_p, last = a.length - 1 - p0;
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const int p = min(p0 + 64 * w + lane, a.length - 1);
            next_ok[w] = shown_at[valid ? p : 0];
            next_delta[w] = f.delta[stat + static_cast<int64_t>(next_head) * a.length + p];
        }
#pragma unroll
        for (int i = 0; i < SE; ++i) {
            const int n = static_cast<int>(threadIdx.x) + i * kThreads;
            next_stat[i] = (n / RT % 2 ? f.delta : f.lse)[stat + static_cast<int64_t>(next_head) * a.length + p0 + min(n % RT, last)];
        }
        next_q.load(q + next_head * a.qs.head + p0 * a.qs.position, a.qs.position, last, a.width);
        next_g.load(d_out + static_cast<int64_t>(next_head) * a.width + p0 * out_row, out_row, last, a.width);
        next_p += RT;
        if (next_p >= to) next_p = first, ++next_head;
    };
    int p0 = next_p;
    if (t0 < t1) fetch();
    for (int t = t0; t < t1; ++t, p0 = p0 + RT >= to ? first : p0 + RT) {
        uint64_t shown[RW], alone[RW];  // alone: see one key
        bool every = true, some = false, any_alone = false;
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const int r = 64 * w + lane;
            shown[w] = __ballot(r < RT && p0 + r < a.length && (!valid || next_ok[w]));
            alone[w] = __ballot(__float_as_uint(next_delta[w]) == kAlone);
            every = every && shown[w] == low_bits(RT - 64 * w), some = some || shown[w], any_alone = any_alone || alone[w];
        }
        // every key of the workgroup is seen by every row of the tile
        const bool all = !far && every && !valid && p0 >= begins(key0 + kOwn - 1) && p0 + RT <= ends(key0) && key0 + kOwn <= a.total;
        __syncthreads();
        if (!all) {
            const bool bad_q = next_q.keep(shown), bad_g = next_g.keep(shown);
            if (bad_q || bad_g) bad_tile = t;
        }
        next_q.store(q_tile, a.width);
        next_g.store(g_tile, a.width);
#pragma unroll
        for (int i = 0; i < SE; ++i) {
            const int n = static_cast<int>(threadIdx.x) + i * kThreads;
            if (n < 2 * RT) stats[n / RT][n % RT] = next_stat[i];
        }
        __syncthreads();
        if (t + 1 < t1) fetch();
        if (!some || !wave_keys) continue;
        auto products = [&](int rb, f32x16& s, f32x16& d) {
            s = d = f32x16(0.0f);
            mma_rows<T, NB>(s, q_tile, rb * 32, kf);
            mma_rows<T, NB>(d, g_tile, rb * 32, vf);
        };
        auto terms = [&](int rb, f32x16& s, f32x16& d) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float4 lse = *reinterpret_cast<const float4*>(&stats[0][rb * 32 + 8 * n + 4 * half]);
                const float4 del = *reinterpret_cast<const float4*>(&stats[1][rb * 32 + 8 * n + 4 * half]);
                const float x[4] = {lse.x, lse.y, lse.z, lse.w}, y[4] = {del.x, del.y, del.z, del.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[4 * n + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * n + i], c, kLift<T> - x[i]));
                    d[4 * n + i] = s[4 * n + i] * (d[4 * n + i] - y[i]);
                }
            }
        };
        auto block = [&](int rb, uint32_t block_shown, uint32_t block_alone) {
            const int pb = p0 + rb * 32;
            if (far ? pb + 32 <= wave_end : (pb + 32 <= wave_begin || pb >= wave_last_end)) return;
            const bool masked = far || !(block_shown == ~0u && !block_alone && wave_whole && pb >= wave_last_begin && pb + 32 <= wave_end);
            f32x16 s, d;
            products(rb, s, d);
            terms(rb, s, d);
            uint32_t seen = ~0u;
            if (masked) {
                const uint64_t by_place = far ? ~low_bits(key_end - pb) : ~low_bits(key_begin - pb) & low_bits(key_end - pb);
                seen = key_ok ? static_cast<uint32_t>(by_place) & block_shown : 0u;
                const uint32_t mine = seen >> (4 * half), moved = (seen & ~block_alone) >> (4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = where_seen(mine, r, s[r], 0.0f);
                    d[r] = where_seen(moved, r, d[r], 0.0f);
                }
            }
            range.fit(d, dk);
            if (masked && bad_tile == t) {
                seen_acc<T, NB>(dv, g_tile, rb * 32, s, seen, scratch[wave]);
                seen_acc<T, NB>(dk, q_tile, rb * 32, d, seen & ~block_alone, scratch[wave]);
            } else {
                mma_acc<T, NB>(dv, g_tile, rb * 32, s);
                mma_acc<T, NB>(dk, q_tile, rb * 32, d);
            }
        };
        if (SHARE) {
            const int rb = (wave - t * RB) & (kWaves - 1);
            const int w = RW > 1 ? rb / 2 : 0;
            if (rb < RB) block(rb, static_cast<uint32_t>(shown[w] >> (32 * (rb & 1))), static_cast<uint32_t>(alone[w] >> (32 * (rb & 1))));
        } else if (NB <= 2 && every && !any_alone && wave_whole && p0 >= wave_last_begin && p0 + RT <= wave_end) {
            // all seen: without a branch, so that one block's products run beside the other's terms (heads of 64: 158 ->
            // 153 us; wider ones have no registers for both blocks)
            f32x16 s[RB], d[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) products(rb, s[rb], d[rb]);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                terms(rb, s[rb], d[rb]);
                range.fit(d[rb], dk);
                mma_acc<T, NB>(dv, g_tile, rb * 32, s[rb]);
                mma_acc<T, NB>(dk, q_tile, rb * 32, d[rb]);
            }
        } else if (NB <= 2) {
#pragma unroll 1
            for (int rb = 0; rb < RB; ++rb) block(rb, static_cast<uint32_t>(shown[0] >> (32 * rb)), static_cast<uint32_t>(alone[0] >> (32 * rb)));
        } else {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) block(rb, static_cast<uint32_t>(shown[0] >> (32 * rb)), static_cast<uint32_t>(alone[0] >> (32 * rb)));
        }
    }
    const float unlift = std::is_same<T, f16>::value ? 1.0f / 256.0f : 1.0f;
    const float by = a.scale * range.back() * unlift;
    const int64_t far_keys = static_cast<int64_t>(f.far_tiles) * 32;
    if constexpr (SHARE) {
        // [32 keys][2][32 NB] floats in the tiles' place
        static_assert(2 * RT * L::kStride >= 32 * 2 * 32 * NB * 4, "the waves' sums need the tiles' room");
        float* sums = reinterpret_cast<float*>(tiles);
        for (int w = 0; w < kWaves; ++w) {
            __syncthreads();
            if (w != wave) continue;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float* x = sums + col * (64 * NB) + 32 * n + 8 * (r / 4) + 4 * half + r % 4;
                    const float k0 = w ? x[0] : 0.0f, v0 = w ? x[32 * NB] : 0.0f;
                    x[0] = k0 + dk[n][r] * by;
                    x[32 * NB] = v0 + dv[n][r] * unlift;
                }
        }
        __syncthreads();
        if (far) {
            float* part = f.far_parts + (((static_cast<int64_t>(chunk) * a.batch + b) * a.groups + g) * far_keys + wave_key) * 2 * a.width;
            for (int i = threadIdx.x; i < 64 * a.width; i += kThreads) {
                const int line = i / a.width;
                part[i] = sums[line * 32 * NB + i - line * a.width];
            }
            return;
        }
        const float* part = f.far_parts + ((static_cast<int64_t>(b) * a.groups + g) * far_keys + key0) * 2 * a.width;
        for (int i = threadIdx.x; i < 64 * (8 * NB); i += kThreads) {  // four columns of a key's dk or dv each
            const int line = i / (8 * NB), e = i % (8 * NB) * 4, at = key0 + line / 2;
            T* out = static_cast<T*>(line % 2 ? f.dv : f.dk);
            if (at >= a.total || e >= a.width || !out) continue;
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = sums[line * 32 * NB + e + j] + (key0 < far_keys ? part[line * a.width + e + j] : 0.0f);
            store_four(out + ((static_cast<int64_t>(b) * a.total + at) * a.groups + g) * a.width, e, a.width, x);
        }
        return;
    }
    if (key >= a.total) return;
    const float* part = f.far_parts + (((static_cast<int64_t>(b) * a.groups + g) * far_keys + key) * 2) * a.width;
    const int64_t cell = ((static_cast<int64_t>(b) * a.total + key) * a.groups + g) * a.width;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int qd = 0; qd < 4; ++qd) {
            const int e = 32 * n + 8 * qd + 4 * half;
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = dk[n][4 * qd + i] * by, y[i] = dv[n][4 * qd + i] * unlift;
            if (key < far_keys && e < a.width) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += part[e + i], y[i] += part[a.width + e + i];
            }
            if (f.dk) store_four(static_cast<T*>(f.dk) + cell, e, a.width, x);
            if (f.dv) store_four(static_cast<T*>(f.dv) + cell, e, a.width, y);
        }
}

// The chunks' sums of the sinks' keys, added in order into the first chunk's.
__global__ __launch_bounds__(kThreads) void window_far_kernel(float* parts, int chunks, int64_t each) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= each) return;
    float sum = parts[i];
#pragma unroll 8
    for (int p = 1; p < chunks; ++p) sum += parts[p * each + i];
    parts[i] = sum;
}

// The sinks' rows past their window, in chunks: two workgroups for each compute unit where
// the rows suffice, none under two tiles of 128.
void far_of(const Shape& s, Backward& f) {
    const int64_t before = s.total - s.length, first = std::max<int64_t>(s.window - before, 0);
    if (s.sinks == 0 || first >= s.length) return;
    f.far_tiles = (s.sinks + 31) / 32;
    f.far_first = static_cast<int>(first);
    const int64_t span = (s.length - first) * s.shared, heads = static_cast<int64_t>(s.batch) * s.groups * f.far_tiles;
    f.far_chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((span + 255) / 256, (512 + heads - 1) / heads)));
}

int64_t far_each(const Shape& s, const Backward& f) {
    return static_cast<int64_t>(s.batch) * s.groups * f.far_tiles * 32 * 2 * s.width;
}
size_t far_values(const Shape& s, const Backward& f) { return static_cast<size_t>(f.far_chunks) * far_each(s, f); }


template <typename T, int NB>
int run(const Backward& f, hipStream_t stream) {
    const int64_t heads = static_cast<int64_t>(f.s.batch) * f.s.groups;
    const char* what = "koemi_window_attention_backward";
    int rc = KOEMI_OK;
    if (f.row_tiles) {
        hipLaunchKernelGGL((window_dq_kernel<T, NB>), dim3(static_cast<unsigned>(heads * f.row_tiles)), dim3(kThreads), 0, stream, f);
        rc = check_launch(what);
    }
    if (rc != KOEMI_OK || (!f.dk && !f.dv)) return rc;
    if (f.far_chunks) {
        hipLaunchKernelGGL((window_dkv_kernel<T, NB, true>), dim3(static_cast<unsigned>(heads * f.far_tiles * f.far_chunks)),
                           dim3(kThreads), 0, stream, f, 1);
        rc = check_launch(what);
        if (rc != KOEMI_OK) return rc;
        if (f.far_chunks > 1) {
            const int64_t each = far_each(f.s, f);
            hipLaunchKernelGGL(window_far_kernel, dim3(grid_for(each, kThreads)), dim3(kThreads), 0, stream, f.far_parts, f.far_chunks, each);
            rc = check_launch(what);
            if (rc != KOEMI_OK) return rc;
        }
    }
    // Shared keys cost about 1.5 times the work on a full chip ([1, 16384], 256 wide workgroups: 1598 us against 1063)
    // and spread it where the wide ones leave compute units idle (70 of them at [5, 777]: 35.5 us against 52.5; 24 at
    // [2, 1500] in fp32: 80 against 256).
    const int64_t wide = heads * ((f.s.total + kRows - 1) / kRows);
    if (wide < 160)
        hipLaunchKernelGGL((window_dkv_kernel<T, NB, true>), dim3(static_cast<unsigned>(heads * ((f.s.total + 31) / 32))),
                           dim3(kThreads), 0, stream, f, 0);
    else
        hipLaunchKernelGGL((window_dkv_kernel<T, NB, false>), dim3(static_cast<unsigned>(wide)), dim3(kThreads), 0, stream, f, 0);
    return check_launch(what);
}

template <typename T>
int by_width(const Backward& f, hipStream_t stream) {
    const int nb = (f.s.width + 31) / 32;
    if (nb <= 1) return run<T, 1>(f, stream);
    if (nb <= 2) return run<T, 2>(f, stream);
    if (nb <= 3) return run<T, 3>(f, stream);
    if (nb <= 4) return run<T, 4>(f, stream);
    if (nb <= 6) return run<T, 6>(f, stream);
    return run<T, 8>(f, stream);
}

}  // namespace
}  // namespace window_attention
}  // namespace koemi

using namespace koemi;
using namespace koemi::window_attention;

extern "C" size_t koemi_window_attention_backward_workspace_bytes(int64_t batch, int64_t length, int64_t total, int64_t heads,
                                                                  int64_t groups, int64_t width, int64_t window, int64_t sinks,
                                                                  int dtype) {
    Backward f{};
    if (shape_of("koemi_window_attention_backward_workspace_bytes", nullptr, nullptr, nullptr, nullptr, nullptr, 0, length, total,
                 heads, groups, width, window, sinks, 1.0f, dtype, f.s) != KOEMI_OK || batch < 1) {
        clear_error();
        return 0;
    }
    f.s.batch = static_cast<int>(batch);
    far_of(f.s, f);
    return (static_cast<size_t>(batch) * heads * length + far_values(f.s, f)) * 4;
}

extern "C" int koemi_window_attention_backward(const void* queries, const void* keys, const void* values, const uint8_t* valid,
                                               const int64_t* strides, const void* output, const void* rest, const float* lse,
                                               const void* grad_output, void* grad_queries, void* grad_keys, void* grad_values,
                                               int64_t batch, int64_t length, int64_t total, int64_t heads, int64_t groups,
                                               int64_t width, int64_t window, int64_t sinks, float scale, int dtype,
                                               void* workspace, size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_window_attention_backward";
    Backward f{};
    const int rc = shape_of(what, queries, keys, values, valid, strides, batch, length, total, heads, groups, width, window, sinks,
                            scale, dtype, f.s);
    if (rc != KOEMI_OK || batch == 0 || total == 0) return rc;
    if (length && (!output || !lse || !grad_output)) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    f.out = output, f.rest = dtype == KOEMI_F32 ? nullptr : rest, f.lse = lse, f.d_out = grad_output, f.dq = grad_queries, f.dk = grad_keys, f.dv = grad_values;
    f.row_tiles = static_cast<int>((length * f.s.shared + kRows - 1) / kRows);
    far_of(f.s, f);
    if (batch * groups * f.far_tiles * f.far_chunks >= (int64_t(1) << 32) / kThreads)
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: too many sinks for gradients: a launch has fewer than 2^32 threads", what);
    const size_t cells = static_cast<size_t>(batch) * heads * length;
    const size_t need = (cells + far_values(f.s, f)) * 4;
    if (need && (!workspace || workspace_bytes < need)) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    f.delta = static_cast<float*>(workspace);
    f.far_parts = f.delta + cells;
    if (dtype == KOEMI_F32) return by_width<float>(f, as_stream(stream));
    if (dtype == KOEMI_F16) return by_width<f16>(f, as_stream(stream));
    return by_width<bf16>(f, as_stream(stream));
}
