// The next id of every row: temperature, top-k, top-p and min-p, and a draw from a given
// uniform number.
//
//   w_j = exp((z_j - max z) / T), of the ids with a score (not excluded, not -inf, not NaN)
//   top-k: z_j at least the k-th largest;  top-p: the w of all better scores, among those,
//   below p of their sum;  min-p: w_j >= m.  Equal scores stay together.
//   id = the first j whose running sum of the kept w exceeds u times the whole
//
// Sums decide ids, so they do not depend on an order: weights are formed in 64 bits and
// added as whole multiples of 2^-44 (a weight below 2^-45 of the largest is never drawn).
// A workgroup owns a row and walks it in tiles of 512 (a wave each): the maximum; a
// histogram of counts and weights over 2048 steps of (max - z) / T; the step that a
// limit falls into, whose scores are then ranked by their bits, eight at a time, from a list
// in LDS (or from the row where they are too many); the tiles' kept weights; the tile that
// u falls into. A row stays in its XCD's L2 between the walks. Few long rows are walked by
// several workgroups each, one launch a phase; a row of one tile stays in a wave's registers.
// Bound by the two passes of exponentials: 128 rows of 131072 bf16 scores with top-p and min-p
// take 7 us for the maximum, 26 the histogram, 9 + 13 + 10 the limit, 20 the kept weights, 6 the pick;
// one read of the scores takes 7.
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace koemi {
namespace {

constexpr int kBins = 2048;        // steps of the histogram
constexpr int kList = 4096;        // scores of one step that LDS holds
constexpr int kTile = 512;         // scores of a wave and step: eight a lane
constexpr int64_t kMaxVocab = 1 << 19;  // 2^44 x 2^19 fits 64 bits
constexpr double kLog2eD = 1.4426950408889634074;

struct Draw {
    const void* logits;
    int64_t row_stride, exclude;
    const float* uniforms;
    int64_t* ids;
    float* probabilities;  // [rows, vocab] or null
    double slope;          // log2(e) / temperature
    double top_p, min_p;
    int64_t top_k;         // 0: none
    int vocab, vector;
};

// 2^x for x <= 0 by the Taylor series of 2^f, |f| <= 1/2, to the 12th power (the 13th adds
// below 2^-52).
__device__ __forceinline__ double pow2(double x) {
    const double n = __builtin_rint(x), f = (x - n) * 0.69314718055994530942;
    double p = 1.0 / 479001600.0;
    p = fma(p, f, 1.0 / 39916800.0);
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}

// The same from 2^(i / 32), i < 32: the series of 2^(f / 32) to the 5th power (the 6th adds below
// 2^-48). Fourteen 64-bit operations a weight instead of twenty-one.
constexpr int kTable = 32;
__device__ __forceinline__ double pow2(double x, const double* table) {
    constexpr double c = 0.69314718055994530942 / kTable;
    const double y = x * kTable, n = __builtin_rint(y), f = y - n;
    const int i = static_cast<int>(n);
    double p = c * c * c * c * c / 120.0;
    p = fma(p, f, c * c * c * c / 24.0);
    p = fma(p, f, c * c * c / 6.0);
    p = fma(p, f, c * c / 2.0);
    p = fma(p, f, c);
    p = fma(p, f, 1.0);
    return ldexp(p * table[i & (kTable - 1)], i >> 5);
}

// A row's scores, in tiles.
template <typename T>
struct Row {
    const T* z;
    int vocab, exclude;
    bool vector, infinite;  // infinite: the largest is +inf, and only such ones count
    double top, slope;
    const double* table;    // 2^(i / 32), or null

    static constexpr int kWords = static_cast<int>(sizeof(T)) / 2;  // of 16 bytes, for eight scores

    // Scores as they count: -inf where there is none, zeros of one sign.
    __device__ __forceinline__ void clean(int j, float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = x[i] != x[i] || j + i == exclude ? -INFINITY : x[i] + 0.0f;
            if (infinite) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        }
    }
    // Scores j .. j + 7.
    __device__ __forceinline__ void load(int j, float (&x)[8]) const {
        alignas(16) T e[8];
        if (vector && j + 8 <= vocab) {
#pragma unroll
            for (int h = 0; h < kWords; ++h) reinterpret_cast<uint4*>(e)[h] = reinterpret_cast<const uint4*>(z + j)[h];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = j + i < vocab ? to_f32(z[j + i]) : -INFINITY;
        }
        clean(j, x);
    }
    // take(tile, a lane's eight scores) for tiles first, first + step .. below last. Tiles loaded
    // ahead gain nothing: the exponentials bound the walks, not the loads.
    template <typename Take>
    __device__ __forceinline__ void walk(int first, int last, int step, Take take) const {
#pragma unroll 1
        for (int t = first; t < last; t += step) {
            float x[8];
            load(t * kTile + lane_id() * 8, x);
            take(t, x);
        }
    }
    __device__ __forceinline__ double weight(float x) const {
        const double e = (static_cast<double>(x) - top) * slope;
        return e > -100.0 ? (table ? pow2(e, table) : pow2(e)) : 0.0;
    }
    // w in steps of 2^-44, 0 <= w <= 1: the last bits of 2^52 plus it.
    static __device__ __forceinline__ uint64_t whole(double w) {
        return __builtin_bit_cast(uint64_t, fma(w, 17592186044416.0, 4503599627370496.0)) & 0xfffffffffffffull;
    }
    // The histogram's step: falls with the score, never rises.
    __device__ __forceinline__ int bin(float x) const {
        const float e = (static_cast<float>(top) - x) * (static_cast<float>(slope) * (kBins / 64.0f));
        return e < static_cast<float>(kBins - 1) ? static_cast<int>(e) : kBins - 1;
    }
};

// Bits whose order as whole numbers is the scores', and back.
__device__ __forceinline__ uint32_t rank_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ (u >> 31 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t r) { return __uint_as_float(r ^ (r >> 31 ? 0x80000000u : ~0u)); }

template <int THREADS>
struct Shared {
    uint64_t mass[kBins];
    double table[kTable];
    uint32_t count[kBins];
    uint32_t list[kList];
    float gathered[THREADS / kWave][kTile];
    uint64_t scan[THREADS / kWave];
    float wave_top[THREADS / kWave];
    uint64_t before;
    int found, listed;
};

// The first of n entries, in the order of `at`, at which the running sum of value(at)
// reaches target, and the sum before it. THREADS threads; n a multiple of them or below.
template <int THREADS, typename Value>
__device__ __forceinline__ int reach(Shared<THREADS>& sh, int n, Value value, double target, uint64_t base, uint64_t& before) {
    const int per = (n + THREADS - 1) / THREADS, first = static_cast<int>(threadIdx.x) * per;
    uint64_t own = 0;
    for (int i = first; i < min(first + per, n); ++i) own += value(i);
    uint64_t total;
    uint64_t run = base + block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, total);
    if (threadIdx.x == 0) sh.found = n - 1, sh.before = 0;
    __syncthreads();
    if (own && static_cast<double>(run) < target && !(static_cast<double>(run + own) < target)) {
        for (int i = first; i < min(first + per, n); ++i) {
            const uint64_t v = value(i);
            if (!(static_cast<double>(run + v) < target)) {
                sh.found = i, sh.before = run;
                break;
            }
            run += v;
        }
    }
    __syncthreads();
    const int found = sh.found;
    before = sh.before;
    __syncthreads();
    return found;
}

// take(score) for every score of a step among tiles first .. last - 1.
template <int THREADS, typename T, typename Take>
__device__ __forceinline__ void of_step(const Row<T>& row, int bin, int first, int last, Take take) {
    row.walk(first + static_cast<int>(threadIdx.x) / kWave, last, THREADS / kWave, [&](int, const float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (x[i] != -INFINITY && row.bin(x[i]) == bin) take(x[i]);
    });
}

// The step in which the running sum (of ones, or of weights) over falling scores reaches
// target, and the sum before it.
template <int THREADS, bool MASS>
__device__ __forceinline__ int step_of(Shared<THREADS>& sh, double target, uint64_t& before) {
    return reach<THREADS>(sh, kBins, [&](int i) { return MASS ? sh.mass[i] : static_cast<uint64_t>(sh.count[i]); }, target, 0, before);
}

// The ranks of a step's scores among tiles first .. last - 1 into the list, as many as fit; how many there are.
template <int THREADS, typename T>
__device__ __forceinline__ int list_step(const Row<T>& row, Shared<THREADS>& sh, int bin, int first, int last) {
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    of_step<THREADS>(row, bin, first, last, [&](float x) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < kList) sh.list[at] = rank_of(x);
    });
    __syncthreads();
    return sh.listed;
}

// The score of a step at which that sum reaches target; `many` scores, from the list where it holds them all.
template <int THREADS, bool MASS, typename T>
__device__ float score_in(const Row<T>& row, Shared<THREADS>& sh, int bin, int many, double target, uint64_t before) {
    __shared__ unsigned long long digits[256];
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += THREADS) digits[i] = 0;
        __syncthreads();
        auto add = [&](uint32_t r) {
            if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8))
                atomicAdd(&digits[255 - ((r >> shift) & 255)], MASS ? Row<T>::whole(row.weight(score_of(r))) : 1ull);
        };
        if (many <= kList) {
            for (int i = threadIdx.x; i < many; i += THREADS) add(sh.list[i]);
        } else {
            of_step<THREADS>(row, bin, 0, (row.vocab + kTile - 1) / kTile, [&](float x) { add(rank_of(x)); });
        }
        __syncthreads();
        const int digit = reach<THREADS>(sh, 256, [&](int i) { return static_cast<uint64_t>(digits[i]); }, target, before, before);
        prefix |= static_cast<uint32_t>(255 - digit) << shift;
    }
    return score_of(prefix);
}

// What the phases of a row share: the largest score found, the limits, the kept weights.
template <int THREADS, typename T>
struct Phases {
    static constexpr int kWaves = THREADS / kWave;
    const Draw& f;
    Shared<THREADS>& sh;
    Row<T> row;
    int64_t r;
    int tiles, lane, wave;
    bool none, by_k, by_p;

    __device__ __forceinline__ Phases(const Draw& draw, Shared<THREADS>& shared, int64_t index)
        : f(draw), sh(shared),
          row{static_cast<const T*>(draw.logits) + index * draw.row_stride, draw.vocab, static_cast<int>(draw.exclude), draw.vector != 0, false, 0.0, draw.slope, shared.table},
          r(index), tiles((draw.vocab + kTile - 1) / kTile), lane(lane_id()), wave(static_cast<int>(threadIdx.x) / kWave) {
        if (threadIdx.x < kTable) sh.table[threadIdx.x] = pow2(-1.0 + threadIdx.x / static_cast<double>(kTable)) * 2.0;
        __syncthreads();
    }

    // The largest of tiles first .. last - 1, in every thread.
    __device__ __forceinline__ float largest(int first, int last) {
        float top = -INFINITY;
        row.walk(first + wave, last, kWaves, [&](int, const float (&x)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
        });
        top = wave_max_xor(top);
        if (lane == 0) sh.wave_top[wave] = top;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sh.wave_top[w]);
        return top;
    }
    __device__ __forceinline__ void begin(float top) {
        row.infinite = top == INFINITY;
        row.top = row.infinite ? 0.0 : static_cast<double>(top);
        none = top == -INFINITY;
        by_k = !none && f.top_k > 0 && f.top_k < f.vocab, by_p = !none && f.top_p < 1.0;
    }
    __device__ __forceinline__ void histogram(int first, int last) {
        for (int i = threadIdx.x; i < kBins; i += THREADS) sh.mass[i] = 0, sh.count[i] = 0;
        __syncthreads();
        row.walk(first + wave, last, kWaves, [&](int, const float (&x)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (x[i] != -INFINITY) {
                    const int b = row.bin(x[i]);
                    if (by_k) atomicAdd(&sh.count[b], 1u);
                    if (by_p) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[b]), static_cast<unsigned long long>(Row<T>::whole(row.weight(x[i]))));
                }
        });
        __syncthreads();
    }
    // Scores counted in the whole row's histogram.
    __device__ __forceinline__ uint64_t available() {
        uint64_t own = 0, all;
        for (int i = threadIdx.x; i < kBins; i += THREADS) own += sh.count[i];
        block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, all);
        return all;
    }
    // The weight of all scores from the limit `at` up, which lies in step `edge` (kBins: no limit); `many`
    // of that step are listed.
    __device__ __forceinline__ uint64_t mass_from(float at, int edge, int many) {
        uint64_t own = 0, total;
        for (int i = threadIdx.x; i < edge; i += THREADS) own += sh.mass[i];
        auto add = [&](float x) {
            if (x >= at) own += Row<T>::whole(row.weight(x));
        };
        if (edge < kBins && many <= kList) {
            for (int i = threadIdx.x; i < many; i += THREADS) add(score_of(sh.list[i]));
        } else if (edge < kBins) {
            of_step<THREADS>(row, edge, 0, tiles, add);
        }
        block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, total);
        return total;
    }
    // The least kept score by top-k and top-p, from the whole row's histogram.
    __device__ __forceinline__ float least() {
        float at = -INFINITY;
        int edge = kBins, many = 0;
        uint64_t before;
        if (by_k && static_cast<uint64_t>(f.top_k) < available()) {
            const double target = static_cast<double>(f.top_k);
            edge = step_of<THREADS, false>(sh, target, before);
            many = list_step<THREADS>(row, sh, edge, 0, tiles);
            at = score_in<THREADS, false>(row, sh, edge, many, target, before);
        }
        if (by_p) {
            const double target = f.top_p * static_cast<double>(mass_from(at, edge, many));
            const int step = step_of<THREADS, true>(sh, target, before);
            if (step != edge) many = list_step<THREADS>(row, sh, step, 0, tiles);
            at = fmaxf(at, score_in<THREADS, true>(row, sh, step, many, target, before));
        }
        return at;
    }
    __device__ __forceinline__ double kept(float x, float least) const {
        if (x == -INFINITY || x < least) return 0.0;
        const double w = row.weight(x);
        return w >= f.min_p ? w : 0.0;
    }
    // The kept weight of tiles first .. last - 1, to `sums`: a wave first gathers its tile's kept
    // scores, often few, so that their exponentials fill its lanes.
    __device__ __forceinline__ void tile_sums(int first, int last, float least, uint64_t* sums) {
        row.walk(first + wave, last, kWaves, [&](int t, const float (&x)[8]) {
            uint64_t sum = 0;
            int count = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = x[i] != -INFINITY && x[i] >= least;
                const uint64_t mask = __ballot(in);
                if (in) sh.gathered[wave][count + __popcll(mask & lanemask_lt())] = x[i];
                count += __popcll(mask);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int i = lane; i < count; i += kWave) sum += Row<T>::whole(kept(sh.gathered[wave][i], least));
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
            if (lane == 0) sums[t] = sum;
        });
    }
    __device__ __forceinline__ uint64_t whole_sum(const uint64_t* sums) {
        uint64_t own = 0, total;
        for (int t = threadIdx.x; t < tiles; t += THREADS) own += sums[t];
        block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, total);
        return total;
    }
    __device__ __forceinline__ void distribution(int first, int last, float least, uint64_t total) {
        const double share = total ? 17592186044416.0 / static_cast<double>(total) : 0.0;
        float* out = f.probabilities + r * f.vocab;
        row.walk(first + wave, last, kWaves, [&](int t, const float (&x)[8]) {
            const int j = t * kTile + lane * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < f.vocab) out[j + i] = static_cast<float>(kept(x[i], least) * share);
        });
    }
    // The first running sum beyond u of the whole; sums are whole, so beyond it means not below the next double.
    __device__ __forceinline__ void pick(float least, const uint64_t* sums, uint64_t total) {
        const float u = f.uniforms[r];
        const double target = static_cast<double>(u > 0.0f ? fminf(u, 0.999999940395355f) : 0.0f) * static_cast<double>(total);
        uint64_t before;
        const int tile = reach<THREADS>(sh, tiles, [&](int i) { return sums[i]; }, nextafter(target, 1e300), 0, before);
        if (wave) return;
        float x[8];
        const int j = tile * kTile + lane * 8;
        row.load(j, x);
        uint64_t w[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = Row<T>::whole(kept(x[i], least)), sum += w[i];
        uint64_t incl = sum;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const uint64_t up = __shfl_up(incl, off, kWave);
            if (lane >= off) incl += up;
        }
        uint64_t run = before + incl - sum;
        int id = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            run += w[i];
            if (id < 0 && static_cast<double>(run) > target) id = j + i;
        }
        const uint64_t hit = __ballot(id >= 0);
        const int chosen = hit ? __shfl(id, __ffsll(static_cast<unsigned long long>(hit)) - 1, kWave) : 0;
        if (lane == 0) f.ids[r] = none ? 0 : chosen;
    }
};

// A row in one workgroup.
template <int THREADS, typename T>
__global__ __launch_bounds__(THREADS) void sample_filtered_kernel(Draw f) {
    __shared__ Shared<THREADS> sh;
    Phases<THREADS, T> p(f, sh, blockIdx.x);
    p.begin(p.largest(0, p.tiles));
    float least = -INFINITY;
    if (p.by_k || p.by_p) {
        p.histogram(0, p.tiles);
        least = p.least();
    }
    __syncthreads();
    p.tile_sums(0, p.tiles, least, sh.mass);  // in the histogram's place
    __syncthreads();
    const uint64_t total = p.whole_sum(sh.mass);
    if (f.probabilities) p.distribution(0, p.tiles, least, total);
    p.pick(least, sh.mass, total);
}

// The limit that a row looks for: the running sum (of weights, or of ones) that reaches target in step
// `bin` (-1: none), of which `listed` scores were found.
struct Limit {
    double target;
    uint64_t before;
    int bin, listed, mass;
};

// A long row in several workgroups, a launch for each phase. `parts` of a row's tiles each.
struct Parted {
    Draw f;
    int parts;
    float* tops;      // [rows, parts]
    float* least;     // [rows]: of the limits found so far
    Limit* limits;    // [rows]
    uint32_t* list;   // [rows, kList]: ranks of a step's scores
    uint64_t* total;  // [rows]
    uint64_t* mass;   // [rows, parts, kBins]
    uint32_t* count;  // [rows, parts, kBins]
    uint64_t* sums;   // [rows, tiles]
};
constexpr int kPartThreads = 1024;  // of a part; a row's own steps are chains of barriers, cheaper among four waves
constexpr int kRowThreads = 256;

template <int THREADS, typename T>
__device__ __forceinline__ void begin_part(Phases<THREADS, T>& p, const Parted& d) {
    float top = -INFINITY;
    for (int i = 0; i < d.parts; ++i) top = fmaxf(top, d.tops[p.r * d.parts + i]);
    p.begin(top);
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_top_kernel(Parted d) {
    __shared__ Shared<kPartThreads> sh;
    Phases<kPartThreads, T> p(d.f, sh, blockIdx.x / d.parts);
    const int part = static_cast<int>(blockIdx.x % d.parts);
    const float top = p.largest(p.tiles * part / d.parts, p.tiles * (part + 1) / d.parts);
    if (threadIdx.x == 0) d.tops[blockIdx.x] = top;
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_histogram_kernel(Parted d) {
    __shared__ Shared<kPartThreads> sh;
    Phases<kPartThreads, T> p(d.f, sh, blockIdx.x / d.parts);
    const int part = static_cast<int>(blockIdx.x % d.parts);
    begin_part(p, d);
    p.histogram(p.tiles * part / d.parts, p.tiles * (part + 1) / d.parts);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kBins;
    for (int i = threadIdx.x; i < kBins; i += kPartThreads) {
        if (p.by_p) d.mass[at + i] = sh.mass[i];
        if (p.by_k) d.count[at + i] = sh.count[i];
    }
}

// The parts' histograms added into the first one's, and the step of the first limit.
template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_step_kernel(Parted d) {
    __shared__ Shared<kPartThreads> sh;
    Phases<kPartThreads, T> p(d.f, sh, blockIdx.x);
    begin_part(p, d);
    for (int i = threadIdx.x; i < kBins; i += kPartThreads) {
        const int64_t first = p.r * d.parts * kBins + i;
        uint64_t mass = 0;
        uint32_t count = 0;
#pragma unroll 4
        for (int part = 0; part < d.parts; ++part) {
            if (p.by_p) mass += d.mass[first + static_cast<int64_t>(part) * kBins];
            if (p.by_k) count += d.count[first + static_cast<int64_t>(part) * kBins];
        }
        sh.mass[i] = mass, sh.count[i] = count;
        if (p.by_p) d.mass[first] = mass;
    }
    __syncthreads();
    Limit limit{0.0, 0, -1, 0, 0};
    if (p.by_k && static_cast<uint64_t>(d.f.top_k) < p.available()) {
        limit.target = static_cast<double>(d.f.top_k);
        limit.bin = step_of<kPartThreads, false>(sh, limit.target, limit.before);
    } else if (p.by_p) {
        limit.mass = 1;
        limit.target = d.f.top_p * static_cast<double>(p.mass_from(-INFINITY, kBins, 0));
        limit.bin = step_of<kPartThreads, true>(sh, limit.target, limit.before);
    }
    if (threadIdx.x == 0) d.limits[p.r] = limit, d.least[p.r] = -INFINITY;
}

// That step's scores, in any order: what is summed of them is whole.
template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_list_kernel(Parted d) {
    __shared__ Shared<kPartThreads> sh;
    __shared__ int base;
    Phases<kPartThreads, T> p(d.f, sh, blockIdx.x / d.parts);
    const int part = static_cast<int>(blockIdx.x % d.parts);
    Limit& limit = d.limits[p.r];
    if (limit.bin < 0) return;
    begin_part(p, d);
    const int many = list_step<kPartThreads>(p.row, sh, limit.bin, p.tiles * part / d.parts, p.tiles * (part + 1) / d.parts);
    if (threadIdx.x == 0) base = many ? atomicAdd(&limit.listed, many) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < min(many, kList) && base + i < kList; i += kPartThreads) d.list[p.r * kList + base + i] = sh.list[i];
}

// The limit among them; after top-k's, top-p's or the step of it, if that is another one.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_limit_kernel(Parted d) {
    __shared__ Shared<kRowThreads> sh;
    Phases<kRowThreads, T> p(d.f, sh, blockIdx.x);
    Limit limit = d.limits[p.r];
    if (limit.bin < 0) return;
    begin_part(p, d);
    const int many = limit.listed;
    if (many <= kList)
        for (int i = threadIdx.x; i < many; i += kRowThreads) sh.list[i] = d.list[p.r * kList + i];
    const bool then = !limit.mass && p.by_p;
    if (then)
        for (int i = threadIdx.x; i < kBins; i += kRowThreads) sh.mass[i] = d.mass[p.r * d.parts * kBins + i];
    __syncthreads();
    float at = limit.mass ? score_in<kRowThreads, true>(p.row, sh, limit.bin, many, limit.target, limit.before)
                          : score_in<kRowThreads, false>(p.row, sh, limit.bin, many, limit.target, limit.before);
    Limit next{0.0, 0, -1, 0, 1};
    if (then) {
        next.target = d.f.top_p * static_cast<double>(p.mass_from(at, limit.bin, many));
        next.bin = step_of<kRowThreads, true>(sh, next.target, next.before);
        if (next.bin == limit.bin) {
            at = fmaxf(at, score_in<kRowThreads, true>(p.row, sh, next.bin, many, next.target, next.before));
            next.bin = -1;
        }
    }
    if (threadIdx.x == 0) d.limits[p.r] = next, d.least[p.r] = fmaxf(d.least[p.r], at);
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_kept_kernel(Parted d) {
    __shared__ Shared<kPartThreads> sh;
    Phases<kPartThreads, T> p(d.f, sh, blockIdx.x / d.parts);
    const int part = static_cast<int>(blockIdx.x % d.parts);
    begin_part(p, d);
    const float least = p.by_k || p.by_p ? d.least[p.r] : -INFINITY;
    p.tile_sums(p.tiles * part / d.parts, p.tiles * (part + 1) / d.parts, least, d.sums + p.r * p.tiles);
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_pick_kernel(Parted d) {
    __shared__ Shared<kRowThreads> sh;
    Phases<kRowThreads, T> p(d.f, sh, blockIdx.x);
    begin_part(p, d);
    const float least = p.by_k || p.by_p ? d.least[p.r] : -INFINITY;
    const uint64_t* sums = d.sums + p.r * p.tiles;
    const uint64_t total = p.whole_sum(sums);
    if (threadIdx.x == 0) d.total[p.r] = total;
    p.pick(least, sums, total);
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_distribution_kernel(Parted d) {
    __shared__ Shared<kPartThreads> sh;
    Phases<kPartThreads, T> p(d.f, sh, blockIdx.x / d.parts);
    const int part = static_cast<int>(blockIdx.x % d.parts);
    begin_part(p, d);
    const float least = p.by_k || p.by_p ? d.least[p.r] : -INFINITY;
    p.distribution(p.tiles * part / d.parts, p.tiles * (part + 1) / d.parts, least, d.total[p.r]);
}

// Over a wave's 64 lanes, the result in each: neighbours, quads, half rows and rows by
// data-parallel moves, then the rows of sixteen and the halves.
template <typename V, typename Op>
__device__ __forceinline__ V over_wave(V x, Op op) {
    constexpr int N = sizeof(V) / 4;
    struct Words {
        int w[N];
    };
    auto step = [&](auto move) {
        Words a = __builtin_bit_cast(Words, x);
#pragma unroll
        for (int i = 0; i < N; ++i) a.w[i] = move(a.w[i]);
        x = op(x, __builtin_bit_cast(V, a));
    };
    step([](int w) { return __builtin_amdgcn_update_dpp(0, w, 0xb1, 0xf, 0xf, true); });   // lane ^ 1
    step([](int w) { return __builtin_amdgcn_update_dpp(0, w, 0x4e, 0xf, 0xf, true); });   // lane ^ 2
    step([](int w) { return __builtin_amdgcn_update_dpp(0, w, 0x141, 0xf, 0xf, true); });  // 7 - lane in eight
    step([](int w) { return __builtin_amdgcn_update_dpp(0, w, 0x140, 0xf, 0xf, true); });  // 15 - lane in sixteen
    auto halves = [&](auto swap) {
        const Words a = __builtin_bit_cast(Words, x);
        Words lo, hi;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const auto both = swap(static_cast<uint32_t>(a.w[i]));
            lo.w[i] = static_cast<int>(both[0]), hi.w[i] = static_cast<int>(both[1]);
        }
        x = op(__builtin_bit_cast(V, lo), __builtin_bit_cast(V, hi));
    };
    halves([](uint32_t w) { return __builtin_amdgcn_permlane16_swap(w, w, false, false); });
    halves([](uint32_t w) { return __builtin_amdgcn_permlane32_swap(w, w, false, false); });
    return x;
}

// Rows of one tile: a wave holds all scores, and finds the limits bit by bit from how many
// scores, or what weight, lie at or above a candidate, until only one score lies between what
// is known to be kept and what is not. 2^44 x 512 = 2^53: sums of whole weights are exact in double.
template <typename T>
__global__ __launch_bounds__(kWave) void sample_narrow_kernel(Draw f) {
    const int lane = lane_id(), j = lane * 8;
    const int64_t r = blockIdx.x;
    Row<T> row{static_cast<const T*>(f.logits) + r * f.row_stride, f.vocab, static_cast<int>(f.exclude), f.vector != 0, false, 0.0, f.slope, nullptr};
    const float u = f.uniforms[r];
    float x[8], top = -INFINITY;
    row.load(j, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
    top = over_wave(top, [](float a, float b) { return fmaxf(a, b); });
    if (top == INFINITY) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        top = 0.0f;
    }
    row.top = static_cast<double>(top);
    const auto add = [](double a, double b) { return a + b; };
    uint32_t rank[8];
    double exact[8], w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool here = x[i] != -INFINITY;
        rank[i] = here ? rank_of(x[i]) : 0u;
        exact[i] = here ? row.weight(x[i]) : 0.0;
        w[i] = static_cast<double>(Row<T>::whole(exact[i]));
    }
    const auto at_least = [&](uint32_t candidate) {
        int count = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) count += __popcll(__ballot(rank[i] >= candidate));
        return count;
    };
    uint32_t least = 1;  // of the kept ranks; no score has rank 0
    if (f.top_k > 0 && f.top_k < f.vocab) {
        uint32_t at = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = at | 1u << bit;
            const int count = at_least(next);
            if (count >= f.top_k) at = next;
            if (count == f.top_k) break;  // the same scores lie at or above the k-th
        }
        least = max(at, 1u);
    }
    if (f.top_p < 1.0) {
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) total += rank[i] >= least ? w[i] : 0.0;
        const double target = f.top_p * over_wave(total, add);
        uint32_t at = 0;
        int above = 0, from = at_least(0);  // scores known to lie above the border, and at or above `at`
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = at | 1u << bit;
            double part[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) part[i] = rank[i] >= next ? w[i] : 0.0;
            const double sum = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
            const int count = at_least(next);
            if (!(over_wave(sum, add) < target))
                at = next, from = count;
            else
                above = count;
            if (from == above + 1) break;
        }
        least = max(least, at);
    }
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (rank[i] < least || !(exact[i] >= f.min_p)) exact[i] = w[i] = 0.0;
        own += w[i];
    }
    double run = own;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const double up = __shfl_up(run, off, kWave);
        if (lane >= off) run += up;
    }
    const double total = __shfl(run, kWave - 1, kWave);
    run -= own;
    if (f.probabilities) {
        const double share = total > 0.0 ? 17592186044416.0 / total : 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j + i < f.vocab) f.probabilities[r * f.vocab + j + i] = static_cast<float>(exact[i] * share);
    }
    const double target = static_cast<double>(u > 0.0f ? fminf(u, 0.999999940395355f) : 0.0f) * total;
    int id = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        run += w[i];
        if (id < 0 && run > target) id = j + i;
    }
    const uint64_t hit = __ballot(id >= 0);
    const int chosen = hit ? __shfl(id, __ffsll(static_cast<unsigned long long>(hit)) - 1, kWave) : 0;
    if (lane == 0) f.ids[r] = chosen;
}

// Workgroups of a row in the walks: one, or for at most 128 rows of 65536 scores and more so many
// that all rows have about 512, none under eight tiles. Seven launches instead of one, in us with
// top-p and min-p, parted against one workgroup a row: 8 x 131072 67 | 119, 128 x 131072 87 | 124,
// 64 x 65536 56 | 72, 128 x 65536 62 | 71, but 8 x 32768 42 | 45, 128 x 32768 52 | 46. Past 128 rows three parts (to
// 170 rows) would still gain, two (192 and more) no longer: 129 x 131072 98 | 126, 160 x 131072 99 | 129, 192 x 131072 127 | 129,
// 256 x 131072 130 | 130, 129 x 65536 66 | 73, 160 x 65536 67 | 75, 192 x 65536 83 | 75, 256 x 65536 83 | 71.
int parts_for(int64_t rows, int64_t vocab) {
    if (vocab < 65536 || rows > 128) return 1;
    const int64_t tiles = (vocab + kTile - 1) / kTile;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({64, tiles / 8, 512 / std::max<int64_t>(rows, 1)})));
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// The parted form's workspace from `base` on; returns its bytes.
size_t lay_out(Parted& d, char* base, int64_t rows, int64_t vocab) {
    const size_t tiles = (vocab + kTile - 1) / kTile, cells = static_cast<size_t>(rows) * d.parts;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* p = base + at;
        at += align256(bytes);
        return p;
    };
    d.total = reinterpret_cast<uint64_t*>(take(rows * 8));
    d.sums = reinterpret_cast<uint64_t*>(take(rows * tiles * 8));
    d.mass = reinterpret_cast<uint64_t*>(take(cells * kBins * 8));
    d.count = reinterpret_cast<uint32_t*>(take(cells * kBins * 4));
    d.tops = reinterpret_cast<float*>(take(cells * 4));
    d.least = reinterpret_cast<float*>(take(rows * 4));
    d.limits = reinterpret_cast<Limit*>(take(rows * sizeof(Limit)));
    d.list = reinterpret_cast<uint32_t*>(take(rows * kList * 4));
    return at;
}

// Threads of a row in one workgroup: a wave takes 512 scores a step, sixteen waves where a row has more than four such tiles.
int threads_for(int64_t vocab) { return vocab <= kTile ? kWave : vocab <= 2048 ? 256 : 1024; }

template <typename T>
int draw(const Draw& f, int64_t rows, void* workspace, hipStream_t stream) {
    const char* what = "koemi_sample_filtered";
    const unsigned grid = static_cast<unsigned>(rows);
    Parted d{};
    d.f = f;
    d.parts = parts_for(rows, f.vocab);
    if (d.parts == 1) {
        if (threads_for(f.vocab) == kWave)
            hipLaunchKernelGGL((sample_narrow_kernel<T>), dim3(grid), dim3(kWave), 0, stream, f);
        else if (threads_for(f.vocab) == 256)
            hipLaunchKernelGGL((sample_filtered_kernel<256, T>), dim3(grid), dim3(256), 0, stream, f);
        else
            hipLaunchKernelGGL((sample_filtered_kernel<1024, T>), dim3(grid), dim3(1024), 0, stream, f);
        return check_launch(what);
    }
    lay_out(d, static_cast<char*>(workspace), rows, f.vocab);
    const dim3 wide(static_cast<unsigned>(rows * d.parts)), threads(kPartThreads);
    hipLaunchKernelGGL((sample_top_kernel<T>), wide, threads, 0, stream, d);
    const int limits = (f.top_k > 0 && f.top_k < f.vocab) + (f.top_p < 1.0);
    if (limits) {
        hipLaunchKernelGGL((sample_histogram_kernel<T>), wide, threads, 0, stream, d);
        hipLaunchKernelGGL((sample_step_kernel<T>), dim3(grid), threads, 0, stream, d);
    }
    for (int i = 0; i < limits; ++i) {
        hipLaunchKernelGGL((sample_list_kernel<T>), wide, threads, 0, stream, d);
        hipLaunchKernelGGL((sample_limit_kernel<T>), dim3(grid), dim3(kRowThreads), 0, stream, d);
    }
    hipLaunchKernelGGL((sample_kept_kernel<T>), wide, threads, 0, stream, d);
    hipLaunchKernelGGL((sample_pick_kernel<T>), dim3(grid), dim3(kRowThreads), 0, stream, d);
    if (f.probabilities) hipLaunchKernelGGL((sample_distribution_kernel<T>), wide, threads, 0, stream, d);
    return check_launch(what);
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_sample_filtered_workspace_bytes(int64_t rows, int64_t vocab) {
    if (rows < 1 || vocab < 1 || vocab > kMaxVocab || rows > 0x7fffffff) return 0;
    Parted d{};
    d.parts = parts_for(rows, vocab);
    return d.parts == 1 ? 0 : lay_out(d, nullptr, rows, vocab);
}

extern "C" int koemi_sample_filtered(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab,
                                     int64_t exclude, double temperature, int64_t top_k, double top_p, double min_p,
                                     const float* uniforms, int64_t* ids, float* probabilities, void* workspace,
                                     size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_sample_filtered";
    if (rows < 0 || vocab < 1) return fail(KOEMI_ERR_INVALID, "%s: rows must not be negative and the vocabulary positive", what);
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16, not %s", what, dtype_name(dtype));
    if (vocab > kMaxVocab) return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^19 ids", what);
    if (rows >= (int64_t(1) << 32) / threads_for(vocab))
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: too many rows: a launch has fewer than 2^32 threads", what);
    if (!(temperature >= 1e-30 && temperature <= 1e30)) return fail(KOEMI_ERR_INVALID, "%s: temperature must be positive and finite", what);
    if (top_k < 0 || !(top_p > 0.0 && top_p <= 1.0) || !(min_p >= 0.0 && min_p <= 1.0))
        return fail(KOEMI_ERR_INVALID, "%s: top_k must not be negative, top_p above 0 and min_p from 0, both at most 1", what);
    if (row_stride == 0) row_stride = vocab;
    if (rows > 1 && row_stride < vocab) return fail(KOEMI_ERR_INVALID, "%s: row stride below the vocabulary", what);
    if (rows == 0) return KOEMI_OK;
    if (!logits || !uniforms || !ids) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    const int64_t size = dtype == KOEMI_F32 ? 4 : 2;
    Draw f{};
    f.logits = logits, f.row_stride = row_stride, f.exclude = exclude >= 0 && exclude < vocab ? exclude : -1;
    f.uniforms = uniforms, f.ids = ids, f.probabilities = probabilities;
    f.slope = kLog2eD / temperature, f.top_p = top_p, f.min_p = min_p, f.top_k = top_k, f.vocab = static_cast<int>(vocab);
    f.vector = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (rows == 1 || row_stride * size % 16 == 0);
    const size_t need = koemi_sample_filtered_workspace_bytes(rows, vocab);
    if (need && (!workspace || workspace_bytes < need)) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    if (dtype == KOEMI_F32) return draw<float>(f, rows, workspace, as_stream(stream));
    if (dtype == KOEMI_F16) return draw<f16>(f, rows, workspace, as_stream(stream));
    return draw<bf16>(f, rows, workspace, as_stream(stream));
}
