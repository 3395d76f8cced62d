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
// u falls into. A row stays in its XCD's L2 between the walks. Bound by the two passes of
// exponentials (about 25 64-bit operations a score).
#include "common.hpp"

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

// A row's scores, in tiles.
template <typename T>
struct Row {
    const T* z;
    int vocab, exclude;
    bool vector, infinite;  // infinite: the largest is +inf, and only such ones count
    double top, slope;

    // Scores 8 i .. 8 i + 7 of a tile's lane, -inf where there is none.
    __device__ __forceinline__ void load(int j, float (&x)[8]) const {
        alignas(16) T e[8];
        if (vector && j + 8 <= vocab) {
#pragma unroll
            for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
                reinterpret_cast<uint4*>(e)[h] = reinterpret_cast<const uint4*>(z + j)[h];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = j + i < vocab ? to_f32(z[j + i]) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = x[i] != x[i] || j + i == exclude ? -INFINITY : x[i] + 0.0f;  // no negative zero
            if (infinite) x[i] = x[i] == INFINITY ? 0.0f : -INFINITY;
        }
    }
    __device__ __forceinline__ double weight(float x) const {
        const double e = (static_cast<double>(x) - top) * slope;
        return e > -100.0 ? pow2(e) : 0.0;
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

// The score at which the running sum (of ones, or of weights) over falling scores
// reaches target.
template <int THREADS, bool MASS, typename T>
__device__ float limit(const Row<T>& row, Shared<THREADS>& sh, double target) {
    constexpr int kWaves = THREADS / kWave;
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    uint64_t before;
    const int bin = reach<THREADS>(sh, kBins, [&](int i) { return MASS ? sh.mass[i] : static_cast<uint64_t>(sh.count[i]); },
                                   target, 0, before);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    auto each = [&](auto take) {  // every score of the step
        for (int t = wave; t * kTile < row.vocab; t += kWaves) {
            float x[8];
            row.load(t * kTile + lane * 8, x);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (x[i] != -INFINITY && row.bin(x[i]) == bin) take(x[i]);
        }
    };
    each([&](float x) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < kList) sh.list[at] = rank_of(x);
    });
    __syncthreads();
    const int many = sh.listed;
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
            each([&](float x) { add(rank_of(x)); });
        }
        __syncthreads();
        const int digit = reach<THREADS>(sh, 256, [&](int i) { return static_cast<uint64_t>(digits[i]); }, target, before, before);
        prefix |= static_cast<uint32_t>(255 - digit) << shift;
    }
    return score_of(prefix);
}

template <int THREADS, typename T>
__global__ __launch_bounds__(THREADS) void sample_filtered_kernel(Draw f) {
    constexpr int kWaves = THREADS / kWave;
    __shared__ Shared<THREADS> sh;
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    const int64_t r = blockIdx.x;
    Row<T> row{static_cast<const T*>(f.logits) + r * f.row_stride, f.vocab, static_cast<int>(f.exclude), f.vector != 0, false, 0.0, f.slope};
    const int tiles = (f.vocab + kTile - 1) / kTile;
    float top = -INFINITY;
    for (int t = wave; t < tiles; t += kWaves) {
        float x[8];
        row.load(t * kTile + lane * 8, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
    }
    top = wave_max_xor(top);
    if (lane == 0) sh.wave_top[wave] = top;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sh.wave_top[w]);
    row.infinite = top == INFINITY;
    row.top = row.infinite ? 0.0 : static_cast<double>(top);
    const bool none = top == -INFINITY;
    const bool by_k = !none && f.top_k > 0 && f.top_k < f.vocab, by_p = !none && f.top_p < 1.0;
    float least = -INFINITY;  // of the kept scores
    if (by_k || by_p) {
        for (int i = threadIdx.x; i < kBins; i += THREADS) sh.mass[i] = 0, sh.count[i] = 0;
        __syncthreads();
        for (int t = wave; t < tiles; t += kWaves) {
            float x[8];
            row.load(t * kTile + lane * 8, x);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (x[i] != -INFINITY) {
                    const int b = row.bin(x[i]);
                    if (by_k) atomicAdd(&sh.count[b], 1u);
                    if (by_p) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[b]), static_cast<unsigned long long>(Row<T>::whole(row.weight(x[i]))));
                }
        }
        __syncthreads();
        if (by_k) {
            uint64_t own = 0, available;
            for (int i = threadIdx.x; i < kBins; i += THREADS) own += sh.count[i];
            block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, available);
            if (static_cast<uint64_t>(f.top_k) < available) least = limit<THREADS, false>(row, sh, static_cast<double>(f.top_k));
        }
        if (by_p) {
            // the sum that p is of: of what top-k leaves
            uint64_t own = 0, total;
            const int edge = least == -INFINITY ? kBins : row.bin(least);
            for (int i = threadIdx.x; i < edge; i += THREADS) own += sh.mass[i];
            if (edge < kBins) {
                for (int t = wave; t < tiles; t += kWaves) {
                    float x[8];
                    row.load(t * kTile + lane * 8, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (x[i] >= least && row.bin(x[i]) == edge) own += Row<T>::whole(row.weight(x[i]));
                }
            }
            block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, total);
            least = fmaxf(least, limit<THREADS, true>(row, sh, f.top_p * static_cast<double>(total)));
        }
    }
    // the kept weights of every tile, in the histogram's place: a wave first gathers its tile's
    // kept scores, often few, so that their exponentials fill its lanes
    __syncthreads();
    auto kept = [&](float x) {
        if (x == -INFINITY || x < least) return 0.0;
        const double w = row.weight(x);
        return w >= f.min_p ? w : 0.0;
    };
    for (int t = wave; t < tiles; t += kWaves) {
        float x[8];
        row.load(t * kTile + lane * 8, x);
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
        for (int i = lane; i < count; i += kWave) sum += Row<T>::whole(kept(sh.gathered[wave][i]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
        if (lane == 0) sh.mass[t] = sum;
    }
    __syncthreads();
    uint64_t own = 0, total;
    for (int t = threadIdx.x; t < tiles; t += THREADS) own += sh.mass[t];
    block_exclusive_scan<THREADS, uint64_t>(own, sh.scan, total);
    if (f.probabilities) {
        const double share = total ? 17592186044416.0 / static_cast<double>(total) : 0.0;
        float* out = f.probabilities + r * f.vocab;
        for (int t = wave; t < tiles; t += kWaves) {
            float x[8];
            const int j = t * kTile + lane * 8;
            row.load(j, x);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < f.vocab) out[j + i] = static_cast<float>(kept(x[i]) * share);
        }
    }
    // the first running sum beyond u of the whole; sums are whole, so beyond it means not below the next double
    const float u = f.uniforms[r];
    const double target = static_cast<double>(u > 0.0f ? fminf(u, 0.999999940395355f) : 0.0f) * static_cast<double>(total);
    uint64_t before;
    const int tile = reach<THREADS>(sh, tiles, [&](int i) { return sh.mass[i]; }, nextafter(target, 1e300), 0, before);
    if (wave) return;
    float x[8];
    const int j = tile * kTile + lane * 8;
    row.load(j, x);
    uint64_t w[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = Row<T>::whole(kept(x[i])), sum += w[i];
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
// scores, or what weight, lie at or above a candidate. 2^44 x 512 = 2^53: sums of whole
// weights are exact in double.
template <typename T>
__global__ __launch_bounds__(kWave) void sample_narrow_kernel(Draw f) {
    const int lane = lane_id(), j = lane * 8;
    const int64_t r = blockIdx.x;
    Row<T> row{static_cast<const T*>(f.logits) + r * f.row_stride, f.vocab, static_cast<int>(f.exclude), f.vector != 0, false, 0.0, f.slope};
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
    uint32_t least = 1;  // of the kept ranks; no score has rank 0
    if (f.top_k > 0 && f.top_k < f.vocab) {
        uint32_t at = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = at | 1u << bit;
            int64_t count = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) count += __popcll(__ballot(rank[i] >= next));
            if (count >= f.top_k) at = next;
        }
        least = max(at, 1u);
    }
    if (f.top_p < 1.0) {
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) total += rank[i] >= least ? w[i] : 0.0;
        const double target = f.top_p * over_wave(total, add);
        uint32_t at = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = at | 1u << bit;
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += rank[i] >= next ? w[i] : 0.0;
            if (!(over_wave(sum, add) < target)) at = next;
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

template <typename T>
int draw(const Draw& f, int64_t rows, hipStream_t stream) {
    // a wave takes 512 scores a step: sixteen waves where a row has more than four such tiles
    if (f.vocab <= kTile)
        hipLaunchKernelGGL((sample_narrow_kernel<T>), dim3(static_cast<unsigned>(rows)), dim3(kWave), 0, stream, f);
    else if (f.vocab <= 2048)
        hipLaunchKernelGGL((sample_filtered_kernel<256, T>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, f);
    else
        hipLaunchKernelGGL((sample_filtered_kernel<1024, T>), dim3(static_cast<unsigned>(rows)), dim3(1024), 0, stream, f);
    return check_launch("koemi_sample_filtered");
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" int koemi_sample_filtered(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab,
                                     int64_t exclude, double temperature, int64_t top_k, double top_p, double min_p,
                                     const float* uniforms, int64_t* ids, float* probabilities, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_sample_filtered";
    if (rows < 0 || vocab < 1) return fail(KOEMI_ERR_INVALID, "%s: rows must not be negative and the vocabulary positive", what);
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: float32, float16 or bfloat16, not %s", what, dtype_name(dtype));
    if (vocab > kMaxVocab) return fail(KOEMI_ERR_UNSUPPORTED, "%s: at most 2^19 ids", what);
    if (rows > 0x7fffffff) return fail(KOEMI_ERR_UNSUPPORTED, "%s: too many rows", what);
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
    if (dtype == KOEMI_F32) return draw<float>(f, rows, as_stream(stream));
    if (dtype == KOEMI_F16) return draw<f16>(f, rows, as_stream(stream));
    return draw<bf16>(f, rows, as_stream(stream));
}
