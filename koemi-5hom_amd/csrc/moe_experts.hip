// The experts' gated feed-forward of every routed pair, weighted and summed per token,
// with its gradients.
//
//   g = W_g x + b_g, v = W_v x + b_v, h = silu(g) v, y = W_o h + b_o of each pair's expert
//   out_t = sum_s w_ts y_ts
//   d' = W_o^T dout_t (not weighted), dw = <d', h> + <dout_t, b_o>,
//   dv = w d' silu(g), dg = w d' v s (1 + g (1 - s)), s = sigmoid(g),
//   dx_t = sum_s W_g^T dg + W_v^T dv,
//   dW_g = sum dg x^T, dW_v = sum dv x^T, dW_o = sum dout (w h)^T, db_g = sum dg,
//   db_v = sum dv, db_o = sum w dout  (sums over the expert's pairs)
//
// (LearnedExpertMixture.combine, model/router.py:61-97 of the reference, before its
// normalizer, and what its autograd forms.) dw needs no y: it is the row sum of d' h, and
// the weighted products take the weight on h's side, so that dout enters them as it came.
//
// The pairs of an expert are consecutive rows of the sorted order, so each product is
// a grouped matrix product: six in all, two of them (W_g and W_v) doubled. The forward
// keeps g and v in fp32: what dw is made of would otherwise be as inexact as 16-bit
// values are, and forming them again would cost two of the products.
//
// Any type, width and alignment runs on the tiles of split_gemm.hpp, which read an
// operand either along K or across it; what lies between two products stays fp32 there
// (two bf16 planes of it are multiplied where the result is 16-bit).
#include "common.hpp"
#include "few_rows_mlp.hpp"
#include "mfma_across.hpp"
#include "split_gemm.hpp"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace koemi {
namespace {

using split_gemm::acc_column;

inline size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t padded_hidden(int64_t hidden) { return (hidden + 7) / 8 * 8; }  // rows of whole 32-byte octets

// sigmoid and 1 - sigmoid. The exponential stays finite (an infinite one would make 0 x inf of
// 1 - s); past its end s is 0, so that g s vanishes however far below zero g lies. NaN stays
// NaN. The product with log2 e is rounded: s for g < 0 and 1 - s for g > 0 are within
// 1.3 |g| + 8 units of 2^-24 of themselves, the other within 4.
__device__ __forceinline__ void sigmoid_pair(float g, float& s, float& rest) {
    const float x = g * -1.44269504088896341f;
    const float e = __builtin_amdgcn_exp2f(x > 126.0f ? 126.0f : x), r = __builtin_amdgcn_rcpf(1.0f + e);
    s = x > 126.0f ? 0.0f : r;
    rest = e * r;
}
__device__ __forceinline__ float glu(float g, float v) {
    float s, rest;
    sigmoid_pair(g, s, rest);
    return g * s * v;
}
// From d' of one hidden unit: dg, dv, w h, and what it adds to dw.
struct GluGradient {
    float dg, dv, wh, dw;
};
__device__ __forceinline__ GluGradient glu_gradient(float g, float v, float d, float w) {
    float s, rest;
    sigmoid_pair(g, s, rest);
    const float silu = g * s, wd = w * d;
    GluGradient o;
    o.dw = d * (silu * v);
    o.dg = wd * v * (s * fmaf(g, rest, 1.0f));
    o.dv = wd * silu;
    o.wh = w * (silu * v);
    return o;
}

// ------------------------------------------------------------------- slots ---
// A slot is up to `rows` consecutive pairs of one expert. expert[count] holds the
// number of slots in use; first[e] the first slot of expert e (experts + 1 of them).
struct Slots {
    int32_t* expert;
    int32_t* first;
    int64_t* row;
    int64_t* end;
};
constexpr int kSlotThreads = 1024;

__global__ __launch_bounds__(kSlotThreads) void slots_kernel(const int64_t* __restrict__ offsets, int64_t experts,
                                                             int64_t pairs, int64_t rows, int64_t max_slots, Slots s) {
    __shared__ int32_t wave_tot[kSlotThreads / kWave];
    int32_t before = 0;
    for (int64_t e0 = 0; e0 < experts; e0 += kSlotThreads) {
        const int64_t e = e0 + threadIdx.x;
        int64_t lo = 0, hi = 0;
        if (e < experts) {
            lo = min(max(offsets[e], int64_t(0)), pairs);
            hi = min(max(offsets[e + 1], lo), pairs);
        }
        const int32_t n = static_cast<int32_t>((hi - lo + rows - 1) / rows);
        int32_t total;
        const int32_t at = before + block_exclusive_scan<kSlotThreads>(n, wave_tot, total);
        if (e < experts) s.first[e] = at;
        for (int32_t i = 0; i < n && at + i < max_slots; ++i) {
            s.expert[at + i] = static_cast<int32_t>(e);
            s.row[at + i] = lo + i * rows;
            s.end[at + i] = hi;
        }
        before += total;
    }
    if (threadIdx.x == 0) {
        s.first[experts] = before;
        s.expert[max_slots] = static_cast<int32_t>(min(static_cast<int64_t>(before), max_slots));
    }
}

// The (slot, column tile) of a workgroup, or false: workgroup b runs on XCD b % 8, and each
// XCD takes a contiguous range of tiles in groups of kGroup slots, so that tiles that
// run at once share operands in its L2.
constexpr uint32_t kGroup = 4;
__device__ __forceinline__ bool slot_tile(const Slots& s, int64_t max_slots, uint32_t n_tiles, uint32_t& slot,
                                          uint32_t& tile_n) {
    const uint32_t slots = static_cast<uint32_t>(s.expert[max_slots]), tiles = slots * n_tiles, per = (tiles + 7) / 8;
    const uint32_t i = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || i >= tiles) return false;
    const uint32_t group = kGroup * n_tiles, first = i / group * kGroup, width = min(kGroup, slots - first);
    slot = first + i % group % width;
    tile_n = i % group / width;
    return true;
}

// --------------------------------------------------- any type and any shape ---
// Rows of a tile: 64 where the experts' segments are mostly shorter than a tile of 128.
inline int any_rows(int64_t pairs, int64_t experts) { return pairs <= 96 * experts ? 64 : 128; }
// Such calls have few tiles too: those of 64 rows are 64 columns wide and have four K steps
// under way (64 tokens bf16, 2048 -> 1024: 53 us with 128 columns and one step).
__host__ __device__ constexpr int any_cols(int rows) { return rows == 64 ? 64 : 128; }
__host__ __device__ constexpr int any_depth(int rows) { return rows == 64 ? 4 : 1; }

// The gradients' tiles are 64 columns wide throughout: more of them, and more workgroups a CU
// (fp16 3000 tokens, 768 -> 2000: hidden 130 us and input 276 with 128 columns, 91 and 241 with
// 64). Where the rows that lie across K allow it they are read eight columns at once: hidden
// 75 us, input 200, each weight's 109 -> 72.
constexpr int kGradientCols = 64;
using split_gemm::kAcross;
using split_gemm::kStrided;
// The column that a thread reads from, of `columns` across K: for those past the last, the last octet (kAcross) or the last.
template <int LIES>
__device__ __forceinline__ int64_t column_of(int64_t c, int64_t columns) {
    return min(c, columns - (LIES == kAcross ? 8 : 1));
}

// What lies between two products, as their operand beside T: fp32 in memory.
template <typename T>
using Between = std::conditional_t<std::is_same<T, float>::value, float, split_gemm::coarse_f32>;
// The LDS of a tile and, after its products, of four waves' output regions.
template <typename G>
constexpr int any_lds(int region) {
    return G::kLdsBytes > 4 * region ? G::kLdsBytes : 4 * region;
}

// g, v (fp32, kept where wanted) and h (fp32) of a slot's pairs x 64 hidden units; rows
// are ld apart, zeros from `hidden` on. B rows 0-63 of the tile are W_g's, 64-127 W_v's.
template <typename T, int BM, int BYTES>
__global__ __launch_bounds__(split_gemm::kThreads, 2) void any_hidden_kernel(
    const T* __restrict__ x, const int64_t* __restrict__ rows, int64_t tokens, const T* __restrict__ Wg,
    const T* __restrict__ bg, const T* __restrict__ Wv, const T* __restrict__ bv, float* __restrict__ keep_g,
    float* __restrict__ keep_v, float* __restrict__ h, Slots slots, int64_t max_slots, int64_t width, int64_t hidden,
    int64_t ld, uint32_t n_tiles) {
    using G = split_gemm::Tile<T, T, BM, 128, split_gemm::kAlong, split_gemm::kAlong, BM == 64 ? 2 : 1>;
    constexpr int kRegion = split_gemm::store_bytes<float, 1>();
    __shared__ __attribute__((aligned(16))) char lds[any_lds<G>(kRegion)];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * 64;
    const int wave = threadIdx.x / kWave, wm = wave >> 1, wn = wave & 1;
    const T* w0 = Wg + e * hidden * width;
    const T* w1 = Wv + e * hidden * width;
    auto a_row = [&](int r) { return x + min(max(rows[min(row0 + r, end - 1)], int64_t(0)), tokens - 1) * width; };
    G tile;
    uint64_t chains = tile.template run<BYTES, BYTES>(
        lds, width, width, 0, ceil_div(width, G::BK) * G::BK, a_row,
        [&](int r) { return (r < 64 ? w0 : w1) + min(n0 + (r & 63), hidden - 1) * width; },
        [&](int t) { return t * 64 + wn * 32; });
    if constexpr (G::kNative) split_gemm::lds_barrier();
    const int64_t first = n0 + wn * 32;
    float b0[16], b1[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int64_t c = e * hidden + min(first + acc_column(v), hidden - 1);
        b0[v] = to_f32(bg[c]);
        b1[v] = to_f32(bv[c]);
    }
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        const int64_t r = row0 + wm * (BM / 2) + i * 32;
        float og[1][16], ov[1][16], oh[1][16];
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const bool in = first + acc_column(v) < hidden;
            og[0][v] = in ? tile.acc[i][0][v] + b0[v] : 0.0f;
            ov[0][v] = in ? tile.acc[i][G::NT - 1][v] + b1[v] : 0.0f;
            oh[0][v] = glu(og[0][v], ov[0][v]);
        }
        char* region = lds + wave * kRegion;
        if (keep_g) {
            split_gemm::store_rows<float, 1>(region, og, keep_g + r * ld + first, ld, end - r, ld - first, true);
            split_gemm::store_rows<float, 1>(region, ov, keep_v + r * ld + first, ld, end - r, ld - first, true);
        }
        split_gemm::store_rows<float, 1>(region, oh, h + r * ld + first, ld, end - r, ld - first, true);
    }
    if constexpr (!G::kNative) {
        chains |= chains >> 16 | chains << 16;
        split_gemm::fix_chains(chains, [&](int block, int v) {
            if (block % G::NT != 0) return;
            const int64_t r = wm * (BM / 2) + block / G::NT * 32 + (lane_id() & 31), c = first + acc_column(v);
            if (row0 + r >= end || c >= hidden) return;
            const float g = split_gemm::scalar_dot(a_row(static_cast<int>(r)), w0 + c * width, width, to_f32(bg[e * hidden + c]));
            const float u = split_gemm::scalar_dot(a_row(static_cast<int>(r)), w1 + c * width, width, to_f32(bv[e * hidden + c]));
            const int64_t o = (row0 + r) * ld + c;
            if (keep_g) keep_g[o] = g, keep_v[o] = u;
            h[o] = glu(g, u);
        });
    }
}

// y = W_o h + b_o of a slot's pairs x a tile's columns, fp32.
template <typename T, int BM, int BYTES>
__global__ __launch_bounds__(split_gemm::kThreads, 2) void any_output_kernel(
    const Between<T>* __restrict__ h, const T* __restrict__ Wo, const T* __restrict__ bo, float* __restrict__ y, Slots slots,
    int64_t max_slots, int64_t width, int64_t hidden, int64_t ld, uint32_t n_tiles) {
    constexpr int BN = any_cols(BM);
    using G = split_gemm::Tile<Between<T>, T, BM, BN, split_gemm::kAlong, split_gemm::kAlong, any_depth(BM)>;
    constexpr int kRegion = split_gemm::store_bytes<float, 1>();
    __shared__ __attribute__((aligned(16))) char lds[any_lds<G>(kRegion)];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * BN;
    const int wave = threadIdx.x / kWave, wm = wave >> 1, wn = wave & 1;
    const T* w = Wo + e * width * hidden;
    G tile;
    const uint64_t chains = tile.template run<16, BYTES>(
        lds, ld, hidden, 0, ceil_div(hidden, G::BK) * G::BK, [&](int r) { return h + min(row0 + r, end - 1) * ld; },
        [&](int r) { return w + min(n0 + r, width - 1) * hidden; }, [&](int t) { return wn * (BN / 2) + t * 32; });
    const int64_t first = n0 + wn * (BN / 2);
#pragma unroll
    for (int j = 0; j < G::NT; ++j)
#pragma unroll
        for (int i = 0; i < G::MT; ++i) {
            const int64_t r = row0 + wm * (BM / 2) + i * 32, c = first + j * 32;
            float o[1][16];
#pragma unroll
            for (int v = 0; v < 16; ++v)
                o[0][v] = tile.acc[i][j][v] + to_f32(bo[e * width + min(c + acc_column(v), width - 1)]);
            split_gemm::store_rows<float, 1>(lds + wave * kRegion, o, y + r * width + c, width, end - r, width - c, width % 8 == 0);
        }
    split_gemm::fix_chains(chains, [&](int block, int v) {
        const int64_t r = row0 + wm * (BM / 2) + block / G::NT * 32 + (lane_id() & 31);
        const int64_t c = first + block % G::NT * 32 + acc_column(v);
        if (r >= end || c >= width) return;
        y[r * width + c] = split_gemm::scalar_dot(h + r * ld, w + c * hidden, hidden, to_f32(bo[e * width + c]));
    });
}

// d' = W_o^T dout of a slot's pairs x a tile's hidden units and what follows from it: dg, dv
// and w h (fp32, rows ld apart, zeros from `hidden` on), and each row's part of dw from
// a wave's half of them: dw_part[(2 tile + wave column) pairs + row].
template <typename T, int BM, int BYTES, int LIES>
__global__ __launch_bounds__(split_gemm::kThreads, 2) void any_hidden_gradient_kernel(
    const T* __restrict__ d_out, const int64_t* __restrict__ rows, int64_t tokens, const T* __restrict__ Wo,
    const float* __restrict__ keep_g, const float* __restrict__ keep_v, const float* __restrict__ sorted_w, float share,
    float* __restrict__ dg, float* __restrict__ dv, float* __restrict__ wh, float* __restrict__ dw_part, Slots slots,
    int64_t max_slots, int64_t pairs, int64_t width, int64_t hidden, int64_t ld, uint32_t n_tiles) {
    constexpr int BN = kGradientCols;
    using G = split_gemm::Tile<T, T, BM, BN, split_gemm::kAlong, LIES, any_depth(BM)>;
    constexpr int kRegion = split_gemm::store_bytes<float, 1>();
    __shared__ __attribute__((aligned(16))) char lds[any_lds<G>(kRegion)];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * BN;
    const int wave = threadIdx.x / kWave, wm = wave >> 1, wn = wave & 1;
    const T* w = Wo + e * width * hidden;
    auto a_row = [&](int r) { return d_out + min(max(rows[min(row0 + r, end - 1)], int64_t(0)), tokens - 1) * width; };
    G tile;
    const uint64_t chains = tile.template run<BYTES, 16>(
        lds, width, width, 0, ceil_div(width, G::BK) * G::BK, a_row, [&](int r) { return w + column_of<LIES>(n0 + r, hidden); },
        [&](int t) { return wn * (BN / 2) + t * 32; }, 1, hidden);
    if constexpr (G::kNative) split_gemm::lds_barrier();
    char* region = lds + wave * kRegion;
    const int64_t first = n0 + wn * (BN / 2);
    float* part = dw_part + (2 * static_cast<int64_t>(tile_n) + wn) * pairs;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        const int64_t r = row0 + wm * (BM / 2) + i * 32, mine = min(r + (lane_id() & 31), end - 1);
        const float weight = sorted_w ? sorted_w[mine] : share;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < G::NT; ++j) {
            const int64_t c = first + j * 32;
            float a[1][16], b[1][16], h[1][16];
            float kg[16], kv[16];
#pragma unroll
            for (int v = 0; v < 16; v += 4) {  // four units at once: rows are padded to eight
                const int64_t at = mine * ld + min(c + acc_column(v), ld - 4);
                const float4 g4 = load4(keep_g + at), v4 = load4(keep_v + at);
                kg[v] = g4.x, kg[v + 1] = g4.y, kg[v + 2] = g4.z, kg[v + 3] = g4.w;
                kv[v] = v4.x, kv[v + 1] = v4.y, kv[v + 2] = v4.z, kv[v + 3] = v4.w;
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int64_t at = min(c + acc_column(v), hidden - 1);
                float d = tile.acc[i][j][v];
                if constexpr (!G::kNative)
                    if (__builtin_expect(chains >> ((i * G::NT + j) * 16 + v) & 1, 0))
                        d = split_gemm::scalar_dot(a_row(static_cast<int>(mine - row0)), w + at, width, 0.0f, 1, hidden);
                const GluGradient o = glu_gradient(kg[v], kv[v], d, weight);
                const bool in = c + acc_column(v) < hidden;
                a[0][v] = in ? o.dg : 0.0f;
                b[0][v] = in ? o.dv : 0.0f;
                h[0][v] = in ? o.wh : 0.0f;
                sum += in ? o.dw : 0.0f;
            }
            split_gemm::store_rows<float, 1>(region, a, dg + r * ld + c, ld, end - r, ld - c, true);
            split_gemm::store_rows<float, 1>(region, b, dv + r * ld + c, ld, end - r, ld - c, true);
            split_gemm::store_rows<float, 1>(region, h, wh + r * ld + c, ld, end - r, ld - c, true);
        }
        sum += __shfl_xor(sum, 32, kWave);
        if (lane_id() < 32 && r + lane_id() < end) part[r + lane_id()] = sum;
    }
}

// dx of a slot's pairs x a tile's columns: dg W_g, then (ADD) dv W_v added to it, fp32. In one
// launch the first product's sums beside the second's spill (fp16 3000 tokens: 301 us).
template <typename T, int BM, int LIES, bool ADD>
__global__ __launch_bounds__(split_gemm::kThreads, 2) void any_input_gradient_kernel(
    const Between<T>* __restrict__ d, const T* __restrict__ W, float* __restrict__ dx, Slots slots, int64_t max_slots,
    int64_t width, int64_t hidden, int64_t ld, uint32_t n_tiles) {
    constexpr int BN = kGradientCols;
    using G = split_gemm::Tile<Between<T>, T, BM, BN, split_gemm::kAlong, LIES, any_depth(BM)>;
    constexpr int kRegion = split_gemm::store_bytes<float, 1>();
    __shared__ __attribute__((aligned(16))) char lds[any_lds<G>(kRegion)];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * BN;
    const int wave = threadIdx.x / kWave, wm = wave >> 1, wn = wave & 1;
    const T* w = W + e * hidden * width;
    G tile;
    const uint64_t chains = tile.template run<16, 16>(
        lds, ld, hidden, 0, ceil_div(hidden, G::BK) * G::BK, [&](int r) { return d + min(row0 + r, end - 1) * ld; },
        [&](int r) { return w + column_of<LIES>(n0 + r, width); }, [&](int t) { return wn * (BN / 2) + t * 32; }, 1, width);
    const int64_t first = n0 + wn * (BN / 2);
#pragma unroll
    for (int j = 0; j < G::NT; ++j)
#pragma unroll
        for (int i = 0; i < G::MT; ++i) {
            const int64_t r = row0 + wm * (BM / 2) + i * 32, c = first + j * 32, mine = min(r + (lane_id() & 31), end - 1);
            float o[1][16];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int64_t at = min(c + acc_column(v), width - 1);
                float sum = tile.acc[i][j][v];
                if (__builtin_expect(chains >> ((i * G::NT + j) * 16 + v) & 1, 0))
                    sum = split_gemm::scalar_dot(d + mine * ld, w + at, hidden, 0.0f, 1, width);
                o[0][v] = ADD ? dx[mine * width + at] + sum : sum;
            }
            split_gemm::store_rows<float, 1>(lds + wave * kRegion, o, dx + r * width + c, width, end - r, width - c, width % 8 == 0);
        }
}

// Every expert's C[m, n] = sum over its pairs of A[pair, m] B[pair, n] (rows lda and ldb
// apart), in type T; zeros for an expert without pairs. Up to three products of the same
// types in one launch, since small ones leave CUs idle (fp32 500 tokens, 201 -> 333: three
// launches 26 us, one 15; fp16 3000, 768 -> 2000: two 150, one 131).
template <typename T, typename TA, typename TB>
struct WeightProducts {
    struct One {
        const TA* a;
        const TB* b;
        T* c;
        int64_t M, N, lda, ldb;
        uint32_t end, n_tiles;  // of an expert's tiles, those of this product and the ones before it
    } one[3];
    int count = 0;
    void add(const TA* a, const TB* b, void* c, int64_t M, int64_t N, int64_t lda, int64_t ldb, int64_t side) {
        const uint32_t nt = static_cast<uint32_t>(ceil_div(N, side)), mt = static_cast<uint32_t>(ceil_div(M, side));
        one[count] = {a, b, static_cast<T*>(c), M, N, lda, ldb, tiles() + mt * nt, nt};
        ++count;
    }
    uint32_t tiles() const { return count ? one[count - 1].end : 0; }
};
template <typename T, typename TA, typename TB, int BM, int A_LIES, int B_LIES>
__global__ __launch_bounds__(split_gemm::kThreads, 2) void any_weight_gradient_kernel(
    WeightProducts<T, TA, TB> products, uint32_t per, const int64_t* __restrict__ offsets, int64_t pairs) {
    using G = split_gemm::Tile<TA, TB, BM, BM, A_LIES, B_LIES, BM == 64 ? 2 : 1>;
    constexpr int kRegion = split_gemm::store_bytes<T, 1>();
    __shared__ __attribute__((aligned(16))) char lds[any_lds<G>(kRegion)];
    const uint32_t e = blockIdx.x / per;
    uint32_t within = blockIdx.x % per;
    int which = 0;
    while (which + 1 < products.count && within >= products.one[which].end) ++which;
    if (which) within -= products.one[which - 1].end;
    const auto& one = products.one[which];
    const int64_t M = one.M, N = one.N, lda = one.lda, ldb = one.ldb;
    T* const C = one.c;
    const int64_t m0 = static_cast<int64_t>(within / one.n_tiles) * BM, n0 = static_cast<int64_t>(within % one.n_tiles) * BM;
    const int64_t lo = min(max(offsets[e], int64_t(0)), pairs), K = min(max(offsets[e + 1], lo), pairs) - lo;
    const int wave = threadIdx.x / kWave, wm = wave >> 1, wn = wave & 1;
    T* out = C + static_cast<int64_t>(e) * M * N;
    const TA* a = one.a + lo * lda;
    const TB* b = one.b + lo * ldb;
    G tile;
    uint64_t chains = 0;
    if (K > 0) {
        chains = tile.template run<16, 16>(
            lds, K, K, 0, ceil_div(K, G::BK) * G::BK, [&](int r) { return a + column_of<A_LIES>(m0 + r, M); },
            [&](int r) { return b + column_of<B_LIES>(n0 + r, N); }, [&](int t) { return wn * (BM / 2) + t * 32; }, lda, ldb);
    } else {
#pragma unroll
        for (int i = 0; i < G::MT; ++i)
#pragma unroll
            for (int j = 0; j < G::NT; ++j) tile.acc[i][j] = split_gemm::f32x16{};
    }
    if constexpr (G::kNative) split_gemm::lds_barrier();
    const int64_t first = n0 + wn * (BM / 2);
#pragma unroll
    for (int j = 0; j < G::NT; ++j)
#pragma unroll
        for (int i = 0; i < G::MT; ++i) {
            const int64_t r = m0 + wm * (BM / 2) + i * 32, c = first + j * 32;
            float o[1][16];
#pragma unroll
            for (int v = 0; v < 16; ++v) o[0][v] = tile.acc[i][j][v];
            split_gemm::store_rows<T, 1>(lds + wave * kRegion, o, out + r * N + c, N, M - r, N - c,
                                         N % 8 == 0 && reinterpret_cast<uintptr_t>(C) % 16 == 0);
        }
    if constexpr (!G::kNative)
        split_gemm::fix_chains(chains, [&](int block, int v) {
            const int64_t r = m0 + wm * (BM / 2) + block / G::NT * 32 + (lane_id() & 31);
            const int64_t c = first + block % G::NT * 32 + acc_column(v);
            if (r < M && c < N) out[r * N + c] = from_f32<T>(split_gemm::scalar_dot(a + r, b + c, K, 0.0f, lda, ldb));
        });
}

// ------------------------------------------------------------ the bf16 tiles ---
// Width and hidden multiples of 64: 256 x 256 tiles of mfma_stage.hpp and mfma_across.hpp
// (four waves in 2 x 2, 128 x 128 outputs each, operands through a ring of four LDS
// stages filled by direct copies). What lies between two products (h, dg, dv, w h) is bf16: as
// two planes it would double four of the six products, for 1.7e-3 from float64 (the results'
// own rounding) instead of 2.3e-3; bf16 torch operations, which round g, v, silu and y too, are at
// 4.7e-3 to 5.8e-3 (4096 tokens, 1024 -> 2048). g, v, y, dx and every sum are fp32. A slot is up to 256 pairs of one expert; the backward works on rows padded to
// whole slots (row 256 slot + r), so that sums over an expert's pairs take whole K steps:
// rows past its pairs are zeros.
using mfma_stage::across_fragment;
using mfma_stage::along_fragment;
using mfma_stage::f32x16;
using mfma_stage::kOperandBytes;
using mfma_stage::uniform_ptr;
constexpr int kTile = 256;
constexpr int kTileK = mfma_stage::kBK;
// Columns of the tiles that write g and v: 128, two workgroups a CU, so that one's epilogue
// runs under the other's products (256 with one: 5% slower here, 10% faster where g and v
// are read, whose workgroups need the registers to have loads under way).
constexpr int kHiddenTile = 128;
template <int BNT>
constexpr uint32_t kTileLds = mfma_stage::TileShape<BNT>::kStages * mfma_stage::TileShape<BNT>::kStageBytes;

template <int BNT>
struct TilePlace {
    static constexpr int NT = BNT / 64;
    int lane, wave, wm, wn;
    uint32_t a_lds, b_lds;
    __device__ __forceinline__ explicit TilePlace(char* lds) {
        lane = lane_id();
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);  // scalar, and what follows from it
        wm = wave >> 1;
        wn = wave & 1;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        a_lds = __builtin_amdgcn_readfirstlane(lds0 + wave * 4 * 1024);
        b_lds = __builtin_amdgcn_readfirstlane(lds0 + kOperandBytes + wave * NT * 1024);
    }
    // Offsets of the wave's copies of an operand along K: row(r) is the memory row of the
    // tile's row r, ld elements long.
    template <int N, typename Row>
    __device__ __forceinline__ void along(uint32_t (&off)[N], int64_t ld, Row row) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (wave * N + i) * 16 + (lane >> 2), g = (lane & 3) ^ mfma_stage::slot_swizzle(r);
            off[i] = (static_cast<uint32_t>(row(r)) * static_cast<uint32_t>(ld) + g * 8) * 2u;
        }
    }
    // Of an operand across K: columns from `first` on (those past `columns`, a multiple of 8, repeat the last).
    template <int N>
    __device__ __forceinline__ void across(uint32_t (&off)[N], int64_t ld, int64_t first, int64_t columns) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int k, c;
            mfma_stage::across_source<N * 64>(wave * N + i, lane, k, c);
            off[i] = (static_cast<uint32_t>(k) * static_cast<uint32_t>(ld) + static_cast<uint32_t>(min(first + c, columns - 8))) * 2u;
        }
    }
    template <int N>
    __device__ __forceinline__ void fragments(uint32_t (&off)[N], bool across, int first) const {
#pragma unroll
        for (int t = 0; t < N; ++t) off[t] = across ? across_fragment<N * 64>(first + t * 32) : along_fragment(first + t * 32);
    }
};
template <int NT>
__device__ __forceinline__ void clear(f32x16 (&acc)[4][NT]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x16{};
}

// A wave's 128 x (32 TILES) outputs as whole bf16 rows. They pass through the wave's own
// LDS region (chunk c of row r at c ^ r, so that rows are read without bank conflicts),
// four consecutive columns c of a row at a time, and leave in 16-byte pieces.
template <int TILES>
__device__ __forceinline__ void put_four(char* region, int r, int c, float v0, float v1, float v2, float v3) {
    constexpr int kRowBytes = TILES * 64, kSwz = kRowBytes / 16 - 1;
    store4(reinterpret_cast<bf16*>(region + r * kRowBytes + ((c >> 3) ^ (r & kSwz)) * 16 + (c & 4) * 2), v0, v1, v2, v3);
}
// rows, cols (a multiple of 8): how many of the region's ROWS and its columns exist from
// out's first element on.
template <int TILES, int ROWS = 128>
__device__ __forceinline__ void flush_wave(const char* region, bf16* out, int64_t ld, int64_t rows, int64_t cols) {
    constexpr int kRowBytes = TILES * 64, kChunks = kRowBytes / 16, kSwz = kChunks - 1;
    constexpr int kIters = ROWS * kChunks / kWave, kBatch = kIters < 8 ? kIters : 8;
    constexpr int kStep = kWave / kChunks;  // rows of one store
    int lane = lane_id();
    asm volatile("" : "+v"(lane));  // addresses formed here: shared with other calls they are kept, and spill
    const int r0 = lane / kChunks, c = lane % kChunks;
    const uint32_t off = (static_cast<uint32_t>(r0) * static_cast<uint32_t>(ld) + c * 8) * 2u;  // below 64 rows
#pragma unroll
    for (int b = 0; b < kIters; b += kBatch) {
        uint4 piece[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = (b + i) * kStep + r0;
            piece[i] = *reinterpret_cast<const uint4*>(region + r * kRowBytes + ((c ^ (r & kSwz)) * 16));
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = (b + i) * kStep + r0;
            char* base = reinterpret_cast<char*>(out + (b + i) * kStep * ld);
            if (r < rows && c * 8 < cols) *reinterpret_cast<uint4*>(base + off) = piece[i];
        }
    }
}
// Both, of value(mt, t, v), element v of the wave's tile (mt, t).
template <int TILES, typename Value>
__device__ __forceinline__ void store_wave(char* region, bf16* out, int64_t ld, int64_t rows, int64_t cols, Value value) {
    const int lane = lane_id();
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            __builtin_amdgcn_sched_barrier(0);  // a tile at a time: all at once they spill
#pragma unroll
            for (int j = 0; j < 4; ++j)
                put_four<TILES>(region, mt * 32 + (lane & 31), t * 32 + (lane >> 5) * 4 + j * 8, value(mt, t, j * 4),
                                value(mt, t, j * 4 + 1), value(mt, t, j * 4 + 2), value(mt, t, j * 4 + 3));
        }
    flush_wave<TILES>(region, out, ld, rows, cols);
}
// A wave's 128 x 128 outputs in fp32, each lane four consecutive columns at a time.
template <typename Value>
__device__ __forceinline__ void store_wave_f32(float* out, int64_t ld, int64_t rows, int64_t cols, Value value) {
    const int lane = lane_id(), r0 = lane & 31, c0 = (lane >> 5) * 4;
    const uint32_t off = (static_cast<uint32_t>(r0) * static_cast<uint32_t>(ld) + c0) * 4u;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                char* base = reinterpret_cast<char*>(out + mt * 32 * ld + t * 32 + j * 8);
                if (mt * 32 + r0 < rows && t * 32 + j * 8 + c0 < cols)
                    store4(reinterpret_cast<float*>(base + off), value(mt, t, j * 4), value(mt, t, j * 4 + 1),
                           value(mt, t, j * 4 + 2), value(mt, t, j * 4 + 3));
            }
        }
}

// g and v are kept in the order of the accumulators: float4 (slot, 32-column block, 32-row
// block, j, lane) holds elements 4 j .. 4 j + 3, so that a wave reads and writes 1 KiB at
// once. The first float of (slot, column block, row block): j and the lane add to it.
__device__ __forceinline__ int64_t kept_at(int64_t slot, int64_t blocks, int64_t c32, int m32) {
    return ((slot * blocks + c32) * 8 + m32) * (4 * kWave * 4);
}
__device__ __forceinline__ uint32_t kept_lane(int j) { return static_cast<uint32_t>((j * kWave + lane_id()) * 4); }
// Past the caches: they are read a whole backward pass later, and once (16384 tokens, 1024
// -> 2048: written 389 us, 365 so; read 331, 306 so).
__device__ __forceinline__ float4 kept4(const float* p) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
    return make_float4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void keep4(float* p, float a, float b, float c, float d) {
    store16_nt(p, make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d)));
}

// g, v and h of a slot's pairs x BNT / 2 hidden units: the first half of the B rows are
// W_g's, the other W_v's.
template <int BNT>
__global__ __launch_bounds__(mfma_stage::kThreads, mfma_stage::TileShape<BNT>::kWgPerCu) void tile_hidden_kernel(
    const bf16* __restrict__ x, const int64_t* __restrict__ rows, int64_t tokens, const bf16* __restrict__ Wg,
    const bf16* __restrict__ bg, const bf16* __restrict__ Wv, const bf16* __restrict__ bv, float* __restrict__ keep_g,
    float* __restrict__ keep_v, bf16* __restrict__ h, Slots slots, int64_t max_slots, int64_t width, int64_t hidden,
    uint32_t n_tiles) {
    constexpr int NT = BNT / 64;
    __shared__ __attribute__((aligned(1024))) char lds[kTileLds<BNT>];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * (BNT / 2);
    const TilePlace<BNT> at(lds);
    const bf16* a = static_cast<const bf16*>(uniform_ptr(x));
    const bf16* b = static_cast<const bf16*>(uniform_ptr((at.wave >= 2 ? Wv : Wg) + static_cast<int64_t>(e) * hidden * width));
    uint32_t a_off[4], b_off[NT], a_frag[4], b_frag[NT];
    at.along(a_off, width, [&](int r) { return min(max(rows[min(row0 + r, end - 1)], int64_t(0)), tokens - 1); });
    at.along(b_off, width, [&](int r) { return min(n0 + (r & (BNT / 2 - 1)), hidden - 1); });
    at.fragments(a_frag, false, at.wm * 128);
#pragma unroll
    for (int t = 0; t < NT; ++t)
        b_frag[t] = along_fragment((t < NT / 2 ? 0 : BNT / 2) + at.wn * (BNT / 4) + t % (NT / 2) * 32);
    f32x16 acc[4][NT];
    clear(acc);
    mfma_stage::across_loop<BNT, false, false>(
        lds, [&](int kt) { return a + kt * kTileK; }, [&](int kt) { return b + kt * kTileK; }, a_off, b_off, at.a_lds,
        at.b_lds, a_frag, b_frag, static_cast<int>(width / kTileK), acc);
    __syncthreads();  // every wave is done reading the stages
    const int64_t first = n0 + at.wn * (BNT / 4), blocks = hidden / 32;
#pragma unroll
    for (int t = 0; t < NT / 2; ++t) {
        if (first + t * 32 >= hidden) break;
        float b0[16], b1[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int64_t c = static_cast<int64_t>(e) * hidden + first + t * 32 + acc_column(v);
            b0[v] = to_f32(bg[c]);
            b1[v] = to_f32(bv[c]);
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                acc[mt][t][v] += b0[v];
                acc[mt][t + NT / 2][v] += b1[v];
            }
            if (keep_g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t o = kept_at(slot, blocks, first / 32 + t, at.wm * 4 + mt);
                    keep4(keep_g + o + kept_lane(j), acc[mt][t][j * 4], acc[mt][t][j * 4 + 1], acc[mt][t][j * 4 + 2], acc[mt][t][j * 4 + 3]);
                    keep4(keep_v + o + kept_lane(j), acc[mt][t + NT / 2][j * 4], acc[mt][t + NT / 2][j * 4 + 1], acc[mt][t + NT / 2][j * 4 + 2],
                          acc[mt][t + NT / 2][j * 4 + 3]);
                }
        }
    }
    store_wave<NT / 2>(lds + at.wave * (128 * 32 * NT), h + (row0 + at.wm * 128) * hidden + first, hidden, end - row0 - at.wm * 128,
                  hidden - first, [&](int mt, int t, int v) { return glu(acc[mt][t][v], acc[mt][t + NT / 2][v]); });
}

// y = W_o h + b_o of a slot's pairs x 256 columns.
__global__ __launch_bounds__(mfma_stage::kThreads, 1) void tile_output_kernel(
    const bf16* __restrict__ h, const bf16* __restrict__ Wo, const bf16* __restrict__ bo, float* __restrict__ y, Slots slots,
    int64_t max_slots, int64_t width, int64_t hidden, uint32_t n_tiles) {
    __shared__ __attribute__((aligned(1024))) char lds[kTileLds<256>];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * kTile;
    const TilePlace<256> at(lds);
    const bf16* a = static_cast<const bf16*>(uniform_ptr(h + row0 * hidden));
    const bf16* b = static_cast<const bf16*>(uniform_ptr(Wo + static_cast<int64_t>(e) * width * hidden));
    uint32_t a_off[4], b_off[4], a_frag[4], b_frag[4];
    at.along(a_off, hidden, [&](int r) { return min(static_cast<int64_t>(r), end - row0 - 1); });
    at.along(b_off, hidden, [&](int r) { return min(n0 + r, width - 1); });
    at.fragments(a_frag, false, at.wm * 128);
    at.fragments(b_frag, false, at.wn * 128);
    f32x16 acc[4][4];
    clear(acc);
    mfma_stage::across_loop<256, false, false>(
        lds, [&](int kt) { return a + kt * kTileK; }, [&](int kt) { return b + kt * kTileK; }, a_off, b_off, at.a_lds,
        at.b_lds, a_frag, b_frag, static_cast<int>(hidden / kTileK), acc);
    const int64_t first = n0 + at.wn * 128, r0 = row0 + at.wm * 128;
    float bias[4][16];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
            bias[t][v] = to_f32(bo[static_cast<int64_t>(e) * width + min(first + t * 32 + acc_column(v), width - 1)]);
    store_wave_f32(y + r0 * width + first, width, end - r0, width - first,
                   [&](int mt, int t, int v) { return acc[mt][t][v] + bias[t][v]; });
}

// The pairs' rows of x and dout, padded to whole slots with zeros; the rows' parts of <dout,
// b_o> and the column sums of w dout, both from the values as they pass. A workgroup takes
// 64 rows and 512 columns, a wave every fourth row, a lane eight columns.
constexpr int kGatherRows = 64, kGatherColumns = 512;
__global__ __launch_bounds__(256) void tile_gather_kernel(const bf16* __restrict__ x, const bf16* __restrict__ d_out,
                                                          const int64_t* __restrict__ rows, const bf16* __restrict__ bo,
                                                          const float* __restrict__ sorted_w, float share,
                                                          bf16* __restrict__ xs, bf16* __restrict__ ds,
                                                          float* __restrict__ dot_part, float* __restrict__ sums, Slots slots,
                                                          int64_t max_slots, int64_t pairs, int64_t tokens, int64_t width) {
    __shared__ float sh[3][kWave][8];
    const int64_t quarter = blockIdx.x, slot = quarter / (kTile / kGatherRows);
    if (slot >= slots.expert[max_slots]) return;
    const int wave = threadIdx.x / kWave, lane = lane_id();
    const int64_t c = static_cast<int64_t>(blockIdx.y) * kGatherColumns + lane * 8, e = slots.expert[slot];
    const int64_t p0 = slots.row[slot] + quarter % (kTile / kGatherRows) * kGatherRows, end = slots.end[slot];
    const bool in = c < width;
    auto spread = [](const uint4& u, float (&f)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    };
    float bias[8] = {}, sum[8] = {};
    if (dot_part && in) spread(*reinterpret_cast<const uint4*>(bo + e * width + c), bias);
    constexpr int kTurn = 4;  // rows of a wave whose loads are under way at once
    for (int i0 = wave; i0 < kGatherRows; i0 += 4 * kTurn) {
        uint4 a[kTurn], d[kTurn];
        float w[kTurn];
#pragma unroll
        for (int u = 0; u < kTurn; ++u) {
            const int64_t p = p0 + i0 + 4 * u;
            const bool real = p < end;
            const int64_t t = real ? min(max(rows[p], int64_t(0)), tokens - 1) : 0;
            a[u] = d[u] = make_uint4(0, 0, 0, 0);
            if (real && in) {
                if (xs) a[u] = *reinterpret_cast<const uint4*>(x + t * width + c);
                d[u] = *reinterpret_cast<const uint4*>(d_out + t * width + c);
            }
            w[u] = !real ? 0.0f : sorted_w ? sorted_w[p] : share;
        }
#pragma unroll
        for (int u = 0; u < kTurn; ++u) {
            const int64_t p = p0 + i0 + 4 * u, padded = quarter * kGatherRows + i0 + 4 * u;
            const bool real = p < end;
            if (in) {
                if (xs) *reinterpret_cast<uint4*>(xs + padded * width + c) = a[u];
                *reinterpret_cast<uint4*>(ds + padded * width + c) = d[u];
            }
            float f[8], dot = 0.0f;
            spread(d[u], f);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                dot = fmaf(f[q], bias[q], dot);
                sum[q] = real ? fmaf(w[u], f[q], sum[q]) : sum[q];
            }
            if (dot_part) {
                dot = wave_sum_xor(dot);
                if (lane == 0 && real) dot_part[blockIdx.y * pairs + p] = dot;
            }
        }
    }
    if (!sums) return;
    if (wave > 0)
#pragma unroll
        for (int q = 0; q < 8; ++q) sh[wave - 1][lane][q] = sum[q];
    __syncthreads();
    if (wave != 0 || !in) return;
#pragma unroll
    for (int q = 0; q < 8; ++q) sum[q] = (sum[q] + sh[0][lane][q]) + (sh[1][lane][q] + sh[2][lane][q]);
    store4(sums + quarter * width + c, sum[0], sum[1], sum[2], sum[3]);
    store4(sums + quarter * width + c + 4, sum[4], sum[5], sum[6], sum[7]);
}

// Adds the column sums of a wave's region of ROWS rows x 32 columns (put_four<1>), as
// products with ones on the matrix cores: the region's rows are K, read transposed. Every
// column of the result is the sums.
template <int ROWS>
__device__ __forceinline__ void region_sums(const char* region, f32x16& acc) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int lane = lane_id(), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    mfma_stage::bf16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<bf16>(1.0f);
#pragma unroll
    for (int k0 = 0; k0 < ROWS; k0 += 16) {
        union {
            s16x4 half[2];
            mfma_stage::bf16x8 whole;
        } u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = k0 + 8 * (lane >> 5) + 4 * j + ((lane & 15) >> 2);
            u.half[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(region + r * 64 + ((chunk ^ (r & 3)) * 16) + (lane & 1) * 8));
        }
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.whole, ones, acc, 0, 0, 0);
    }
}
__device__ __forceinline__ void store_sums(const f32x16& acc, float* out) {
    const int lane = lane_id();
    if ((lane & 31) == 0)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            store4(out + (lane >> 5) * 4 + j * 8, acc[j * 4], acc[j * 4 + 1], acc[j * 4 + 2], acc[j * 4 + 3]);
}

// d' of a slot x 256 hidden units and what follows: dg and dv side by side (rows of 2
// hidden), w h, all padded, each pair's part of dw from a wave's 128 units, and (sums,
// NULL: not wanted) the column sums of dg and dv over a wave's 128 rows.
__global__ __launch_bounds__(mfma_stage::kThreads, 1) void tile_hidden_gradient_kernel(
    const bf16* __restrict__ ds, const bf16* __restrict__ Wo, const float* __restrict__ keep_g, const float* __restrict__ keep_v,
    const float* __restrict__ sorted_w, float share, bf16* __restrict__ dgv, bf16* __restrict__ wh,
    float* __restrict__ dw_part, float* __restrict__ sums, Slots slots, int64_t max_slots, int64_t pairs, int64_t width,
    int64_t hidden, uint32_t n_tiles) {
    constexpr int NT = kTile / 64, kRows = 64;
    __shared__ __attribute__((aligned(1024))) char lds[kTileLds<kTile>];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * kTile;
    const int64_t padded = static_cast<int64_t>(slot) * kTile;
    const TilePlace<kTile> at(lds);
    const bf16* a = static_cast<const bf16*>(uniform_ptr(ds + padded * width));
    const bf16* b = static_cast<const bf16*>(uniform_ptr(Wo + static_cast<int64_t>(e) * width * hidden));
    uint32_t a_off[4], b_off[NT], a_frag[4], b_frag[NT];
    at.along(a_off, width, [&](int r) { return r; });
    at.across(b_off, hidden, n0, hidden);
    at.fragments(a_frag, false, at.wm * 128);
    at.fragments(b_frag, true, at.wn * (kTile / 2));
    f32x16 acc[4][NT];
    clear(acc);
    mfma_stage::across_loop<kTile, false, true>(
        lds, [&](int kt) { return a + kt * kTileK; }, [&](int kt) { return b + kt * kTileK * hidden; }, a_off, b_off, at.a_lds,
        at.b_lds, a_frag, b_frag, static_cast<int>(width / kTileK), acc);
    const int64_t first = n0 + at.wn * (kTile / 2), blocks = hidden / 32;
    // block 4 t + mt of kept g and v, loaded while the block before is worked on
    struct Kept {
        float4 g[4], v[4];
    } kept[2];
    auto fetch = [&](int block, Kept& k) {
        const int64_t o = kept_at(slot, blocks, min(first / 32 + block / 4, blocks - 1), at.wm * 4 + block % 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k.g[j] = kept4(keep_g + o + kept_lane(j));
            k.v[j] = kept4(keep_v + o + kept_lane(j));
        }
    };
    fetch(0, kept[0]);
    __syncthreads();  // every wave is done reading the stages
    // 64 rows x 32 columns at a time: dg, dv and w h in three regions, so that no product is kept beside its sums
    constexpr int kRegion = kRows * 64;
    static_assert(4 * 3 * kRegion <= kTileLds<kTile>, "the output regions fit the stages");
    char* region = lds + at.wave * (3 * kRegion);
    const int64_t r0 = padded + at.wm * 128;
    float* part = dw_part + (2 * static_cast<int64_t>(tile_n) + at.wn) * pairs;
    float weight[4], sum[4] = {};
    bool real[4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
        const int64_t p = row0 + at.wm * 128 + mt * 32 + (at.lane & 31);
        real[mt] = p < end;
        weight[mt] = !real[mt] ? 0.0f : sorted_w ? sorted_w[p] : share;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (first + t * 32 >= hidden) break;  // the same for the wave
        f32x16 g_sums = {}, v_sums = {};
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            __builtin_amdgcn_sched_barrier(0);
            const Kept& k = kept[mt % 2];
            if (t * 4 + mt < 4 * NT - 1) fetch(t * 4 + mt + 1, kept[(mt + 1) % 2]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float g[4] = {k.g[j].x, k.g[j].y, k.g[j].z, k.g[j].w}, v[4] = {k.v[j].x, k.v[j].y, k.v[j].z, k.v[j].w};
                float dg[4], dv[4], h[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const GluGradient o4 = glu_gradient(g[q], v[q], acc[mt][t][j * 4 + q], weight[mt]);
                    sum[mt] += real[mt] ? o4.dw : 0.0f;
                    dg[q] = real[mt] ? o4.dg : 0.0f;
                    dv[q] = real[mt] ? o4.dv : 0.0f;
                    h[q] = real[mt] ? o4.wh : 0.0f;
                }
                const int r = mt * 32 % kRows + (at.lane & 31), c = (at.lane >> 5) * 4 + j * 8;
                put_four<1>(region, r, c, dg[0], dg[1], dg[2], dg[3]);
                put_four<1>(region + kRegion, r, c, dv[0], dv[1], dv[2], dv[3]);
                put_four<1>(region + 2 * kRegion, r, c, h[0], h[1], h[2], h[3]);
            }
            if ((mt + 1) * 32 % kRows != 0) continue;
            if (sums) {
                region_sums<kRows>(region, g_sums);
                region_sums<kRows>(region + kRegion, v_sums);
            }
            const int64_t row = r0 + mt * 32 / kRows * kRows;
            bf16* out = dgv + row * 2 * hidden + first + t * 32;
            flush_wave<1, kRows>(region, out, 2 * hidden, kRows, 32);
            flush_wave<1, kRows>(region + kRegion, out + hidden, 2 * hidden, kRows, 32);
            flush_wave<1, kRows>(region + 2 * kRegion, wh + row * hidden + first + t * 32, hidden, kRows, 32);
        }
        if (sums) {
            float* to = sums + (2 * static_cast<int64_t>(slot) + at.wm) * 2 * hidden + first + t * 32;
            store_sums(g_sums, to);
            store_sums(v_sums, to + hidden);
        }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
        sum[mt] += __shfl_xor(sum[mt], 32, kWave);
        if (at.lane < 32 && real[mt]) part[row0 + at.wm * 128 + mt * 32 + at.lane] = sum[mt];
    }
}

// dx of a slot's pairs x 256 columns: [dg dv] [W_g ; W_v], one sum over 2 hidden.
__global__ __launch_bounds__(mfma_stage::kThreads, 1) void tile_input_gradient_kernel(
    const bf16* __restrict__ dgv, const bf16* __restrict__ Wg, const bf16* __restrict__ Wv, float* __restrict__ dx, Slots slots,
    int64_t max_slots, int64_t width, int64_t hidden, uint32_t n_tiles) {
    __shared__ __attribute__((aligned(1024))) char lds[kTileLds<256>];
    uint32_t slot, tile_n;
    if (!slot_tile(slots, max_slots, n_tiles, slot, tile_n)) return;
    const int e = slots.expert[slot];
    const int64_t row0 = slots.row[slot], end = slots.end[slot], n0 = static_cast<int64_t>(tile_n) * kTile;
    const TilePlace<256> at(lds);
    const bf16* a = static_cast<const bf16*>(uniform_ptr(dgv + static_cast<int64_t>(slot) * kTile * 2 * hidden));
    const bf16* b0 = static_cast<const bf16*>(uniform_ptr(Wg + static_cast<int64_t>(e) * hidden * width));
    const bf16* b1 = static_cast<const bf16*>(uniform_ptr(Wv + static_cast<int64_t>(e) * hidden * width));
    uint32_t a_off[4], b_off[4], a_frag[4], b_frag[4];
    at.along(a_off, 2 * hidden, [&](int r) { return r; });
    at.across(b_off, width, n0, width);
    at.fragments(a_frag, false, at.wm * 128);
    at.fragments(b_frag, true, at.wn * 128);
    f32x16 acc[4][4];
    clear(acc);
    const int steps = static_cast<int>(hidden / kTileK);
    mfma_stage::across_loop<256, false, true>(
        lds, [&](int kt) { return a + kt * kTileK; },
        [&](int kt) { return kt < steps ? b0 + kt * kTileK * width : b1 + (kt - steps) * kTileK * width; }, a_off, b_off,
        at.a_lds, at.b_lds, a_frag, b_frag, 2 * steps, acc);
    const int64_t first = n0 + at.wn * 128, r0 = row0 + at.wm * 128;
    store_wave_f32(dx + r0 * width + first, width, end - r0, width - first,
                   [&](int mt, int t, int v) { return acc[mt][t][v]; });
}

// The three weights' gradients of every expert, in tiles of 256 x 256: sums over its
// padded rows. `which` 0: dW_g, 1: dW_v, 2: dW_o; a NULL one is not wanted.
__global__ __launch_bounds__(mfma_stage::kThreads, 1) void tile_weight_gradient_kernel(
    const bf16* __restrict__ dgv, const bf16* __restrict__ wh, const bf16* __restrict__ xs, const bf16* __restrict__ ds,
    const int64_t* __restrict__ offsets, Slots slots, bf16* __restrict__ dWg, bf16* __restrict__ dWv, bf16* __restrict__ dWo,
    int64_t pairs, int64_t width, int64_t hidden, uint32_t w_tiles, uint32_t h_tiles, uint32_t tiles) {
    __shared__ __attribute__((aligned(1024))) char lds[kTileLds<256>];
    const uint32_t per = (tiles + 7) / 8, i = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || i >= tiles) return;
    const uint32_t one = w_tiles * h_tiles, e = i / (3 * one), which = i % (3 * one) / one, within = i % one;
    bf16* C = which == 0 ? dWg : which == 1 ? dWv : dWo;
    if (!C) return;
    const bool out = which == 2;
    const int64_t M = out ? width : hidden, N = out ? hidden : width;
    const uint32_t n_tiles = out ? h_tiles : w_tiles;
    const int64_t m0 = static_cast<int64_t>(within / n_tiles) * kTile, n0 = static_cast<int64_t>(within % n_tiles) * kTile;
    const int64_t lo = min(max(offsets[e], int64_t(0)), pairs), count = min(max(offsets[e + 1], lo), pairs) - lo;
    const int64_t row = static_cast<int64_t>(slots.first[e]) * kTile;
    const int64_t lda = out ? width : 2 * hidden, ldb = out ? hidden : width;
    const TilePlace<256> at(lds);
    const bf16* a = static_cast<const bf16*>(uniform_ptr((out ? ds : dgv + (which == 1 ? hidden : 0)) + row * lda));
    const bf16* b = static_cast<const bf16*>(uniform_ptr((out ? wh : xs) + row * ldb));
    uint32_t a_off[4], b_off[4], a_frag[4], b_frag[4];
    at.across(a_off, lda, m0, M);
    at.across(b_off, ldb, n0, N);
    at.fragments(a_frag, true, at.wm * 128);
    at.fragments(b_frag, true, at.wn * 128);
    f32x16 acc[4][4];
    clear(acc);
    const int nk = static_cast<int>((count + kTileK - 1) / kTileK);
    if (nk > 0)  // the same for the workgroup
        mfma_stage::across_loop<256, true, true>(
            lds, [&](int kt) { return a + kt * kTileK * lda; }, [&](int kt) { return b + kt * kTileK * ldb; }, a_off, b_off,
            at.a_lds, at.b_lds, a_frag, b_frag, nk, acc);
    __syncthreads();  // every wave is done reading the stages
    const int64_t r = m0 + at.wm * 128, c = n0 + at.wn * 128;
    store_wave<4>(lds + at.wave * (128 * 256), C + static_cast<int64_t>(e) * M * N + r * N + c, N, M - r, N - c,
                  [&](int mt, int t, int v) { return acc[mt][t][v]; });
}

// ------------------------------------------------------- rows and columns ---
// out[t] = sum over the token's pairs of weight x row, in the order of its slots, rounded
// once; pairs past the valid ones count nothing. weights NULL: `share` each.
template <typename T>
__global__ __launch_bounds__(256) void combine_rows_kernel(const float* __restrict__ rows, const int64_t* __restrict__ positions,
                                                           const int64_t* __restrict__ valid_end, const float* __restrict__ weights,
                                                           float share, T* __restrict__ out, int64_t tokens, int64_t width,
                                                           int top_k) {
    const int64_t per_row = (width + 3) / 4, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t t = i / per_row, c = i % per_row * 4;
    if (t >= tokens) return;
    const int64_t end = *valid_end;
    float o[4] = {};
    for (int s = 0; s < top_k; ++s) {
        const int64_t p = positions[t * top_k + s];
        if (p < 0 || p >= end) continue;
        const float w = weights ? weights[t * top_k + s] : share;
        const float* r = rows + p * width + c;
        if (width % 4 == 0) {
            const float4 v = load4(r);
            o[0] = fmaf(w, v.x, o[0]), o[1] = fmaf(w, v.y, o[1]), o[2] = fmaf(w, v.z, o[2]), o[3] = fmaf(w, v.w, o[3]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < width) o[q] = fmaf(w, r[q], o[q]);
        }
    }
    T* y = out + t * width + c;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (c + q < width) y[q] = from_f32<T>(o[q]);
}

// The rows of x and dout that the pairs came from, in sorted order (either NULL: not
// wanted), and <dout, b_o> of each pair. A wave per pair, a lane VEC columns at a time (fp16
// 3000 tokens of 768: one 18 us, eight 9).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void gather_pairs_kernel(const T* __restrict__ x, const T* __restrict__ d_out,
                                                           const int64_t* __restrict__ rows, const int64_t* __restrict__ offsets,
                                                           int64_t experts, const T* __restrict__ bo,
                                                           const int64_t* __restrict__ pair_experts, T* __restrict__ xs,
                                                           T* __restrict__ ds, float* __restrict__ dot, int64_t pairs,
                                                           int64_t tokens, int64_t width) {
    struct alignas(sizeof(T) * VEC) Piece {
        T v[VEC];
    };
    const int64_t p = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (p >= pairs || p >= offsets[experts]) return;
    const int64_t t = min(max(rows[p], int64_t(0)), tokens - 1), e = min(max(pair_experts[p], int64_t(0)), experts - 1);
    float sum = 0.0f;
    for (int64_t c = lane_id() * VEC; c < width; c += kWave * VEC) {
        auto piece = [&](const T* from) { return *reinterpret_cast<const Piece*>(from + c); };
        if (xs) *reinterpret_cast<Piece*>(xs + p * width + c) = piece(x + t * width);
        const Piece d = piece(d_out + t * width);
        if (ds) *reinterpret_cast<Piece*>(ds + p * width + c) = d;
        if (dot) {
            const Piece b = piece(bo + e * width);
#pragma unroll
            for (int v = 0; v < VEC; ++v) sum = fmaf(to_f32(d.v[v]), to_f32(b.v[v]), sum);
        }
    }
    if (dot) {
        sum = wave_sum_xor(sum);
        if (lane_id() == 0) dot[p] = sum;
    }
}

// dw of every pair: the parts of its row's <d', h> and <dout, b_o> in order, 0 past the valid
// pairs. A thread per sorted row (the parts lie in that order), which looks for its slot
// among its token's.
__global__ __launch_bounds__(256) void weight_gradient_kernel(const float* __restrict__ part, int parts,
                                                              const float* __restrict__ dot, int dot_parts,
                                                              const int64_t* __restrict__ rows,
                                                              const int64_t* __restrict__ positions,
                                                              const int64_t* __restrict__ valid_end, float* __restrict__ dw,
                                                              int64_t pairs, int top_k) {
    const int64_t p = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (p >= pairs) return;
    float sum = 0.0f;
    if (p < *valid_end) {
        constexpr int kAhead = 16;  // loads under way at once
        for (int j = 0; j < parts; j += kAhead) {
            float v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) v[i] = part[min(j + i, parts - 1) * pairs + p];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) sum += j + i < parts ? v[i] : 0.0f;
        }
        for (int j = 0; j < dot_parts; ++j) sum += dot[j * pairs + p];
    }
    const int64_t t = min(max(rows[p], int64_t(0)), pairs / top_k - 1);
    for (int s = 0; s < top_k; ++s)
        if (positions[t * top_k + s] == p) dw[t * top_k + s] = sum;
}

// Column sums of each expert's rows, for the three biases in one launch each (blockIdx.z; an
// out of NULL is not wanted). First each slot's (a workgroup per slot and 64 columns, four
// waves over the rows), then each expert's slots in order.
struct ColumnSums {
    const void* a;     // rows of float (T for the third), lda apart
    float* part;       // `per` rows a slot, ld apart
    void* out;         // [experts, columns]
    int64_t lda, ld, columns;
    int per;
};
struct ThreeSums {
    ColumnSums s[3];
};
template <typename TA>
__device__ __forceinline__ float column_sum(const TA* a, int64_t lda, const float* weights, float share, bool weighted,
                                            int64_t begin, int64_t end) {
    float sum = 0.0f;
#pragma unroll 8
    for (int64_t r = begin; r < end; r += 4)
        sum = fmaf(weighted ? (weights ? weights[r] : share) : 1.0f, to_f32(a[r * lda]), sum);
    return sum;
}
template <typename T>
__global__ __launch_bounds__(256) void slot_sums_kernel(ThreeSums all, const float* __restrict__ weights, float share,
                                                        Slots slots, int64_t max_slots, int64_t rows) {
    const ColumnSums& s = all.s[blockIdx.z];
    const int64_t slot = blockIdx.x;
    if (!s.out || slot >= slots.expert[max_slots] || static_cast<int64_t>(blockIdx.y) * kWave >= s.columns) return;
    __shared__ float sh[4][kWave];
    const int wave = threadIdx.x / kWave;
    const int64_t c = static_cast<int64_t>(blockIdx.y) * kWave + lane_id();
    const int64_t r0 = slots.row[slot], end = min(slots.end[slot], r0 + rows);
    float sum = 0.0f;
    if (c < s.columns)
        sum = blockIdx.z == 2 ? column_sum(static_cast<const T*>(s.a) + c, s.lda, weights, share, true, r0 + wave, end)
                              : column_sum(static_cast<const float*>(s.a) + c, s.lda, weights, share, false, r0 + wave, end);
    sh[wave][lane_id()] = sum;
    __syncthreads();
    if (wave == 0 && c < s.columns)
        s.part[slot * s.ld + c] = (sh[0][lane_id()] + sh[1][lane_id()]) + (sh[2][lane_id()] + sh[3][lane_id()]);
}
template <typename T>
__global__ __launch_bounds__(256) void expert_sums_kernel(ThreeSums all, const int32_t* __restrict__ first) {
    const ColumnSums& s = all.s[blockIdx.z];
    const int64_t e = blockIdx.y, c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (!s.out || c >= s.columns) return;
    const int64_t end = static_cast<int64_t>(first[e + 1]) * s.per;
    float sum = 0.0f;
#pragma unroll 8
    for (int64_t i = static_cast<int64_t>(first[e]) * s.per; i < end; ++i) sum += s.part[i * s.ld + c];
    static_cast<T*>(s.out)[e * s.columns + c] = from_f32<T>(sum);
}

// --------------------------------------------------------------- the calls ---
struct Shape {
    int64_t pairs, tokens, width, hidden, experts, top_k;
    int dtype;
};
inline size_t element(int dtype) { return dtype == KOEMI_F32 ? 4 : 2; }
// Which path a shape takes: the bf16 tiles where their alignment holds, their 32-bit
// offsets reach and the experts' segments average at least a quarter of a tile's rows.
inline bool tile_shape(const Shape& s) {
    const int64_t reach = int64_t(1) << 31;
    return s.dtype == KOEMI_BF16 && s.width % 64 == 0 && s.hidden % 64 == 0 && s.pairs >= 64 * s.experts &&
           s.tokens * s.width < reach && s.hidden * s.width < reach && 512 * s.hidden < reach;
}
inline int64_t slot_rows(const Shape& s) { return tile_shape(s) ? kTile : any_rows(s.pairs, s.experts); }
inline int64_t most_slots(const Shape& s) { return ceil_div(s.pairs, slot_rows(s)) + s.experts; }

// Rows of the gathered operands of the backward: whole slots for the tiles.
inline int64_t gathered_rows(const Shape& s) { return tile_shape(s) ? most_slots(s) * kTile : s.pairs; }
// Floats of g (and of v) that the forward keeps.
inline int64_t kept_floats(const Shape& s) {
    return tile_shape(s) ? most_slots(s) * kTile * s.hidden : s.pairs * padded_hidden(s.hidden);
}

// Carves a workspace, or only measures it (base null).
struct Carver {
    char* base;
    size_t used = 0;
    template <typename V>
    V* take(int64_t n) {
        V* p = base ? reinterpret_cast<V*>(base + used) : nullptr;
        used += align256(static_cast<size_t>(std::max<int64_t>(n, 1)) * sizeof(V));
        return p;
    }
    Slots slots(const Shape& s) {
        Slots o;
        o.expert = take<int32_t>(most_slots(s) + 1);
        o.first = take<int32_t>(s.experts + 1);
        o.row = take<int64_t>(most_slots(s));
        o.end = take<int64_t>(most_slots(s));
        return o;
    }
};
// What the forward keeps: g, v and the slots.
struct SavedSpace {
    float* keep;
    Slots slots;
    size_t bytes;
};
inline SavedSpace saved_space(const Shape& s, void* base) {
    Carver c{static_cast<char*>(base)};
    SavedSpace w;
    w.keep = c.take<float>(2 * kept_floats(s));
    w.slots = c.slots(s);
    w.bytes = c.used;
    return w;
}
struct ForwardSpace {
    Slots slots;  // in `saved` where that is given
    float *h, *y;
    size_t bytes;
};
inline ForwardSpace forward_space(const Shape& s, void* base) {
    Carver c{static_cast<char*>(base)};
    ForwardSpace w;
    w.slots = c.slots(s);
    w.h = c.take<float>(tile_shape(s) ? s.pairs * s.hidden / 2 : s.pairs * padded_hidden(s.hidden));
    w.y = c.take<float>(s.pairs * s.width);
    w.bytes = c.used;
    return w;
}
struct BackwardSpace {
    Slots slots;  // the forward's, in `saved`
    float *dg, *dv, *wh, *dx, *dw_part, *dot, *sums, *out_sums;
    void *xs, *ds;
    size_t bytes;
};
inline BackwardSpace backward_space(const Shape& s, void* base) {
    Carver c{static_cast<char*>(base)};
    BackwardSpace w;
    const int64_t ld = padded_hidden(s.hidden), rows = gathered_rows(s);
    if (tile_shape(s)) {  // dg and dv as bf16 side by side, w h bf16
        w.dg = c.take<float>(rows * s.hidden);
        w.dv = nullptr;
        w.wh = c.take<float>(rows * s.hidden / 2);
    } else {
        w.dg = c.take<float>(rows * ld);
        w.dv = c.take<float>(rows * ld);
        w.wh = c.take<float>(rows * ld);
    }
    w.dx = c.take<float>(s.pairs * s.width);
    w.dw_part = c.take<float>(2 * ceil_div(s.hidden, tile_shape(s) ? kTile : kGradientCols) * s.pairs);
    if (tile_shape(s)) {
        w.dot = c.take<float>(ceil_div(s.width, kGatherColumns) * s.pairs);
        w.sums = c.take<float>(most_slots(s) * 4 * s.hidden);
        w.out_sums = c.take<float>(most_slots(s) * (kTile / kGatherRows) * s.width);
    } else {
        w.dot = c.take<float>(s.pairs);
        w.sums = c.take<float>(most_slots(s) * 2 * s.hidden);
        w.out_sums = c.take<float>(most_slots(s) * s.width);
    }
    w.xs = c.take<char>(rows * s.width * static_cast<int64_t>(element(s.dtype)));
    w.ds = c.take<char>(rows * s.width * static_cast<int64_t>(element(s.dtype)));
    w.bytes = c.used;
    return w;
}

int check_shape(const char* what, const Shape& s) {
    if (!float_dtype(s.dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(s.dtype));
    if (s.tokens < 0 || s.width < 1 || s.hidden < 1 || s.experts < 1 || s.top_k < 1)
        return fail(KOEMI_ERR_INVALID, "%s: bad dimension", what);
    if (s.tokens >= (int64_t(1) << 26) || s.top_k > 256 || s.pairs >= (int64_t(1) << 26) || s.width >= (1 << 22) ||
        s.hidden >= (1 << 22) || s.experts >= (1 << 16))
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: shape too large", what);
    // a launch has fewer than 2^32 threads along a dimension: 2^24 workgroups of 256
    const int64_t most = (int64_t(1) << 24) - 8, most_columns = ceil_div(std::max(s.width, s.hidden), 64);
    if (most_slots(s) * most_columns > most || 3 * s.experts * ceil_div(s.width, 64) * ceil_div(s.hidden, 64) > most ||
        s.tokens * ceil_div(s.width, 4) >= (int64_t(1) << 32) - 256)
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: shape too large", what);
    return KOEMI_OK;
}
inline unsigned tiles_grid(int64_t slots, int64_t n_tiles) { return static_cast<unsigned>(ceil_div(slots * n_tiles, 8) * 8); }

// Runs f(BM) for the tile rows of the shape and f's load bytes of a row of `width` elements at base.
template <typename F>
void by_rows(const Shape& s, F f) {
    if (any_rows(s.pairs, s.experts) == 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}
// Whether 16 bytes can be read and written at once from each.
inline bool aligned16(std::initializer_list<const void*> pointers) {
    uintptr_t all = 0;
    for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
    return all % 16 == 0;
}
// Whether the rows of an operand across K can be read eight columns at once.
template <typename T>
bool octets(const void* base, int64_t columns, int64_t ld) {
    return columns % 8 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld * sizeof(T) % 16 == 0;
}
template <typename F>
void by_lies(bool across, F f) {
    if (across) f(std::integral_constant<int, kAcross>{});
    else f(std::integral_constant<int, kStrided>{});
}
template <typename F>
void by_bytes(int bytes, F f) {
    if (bytes == 16) f(std::integral_constant<int, 16>{});
    else if (bytes == 8) f(std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, split_gemm::kElementLoads>{});
}
void find_slots(const Shape& s, const int64_t* offsets, const Slots& slots, hipStream_t q) {
    hipLaunchKernelGGL(slots_kernel, dim3(1), dim3(kSlotThreads), 0, q, offsets, s.experts, s.pairs,
                       slot_rows(s), most_slots(s), slots);
}
template <typename T>
void combine(const float* rows, const int64_t* positions, const int64_t* offsets, const float* weights, float share, void* out,
             const Shape& s, hipStream_t q) {
    hipLaunchKernelGGL(combine_rows_kernel<T>, dim3(grid_for(s.tokens * ceil_div(s.width, 4), 256)), dim3(256), 0, q, rows,
                       positions, offsets + s.experts, weights, share, static_cast<T*>(out), s.tokens, s.width,
                       static_cast<int>(s.top_k));
}

template <typename T>
Between<T>* between(float* p) {
    return reinterpret_cast<Between<T>*>(p);
}

struct Weights {
    const void *Wg, *bg, *Wv, *bv, *Wo, *bo;
};
struct Gradients {
    void *x, *Wg, *bg, *Wv, *bv, *Wo, *bo;
    float* weights;
};

template <typename T>
int any_forward(const Shape& s, const void* x, const int64_t* rows, const int64_t* offsets, const int64_t* positions,
                const float* pair_weights, const Weights& m, void* out, float* keep, const ForwardSpace& w, hipStream_t q) {
    const int64_t ld = padded_hidden(s.hidden), slots = most_slots(s);
    float* keep_v = keep ? keep + s.pairs * ld : nullptr;
    find_slots(s, offsets, w.slots, q);
    by_rows(s, [&](auto rows_tag) {
        constexpr int BM = decltype(rows_tag)::value;
        const int in_bytes = std::min({split_gemm::load_bytes<T>(x, s.width), split_gemm::load_bytes<T>(m.Wg, s.width),
                                       split_gemm::load_bytes<T>(m.Wv, s.width)});
        by_bytes(in_bytes, [&](auto bytes) {
            const uint32_t n = static_cast<uint32_t>(ceil_div(s.hidden, 64));
            hipLaunchKernelGGL((any_hidden_kernel<T, BM, decltype(bytes)::value>), dim3(tiles_grid(slots, n)),
                               dim3(split_gemm::kThreads), 0, q, static_cast<const T*>(x), rows, s.tokens,
                               static_cast<const T*>(m.Wg), static_cast<const T*>(m.bg), static_cast<const T*>(m.Wv),
                               static_cast<const T*>(m.bv), keep, keep_v, w.h, w.slots, slots, s.width, s.hidden, ld, n);
        });
        by_bytes(split_gemm::load_bytes<T>(m.Wo, s.hidden), [&](auto bytes) {
            const uint32_t n = static_cast<uint32_t>(ceil_div(s.width, any_cols(BM)));
            hipLaunchKernelGGL((any_output_kernel<T, BM, decltype(bytes)::value>), dim3(tiles_grid(slots, n)),
                               dim3(split_gemm::kThreads), 0, q, between<T>(w.h), static_cast<const T*>(m.Wo),
                               static_cast<const T*>(m.bo), w.y, w.slots, slots, s.width, s.hidden, ld, n);
        });
    });
    combine<T>(w.y, positions, offsets, pair_weights, 1.0f / static_cast<float>(s.top_k), out, s, q);
    return check_launch("koemi_moe_experts_forward");
}

template <typename T>
int any_backward(const Shape& s, const void* d_out, const void* x, const int64_t* rows, const int64_t* pair_experts,
                 const int64_t* offsets, const int64_t* positions, const float* sorted_w, const Weights& m, const float* keep,
                 const Gradients& d, const BackwardSpace& w, hipStream_t q) {
    const int64_t ld = padded_hidden(s.hidden), slots = most_slots(s);
    const float share = 1.0f / static_cast<float>(s.top_k);
    const T* dy = static_cast<const T*>(d_out);
    T *xs = static_cast<T*>(w.xs), *ds = static_cast<T*>(w.ds);
    const bool want_in = d.Wg || d.Wv, want_out = d.Wo || d.bo;
    if (want_in || want_out || d.weights) {
        auto gather = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(grid_for(s.pairs, 4)), dim3(256), 0, q, static_cast<const T*>(x), dy, rows, offsets,
                               s.experts, static_cast<const T*>(m.bo), pair_experts, want_in ? xs : nullptr,
                               want_out ? ds : nullptr, d.weights ? w.dot : nullptr, s.pairs, s.tokens, s.width);
        };
        constexpr int kPiece = 16 / sizeof(T);
        if (s.width % kPiece == 0 && aligned16({x, d_out, m.bo})) gather(gather_pairs_kernel<T, kPiece>);
        else gather(gather_pairs_kernel<T, 1>);
    }
    const uint32_t h_tiles = static_cast<uint32_t>(ceil_div(s.hidden, kGradientCols));
    const uint32_t w_tiles = static_cast<uint32_t>(ceil_div(s.width, kGradientCols));
    by_rows(s, [&](auto rows_tag) {
        constexpr int BM = decltype(rows_tag)::value;
        by_bytes(split_gemm::load_bytes<T>(d_out, s.width), [&](auto bytes) {
            by_lies(octets<T>(m.Wo, s.hidden, s.hidden), [&](auto lies) {
                hipLaunchKernelGGL((any_hidden_gradient_kernel<T, BM, decltype(bytes)::value, decltype(lies)::value>),
                                   dim3(tiles_grid(slots, h_tiles)), dim3(split_gemm::kThreads), 0, q, dy, rows, s.tokens,
                                   static_cast<const T*>(m.Wo), keep, keep + s.pairs * ld, sorted_w, share, w.dg, w.dv, w.wh,
                                   w.dw_part, w.slots, slots, s.pairs, s.width, s.hidden, ld, h_tiles);
            });
        });
        if (d.x) by_lies(octets<T>(m.Wg, s.width, s.width) && octets<T>(m.Wv, s.width, s.width), [&](auto lies) {
            constexpr int kLies = decltype(lies)::value;
            const dim3 grid(tiles_grid(slots, w_tiles)), threads(split_gemm::kThreads);
            hipLaunchKernelGGL((any_input_gradient_kernel<T, BM, kLies, false>), grid, threads, 0, q, between<T>(w.dg),
                               static_cast<const T*>(m.Wg), w.dx, w.slots, slots, s.width, s.hidden, ld, w_tiles);
            hipLaunchKernelGGL((any_input_gradient_kernel<T, BM, kLies, true>), grid, threads, 0, q, between<T>(w.dv),
                               static_cast<const T*>(m.Wv), w.dx, w.slots, slots, s.width, s.hidden, ld, w_tiles);
        });
    });
    if (d.x) combine<T>(w.dx, positions, offsets, nullptr, 1.0f, d.x, s, q);
    if (d.weights)
        hipLaunchKernelGGL(weight_gradient_kernel, dim3(grid_for(s.pairs, 256)), dim3(256), 0, q, w.dw_part,
                           static_cast<int>(2 * h_tiles), w.dot, 1, rows, positions, offsets + s.experts, d.weights, s.pairs,
                           static_cast<int>(s.top_k));
    // tiles of 64 x 64 where those of 128 x 128 would leave CUs idle
    const int side = s.experts * ceil_div(s.width, 128) * ceil_div(s.hidden, 128) < 256 ? 64 : 128;
    auto multiply = [&](const auto& products) {
        using P = std::decay_t<decltype(products)>;
        using TA = std::remove_const_t<std::remove_pointer_t<decltype(products.one[0].a)>>;
        using TB = std::remove_const_t<std::remove_pointer_t<decltype(products.one[0].b)>>;
        if (!products.count) return;
        auto launch = [&](void (*kernel)(P, uint32_t, const int64_t*, int64_t)) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(s.experts * products.tiles())), dim3(split_gemm::kThreads), 0, q,
                               products, products.tiles(), offsets, s.pairs);
        };
        // the workspace's rows are aligned: both widths in whole octets, or none read as such
        by_lies(s.hidden % 8 == 0 && s.width % 8 == 0, [&](auto lies) {
            constexpr int kLies = decltype(lies)::value;
            if (side == 64) launch(any_weight_gradient_kernel<T, TA, TB, 64, kLies, kLies>);
            else launch(any_weight_gradient_kernel<T, TA, TB, 128, kLies, kLies>);
        });
    };
    WeightProducts<T, Between<T>, T> in;
    WeightProducts<T, T, Between<T>> out;
    if (d.Wg) in.add(between<T>(w.dg), xs, d.Wg, s.hidden, s.width, ld, s.width, side);
    if (d.Wv) in.add(between<T>(w.dv), xs, d.Wv, s.hidden, s.width, ld, s.width, side);
    if constexpr (std::is_same<T, float>::value) {
        if (d.Wo) in.add(ds, w.wh, d.Wo, s.width, s.hidden, s.width, ld, side);
    } else if (d.Wo) {
        out.add(ds, between<T>(w.wh), d.Wo, s.width, s.hidden, s.width, ld, side);
    }
    multiply(in);
    if constexpr (!std::is_same<T, float>::value) multiply(out);
    if (d.bg || d.bv || d.bo) {
        const int64_t most = std::max(s.hidden, s.width);
        const ThreeSums sums{{{w.dg, w.sums, d.bg, ld, 2 * s.hidden, s.hidden, 1},
                              {w.dv, w.sums + s.hidden, d.bv, ld, 2 * s.hidden, s.hidden, 1},
                              {ds, w.out_sums, d.bo, s.width, s.width, s.width, 1}}};
        hipLaunchKernelGGL(slot_sums_kernel<T>, dim3(static_cast<unsigned>(slots), static_cast<unsigned>(ceil_div(most, kWave)), 3),
                           dim3(256), 0, q, sums, sorted_w, share, w.slots, slots, slot_rows(s));
        hipLaunchKernelGGL(expert_sums_kernel<T>, dim3(grid_for(most, 256), static_cast<unsigned>(s.experts), 3), dim3(256), 0, q,
                           sums, w.slots.first);
    }
    return check_launch("koemi_moe_experts_backward");
}

int tile_forward(const Shape& s, const void* x, const int64_t* rows, const int64_t* offsets, const int64_t* positions,
                 const float* pair_weights, const Weights& m, void* out, float* keep, const ForwardSpace& w, hipStream_t q) {
    const int64_t slots = most_slots(s);
    const uint32_t h_tiles = static_cast<uint32_t>(ceil_div(s.hidden, kHiddenTile / 2)),
                   w_tiles = static_cast<uint32_t>(ceil_div(s.width, kTile));
    bf16* h = reinterpret_cast<bf16*>(w.h);
    find_slots(s, offsets, w.slots, q);
    hipLaunchKernelGGL(tile_hidden_kernel<kHiddenTile>, dim3(tiles_grid(slots, h_tiles)), dim3(mfma_stage::kThreads), 0, q,
                       static_cast<const bf16*>(x), rows, s.tokens, static_cast<const bf16*>(m.Wg),
                       static_cast<const bf16*>(m.bg), static_cast<const bf16*>(m.Wv), static_cast<const bf16*>(m.bv), keep,
                       keep ? keep + kept_floats(s) : nullptr, h, w.slots, slots, s.width, s.hidden, h_tiles);
    hipLaunchKernelGGL(tile_output_kernel, dim3(tiles_grid(slots, w_tiles)), dim3(mfma_stage::kThreads), 0, q, h,
                       static_cast<const bf16*>(m.Wo), static_cast<const bf16*>(m.bo), w.y, w.slots, slots, s.width, s.hidden,
                       w_tiles);
    combine<bf16>(w.y, positions, offsets, pair_weights, 1.0f / static_cast<float>(s.top_k), out, s, q);
    return check_launch("koemi_moe_experts_forward(tiles)");
}

int tile_backward(const Shape& s, const void* d_out, const void* x, const int64_t* rows, const int64_t* offsets,
                  const int64_t* positions, const float* sorted_w, const Weights& m, const float* keep, const Gradients& d,
                  const BackwardSpace& w, hipStream_t q) {
    const int64_t slots = most_slots(s), padded = gathered_rows(s);
    const float share = 1.0f / static_cast<float>(s.top_k);
    const uint32_t h_tiles = static_cast<uint32_t>(ceil_div(s.hidden, kTile)), w_tiles = static_cast<uint32_t>(ceil_div(s.width, kTile));
    bf16 *xs = static_cast<bf16*>(w.xs), *ds = static_cast<bf16*>(w.ds);
    bf16 *dgv = reinterpret_cast<bf16*>(w.dg), *wh = reinterpret_cast<bf16*>(w.wh);
    const dim3 threads(mfma_stage::kThreads);
    const unsigned blocks = static_cast<unsigned>(ceil_div(s.width, kGatherColumns));
    hipLaunchKernelGGL(tile_gather_kernel, dim3(static_cast<unsigned>(padded / kGatherRows), blocks), dim3(256), 0, q,
                       static_cast<const bf16*>(x), static_cast<const bf16*>(d_out), rows, static_cast<const bf16*>(m.bo),
                       sorted_w, share, d.Wg || d.Wv ? xs : nullptr, ds, d.weights ? w.dot : nullptr,
                       d.bo ? w.out_sums : nullptr, w.slots, slots, s.pairs, s.tokens, s.width);
    hipLaunchKernelGGL(tile_hidden_gradient_kernel, dim3(tiles_grid(slots, h_tiles)), threads, 0, q, ds,
                       static_cast<const bf16*>(m.Wo), keep, keep + kept_floats(s), sorted_w, share, dgv, wh, w.dw_part,
                       d.bg || d.bv ? w.sums : nullptr, w.slots, slots, s.pairs, s.width, s.hidden, h_tiles);
    if (d.x) {
        hipLaunchKernelGGL(tile_input_gradient_kernel, dim3(tiles_grid(slots, w_tiles)), threads, 0, q, dgv,
                           static_cast<const bf16*>(m.Wg), static_cast<const bf16*>(m.Wv), w.dx, w.slots, slots, s.width,
                           s.hidden, w_tiles);
        combine<bf16>(w.dx, positions, offsets, nullptr, 1.0f, d.x, s, q);
    }
    if (d.weights)
        hipLaunchKernelGGL(weight_gradient_kernel, dim3(grid_for(s.pairs, 256)), dim3(256), 0, q, w.dw_part,
                           static_cast<int>(2 * h_tiles), w.dot, static_cast<int>(blocks), rows, positions, offsets + s.experts,
                           d.weights, s.pairs, static_cast<int>(s.top_k));
    if (d.Wg || d.Wv || d.Wo) {
        const uint32_t tiles = static_cast<uint32_t>(s.experts) * 3 * w_tiles * h_tiles;
        hipLaunchKernelGGL(tile_weight_gradient_kernel, dim3((tiles + 7) / 8 * 8), threads, 0, q, dgv, wh, xs, ds, offsets,
                           w.slots, static_cast<bf16*>(d.Wg), static_cast<bf16*>(d.Wv), static_cast<bf16*>(d.Wo), s.pairs,
                           s.width, s.hidden, w_tiles, h_tiles, tiles);
    }
    if (d.bg || d.bv || d.bo) {
        const ThreeSums sums{{{nullptr, w.sums, d.bg, 0, 2 * s.hidden, s.hidden, 2},
                              {nullptr, w.sums + s.hidden, d.bv, 0, 2 * s.hidden, s.hidden, 2},
                              {nullptr, w.out_sums, d.bo, 0, s.width, s.width, kTile / kGatherRows}}};
        hipLaunchKernelGGL(expert_sums_kernel<bf16>, dim3(grid_for(std::max(s.hidden, s.width), 256), static_cast<unsigned>(s.experts), 3),
                           dim3(256), 0, q, sums, w.slots.first);
    }
    return check_launch("koemi_moe_experts_backward(tiles)");
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_moe_experts_saved_bytes(int64_t tokens, int64_t top_k, int64_t width, int64_t hidden,
                                                int64_t expert_count, int dtype) {
    const Shape s{tokens * top_k, tokens, width, hidden, expert_count, top_k, dtype};
    if (check_shape("koemi_moe_experts_saved_bytes", s) != KOEMI_OK) return 0;
    return saved_space(s, nullptr).bytes;
}

extern "C" size_t koemi_moe_experts_workspace_bytes(int64_t tokens, int64_t top_k, int64_t width, int64_t hidden,
                                                    int64_t expert_count, int dtype, int backward) {
    const Shape s{tokens * top_k, tokens, width, hidden, expert_count, top_k, dtype};
    if (check_shape("koemi_moe_experts_workspace_bytes", s) != KOEMI_OK) return 0;
    return backward ? backward_space(s, nullptr).bytes : forward_space(s, nullptr).bytes;
}

extern "C" int koemi_moe_experts_forward(const void* context, const int64_t* sorted_rows, const int64_t* segment_offsets,
                                         const int64_t* pair_positions, const float* pair_weights, const void* gate_weights,
                                         const void* gate_biases, const void* value_weights, const void* value_biases,
                                         const void* output_weights, const void* output_biases, void* output, void* saved,
                                         int64_t tokens, int64_t top_k, int64_t width, int64_t hidden, int64_t expert_count,
                                         int dtype, void* workspace, size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_moe_experts_forward";
    const Shape s{tokens * top_k, tokens, width, hidden, expert_count, top_k, dtype};
    const int st = check_shape(what, s);
    if (st != KOEMI_OK || tokens == 0) return st;
    const Weights m{gate_weights, gate_biases, value_weights, value_biases, output_weights, output_biases};
    if (!context || !sorted_rows || !segment_offsets || !pair_positions || !m.Wg || !m.bg || !m.Wv || !m.bv || !m.Wo ||
        !m.bo || !output)
        return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    ForwardSpace w = forward_space(s, workspace);
    if (!workspace || workspace_bytes < w.bytes) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    if (!aligned16({saved, workspace})) return fail(KOEMI_ERR_INVALID, "%s: saved and workspace must be 16-byte aligned", what);
    float* keep = nullptr;
    if (saved) {
        const SavedSpace space = saved_space(s, saved);
        keep = space.keep;
        w.slots = space.slots;
    }
    hipStream_t q = as_stream(stream);
    const bool few = !saved && few_rows_mlp_fits(s.pairs, width, hidden, expert_count, dtype);
    if ((tile_shape(s) || few) && !aligned16({context, m.Wg, m.Wv, m.Wo}))
        return fail(KOEMI_ERR_INVALID, "%s: operands must be 16-byte aligned", what);
    if (few) {  // a decode step: bound by the weights, read once
        const int rc = few_rows_mlp(context, sorted_rows, tokens, segment_offsets, m.Wg, m.bg, m.Wv, m.bv, m.Wo, m.bo, w.h, w.y,
                                    s.pairs, width, hidden, expert_count, q);
        if (rc != KOEMI_OK) return rc;
        combine<bf16>(w.y, pair_positions, segment_offsets, pair_weights, 1.0f / static_cast<float>(top_k), output, s, q);
        return check_launch("koemi_moe_experts_forward(few rows)");
    }
    if (tile_shape(s))
        return tile_forward(s, context, sorted_rows, segment_offsets, pair_positions, pair_weights, m, output, keep, w, q);
    if (dtype == KOEMI_F32)
        return any_forward<float>(s, context, sorted_rows, segment_offsets, pair_positions, pair_weights, m, output, keep, w, q);
    if (dtype == KOEMI_F16)
        return any_forward<f16>(s, context, sorted_rows, segment_offsets, pair_positions, pair_weights, m, output, keep, w, q);
    return any_forward<bf16>(s, context, sorted_rows, segment_offsets, pair_positions, pair_weights, m, output, keep, w, q);
}

extern "C" int koemi_moe_experts_backward(const void* grad_output, const void* context, const int64_t* sorted_rows,
                                          const int64_t* sorted_experts, const int64_t* segment_offsets,
                                          const int64_t* pair_positions, const float* sorted_weights, const void* gate_weights,
                                          const void* value_weights, const void* output_weights, const void* output_biases,
                                          const void* saved, void* grad_context, float* grad_pair_weights,
                                          void* grad_gate_weights, void* grad_gate_biases, void* grad_value_weights,
                                          void* grad_value_biases, void* grad_output_weights, void* grad_output_biases,
                                          int64_t tokens, int64_t top_k, int64_t width, int64_t hidden, int64_t expert_count,
                                          int dtype, void* workspace, size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_moe_experts_backward";
    const Shape s{tokens * top_k, tokens, width, hidden, expert_count, top_k, dtype};
    const int st = check_shape(what, s);
    if (st != KOEMI_OK || tokens == 0) return st;
    const Weights m{gate_weights, nullptr, value_weights, nullptr, output_weights, output_biases};
    if (!grad_output || !context || !sorted_rows || !sorted_experts || !segment_offsets || !pair_positions || !m.Wg ||
        !m.Wv || !m.Wo || !m.bo || !saved)
        return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    const Gradients d{grad_context,       grad_gate_weights,   grad_gate_biases,   grad_value_weights,
                      grad_value_biases,  grad_output_weights, grad_output_biases, grad_pair_weights};
    BackwardSpace w = backward_space(s, workspace);
    if (!workspace || workspace_bytes < w.bytes) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    if (!aligned16({saved, workspace})) return fail(KOEMI_ERR_INVALID, "%s: saved and workspace must be 16-byte aligned", what);
    const SavedSpace space = saved_space(s, const_cast<void*>(saved));  // read alone
    const float* keep = space.keep;
    w.slots = space.slots;
    hipStream_t q = as_stream(stream);
    if (tile_shape(s)) {
        if (!aligned16({grad_output, context, m.Wg, m.Wv, m.Wo, m.bo, d.Wg, d.Wv, d.Wo}))
            return fail(KOEMI_ERR_INVALID, "%s: operands must be 16-byte aligned", what);
        return tile_backward(s, grad_output, context, sorted_rows, segment_offsets, pair_positions, sorted_weights, m, keep, d, w,
                             q);
    }
    if (dtype == KOEMI_F32)
        return any_backward<float>(s, grad_output, context, sorted_rows, sorted_experts, segment_offsets, pair_positions,
                                   sorted_weights, m, keep, d, w, q);
    if (dtype == KOEMI_F16)
        return any_backward<f16>(s, grad_output, context, sorted_rows, sorted_experts, segment_offsets, pair_positions,
                                 sorted_weights, m, keep, d, w, q);
    return any_backward<bf16>(s, grad_output, context, sorted_rows, sorted_experts, segment_offsets, pair_positions,
                              sorted_weights, m, keep, d, w, q);
}
