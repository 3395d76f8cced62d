// The learned softmax top-k route with its statistics and balance loss, to be trained.
//
//   p = softmax(z), the k largest logits in descending order (ties to the lower
//   expert), w_s = p at them, mass_e = sum_t p_te, counts_e = the tokens that chose e,
//   loss = E sum_e (mass_e / max(valid, 1)) (counts_e / max(sum counts, 1))
//   dz_e = p_e (g_e - sum_j p_j g_j),
//   g_e = dmass_e + dloss E counts_e / (max(valid, 1) max(sum counts, 1)) + sum_s [a_s = e] dw_s
//
// (model/router.py:11-22, 43-59 of the reference and its autograd; the counts are
// constants there too.) A token lies on a group of 1 to 64 lanes, each with 4, 8 or 16
// consecutive logits in registers: one read of the logits a direction, the softmax and
// each of the k choices by reductions over the group. Experts at minus infinity are
// never chosen (the slot is -1, its weight 0), and a token with no other is not routed
// at all, like one that is not valid.
//
// A lane always holds the same experts, so the mass adds up in its registers over
// the workgroup's tokens, then over its groups through LDS, then over the workgroups in
// a second launch: every order is fixed (the counts are whole numbers). Bound by the latency
// of a token's reductions for many experts (two waves a SIMD in the forward), by the two
// launches' for a few tokens.
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace koemi {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024;
constexpr int kMaxBlocks = 512;        // workgroups whose partial sums the second launch adds
constexpr int kFinishThreads = 1024;

// e^x for x <= 0 within 1.5 units: the product with log2 e in two parts, since v_exp_f32
// alone would see it rounded (20 units of 2^-24 at x = -30). Below -150 the result is 0
// in fp32, minus infinity included; NaN stays.
__device__ __forceinline__ float exp_nonpos(float x) {
    x = x < -150.0f ? -150.0f : x;
    const float hi = x * 1.44269504088896341f;
    const float lo = fmaf(x, 1.925963033500011e-8f, fmaf(x, 1.44269504088896341f, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e, lo * 0.693147180559945309f, e);
}

// The other lanes of a reduction over aligned groups of lanes: mirrored within 2, 4,
// 8 and 16 lanes by data-parallel moves (a mirror pairs the halves as a butterfly does, once
// each half agrees), then by permutes.
template <int SPAN>
__device__ __forceinline__ uint32_t across(uint32_t v) {
    if constexpr (SPAN == 2) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
    else if constexpr (SPAN == 4) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);   // quad_perm 2 3 0 1
    else if constexpr (SPAN == 8) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);  // row_half_mirror
    else if constexpr (SPAN == 16) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true); // row_mirror
    else return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), SPAN / 2, kWave));
}
// v combined over the group's G lanes, the same bits in each.
template <int G, int SPAN = 2, typename V, typename Op>
__device__ __forceinline__ V over_group(V v, Op op) {
    if constexpr (SPAN <= G) return over_group<G, SPAN * 2>(op(v, __builtin_bit_cast(V, across<SPAN>(__builtin_bit_cast(uint32_t, v)))), op);
    else return v;
}

// A logit's place in the order of choices: greater for a larger logit (+0 and -0
// alike), 0 for one that is not to be chosen. For 16-bit logits the low half holds the
// expert, greater for a lower one, so that the largest key names it.
template <typename T>
__device__ __forceinline__ uint32_t choice_key(float v, int e) {
    if (v == -__builtin_inff()) return 0u;
    v += 0.0f;
    if constexpr (sizeof(T) == 2) {
        const uint32_t b = __builtin_bit_cast(uint16_t, from_f32<T>(v));
        return ((b & 0x8000u ? ~b : b | 0x8000u) & 0xffffu) << 16 | static_cast<uint32_t>(0xffff - e);
    } else {
        const uint32_t b = __float_as_uint(v);
        return b & 0x80000000u ? ~b : b | 0x80000000u;
    }
}
template <typename T>
__device__ __forceinline__ float key_value(uint32_t k) {
    if constexpr (sizeof(T) == 2) {
        k >>= 16;
        return to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(k & 0x8000u ? k & 0x7fffu : ~k)));
    } else {
        return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
    }
}

// n values `step` apart, in eight sums and those in pairs: 64 in a row are off by twice as
// much ([64, 16] fp32, the mass: 1.2e-7 of itself, 5e-8 so).
__device__ __forceinline__ float spaced_sum(const float* p, int step, int n) {
    float s[8] = {};
    for (int i = 0; i < n; i += 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += i + j < n ? p[(i + j) * step] : 0.0f;
    return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// The layout of a token: G lanes of VPL experts each.
template <typename T, int G, int VPL>
struct Token {
    static constexpr int kPerBlock = kThreads / G;
    float z[VPL];

    // Row pointers start aligned to VPL elements and hold a multiple of them (vec), or
    // are read one by one; minus infinity past the experts.
    __device__ __forceinline__ void load(const T* row, int e0, int experts, bool vec) {
        if (vec) {
            if (e0 < experts) {
                struct alignas(sizeof(T) * VPL > 16 ? 16 : sizeof(T) * VPL) Raw {
                    T v[VPL];
                };
                const Raw r = *reinterpret_cast<const Raw*>(row + e0);
#pragma unroll
                for (int v = 0; v < VPL; ++v) z[v] = to_f32(r.v[v]);
                return;
            }
#pragma unroll
            for (int v = 0; v < VPL; ++v) z[v] = -__builtin_inff();
        } else {
#pragma unroll
            for (int v = 0; v < VPL; ++v) z[v] = e0 + v < experts ? to_f32(row[e0 + v]) : -__builtin_inff();
        }
    }
    // p over the group (NaN where a logit is NaN or plus infinity), e^(z - most) times
    // scale; false: no logit above minus infinity, p is 0.
    float most, scale;
    __device__ __forceinline__ bool softmax(float (&p)[VPL]) {
        float m = z[0];
        uint32_t any = 0;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            m = fmaxf(m, z[v]);
            any |= z[v] != -__builtin_inff();
        }
        most = over_group<G>(m, [](float a, float b) { return fmaxf(a, b); });
        any = over_group<G>(any, [](uint32_t a, uint32_t b) { return a | b; });
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            p[v] = exp_nonpos(z[v] - most);
            sum += p[v];
        }
        scale = 1.0f / over_group<G>(sum, [](float a, float b) { return a + b; });
#pragma unroll
        for (int v = 0; v < VPL; ++v) p[v] = any ? p[v] * scale : 0.0f;
        return any != 0;
    }
};

template <typename T, int G, int VPL>
__global__ __launch_bounds__(kThreads) void route_balanced_kernel(
    const T* __restrict__ logits, int64_t row_stride, const uint8_t* __restrict__ valid, int64_t* __restrict__ out_idx,
    float* __restrict__ out_w, int64_t tokens, int experts, int top_k, int vec, float* __restrict__ part_mass,
    uint32_t* __restrict__ part_counts, uint32_t* __restrict__ part_valid) {
    using K = Token<T, G, VPL>;
    __shared__ float mass_sh[kThreads * VPL];
    __shared__ uint32_t counts_sh[G * VPL];
    __shared__ uint32_t valid_sh[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid % G, group = tid / G, e0 = lane * VPL;
    float mass[VPL];
    uint32_t routed_tokens = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) mass[v] = 0.0f;
    for (int e = tid; e < G * VPL; e += kThreads) counts_sh[e] = 0;
    __syncthreads();
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * K::kPerBlock; first < tokens;
         first += static_cast<int64_t>(gridDim.x) * K::kPerBlock) {
        const int64_t t = first + group;
        const bool here = t < tokens && valid[min(t, tokens - 1)] != 0;
        K token;
        token.load(logits + min(t, tokens - 1) * row_stride, e0, experts, vec);
        if (!here)
#pragma unroll
            for (int v = 0; v < VPL; ++v) token.z[v] = -__builtin_inff();
        float p[VPL];
        const bool routed = token.softmax(p);
        uint32_t key[VPL];
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            mass[v] += p[v];
            key[v] = choice_key<T>(token.z[v], e0 + v);
        }
        routed_tokens += routed && lane == 0;
        // the k choices: the largest key of the group; lane s % G keeps choice s
        int64_t my_idx = -1;
        uint32_t my_key = 0;
        for (int s = 0; s < top_k; ++s) {
            uint32_t top = key[0];
#pragma unroll
            for (int v = 1; v < VPL; ++v) top = max(top, key[v]);
            top = over_group<G>(top, [](uint32_t a, uint32_t b) { return max(a, b); });
            uint32_t e;
            if constexpr (sizeof(T) == 2) {
                e = 0xffffu - (top & 0xffffu);
            } else {  // the lowest expert that has it
                e = ~0u;
#pragma unroll
                for (int v = VPL - 1; v >= 0; --v) e = key[v] == top ? e0 + v : e;
                e = over_group<G>(e, [](uint32_t a, uint32_t b) { return min(a, b); });
            }
#pragma unroll
            for (int v = 0; v < VPL; ++v) key[v] = e == static_cast<uint32_t>(e0 + v) ? 0u : key[v];
            if (s % G == lane) {
                my_key = top;
                my_idx = top ? static_cast<int64_t>(e) : -1;
                if (top) atomicAdd(&counts_sh[e], 1u);  // whole numbers: any order
            }
            if ((s % G == G - 1 || s == top_k - 1) && t < tokens && lane <= s % G) {
                const int64_t o = t * top_k + (s - s % G + lane);
                out_idx[o] = my_idx;
                out_w[o] = my_key ? exp_nonpos(key_value<T>(my_key) - token.most) * token.scale : 0.0f;
            }
        }
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) routed_tokens += __shfl_xor(routed_tokens, off, kWave);
    if (lane_id() == 0) valid_sh[tid / kWave] = routed_tokens;
#pragma unroll
    for (int v = 0; v < VPL; ++v) mass_sh[group * (G * VPL) + e0 + v] = mass[v];
    __syncthreads();
    for (int e = tid; e < experts; e += kThreads) {
        const float m = spaced_sum(mass_sh + e, G * VPL, K::kPerBlock);
        part_mass[static_cast<int64_t>(blockIdx.x) * experts + e] = m;
        part_counts[static_cast<int64_t>(blockIdx.x) * experts + e] = counts_sh[e];
    }
    if (tid == 0) {
        uint32_t n = 0;
        for (int w = 0; w < kThreads / kWave; ++w) n += valid_sh[w];
        part_valid[blockIdx.x] = n;
    }
}

// Sums v over the workgroup in a fixed order; every thread gets the total.
template <typename V, int THREADS>
__device__ __forceinline__ V block_sum(V v, V* scratch) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    __syncthreads();
    if (lane_id() == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    V total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) total += scratch[w];
    return total;
}

// Adds the workgroups' partial sums: thread (slice, e) every slices-th of them, the
// slices through LDS, then the loss.
__global__ __launch_bounds__(kFinishThreads) void route_balanced_finish_kernel(
    const float* __restrict__ part_mass, const uint32_t* __restrict__ part_counts, const uint32_t* __restrict__ part_valid,
    int blocks, int experts, int padded, float* __restrict__ mass, float* __restrict__ counts,
    float* __restrict__ valid_count, float* __restrict__ loss) {
    __shared__ float mass_sh[kFinishThreads];
    __shared__ uint32_t counts_sh[kFinishThreads];
    __shared__ uint32_t count_scratch[kFinishThreads / kWave];
    __shared__ float scratch[kFinishThreads / kWave];
    const int tid = threadIdx.x, e = tid % padded, slice = tid / padded, slices = kFinishThreads / padded;
    float m = 0.0f;
    uint32_t c = 0, n = 0;
    if (e < experts)
#pragma unroll 8
        for (int b = slice; b < blocks; b += slices) {
            m += part_mass[static_cast<int64_t>(b) * experts + e];
            c += part_counts[static_cast<int64_t>(b) * experts + e];
        }
    for (int b = tid; b < blocks; b += kFinishThreads) n += part_valid[b];
    mass_sh[tid] = m;
    counts_sh[tid] = c;
    const uint32_t routed = block_sum<uint32_t, kFinishThreads>(n, count_scratch);  // (joins: the slices are in LDS)
    m = 0.0f, c = 0;
    if (tid < experts) {
        m = spaced_sum(mass_sh + tid, padded, slices);
        for (int s = 0; s < slices; ++s) c += counts_sh[s * padded + tid];
    }
    const uint32_t total = block_sum<uint32_t, kFinishThreads>(c, count_scratch);
    const float share = tid < experts ? m / fmaxf(static_cast<float>(routed), 1.0f) *
                                            (static_cast<float>(c) / fmaxf(static_cast<float>(total), 1.0f)) : 0.0f;
    const float sum = block_sum<float, kFinishThreads>(share, scratch);
    if (tid < experts) {
        mass[tid] = m;
        counts[tid] = static_cast<float>(c);
    }
    if (tid == 0) {
        valid_count[0] = static_cast<float>(routed);
        loss[0] = static_cast<float>(experts) * sum;
    }
}

// dloss by mass_e: E counts_e / (max(valid, 1) max(sum counts, 1)), the sum over the whole workgroup.
template <int THREADS>
__device__ __forceinline__ float loss_scale(const float* counts, const float* valid_count, const float* grad_loss,
                                            int experts, float* scratch) {
    float c = 0.0f;
    for (int e = threadIdx.x; e < experts; e += THREADS) c += counts[e];
    const float total = block_sum<float, THREADS>(c, scratch);
    return grad_loss[0] * static_cast<float>(experts) / (fmaxf(valid_count[0], 1.0f) * fmaxf(total, 1.0f));
}

template <typename T, int G, int VPL>
__global__ __launch_bounds__(kThreads) void route_balanced_backward_kernel(
    const T* __restrict__ logits, int64_t row_stride, const uint8_t* __restrict__ valid, const int64_t* __restrict__ idx,
    const float* __restrict__ counts, const float* __restrict__ valid_count, const float* __restrict__ grad_w,
    const float* __restrict__ grad_mass, const float* __restrict__ grad_loss, T* __restrict__ grad_logits, int64_t tokens,
    int experts, int top_k, int vec) {
    using K = Token<T, G, VPL>;
    __shared__ float scratch[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid % G, group = tid / G, e0 = lane * VPL;
    const float scale = grad_loss ? loss_scale<kThreads>(counts, valid_count, grad_loss, experts, scratch) : 0.0f;
    float base[VPL];  // what every token adds to g
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const int e = min(e0 + v, experts - 1);
        base[v] = (grad_mass ? grad_mass[e] : 0.0f) + (grad_loss ? scale * counts[e] : 0.0f);
    }
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * K::kPerBlock; first < tokens;
         first += static_cast<int64_t>(gridDim.x) * K::kPerBlock) {
        const int64_t t = first + group, tc = min(t, tokens - 1);
        const bool here = t < tokens && valid[tc] != 0;
        K token;
        token.load(logits + tc * row_stride, e0, experts, vec);
        if (!here)
#pragma unroll
            for (int v = 0; v < VPL; ++v) token.z[v] = -__builtin_inff();
        float p[VPL], g[VPL];
        const bool routed = token.softmax(p);
#pragma unroll
        for (int v = 0; v < VPL; ++v) g[v] = base[v];
        if (grad_w)
            for (int s = 0; s < top_k; ++s) {
                const int e = static_cast<int>(idx[tc * top_k + s]);
                const float d = grad_w[tc * top_k + s];
#pragma unroll
                for (int v = 0; v < VPL; ++v) g[v] += e == e0 + v ? d : 0.0f;
            }
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) dot += p[v] * g[v];  // past the experts p is 0
        dot = over_group<G>(dot, [](float a, float b) { return a + b; });
        if (t >= tokens) continue;
        T* out = grad_logits + t * experts + e0;
        struct alignas(sizeof(T) * VPL > 16 ? 16 : sizeof(T) * VPL) Raw {
            T v[VPL];
        } r;
#pragma unroll
        for (int v = 0; v < VPL; ++v) r.v[v] = from_f32<T>(routed ? p[v] * (g[v] - dot) : 0.0f);
        if (vec) {
            if (e0 < experts) *reinterpret_cast<Raw*>(out) = r;
        } else {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
                if (e0 + v < experts) out[v] = r.v[v];
        }
    }
}

__global__ __launch_bounds__(kThreads) void balance_loss_backward_kernel(const float* __restrict__ counts,
                                                                         const float* __restrict__ valid_count,
                                                                         const float* __restrict__ grad_loss, int64_t experts,
                                                                         float* __restrict__ grad_mass) {
    __shared__ float scratch[kThreads / kWave];
    const float scale = loss_scale<kThreads>(counts, valid_count, grad_loss, static_cast<int>(experts), scratch);
    for (int64_t e = threadIdx.x; e < experts; e += kThreads) grad_mass[e] = scale * counts[e];
}

// Lanes of a token: the fewest that hold its experts, 4 each up to 32 experts, 8 up to
// 64, else 16: fewer lanes reduce in fewer steps, more give small calls more waves
// ([131072, 128] bf16 with top 4: 107 us with 32 lanes of 4).
struct Layout {
    int lanes, per_lane, blocks;
};
inline Layout layout_of(int64_t tokens, int64_t experts) {
    Layout l;
    l.per_lane = experts <= 32 ? 4 : experts <= 64 ? 8 : 16;
    for (l.lanes = 1; l.lanes * l.per_lane < experts; l.lanes *= 2) {
    }
    const int64_t per_block = kThreads / l.lanes;
    l.blocks = static_cast<int>(std::min<int64_t>((tokens + per_block - 1) / per_block, kMaxBlocks));
    return l;
}
template <typename Run>
void by_layout(const Layout& l, Run run) {
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 16> sixteen;
    const std::integral_constant<int, 8> eight;
    if (l.per_lane == 4) switch (l.lanes) {
            case 1: return run(std::integral_constant<int, 1>{}, four);
            case 2: return run(std::integral_constant<int, 2>{}, four);
            case 4: return run(std::integral_constant<int, 4>{}, four);
            default: return run(eight, four);
        }
    if (l.per_lane == 8) return run(eight, eight);
    switch (l.lanes) {
        case 8: return run(eight, sixteen);
        case 16: return run(sixteen, sixteen);
        case 32: return run(std::integral_constant<int, 32>{}, sixteen);
        default: return run(std::integral_constant<int, 64>{}, sixteen);
    }
}
inline bool rows_vector(const void* base, int64_t stride, int64_t experts, int per_lane, int size) {
    const int64_t bytes = std::min(per_lane * size, 16);
    return experts % per_lane == 0 && reinterpret_cast<uintptr_t>(base) % bytes == 0 && stride * size % bytes == 0;
}

inline size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

int check_route(const char* what, const void* logits, int dtype, int64_t row_stride, int64_t tokens, int64_t experts,
                int64_t top_k) {
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (tokens < 0 || experts < 1 || top_k < 1) return fail(KOEMI_ERR_INVALID, "%s: bad dimension", what);
    if (experts > kMaxExperts) return fail(KOEMI_ERR_UNSUPPORTED, "%s: more than %d experts", what, kMaxExperts);
    if (top_k > experts) return fail(KOEMI_ERR_INVALID, "%s: top_k exceeds the experts", what);
    if (tokens > ((int64_t(1) << 32) - 1) / top_k)  // their counts have 32 bits
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: 2^32 choices or more", what);
    if (tokens > 0 && !logits) return fail(KOEMI_ERR_INVALID, "%s: null logits", what);
    if (tokens > 1 && row_stride < experts) return fail(KOEMI_ERR_INVALID, "%s: logit rows overlap", what);
    return KOEMI_OK;
}

template <typename T>
int route_forward(const Layout& l, const void* logits, int64_t stride, const uint8_t* valid, int64_t* idx, float* w,
                  int64_t tokens, int experts, int top_k, float* pm, uint32_t* pc, uint32_t* pv, hipStream_t s) {
    const int vec = rows_vector(logits, stride, experts, l.per_lane, sizeof(T));
    by_layout(l, [&](auto lanes, auto per) {
        hipLaunchKernelGGL((route_balanced_kernel<T, decltype(lanes)::value, decltype(per)::value>), dim3(l.blocks),
                           dim3(kThreads), 0, s, static_cast<const T*>(logits), stride, valid, idx, w, tokens, experts, top_k,
                           vec, pm, pc, pv);
    });
    return check_launch("koemi_moe_route_balanced_forward");
}
template <typename T>
int route_backward(const Layout& l, const void* logits, int64_t stride, const uint8_t* valid, const int64_t* idx,
                   const float* counts, const float* valid_count, const float* dw, const float* dm, const float* dl,
                   void* out, int64_t tokens, int experts, int top_k, hipStream_t s) {
    const int vec = rows_vector(logits, stride, experts, l.per_lane, sizeof(T)) &&
                    rows_vector(out, experts, experts, l.per_lane, sizeof(T));
    by_layout(l, [&](auto lanes, auto per) {
        hipLaunchKernelGGL((route_balanced_backward_kernel<T, decltype(lanes)::value, decltype(per)::value>),
                           dim3(l.blocks * 4), dim3(kThreads), 0, s, static_cast<const T*>(logits), stride, valid, idx, counts,
                           valid_count, dw, dm, dl, static_cast<T*>(out), tokens, experts, top_k, vec);
    });
    return check_launch("koemi_moe_route_balanced_backward");
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" size_t koemi_moe_route_balanced_workspace_bytes(int64_t tokens, int64_t expert_count) {
    if (tokens <= 0 || expert_count < 1 || expert_count > kMaxExperts) return 0;
    const Layout l = layout_of(tokens, expert_count);
    return 2 * align256(static_cast<size_t>(l.blocks) * expert_count * 4) + align256(static_cast<size_t>(l.blocks) * 4);
}

extern "C" int koemi_moe_route_balanced_forward(const void* router_logits, int dtype, int64_t row_stride,
                                                const uint8_t* valid_mask, int64_t* assignments, float* weights,
                                                float* probability_mass, float* assignment_counts, float* valid_count,
                                                float* balance_loss, int64_t tokens, int64_t expert_count, int64_t top_k,
                                                void* workspace, size_t workspace_bytes, koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_moe_route_balanced_forward";
    const int st = check_route(what, router_logits, dtype, row_stride, tokens, expert_count, top_k);
    if (st != KOEMI_OK) return st;
    if (!probability_mass || !assignment_counts || !valid_count || !balance_loss ||
        (tokens > 0 && (!valid_mask || !assignments || !weights)))
        return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    const size_t need = koemi_moe_route_balanced_workspace_bytes(tokens, expert_count);
    if (need && (!workspace || workspace_bytes < need)) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    const Layout l = layout_of(tokens, expert_count);
    const size_t sums = align256(static_cast<size_t>(l.blocks) * expert_count * 4);
    char* ws = static_cast<char*>(workspace);
    float* pm = reinterpret_cast<float*>(ws);
    uint32_t* pc = reinterpret_cast<uint32_t*>(ws + sums);
    uint32_t* pv = reinterpret_cast<uint32_t*>(ws + 2 * sums);
    hipStream_t s = as_stream(stream);
    const int E = static_cast<int>(expert_count), k = static_cast<int>(top_k);
    if (tokens > 0) {
        int rc;
        if (dtype == KOEMI_F32) rc = route_forward<float>(l, router_logits, row_stride, valid_mask, assignments, weights, tokens, E, k, pm, pc, pv, s);
        else if (dtype == KOEMI_F16) rc = route_forward<f16>(l, router_logits, row_stride, valid_mask, assignments, weights, tokens, E, k, pm, pc, pv, s);
        else rc = route_forward<bf16>(l, router_logits, row_stride, valid_mask, assignments, weights, tokens, E, k, pm, pc, pv, s);
        if (rc != KOEMI_OK) return rc;
    }
    int padded = 64;  // whole waves of experts in the second launch
    while (padded < E) padded *= 2;
    hipLaunchKernelGGL(route_balanced_finish_kernel, dim3(1), dim3(kFinishThreads), 0, s, pm, pc, pv, l.blocks, E, padded,
                       probability_mass, assignment_counts, valid_count, balance_loss);
    return check_launch("koemi_moe_route_balanced_forward(finish)");
}

extern "C" int koemi_moe_route_balanced_backward(const void* router_logits, int dtype, int64_t row_stride,
                                                 const uint8_t* valid_mask, const int64_t* assignments,
                                                 const float* assignment_counts, const float* valid_count,
                                                 const float* grad_weights, const float* grad_mass, const float* grad_loss,
                                                 void* grad_logits, int64_t tokens, int64_t expert_count, int64_t top_k,
                                                 koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_moe_route_balanced_backward";
    const int st = check_route(what, router_logits, dtype, row_stride, tokens, expert_count, top_k);
    if (st != KOEMI_OK || tokens == 0) return st;
    if (!valid_mask || !assignments || !assignment_counts || !valid_count || !grad_logits)
        return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    const Layout l = layout_of(tokens, expert_count);
    const int E = static_cast<int>(expert_count), k = static_cast<int>(top_k);
    hipStream_t s = as_stream(stream);
    if (dtype == KOEMI_F32)
        return route_backward<float>(l, router_logits, row_stride, valid_mask, assignments, assignment_counts, valid_count,
                                     grad_weights, grad_mass, grad_loss, grad_logits, tokens, E, k, s);
    if (dtype == KOEMI_F16)
        return route_backward<f16>(l, router_logits, row_stride, valid_mask, assignments, assignment_counts, valid_count,
                                   grad_weights, grad_mass, grad_loss, grad_logits, tokens, E, k, s);
    return route_backward<bf16>(l, router_logits, row_stride, valid_mask, assignments, assignment_counts, valid_count,
                                grad_weights, grad_mass, grad_loss, grad_logits, tokens, E, k, s);
}

extern "C" int koemi_moe_router_balance_loss_backward(const float* assignment_counts, const float* valid_count,
                                                      const float* grad_loss, int64_t expert_count, float* grad_mass,
                                                      koemi_stream_t stream) {
    clear_error();
    if (expert_count < 1 || expert_count > (1 << 20))
        return fail(KOEMI_ERR_INVALID, "koemi_moe_router_balance_loss_backward: bad expert count");
    if (!assignment_counts || !valid_count || !grad_loss || !grad_mass)
        return fail(KOEMI_ERR_INVALID, "koemi_moe_router_balance_loss_backward: null pointer");
    hipLaunchKernelGGL(balance_loss_backward_kernel, dim3(1), dim3(kThreads), 0, as_stream(stream), assignment_counts,
                       valid_count, grad_loss, expert_count, grad_mass);
    return check_launch("koemi_moe_router_balance_loss_backward");
}
