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
// each of the k choices by butterflies over the group. Experts at minus infinity are
// never chosen (the slot is -1, its weight 0), and a token with no other is not routed
// at all, like one that is not valid.
//
// A lane always holds the same experts, so the statistics add up in its registers over
// the workgroup's tokens, then over its groups through LDS, then over the workgroups in
// a second launch: every order is fixed. Bound by memory for many experts, by the two
// launches' latency for a few tokens.
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

// Ordered like the value it comes from, +0 and -0 alike; never 0, which stands for "not to be chosen".
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
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
            struct alignas(sizeof(T) * VPL > 16 ? 16 : sizeof(T) * VPL) Raw {
                T v[VPL];
            };
            if (e0 < experts) {
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
    // p over the group (NaN where a logit is NaN or plus infinity); false: no logit above
    // minus infinity, p is 0.
    __device__ __forceinline__ bool softmax(float (&p)[VPL]) const {
        float m = z[0];
        bool any = false;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            m = fmaxf(m, z[v]);
            any |= z[v] != -__builtin_inff();
        }
        uint32_t some = any;
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) {
            m = fmaxf(m, __shfl_xor(m, off, kWave));
            some |= __shfl_xor(some, off, kWave);
        }
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            p[v] = exp_nonpos(z[v] - m);
            sum += p[v];
        }
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
#pragma unroll
        for (int v = 0; v < VPL; ++v) p[v] = some ? p[v] / sum : 0.0f;
        return some != 0;
    }
};

template <typename T, int G, int VPL>
__global__ __launch_bounds__(kThreads) void route_balanced_kernel(
    const T* __restrict__ logits, int64_t row_stride, const uint8_t* __restrict__ valid, int64_t* __restrict__ out_idx,
    float* __restrict__ out_w, int64_t tokens, int experts, int top_k, int vec, float* __restrict__ part_mass,
    uint32_t* __restrict__ part_counts, uint32_t* __restrict__ part_valid) {
    using K = Token<T, G, VPL>;
    __shared__ float mass_sh[kThreads * VPL];
    __shared__ uint32_t counts_sh[kThreads * VPL];
    __shared__ uint32_t valid_sh[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid % G, group = tid / G, e0 = lane * VPL;
    float mass[VPL];
    uint32_t counts[VPL], routed_tokens = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) mass[v] = 0.0f, counts[v] = 0;
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
            key[v] = token.z[v] == -__builtin_inff() ? 0u : order_key(token.z[v]);
        }
        routed_tokens += routed && lane == 0;
        // the k choices: each lane's best, then the group's; lane s % G keeps choice s
        int64_t my_idx = -1;
        float my_w = 0.0f;
        for (int s = 0; s < top_k; ++s) {
            uint32_t best = key[0];
            int at = 0;
#pragma unroll
            for (int v = 1; v < VPL; ++v)
                if (key[v] > best) best = key[v], at = v;
            uint64_t top = static_cast<uint64_t>(best) << 32 | static_cast<uint32_t>(~(e0 + at));
#pragma unroll
            for (int off = G / 2; off > 0; off >>= 1) {
                const uint32_t hi = __shfl_xor(static_cast<uint32_t>(top >> 32), off, kWave);
                const uint32_t lo = __shfl_xor(static_cast<uint32_t>(top), off, kWave);
                const uint64_t other = static_cast<uint64_t>(hi) << 32 | lo;
                top = other > top ? other : top;
            }
            const bool chosen = (top >> 32) != 0;
            const int e = static_cast<int>(~static_cast<uint32_t>(top));
            float w = 0.0f;
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const bool mine = chosen && e == e0 + v;
                key[v] = mine ? 0u : key[v];
                counts[v] += mine;
                w = mine ? p[v] : w;
            }
            if constexpr (G > 1) w = __shfl(w, (lane_id() & ~(G - 1)) + (chosen ? e / VPL : 0), kWave);
            if (s % G == lane) my_idx = chosen ? e : -1, my_w = chosen ? w : 0.0f;
            if ((s % G == G - 1 || s == top_k - 1) && t < tokens && lane <= s % G) {
                const int64_t o = t * top_k + (s - s % G + lane);
                out_idx[o] = my_idx;
                out_w[o] = my_w;
            }
        }
    }
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) routed_tokens += __shfl_xor(routed_tokens, off, kWave);
    if (lane_id() == 0) valid_sh[tid / kWave] = routed_tokens;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        mass_sh[group * (G * VPL) + e0 + v] = mass[v];
        counts_sh[group * (G * VPL) + e0 + v] = counts[v];
    }
    __syncthreads();
    for (int e = tid; e < experts; e += kThreads) {
        float m = 0.0f;
        uint32_t c = 0;
        for (int g = 0; g < K::kPerBlock; ++g) m += mass_sh[g * (G * VPL) + e], c += counts_sh[g * (G * VPL) + e];
        part_mass[static_cast<int64_t>(blockIdx.x) * experts + e] = m;
        part_counts[static_cast<int64_t>(blockIdx.x) * experts + e] = c;
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
#pragma unroll 4
        for (int b = slice; b < blocks; b += slices) {
            m += part_mass[static_cast<int64_t>(b) * experts + e];
            c += part_counts[static_cast<int64_t>(b) * experts + e];
        }
    for (int b = tid; b < blocks; b += kFinishThreads) n += part_valid[b];
    mass_sh[tid] = m;
    counts_sh[tid] = c;
    const uint32_t routed = block_sum<uint32_t, kFinishThreads>(n, count_scratch);  // (joins: the slices are in LDS)
    m = 0.0f, c = 0;
    if (tid < experts)
        for (int s = 0; s < slices; ++s) m += mass_sh[s * padded + tid], c += counts_sh[s * padded + tid];
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
                const int64_t e = idx[tc * top_k + s];
                const float d = grad_w[tc * top_k + s];
#pragma unroll
                for (int v = 0; v < VPL; ++v) g[v] += e == e0 + v ? d : 0.0f;
            }
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) dot += e0 + v < experts ? p[v] * g[v] : 0.0f;
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) dot += __shfl_xor(dot, off, kWave);
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

// Lanes of a token: the fewest that hold its experts, 4 each up to 256 experts, then 8 and 16.
struct Layout {
    int lanes, per_lane, blocks;
};
inline Layout layout_of(int64_t tokens, int64_t experts) {
    Layout l;
    l.per_lane = experts <= 256 ? 4 : experts <= 512 ? 8 : 16;
    for (l.lanes = 1; l.lanes * l.per_lane < experts; l.lanes *= 2) {
    }
    const int64_t per_block = kThreads / l.lanes;
    l.blocks = static_cast<int>(std::min<int64_t>((tokens + per_block - 1) / per_block, kMaxBlocks));
    return l;
}
template <typename Run>
void by_layout(const Layout& l, Run run) {
    auto wide = [&](auto per) { run(std::integral_constant<int, 64>{}, per); };
    if (l.per_lane == 16) return wide(std::integral_constant<int, 16>{});
    if (l.per_lane == 8) return wide(std::integral_constant<int, 8>{});
    const std::integral_constant<int, 4> four;
    switch (l.lanes) {
        case 1: return run(std::integral_constant<int, 1>{}, four);
        case 2: return run(std::integral_constant<int, 2>{}, four);
        case 4: return run(std::integral_constant<int, 4>{}, four);
        case 8: return run(std::integral_constant<int, 8>{}, four);
        case 16: return run(std::integral_constant<int, 16>{}, four);
        case 32: return run(std::integral_constant<int, 32>{}, four);
        default: return run(std::integral_constant<int, 64>{}, four);
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
