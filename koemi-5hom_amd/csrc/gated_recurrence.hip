// The bounded recurrent state with its gradients, from gate pre-activations.
//
//   s = sigmoid(r), a = 2^-8 + (1 - 2^-7) s, k = 1 - a, u = tanh(c)
//   h_t = a_t h_{t-1} + k_t u_t                 (a masked position: h_t = h_{t-1})
//   g_t = dh_t + a_{t+1} g_{t+1},  g_{L-1} = dh_{L-1} + dfinal
//   dr_t = g_t (h_{t-1} - u_t) (1 - 2^-7) s (1 - s),  dc_t = g_t k_t (1 - u_t^2),
//   dh0 = a_0 g_0
//
// (model/memory.py:14-30 and network.py:306-310 of the reference, whose
// gradients its autograd forms.) Both directions are scans of affine maps
// x -> p x + q, which compose as (p2, q2) o (p1, q1) = (p2 p1, p2 q1 + q2).
//
// A workgroup owns a strip of columns of one batch row and walks a part of the
// sequence in chunks. A chunk's steps lie on LPC lane groups of eight waves,
// kSteps consecutive steps each, a lane two adjacent columns (one where the layout
// allows no pairs): each lane folds its steps into one map, the groups of a wave
// compose theirs by shuffles, the waves theirs through LDS, and then every lane
// runs its steps again from its own entry state. The next chunk's loads are in
// flight meanwhile. Bound by memory and, for 16-bit inputs, as much by the gates
// (four transcendental instructions and about twenty-five others an element).
//
// The backward pass forms h again instead of reading it: the forward keeps the
// fp32 state before every kKeep-th position (1/64 of an element's traffic),
// and a chunk starts from there. That saves the read of h, and the gradients see the
// fp32 states, not states rounded to 16 bits.
//
// Where even narrow strips do not fill the chip (few long rows), the sequence is cut into
// parts that run at once: a first launch folds each part but the last (first, for the
// gradients) into its map, and each part's workgroup composes the maps before it (after it).
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace koemi {
namespace {

constexpr int kSteps = 8;                     // steps of a lane and chunk
constexpr int kWaves = 8;                     // waves of a workgroup
constexpr int kThreads = kWave * kWaves;
constexpr int kKeep = kSteps * kWaves;        // positions between kept states
constexpr int kMaxParts = 64;                 // parts a sequence is cut into at most

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T e[VEC];
};

// One element's gates. e stays finite (an infinite one would make 0 x inf of k);
// the comparisons keep NaN.
struct Gates {
    float a, k, u;    // retention, 1 - retention, candidate
    float ds, du;     // s (1 - s), 1 - u^2
};
__device__ __forceinline__ void exp_pair(float r, float c, float& e, float& d) {
    const float x = r * -1.44269504088896341f;
    e = __builtin_amdgcn_exp2f(x > 126.0f ? 126.0f : x);
    d = __builtin_amdgcn_exp2f(fabsf(c) * -2.88539008177792682f);
}
// s = 1 / (1 + e) and 1 - s = e / (1 + e), so that k (down to 2^-8) loses nothing to a
// subtraction from 1: a and k within 7 units of 2^-24 (the product with log2 e is rounded,
// which costs s or 1 - s 1.3 |r| units more where that one is small, and 2^-8 is not).
// u = (1 - d) / (1 + d), which cancels next to zero; below 3/8 it is c + c^3 P(c^2), P of
// degree 2 with the least largest error of tanh (7e-8 of it). u is within 2.3 units of 2^-24
// of itself below and 4.2 above; the quotient alone is off by 1.5 / c units ([8, 2048, 1024]
// bf16 forward: 32 us with the quotient alone, 35 with P of degree 1 below 3/16 or with this;
// [1, 32768, 512] fp32 forward 44 and 47 beside its fold).
template <bool GRADIENTS>
__device__ __forceinline__ Gates gates_of(float r, float c) {
    Gates o;
    float e, d;
    exp_pair(r, c, e, d);
    const float s = __builtin_amdgcn_rcpf(1.0f + e), w = __builtin_amdgcn_rcpf(1.0f + d), rest = e * s;
    o.a = fmaf(kGateRetentionSpan, s, kGateMinRetention);
    o.k = fmaf(kGateRetentionSpan, rest, kGateMinRetention);
    const float c2 = c * c, p = fmaf(fmaf(-0.0484872918f, c2, 0.132897262f), c2, -0.333323335f);
    o.u = fabsf(c) < 0.375f ? fmaf(c * c2, p, c) : copysignf((1.0f - d) * w, c);
    if constexpr (GRADIENTS) {
        o.ds = s * rest;
        o.du = 4.0f * d * w * w;
    }
    return o;
}
__device__ __forceinline__ float retention_of(float r) {
    return fmaf(kGateRetentionSpan, gate_sigmoid(r), kGateMinRetention);
}

// All bits where step i of the mask is valid. Selects by it cost one instruction and no
// branch, which the compiler puts around a conditional product, spilling what it needs.
__device__ __forceinline__ uint32_t lane_bits(uint32_t mask, int i) {
    return static_cast<uint32_t>(static_cast<int32_t>(mask << (31 - i)) >> 31);
}
__device__ __forceinline__ float or_zero(float v, uint32_t bits) { return __uint_as_float(__float_as_uint(v) & bits); }
__device__ __forceinline__ float or_one(float v, uint32_t bits) {
    return __uint_as_float((__float_as_uint(v) & bits) | (0x3f800000u & ~bits));
}

// What both directions work on. z: r in the first `width` columns of a row, c in
// the next; rows z_row elements apart, batch rows z_batch.
struct Sequence {
    const void* z;
    int64_t z_batch, z_row;
    const uint8_t* valid;  // [batch, length] or null
    int64_t batch, length, width;
    int64_t strips, parts, part_steps;
};

template <int VEC, int LPC>
struct Place {
    static constexpr int kLanes = kWave / LPC;       // lanes of a group
    static constexpr int kColumns = kLanes * VEC;    // columns of a strip
    static constexpr int kChunk = kKeep * LPC;       // steps of a chunk
    int wave, group, lane;       // lane: of its group
    int64_t b, part;
    uint32_t f;                  // the lane's first column
    bool inside;                 // its columns exist
    uint32_t segment;            // the lane's first step in a chunk

    // Workgroup i runs on XCD i % 8: each XCD takes a contiguous range of
    // (batch row, part, strip), so that strips that share cache lines share an L2.
    __device__ __forceinline__ bool place(const Sequence& q) {
        const uint32_t total = static_cast<uint32_t>(q.batch * q.parts * q.strips), per = (total + 7) / 8;
        const uint32_t i = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        if ((blockIdx.x >> 3) >= per || i >= total) return false;
        const uint32_t strip = i % static_cast<uint32_t>(q.strips), rest = i / static_cast<uint32_t>(q.strips);
        part = rest % static_cast<uint32_t>(q.parts);
        b = rest / static_cast<uint32_t>(q.parts);
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        group = lane_id() / kLanes;
        lane = lane_id() % kLanes;
        f = strip * kColumns + lane * VEC;
        inside = f < q.width;
        if (!inside) f = 0;
        segment = static_cast<uint32_t>((wave * LPC + group) * kSteps);
        return true;
    }
};

// The rows of one chunk of an array as a buffer: row t of the array starts at base + t
// row (elements; base, t0 and end the same for the whole workgroup). Reads past `end`
// give 0 and writes there are dropped, so that a chunk needs no bounds of its own, and
// an address is one 32-bit offset (the entry points bound the rows). A chunk that is
// not there (t0 outside [0, end), or no array) has no rows: its reads give 0 without a
// branch, which would let the compiler move the loads away from where they stand.
template <typename T, int VEC, typename P>
struct Rows {
    __amdgpu_buffer_rsrc_t buffer;
    uint32_t step, first;  // bytes

    __device__ __forceinline__ Rows(const T* base, int64_t row, int64_t t0, int64_t end, const P& at) {
        const int64_t rows = base && t0 >= 0 && t0 < end ? min(end - t0, static_cast<int64_t>(P::kChunk)) : 0;
        step = static_cast<uint32_t>(row) * static_cast<uint32_t>(sizeof(T));
        buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + t0 * row), 0,
                                                   static_cast<int>(static_cast<uint32_t>(rows) * step), 0x00020000);
        first = at.segment * step + at.f * static_cast<uint32_t>(sizeof(T));
        asm volatile("" : "+v"(first));  // the offsets of a step are formed in the chunk: hoisted they cost 24 registers
    }
    __device__ __forceinline__ void load(Pack<T, VEC> (&o)[kSteps]) const {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const uint32_t off = first + i * step;
            if constexpr (sizeof(T) * VEC == 2)
                o[i] = __builtin_bit_cast(Pack<T, VEC>, __builtin_amdgcn_raw_buffer_load_b16(buffer, off, 0, 0));
            else if constexpr (sizeof(T) * VEC == 4)
                o[i] = __builtin_bit_cast(Pack<T, VEC>, __builtin_amdgcn_raw_buffer_load_b32(buffer, off, 0, 0));
            else
                o[i] = __builtin_bit_cast(Pack<T, VEC>, __builtin_amdgcn_raw_buffer_load_b64(buffer, off, 0, 0));
        }
    }
    __device__ __forceinline__ void store(int i, const Pack<T, VEC>& v) const {
        const uint32_t off = first + i * step;
        if constexpr (sizeof(T) * VEC == 2)
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), buffer, off, 0, 0);
        else if constexpr (sizeof(T) * VEC == 4)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), buffer, off, 0, 0);
        else {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), buffer, off, 0, 0);
        }
    }
};
// The valid bytes of a chunk: each of a group's first eight lanes loads one step's, and
// the mask (bit i: the lane's step i is before `end` and valid) is formed when they are
// used, since forming it waits for them.
template <typename P>
struct Valid {
    uint32_t byte, rows;

    __device__ __forceinline__ void load(const uint8_t* valid, int64_t t0, int64_t end, const P& at) {
        rows = static_cast<uint32_t>(t0 >= 0 && t0 < end ? min(end - t0, static_cast<int64_t>(P::kChunk)) : 0);
        const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(valid + t0), 0, static_cast<int>(valid ? rows : 0), 0x00020000);
        byte = __builtin_amdgcn_raw_buffer_load_b8(buffer, at.segment + (at.lane & (kSteps - 1)), 0, 0);
    }
    __device__ __forceinline__ uint32_t mask(const uint8_t* valid, const P& at) const {
        const bool ok = (byte != 0 || !valid) && at.segment + (at.lane & (kSteps - 1)) < rows;
        return static_cast<uint32_t>(__ballot(ok) >> (at.group * P::kLanes)) & ((1u << kSteps) - 1);
    }
};

// (p, q) of this lane's group composed with those of the groups before it
// (REVERSE: after it) in the wave, itself included; before/after alone in (xp, xq).
template <int LPC, bool REVERSE>
__device__ __forceinline__ void scan_groups(float& p, float& q, float& xp, float& xq, int group) {
    constexpr int kLanes = kWave / LPC;
    xp = 1.0f, xq = 0.0f;
    if constexpr (LPC > 1) {
#pragma unroll
        for (int off = 1; off < LPC; off <<= 1) {
            const float op = REVERSE ? __shfl_down(p, off * kLanes, kWave) : __shfl_up(p, off * kLanes, kWave);
            const float oq = REVERSE ? __shfl_down(q, off * kLanes, kWave) : __shfl_up(q, off * kLanes, kWave);
            const bool has = REVERSE ? group + off < LPC : group >= off;
            q = has ? fmaf(p, oq, q) : q;
            p = has ? p * op : p;
        }
        const float op = REVERSE ? __shfl_down(p, kLanes, kWave) : __shfl_up(p, kLanes, kWave);
        const float oq = REVERSE ? __shfl_down(q, kLanes, kWave) : __shfl_up(q, kLanes, kWave);
        const bool has = REVERSE ? group + 1 < LPC : group > 0;
        xp = has ? op : 1.0f;
        xq = has ? oq : 0.0f;
    }
}

// The state before every kKeep-th position lies at kept[(b * rows + t / kKeep) * width + f].
__device__ __forceinline__ int64_t kept_rows(int64_t length) { return (length + kKeep - 1) / kKeep; }

// x through `count` parts' maps, the first at maps[cell], the next `step` after it: eight
// parts' loads are under way at once ([1, 32768, 512] fp32, 32 parts, one by one: forward 51
// us, backward 81; so 43 and 78).
template <int VEC>
__device__ __forceinline__ void through_maps(float (&x)[VEC], const float* __restrict__ maps, int64_t cells, int64_t cell,
                                             int64_t step, int64_t count) {
    constexpr int kAhead = 8;
    for (int64_t j = 0; j < count; j += kAhead) {
        Pack<float, VEC> p[kAhead], q[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t at = cell + min(j + i, count - 1) * step;
            p[i] = *reinterpret_cast<const Pack<float, VEC>*>(maps + at);
            q[i] = *reinterpret_cast<const Pack<float, VEC>*>(maps + cells + at);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) x[v] = j + i < count ? fmaf(p[i].e[v], x[v], q[i].e[v]) : x[v];
    }
}

// Each part's map but the last's (REVERSE: the adjoint's, x -> a (d + x) from the last step to
// the first, but the first's) into maps[2, batch, parts, width] (p, then q). A wave folds an
// eighth of the part by itself and the waves' maps meet once, at the end. [1, 32768, 512]
// fp32, 134 MB either way: 37 us (43 in chunks of the workgroup; half of it the gates) and
// 24; loads two or three blocks ahead 39 to 45 and no faster.
template <typename T, int VEC, int LPC, bool REVERSE>
__global__ __launch_bounds__(kThreads) void recurrence_fold_kernel(Sequence s, const T* __restrict__ d_states,
                                                                   float* __restrict__ maps) {
    using P = Place<VEC, LPC>;
    constexpr int kBlock = kSteps * LPC;
    __shared__ float wave_p[kWaves][P::kColumns], wave_q[kWaves][P::kColumns];
    P at;
    if (!at.place(s)) return;
    if (at.part == (REVERSE ? 0 : s.parts - 1)) return;
    at.segment = static_cast<uint32_t>(at.group * kSteps);
    const int64_t share = s.part_steps / kWaves, begin = at.part * s.part_steps + at.wave * share;
    const int64_t end = min(s.length, begin + share), blocks = max((end - begin + kBlock - 1) / kBlock, int64_t(0));
    const T* zr = static_cast<const T*>(s.z) + at.b * s.z_batch;
    const T* other = REVERSE ? d_states ? d_states + at.b * s.length * s.width : nullptr : zr + s.width;
    const int64_t other_row = REVERSE ? s.width : s.z_row;
    const uint8_t* valid = s.valid ? s.valid + at.b * s.length : nullptr;
    struct Raw {
        Pack<T, VEC> r[kSteps], o[kSteps];
        Valid<P> valid;
    } raw;
    auto fetch = [&](int64_t i) {  // block i in the order of the fold; none past the last: an identity
        const int64_t t0 = i < blocks ? begin + (REVERSE ? blocks - 1 - i : i) * kBlock : -1;
        Rows<T, VEC, P>(zr, s.z_row, t0, end, at).load(raw.r);
        Rows<T, VEC, P>(other, other_row, t0, end, at).load(raw.o);
        raw.valid.load(valid, t0, end, at);
    };
    float whole_p[VEC], whole_q[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) whole_p[v] = 1.0f, whole_q[v] = 0.0f;
    fetch(0);
    for (int64_t i = 0; i < blocks; ++i) {
        float p[VEC], q[VEC], xp[VEC], xq[VEC];
        const uint32_t mask = raw.valid.mask(valid, at);
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[v] = 1.0f, q[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int step = REVERSE ? kSteps - 1 - k : k;
            const uint32_t bits = lane_bits(mask, step);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float r = to_f32(raw.r[step].e[v]), o = to_f32(raw.o[step].e[v]);
                if constexpr (REVERSE) {
                    const float a = or_one(retention_of(r), bits);
                    q[v] = a * (o + q[v]);
                    p[v] *= a;
                } else {
                    const Gates g = gates_of<false>(r, o);
                    const float a = or_one(g.a, bits);
                    q[v] = fmaf(a, q[v], or_zero(g.k * g.u, bits));
                    p[v] *= a;
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // as in the walks: the next loads run under the rest
        fetch(i + 1);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            scan_groups<LPC, REVERSE>(p[v], q[v], xp[v], xq[v], at.group);
            whole_q[v] = fmaf(p[v], whole_q[v], q[v]);  // right in the last group (REVERSE: the first)
            whole_p[v] *= p[v];
        }
    }
    if (at.group == (REVERSE ? 0 : LPC - 1))
#pragma unroll
        for (int v = 0; v < VEC; ++v) wave_p[at.wave][at.lane * VEC + v] = whole_p[v], wave_q[at.wave][at.lane * VEC + v] = whole_q[v];
    __syncthreads();
    if (!at.inside || at.wave != 0 || at.group != 0) return;
    const int64_t cell = (at.b * s.parts + at.part) * s.width + at.f, cells = s.batch * s.parts * s.width;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float p = 1.0f, q = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            const int w = REVERSE ? kWaves - 1 - k : k;
            const float wp = wave_p[w][at.lane * VEC + v];
            q = fmaf(wp, q, wave_q[w][at.lane * VEC + v]);
            p *= wp;
        }
        maps[cell + v] = p;
        maps[cells + cell + v] = q;
    }
}

// Forward, each part from the initial state through the maps before it.
template <typename T, int VEC, int LPC>
__global__ __launch_bounds__(kThreads) void recurrence_forward_kernel(Sequence s, const float* __restrict__ initial,
                                                                      T* __restrict__ states, float* __restrict__ final_state,
                                                                      float* __restrict__ kept, float* __restrict__ maps) {
    using P = Place<VEC, LPC>;
    __shared__ float wave_p[2][kWaves][P::kColumns], wave_q[2][kWaves][P::kColumns];
    P at;
    if (!at.place(s)) return;
    const int64_t begin = at.part * s.part_steps, end = min(s.length, begin + s.part_steps);
    const T* zr = static_cast<const T*>(s.z) + at.b * s.z_batch;
    const T* zc = zr + s.width;
    const uint8_t* valid = s.valid ? s.valid + at.b * s.length : nullptr;
    const int64_t cells = s.batch * s.parts * s.width;
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = !initial || !at.inside ? 0.0f : initial[at.b * s.width + at.f + v];
    struct Raw {
        Pack<T, VEC> r[kSteps], c[kSteps];
        Valid<P> valid;
    };
    auto fetch = [&](int64_t t0, Raw& o) {
        Rows<T, VEC, P>(zr, s.z_row, t0, end, at).load(o.r);
        Rows<T, VEC, P>(zc, s.z_row, t0, end, at).load(o.c);
        o.valid.load(valid, t0, end, at);
    };
    int turn = 0;
    Raw raw;
    if (begin < end) fetch(begin, raw);
    through_maps<VEC>(carry, maps, cells, at.b * s.parts * s.width + at.f, s.width, at.part);
    for (int64_t t0 = begin; t0 < end; t0 += P::kChunk) {
        float a[kSteps][VEC], b[kSteps][VEC], p[VEC], q[VEC], xp[VEC], xq[VEC];
        const uint32_t mask = raw.valid.mask(valid, at);
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[v] = 1.0f, q[v] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const uint32_t bits = lane_bits(mask, i);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gates g = gates_of<false>(to_f32(raw.r[i].e[v]), to_f32(raw.c[i].e[v]));
                a[i][v] = or_one(g.a, bits);
                b[i][v] = or_zero(g.k * g.u, bits);
                q[v] = fmaf(a[i][v], q[v], b[i][v]);
                p[v] *= a[i][v];
            }
        }
        // the gates are formed: the next chunk's loads run under the rest, in the same registers
        __builtin_amdgcn_sched_barrier(0);
        fetch(t0 + P::kChunk, raw);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            scan_groups<LPC, false>(p[v], q[v], xp[v], xq[v], at.group);
            if (at.group == LPC - 1) {
                wave_p[turn][at.wave][at.lane * VEC + v] = p[v];
                wave_q[turn][at.wave][at.lane * VEC + v] = q[v];
            }
        }
        __syncthreads();  // the other buffer's readers are past it: they have written this one
        float in[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float x = carry[v];
            in[v] = x;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                if (w == at.wave) in[v] = x;
                x = fmaf(wave_p[turn][w][at.lane * VEC + v], x, wave_q[turn][w][at.lane * VEC + v]);
            }
            carry[v] = x;
            in[v] = fmaf(xp[v], in[v], xq[v]);
        }
        turn ^= 1;
        if (!at.inside) continue;
        const int64_t t = t0 + at.segment;
        if (kept && t % kKeep == 0 && t < end) {
            Pack<float, VEC> k;
#pragma unroll
            for (int v = 0; v < VEC; ++v) k.e[v] = in[v];
            *reinterpret_cast<Pack<float, VEC>*>(kept + (at.b * kept_rows(s.length) + t / kKeep) * s.width + at.f) = k;
        }
        const Rows<T, VEC, P> out(states + at.b * s.length * s.width, s.width, t0, end, at);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            Pack<T, VEC> h;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                in[v] = fmaf(a[i][v], in[v], b[i][v]);
                h.e[v] = from_f32<T>(in[v]);
            }
            out.store(i, h);
        }
    }
    if (!at.inside || at.wave != 0 || at.group != 0 || at.part != s.parts - 1) return;
#pragma unroll
    for (int v = 0; v < VEC; ++v) final_state[at.b * s.width + at.f + v] = carry[v];
}

// Backward, from the last chunk to the first, through the maps of the parts after. The carry
// is a_{t+1} g_{t+1}.
template <typename T, int VEC, int LPC>
__global__ __launch_bounds__(kThreads) void recurrence_backward_kernel(
    Sequence s, const float* __restrict__ kept, const T* __restrict__ d_states, const float* __restrict__ d_final,
    T* __restrict__ d_z, float* __restrict__ d_initial, float* __restrict__ maps) {
    using P = Place<VEC, LPC>;
    __shared__ float wave_p[2][kWaves][P::kColumns], wave_q[2][kWaves][P::kColumns], wave_h[2][kWaves][P::kColumns];
    P at;
    if (!at.place(s)) return;
    const int64_t begin = at.part * s.part_steps, end = min(s.length, begin + s.part_steps);
    const T* zr = static_cast<const T*>(s.z) + at.b * s.z_batch;
    const T* zc = zr + s.width;
    const T* up = d_states ? d_states + at.b * s.length * s.width : nullptr;
    const uint8_t* valid = s.valid ? s.valid + at.b * s.length : nullptr;
    const int64_t cells = s.batch * s.parts * s.width;
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = !d_final || !at.inside ? 0.0f : d_final[at.b * s.width + at.f + v];
    struct Raw {
        Pack<T, VEC> r[kSteps], c[kSteps], d[kSteps];
        Pack<float, VEC> h;
        Valid<P> valid;
    };
    auto fetch = [&](int64_t t0, Raw& o) {
        Rows<T, VEC, P>(zr, s.z_row, t0, end, at).load(o.r);
        Rows<T, VEC, P>(up, s.width, t0, end, at).load(o.d);
        Rows<T, VEC, P>(zc, s.z_row, t0, end, at).load(o.c);
        const int64_t row = at.b * kept_rows(s.length) + max(t0, int64_t(0)) / kKeep;
        o.h = *reinterpret_cast<const Pack<float, VEC>*>(kept + row * s.width + at.f);
        o.valid.load(valid, t0, end, at);
    };
    int turn = 0;
    Raw raw;
    const int64_t last = begin + (end - begin - 1) / P::kChunk * P::kChunk;
    if (begin < end) fetch(last, raw);
    through_maps<VEC>(carry, maps, cells, ((at.b + 1) * s.parts - 1) * s.width + at.f, -s.width, s.parts - 1 - at.part);
    for (int64_t t0 = last; begin < end && t0 >= begin; t0 -= P::kChunk) {
        // x: an element's increment, then the state before it; cr, cc: what g times
        // (h_{t-1} - u) and g are multiplied by for dr and dc
        float a[kSteps][VEC], d[kSteps][VEC], x[kSteps][VEC], u[kSteps][VEC], cr[kSteps][VEC], cc[kSteps][VEC];
        float p[VEC], q[VEC], fp[VEC], fq[VEC], xp[VEC], xq[VEC], yp[VEC], yq[VEC];
        const uint32_t mask = raw.valid.mask(valid, at);
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[v] = 1.0f, q[v] = 0.0f, fq[v] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const uint32_t bits = lane_bits(mask, i);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Gates g = gates_of<true>(to_f32(raw.r[i].e[v]), to_f32(raw.c[i].e[v]));
                a[i][v] = or_one(g.a, bits);
                x[i][v] = or_zero(g.k * g.u, bits);
                u[i][v] = g.u;
                cr[i][v] = kGateRetentionSpan * g.ds;
                cc[i][v] = g.k * g.du;
                fq[v] = fmaf(a[i][v], fq[v], x[i][v]);
                p[v] *= a[i][v];
                d[i][v] = to_f32(raw.d[i].e[v]);
            }
        }
        float start[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) start[v] = raw.h.e[v];
        // the gates are formed: the next chunk's loads run under the rest, in the same registers
        __builtin_amdgcn_sched_barrier(0);
        fetch(t0 - P::kChunk, raw);
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) q[v] = a[i][v] * (d[i][v] + q[v]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            fp[v] = p[v];
            scan_groups<LPC, true>(p[v], q[v], xp[v], xq[v], at.group);
            scan_groups<LPC, false>(fp[v], fq[v], yp[v], yq[v], at.group);
            if (at.group == 0) {
                wave_p[turn][at.wave][at.lane * VEC + v] = p[v];
                wave_q[turn][at.wave][at.lane * VEC + v] = q[v];
            }
            if (at.group == LPC - 1) wave_h[turn][at.wave][at.lane * VEC + v] = fq[v];
        }
        __syncthreads();  // the other buffer's readers are past it: they have written this one
        float in[VEC], h[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float c = carry[v];
            in[v] = c;
            float y = start[v];
            h[v] = y;
            float wp[kWaves];
#pragma unroll
            for (int w = kWaves - 1; w >= 0; --w) {
                if (w == at.wave) in[v] = c;
                wp[w] = wave_p[turn][w][at.lane * VEC + v];
                c = fmaf(wp[w], c, wave_q[turn][w][at.lane * VEC + v]);
            }
            carry[v] = c;
#pragma unroll
            for (int w = 0; w < kWaves - 1; ++w) {
                y = fmaf(wp[w], y, wave_h[turn][w][at.lane * VEC + v]);
                if (w + 1 == at.wave) h[v] = y;
            }
            in[v] = fmaf(xp[v], in[v], xq[v]);
            h[v] = fmaf(yp[v], h[v], yq[v]);
        }
        turn ^= 1;
        if (!at.inside) continue;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float next = fmaf(a[i][v], h[v], x[i][v]);
                x[i][v] = h[v];
                h[v] = next;
            }
        T* out = d_z + at.b * s.length * 2 * s.width;
        const Rows<T, VEC, P> out_r(out, 2 * s.width, t0, end, at), out_c(out + s.width, 2 * s.width, t0, end, at);
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            Pack<T, VEC> dr, dc;
            const uint32_t bits = lane_bits(mask, i);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float g = d[i][v] + in[v];
                in[v] = a[i][v] * g;
                dr.e[v] = from_f32<T>(or_zero(g * (x[i][v] - u[i][v]) * cr[i][v], bits));
                dc.e[v] = from_f32<T>(or_zero(g * cc[i][v], bits));
            }
            out_r.store(i, dr);
            out_c.store(i, dc);
        }
    }
    if (!at.inside || at.wave != 0 || at.group != 0 || at.part != 0 || !d_initial) return;
#pragma unroll
    for (int v = 0; v < VEC; ++v) d_initial[at.b * s.width + at.f + v] = carry[v];
}

// How a call is laid out: two columns a lane where rows allow it, strips that leave a CU the
// least work, and parts where they leave most of the chip idle.
struct Plan {
    int vec, lpc;
    int64_t strips, parts, part_steps;
};
// whole: workgroups that run at once on 256 CUs. The registers let two of the forward's share
// a CU and one of the backward's (bf16 [16, 2048, 1024] backward: 82 us as 256, 92 as 512).
// Strips have 16 lanes at least, so that [8, 2048, 1024] has 256 workgroups forward too.
// parts: from how many on they pay for the fold (bf16 [4, 2048, 1024] in two: forward 12 + 16 us
// against 26, backward 8 + 23 against 38). They fill the chip once: more only hand on more maps
// (bf16 [1, 32768, 512] backward: 43 us in 32 parts of eight strips, 55 in 64).
struct Fill {
    int64_t whole, parts;
};
constexpr Fill kForwardFill{512, 3}, kBackwardFill{256, 2};
constexpr int64_t kPartFill = 256;
constexpr int64_t kMostGroups = (int64_t(1) << 23) - 8;  // a launch has fewer than 2^32 threads, of 512 a workgroup

inline Plan plan_of(int64_t batch, int64_t length, int64_t width, int vec, int size, Fill fill) {
    Plan p;
    p.vec = vec;
    auto strips_of = [&](int lpc) {
        const int64_t columns = kWave / lpc * vec;
        return (width + columns - 1) / columns;
    };
    int64_t least = 0;
    for (int lpc = 1; lpc <= 4; lpc *= 2) {  // rounds of the chip times columns
        if (lpc > 1 && batch * strips_of(lpc) > kMostGroups) break;  // the widest strips always fit (check_sequence)
        const int64_t cost = (batch * strips_of(lpc) + fill.whole - 1) / fill.whole * (kWave / lpc);
        if (lpc == 1 || cost < least) p.lpc = lpc, least = cost;
    }
    p.strips = strips_of(p.lpc);
    p.parts = 1;
    if (batch * p.strips * fill.parts <= kPartFill) {
        // where parts fill the chip all the same, a strip's row has a cache line's 128 bytes
        // ([1, 32768, 512] fp32 backward: 80 us and 31 for the maps with 64 bytes, 63 and 24)
        const int whole = vec * size / 2;
        if (batch * strips_of(whole) * std::min<int64_t>(kMaxParts, length / (kKeep * whole) / 4) >= kPartFill / 2) {
            p.lpc = whole;
            p.strips = strips_of(whole);
        }
        const int64_t chunks = (length + kKeep * p.lpc - 1) / (kKeep * p.lpc);
        if (chunks >= 8) p.parts = std::min<int64_t>(std::min<int64_t>(kMaxParts, chunks / 4), kPartFill / (batch * p.strips));
    }
    const int64_t chunk = static_cast<int64_t>(kKeep) * p.lpc, chunks = (length + chunk - 1) / chunk;
    p.part_steps = std::max<int64_t>((chunks + p.parts - 1) / p.parts, 1) * chunk;
    p.parts = std::max<int64_t>((length + p.part_steps - 1) / p.part_steps, 1);
    return p;
}
// Every row of the arrays starts where two elements load at once.
inline bool pairs_fit(const void* z, int64_t z_batch, int64_t z_row, int64_t width, int dtype, const void* x,
                      const void* y, const void* kept) {
    const uintptr_t two = dtype == KOEMI_F32 ? 8 : 4;
    const uintptr_t bases = reinterpret_cast<uintptr_t>(z) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
    return width % 2 == 0 && z_batch % 2 == 0 && z_row % 2 == 0 && bases % two == 0 &&
           reinterpret_cast<uintptr_t>(kept) % 8 == 0;
}
inline size_t maps_bytes(const Plan& p, int64_t batch, int64_t width) {
    return p.parts > 1 ? static_cast<size_t>(2 * batch * p.parts * width) * sizeof(float) : 0;
}

int check_sequence(const char* what, const void* z, int64_t z_batch, int64_t z_row, int dtype, int64_t batch, int64_t length,
                   int64_t width) {
    if (!float_dtype(dtype)) return fail(KOEMI_ERR_UNSUPPORTED, "%s: unsupported dtype %s", what, dtype_name(dtype));
    if (batch < 0 || length < 0 || width < 0) return fail(KOEMI_ERR_INVALID, "%s: negative dimension", what);
    if (batch == 0 || width == 0) return KOEMI_OK;
    if (length > 0 && !z) return fail(KOEMI_ERR_INVALID, "%s: null pre-activations", what);
    if (length > 1 && z_row < 2 * width) return fail(KOEMI_ERR_INVALID, "%s: pre-activation rows overlap", what);
    const __int128 cells = static_cast<__int128>(batch) * width * (length + 1) * 8;
    if (cells > (static_cast<__int128>(1) << 60)) return fail(KOEMI_ERR_INVALID, "%s: too many elements", what);
    // plan_of takes strips of 64 columns or more where narrower ones would be too many
    if (static_cast<__int128>(batch) * ((width + 63) / 64) > kMostGroups)
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: more than 2^23 strips of 64 columns", what);
    // offsets inside a chunk of four lane groups of kKeep rows have 32 bits
    const int64_t row = std::max<int64_t>(length > 1 ? z_row : 0, 2 * width);
    if (row > (int64_t(1) << 32) / (4 * kKeep * 4) - 1)
        return fail(KOEMI_ERR_UNSUPPORTED, "%s: rows of more than 2^22 elements", what);
    return KOEMI_OK;
}

unsigned grid_of(const Sequence& s) { return static_cast<unsigned>((s.batch * s.parts * s.strips + 7) / 8 * 8); }

// Calls run(std::integral_constant VEC, LPC) of the plan; MOST: columns of a lane at most.
template <int MOST, typename Run>
void by_plan(const Plan& p, Run run) {
    auto lanes = [&](auto vec) {
        if (p.lpc == 1) run(vec, std::integral_constant<int, 1>{});
        else if (p.lpc == 2) run(vec, std::integral_constant<int, 2>{});
        else run(vec, std::integral_constant<int, 4>{});
    };
    if constexpr (MOST >= 2)
        if (p.vec == 2) return lanes(std::integral_constant<int, 2>{});
    lanes(std::integral_constant<int, 1>{});
}

template <typename T>
int forward(Sequence s, const Plan& p, const float* initial, void* states, float* final_state, float* kept, float* maps,
            hipStream_t stream) {
    by_plan<2>(p, [&](auto vec, auto lpc) {
        constexpr int V = decltype(vec)::value, C = decltype(lpc)::value;
        if (s.parts > 1)
            hipLaunchKernelGGL((recurrence_fold_kernel<T, V, C, false>), dim3(grid_of(s)), dim3(kThreads), 0, stream, s,
                               static_cast<const T*>(nullptr), maps);
        hipLaunchKernelGGL((recurrence_forward_kernel<T, V, C>), dim3(grid_of(s)), dim3(kThreads), 0, stream, s,
                           initial, static_cast<T*>(states), final_state, kept, maps);
    });
    return check_launch("koemi_gated_recurrence_forward");
}
template <typename T>
int backward(Sequence s, const Plan& p, const float* kept, const void* d_states, const float* d_final, void* d_z,
             float* d_initial, float* maps, hipStream_t stream) {
    by_plan<std::is_same<T, float>::value ? 1 : 2>(p, [&](auto vec, auto lpc) {
        constexpr int V = decltype(vec)::value, C = decltype(lpc)::value;
        if (s.parts > 1)
            hipLaunchKernelGGL((recurrence_fold_kernel<T, V, C, true>), dim3(grid_of(s)), dim3(kThreads), 0, stream, s,
                               static_cast<const T*>(d_states), maps);
        hipLaunchKernelGGL((recurrence_backward_kernel<T, V, C>), dim3(grid_of(s)), dim3(kThreads), 0, stream, s,
                           kept, static_cast<const T*>(d_states), d_final, static_cast<T*>(d_z), d_initial, maps);
    });
    return check_launch("koemi_gated_recurrence_backward");
}

}  // namespace
}  // namespace koemi

using namespace koemi;

extern "C" int64_t koemi_gated_recurrence_kept_rows(int64_t length) {
    return length > 0 ? (length + kKeep - 1) / kKeep : 0;
}

extern "C" size_t koemi_gated_recurrence_workspace_bytes(int64_t batch, int64_t length, int64_t width) {
    if (batch <= 0 || length <= 0 || width <= 0) return 0;
    size_t most = 0;  // of every layout: which one a call takes depends on its type and alignment
    for (int vec = 1; vec <= 2; ++vec)
        for (int size = 2; size <= 4; size += 2)
            for (const Fill& fill : {kForwardFill, kBackwardFill})
                most = std::max(most, maps_bytes(plan_of(batch, length, width, vec, size, fill), batch, width));
    return most;
}

extern "C" int koemi_gated_recurrence_forward(const void* preactivations, int64_t batch_stride, int64_t row_stride,
                                              int dtype, const uint8_t* valid, const float* initial, void* states,
                                              float* final_states, float* kept, int64_t batch, int64_t length,
                                              int64_t width, void* workspace, size_t workspace_bytes,
                                              koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_gated_recurrence_forward";
    const int st = check_sequence(what, preactivations, batch_stride, row_stride, dtype, batch, length, width);
    if (st != KOEMI_OK || batch == 0 || width == 0) return st;
    if (length <= 1) row_stride = 2 * width;  // a single row has no next one: Rows takes its size from the stride
    if (!final_states || (length > 0 && !states)) return fail(KOEMI_ERR_INVALID, "%s: null output", what);
    const bool pairs = pairs_fit(preactivations, batch_stride, row_stride, width, dtype, states, nullptr, kept);
    const Plan p = plan_of(batch, length, width, pairs ? 2 : 1, dtype == KOEMI_F32 ? 4 : 2, kForwardFill);
    const size_t need = maps_bytes(p, batch, width);
    if (need && (!workspace || workspace_bytes < need)) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    const Sequence s{preactivations, batch_stride, row_stride, valid, batch, length, width, p.strips, p.parts, p.part_steps};
    float* maps = static_cast<float*>(workspace);
    if (dtype == KOEMI_F32) return forward<float>(s, p, initial, states, final_states, kept, maps, as_stream(stream));
    if (dtype == KOEMI_F16) return forward<f16>(s, p, initial, states, final_states, kept, maps, as_stream(stream));
    return forward<bf16>(s, p, initial, states, final_states, kept, maps, as_stream(stream));
}

extern "C" int koemi_gated_recurrence_backward(const void* preactivations, int64_t batch_stride, int64_t row_stride,
                                               int dtype, const uint8_t* valid, const float* kept,
                                               const void* grad_states, const float* grad_final,
                                               void* grad_preactivations, float* grad_initial, int64_t batch,
                                               int64_t length, int64_t width, void* workspace, size_t workspace_bytes,
                                               koemi_stream_t stream) {
    clear_error();
    const char* what = "koemi_gated_recurrence_backward";
    const int st = check_sequence(what, preactivations, batch_stride, row_stride, dtype, batch, length, width);
    if (st != KOEMI_OK || batch == 0 || width == 0) return st;
    if (length <= 1) row_stride = 2 * width;  // a single row has no next one: Rows takes its size from the stride
    if (length > 0 && (!kept || !grad_preactivations)) return fail(KOEMI_ERR_INVALID, "%s: null pointer", what);
    // fp32 takes one column a lane: two spill ([1, 32768, 512] 101 us against 81 in strips as wide; bf16 [8, 2048, 1024] 57 with one, 47 with two)
    const bool pairs = dtype != KOEMI_F32 && pairs_fit(preactivations, batch_stride, row_stride, width, dtype, grad_states,
                                                       grad_preactivations, kept);
    const Plan p = plan_of(batch, length, width, pairs ? 2 : 1, dtype == KOEMI_F32 ? 4 : 2, kBackwardFill);
    const size_t need = maps_bytes(p, batch, width);
    if (need && (!workspace || workspace_bytes < need)) return fail(KOEMI_ERR_INVALID, "%s: workspace too small", what);
    const Sequence s{preactivations, batch_stride, row_stride, valid, batch, length, width, p.strips, p.parts, p.part_steps};
    float* maps = static_cast<float*>(workspace);
    hipStream_t q = as_stream(stream);
    if (dtype == KOEMI_F32) return backward<float>(s, p, kept, grad_states, grad_final, grad_preactivations, grad_initial, maps, q);
    if (dtype == KOEMI_F16) return backward<f16>(s, p, kept, grad_states, grad_final, grad_preactivations, grad_initial, maps, q);
    return backward<bf16>(s, p, kept, grad_states, grad_final, grad_preactivations, grad_initial, maps, q);
}
