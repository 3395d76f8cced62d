// The bf16 MFMA main loop of mfma_stage.hpp for operands that lie across K: stored
// [K, rows], a K step being 32 rows of memory of which the tile takes 256 columns, as the
// weights of a product's gradient do. Such an operand is staged as it lies, 32 rows of 512
// bytes, and its fragments (eight K values of one column a lane) are read by
// ds_read_b64_tr_b16: of the sixteen lanes of a group, lanes 4 j .. 4 j + 3 address row
// j's sixteen columns, eight bytes each, and lane i receives column i of the four rows.
//
// Bank conflicts: the 32-byte unit u of K row k sits at unit u ^ across_swizzle(k). Its
// low part {0, 2, 5, 7} puts the four rows that sixteen or 32 lanes read into distinct
// banks, bit 3 of k sends the other half wave's rows to the other half of the 512 bytes.
// Copies write 1 KiB (two K rows) from two runs of 512 contiguous bytes. Tiles 128 columns
// wide have rows of 256 bytes, four to a copy, and the low part alone.
#pragma once

#include "mfma_stage.hpp"

namespace koemi {
namespace mfma_stage {

// COLUMNS: 256 or 128 of the tile.
template <int COLUMNS>
constexpr int kAcrossRowBytes = COLUMNS * 2;

template <int COLUMNS>
__device__ __forceinline__ int across_swizzle(int k) {
    const int r = k & 3;
    return (2 * r + (r >> 1)) ^ (COLUMNS == 256 ? k & 8 : 0);
}

// Byte offset in the operand's stage, for K group 0 of a step, of the lane's fragment
// of the 32 columns from `column` on: K rows 8 (lane / 32) + (lane % 16) / 4, columns
// 16 (lane / 16 % 2) + 4 (lane % 4).
template <int COLUMNS>
__device__ __forceinline__ uint32_t across_fragment(int column) {
    const int lane = lane_id(), k = 8 * (lane >> 5) + ((lane & 15) >> 2);
    const int unit = column / 16 + ((lane >> 4) & 1);
    return static_cast<uint32_t>(k * kAcrossRowBytes<COLUMNS> + ((unit ^ across_swizzle<COLUMNS>(k)) << 5) + (lane & 3) * 8);
}
// The same of an operand along K: row `row` + lane % 32, K half lane / 32.
__device__ __forceinline__ uint32_t along_fragment(int row) {
    return stage_slot(row + (lane_id() & 31), lane_id() >> 5);
}

// What lane `lane` of stage copy `chunk` (1 KiB) of an across operand brings: its K row
// and its column.
template <int COLUMNS>
__device__ __forceinline__ void across_source(int chunk, int lane, int& k, int& column) {
    constexpr int kLanes = kAcrossRowBytes<COLUMNS> / 16;  // of a K row
    k = 64 / kLanes * chunk + lane / kLanes;
    const int slot = lane % kLanes;
    column = (((slot >> 1) ^ across_swizzle<COLUMNS>(k)) << 4) + (slot & 1) * 8;
}

template <bool ACROSS, int COLUMNS>
__device__ __forceinline__ bf16x8 read_fragment(const char* operand, uint32_t off, int kk) {
    if constexpr (ACROSS) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const char* p = operand + off + kk * (16 * kAcrossRowBytes<COLUMNS>);
        union {
            s16x4 half[2];
            bf16x8 whole;
        } u;
        u.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
        u.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * kAcrossRowBytes<COLUMNS>));
        return u.whole;
    } else {
        return *reinterpret_cast<const bf16x8*>(operand + (off ^ (kk << 5)));
    }
}

// stage_loop of a 256 x BNT tile with either operand along or across K. a_base(kt),
// b_base(kt): uniform pointers to K step kt; a_off, b_off: byte offsets of this lane's
// 16 bytes of its copies of an operand; a_lds, b_lds: the wave's copy destinations in
// stage 0; a_frag, b_frag: fragment offsets (along_fragment, across_fragment) of the
// wave's four and BNT / 64 tiles of 32. nk >= 1 K steps into acc[A tile][B tile], element v
// of lane l: A row l % 32, B column 8 (v / 4) + 4 (l / 32) + v % 4.
template <int BNT, bool A_ACROSS, bool B_ACROSS, typename ABase, typename BBase>
__device__ __forceinline__ void across_loop(char* lds, ABase a_base, BBase b_base, const uint32_t (&a_off)[4],
                                            const uint32_t (&b_off)[BNT / 64], uint32_t a_lds, uint32_t b_lds,
                                            const uint32_t (&a_frag)[4], const uint32_t (&b_frag)[BNT / 64], int nk,
                                            f32x16 (&acc)[4][BNT / 64]) {
    using TS = TileShape<BNT>;
    constexpr int NT = TS::kNT, kStages = TS::kStages, CPT = TS::kCopies, MK = 4 * NT;
    constexpr uint32_t kStageBytes = TS::kStageBytes;
    auto issue_one = [&](int kt, int stage, int i) {
        if (i < 4) lds_dma16(a_lds + stage * kStageBytes + i * 1024, a_base(kt), a_off[i]);
        else lds_dma16(b_lds + stage * kStageBytes + (i - 4) * 1024, b_base(kt), b_off[i - 4]);
    };
    // Fragment f of a half step, in the order its products use them: A 0, the B ones, A 1 .. 3.
    auto read_frag = [&](int kt, int kk, int f, bf16x8 (&af)[4], bf16x8 (&bfr)[NT]) {
        const char* stage = lds + (kt % kStages) * kStageBytes;
        if (f >= 1 && f <= NT) bfr[f - 1] = read_fragment<B_ACROSS, BNT>(stage + kOperandBytes, b_frag[f - 1], kk);
        else {
            const int t = f == 0 ? 0 : f - NT;
            af[t] = read_fragment<A_ACROSS, 256>(stage, a_frag[t], kk);
        }
    };
    auto mfma_one = [&](int j, const bf16x8 (&af)[4], const bf16x8 (&bfr)[NT]) {
        acc[j / NT][j % NT] =
            __builtin_amdgcn_mfma_f32_32x32x16_bf16(bfr[j % NT], af[j / NT], acc[j / NT][j % NT], 0, 0, 0);
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
        if (s < nk)
#pragma unroll
            for (int i = 0; i < CPT; ++i) issue_one(s, s, i);
    wait_tiles_and_sync<CPT>(min(nk, kStages - 1) - 1);
    bf16x8 a0[4], b0[NT], a1[4], b1[NT];
#pragma unroll
    for (int f = 0; f < 4 + NT; ++f) read_frag(0, 0, f, a0, b0);
    auto k_step = [&](int kt, auto copy_tag) {
        constexpr bool kCopy = decltype(copy_tag)::value;
        if (kCopy) wait_tiles_and_sync<CPT>(kStages - 3);
        else wait_tiles_and_sync<CPT>(max(min(nk - 2 - kt, kStages - 3), 0));
        const int sc = (kt + kStages - 1) % kStages;
#pragma unroll
        for (int j = 0; j < MK; ++j) {
            mfma_one(j, a0, b0);
            if constexpr (NT == 4) {
                if (j % 4 == 0) {
                    if constexpr (kCopy) issue_one(kt + kStages - 1, sc, j / 4);
                } else if (j % 2 == 1) {
                    read_frag(kt, 1, j / 2, a1, b1);
                }
            } else {
                if constexpr (kCopy) {
                    if (j < CPT) issue_one(kt + kStages - 1, sc, j);
                }
                if (j >= 2) read_frag(kt, 1, j - 2, a1, b1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const int kn = min(kt + 1, nk - 1);  // the last step re-reads its own stage harmlessly
#pragma unroll
        for (int j = 0; j < MK; ++j) {
            mfma_one(j, a1, b1);
            if constexpr (NT == 4) {
                if constexpr (kCopy) {
                    if (j % 4 == 0) issue_one(kt + kStages - 1, sc, 4 + j / 4);
                }
                if (j % 2 == 1) read_frag(kn, 0, j / 2, a0, b0);
            } else {
                if (j >= 2) read_frag(kn, 0, j - 2, a0, b0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int kt = 0;
    for (; kt + kStages - 1 < nk; ++kt) k_step(kt, std::true_type{});
    for (; kt < nk; ++kt) k_step(kt, std::false_type{});
}

}  // namespace mfma_stage
}  // namespace koemi
