// Main loop of the 16-bit linear's GEMM (dense.hip): C[BM x BN] += A[BM rows, K] . B[BN rows, K]^T through the two LDS
// stage buffers and the barrier discipline of wl_ring.h -- a stage is 64 values of K of every row, loaded global -> LDS;
// stage p + 1 flies while stage p is computed; one barrier a stage, before its last K step's MFMAs, behind which the
// loads of stage p + 2 and the first fragment reads of stage p + 1 go out between those MFMAs. What differs: each operand
// has a row length of its own and the last stage may be short (its chunks past K load zeros), so strided rows and every
// K that is a multiple of 8 need no copy; and each operand's loads are divided over the waves by themselves.
#pragma once

#include "wl_ring.h"

namespace wf {

typedef float f32x16v __attribute__((ext_vector_type(16)));

template <int VM_, int VN_, int WM_, int WN_>
struct DenseShape {
    static constexpr int VM = VM_, VN = VN_, WM = WM_, WN = WN_;
    static constexpr int NT = 64 * VM * VN, NW = NT / 64;
    static constexpr int BM = VM * WM * 32, BN = VN * WN * 32;
    static constexpr int AW = BM / 8 / NW, BW = BN / 8 / NW;      // 1 KiB loads of each operand a wave and stage
    static constexpr int ASLOTS = BM * 8, SLOTS = (BM + BN) * 8;  // 16-byte slots of a stage buffer, A's first
    static_assert(AW * NW * 8 == BM && BW * NW * 8 == BN, "whole loads for every wave");
    static_assert(2 * SLOTS * 16 <= 160 * 1024, "two stage buffers fit the LDS");
};

// an operand's tile: a buffer over its rows from the tile's first, row bytes, and K in bytes
struct DenseTile {
    __amdgpu_buffer_rsrc_t r;
    uint32_t row, k;
};

// acc[i][j] over the nk stages from stage s0. mma(acc, a, b) returns acc + a . b.
template <typename S, typename Mma>
__device__ __forceinline__ void dense_mainloop(const DenseTile& ta, const DenseTile& tb, int s0, int nk, int wave,
                                               int lane, wl_frag* sb0, wl_frag* sb1, f32x16v (&acc)[S::WM][S::WN],
                                               Mma&& mma) {
    constexpr int WM = S::WM, WN = S::WN, AW = S::AW, BW = S::BW, IPW = AW + BW;
    constexpr int READS = WM + WN, MFMAS = WM * WN;
    const int wm = wave / S::VN, wn = wave % S::VN;
    // load g of an operand covers its rows 8 g .. 8 g + 7; lane l takes row 8 g + l / 8, chunk swz8(row, l % 8), which is
    // swz8(l / 8, l % 8) for even g and that ^ 4 for odd g
    const uint32_t chunk = (uint32_t)swz8(lane / 8, lane % 8) * 16u;
    const uint32_t la = (uint32_t)(lane / 8) * ta.row, lb = (uint32_t)(lane / 8) * tb.row;
    auto issue = [&](wl_frag* st, int kt, auto qc) {               // load q of this wave's IPW of stage kt
        constexpr int q = decltype(qc)::value;
        constexpr bool A = q < AW;
        const int g = A ? wave * AW + q : wave * BW + (q - AW);
        const uint32_t c = chunk ^ ((g & 1) ? 64u : 0u), k0 = (uint32_t)kt * 128u, k = A ? ta.k : tb.k;
        // (a chunk past K goes past every buffer's end: zeros; stages past the last load zeros too)
        const uint32_t at = k0 + c < k ? (A ? la : lb) + (uint32_t)(8 * g) * (A ? ta.row : tb.row) + k0 + c : 0x80000000u;
        lds_dma16(A ? ta.r : tb.r, st + (A ? 0 : S::ASLOTS) + 64 * g, at);
    };
    const int lr = lane & 31, lk = lane >> 5;
    const int arow = wm * WM * 32 + lr, brow = wn * WN * 32 + lr;
    const int abase = arow * 8 + swz8(arow, lk), bbase = S::ASLOTS + brow * 8 + swz8(brow, lk);
    wl_frag fa[2][WM], fb[2][WN];
    auto fread = [&](const wl_frag* st, int ks, int set, auto rc) {    // read rc of a K step: a0, the b's, the other a's
        constexpr int r = decltype(rc)::value;
        if constexpr (r == 0) fa[set][0] = st[abase ^ (2 * ks)];
        else if constexpr (r <= WN) fb[set][r - 1] = (st + (bbase ^ (2 * ks)))[(r - 1) * 256];
        else fa[set][r - WN] = (st + (abase ^ (2 * ks)))[(r - WN) * 256];
    };
    auto kstep = [&](auto load, int set, const wl_frag* st, int ks, wl_frag* free_, int kt) {
        static_for<MFMAS>([&](auto mc) {
            constexpr int m = decltype(mc)::value;
            acc[m / WN][m % WN] = mma(acc[m / WN][m % WN], fa[set][m / WN], fb[set][m % WN]);
            constexpr int r0 = m * READS / MFMAS, r1 = (m + 1) * READS / MFMAS;
            static_for<r1 - r0>([&](auto x) {
                fread(st, ks, set ^ 1, std::integral_constant<int, r0 + decltype(x)::value>{});
            });
            if constexpr (decltype(load)::value) {
                constexpr int q0 = m * IPW / MFMAS, q1 = (m + 1) * IPW / MFMAS;
                static_for<q1 - q0>([&](auto x) {
                    issue(free_, kt, std::integral_constant<int, q0 + decltype(x)::value>{});
                });
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    static_for<IPW>([&](auto q) { issue(sb0, s0, q); });
    static_for<IPW>([&](auto q) { issue(sb1, s0 + 1, q); });
    wait_vm<IPW>();                                      // the first stage landed; the second may be in flight
    wave_barrier_sync();
    static_for<READS>([&](auto rc) { fread(sb0, 0, 0, rc); });
    auto step = [&](int p, wl_frag* cur, wl_frag* oth) {
        kstep(std::false_type{}, 0, cur, 1, nullptr, 0);
        kstep(std::false_type{}, 1, cur, 2, nullptr, 0);
        kstep(std::false_type{}, 0, cur, 3, nullptr, 0);
        wait_vm<0>();                                    // stage p + 1 landed (this wave's loads)
        __builtin_amdgcn_s_waitcnt(0xc07f);              // lgkmcnt(0): this wave's reads of cur are done
        wave_barrier_sync();                             // ... and every wave's: cur is free, p + 1 is whole
        kstep(std::true_type{}, 1, oth, 0, cur, p + 2);
    };
    int p = 0;
    for (; p + 2 <= nk; p += 2) {
        step(s0 + p, sb0, sb1);
        step(s0 + p + 1, sb1, sb0);
    }
    if (p < nk) step(s0 + p, sb0, sb1);
    wait_vm<0>();                                        // the stage buffers are idle from here on
    __builtin_amdgcn_s_waitcnt(0xc07f);
    wave_barrier_sync();
}

}  // namespace wf
