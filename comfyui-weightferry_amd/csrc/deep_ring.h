// A main loop for products too small to fill the chip (dense_ring.h has the one for the others): what they wait for is memory, since a
// workgroup's stage is computed in a tenth of the time that its loads take to arrive. So the ring is four stage buffers deep, three
// stages in flight, one barrier a stage: behind it stage p is whole and the buffer of stage p - 1 is free, and the loads of stage p + 3 go
// out into that before stage p's fragments are read.
//
// us with two buffers / four, of the gated linear where a tile has a CU to itself: 128 x 13824 x 5120 79.5 / 70.5, 700 x 2048 x 5120
// 43.7 / 40.2, 77 x 2608 x 1536 16.9 / 15.2. With two tiles on a CU they hide each other's loads and the second pair of buffers
// only takes room: 512 x 8192 x 2048 38.6 / 43.6.
#pragma once

#include "dense_ring.h"

namespace wf {

constexpr int kDeep = 4;

// acc over the nk stages from stage s0, as dense_loop. sb: the kernel's stage buffers, arrays of their own, so that the compiler tracks the loads
// into each.
template <typename S, typename LA, typename LB, typename TA, typename TB, typename Mma>
__device__ __forceinline__ void deep_loop(const TA& ta, const TB& tb, int s0, int nk, int wave, int lane, wl_frag* const (&sb)[kDeep],
                                          f32x16v (&acc)[S::WM][S::WN], Mma&& mma) {
    constexpr int WM = S::WM, WN = S::WN, AW = S::AW, BW = S::BW, IPW = AW + BW;
    LA a;
    LB b;
    a.init(ta, lane, wave, wave / S::VN * WM);
    b.init(tb, lane, wave, wave % S::VN * WN);
    auto issue = [&](wl_frag* st, int kt) {                        // (stages past the last land where nothing reads them)
        a.begin(kt);
        b.begin(kt);
        static_for<AW>([&](auto q) { a.template load<decltype(q)::value>(st, wave, kt); });
        static_for<BW>([&](auto q) { b.template load<decltype(q)::value>(st + S::ASLOTS, wave, kt); });
    };
    static_for<kDeep - 1>([&](auto i) { issue(sb[decltype(i)::value], s0 + decltype(i)::value); });
    auto step = [&](int p, wl_frag* cur, wl_frag* last) {
        wait_vm<IPW * (kDeep - 2)>();                              // stage p landed (this wave's loads)
        __builtin_amdgcn_s_waitcnt(0xc07f);                        // lgkmcnt(0): this wave's reads of stage p - 1 are done
        wave_barrier_sync();                                       // ... and every wave's: p is whole, p - 1's buffer is free
        issue(last, s0 + p + kDeep - 1);
        static_for<4>([&](auto ks) {
            wl_frag fa[WM], fb[WN];
            static_for<WM>([&](auto i) { fa[decltype(i)::value] = a.template read<decltype(i)::value>(cur, decltype(ks)::value); });
            static_for<WN>([&](auto j) {
                fb[decltype(j)::value] = b.template read<decltype(j)::value>(cur + S::ASLOTS, decltype(ks)::value);
            });
#pragma unroll
            for (int i = 0; i < WM; i++)
#pragma unroll
                for (int j = 0; j < WN; j++) acc[i][j] = mma(acc[i][j], fa[i], fb[j]);
        });
    };
    int p = 0;
    for (; p + kDeep <= nk; p += kDeep)
        static_for<kDeep>([&](auto i) {
            constexpr int I = decltype(i)::value;
            step(p + I, sb[I], sb[(I + kDeep - 1) % kDeep]);
        });
    static_for<kDeep - 1>([&](auto i) {
        constexpr int I = decltype(i)::value;
        if (p + I < nk) step(p + I, sb[I], sb[(I + kDeep - 1) % kDeep]);
    });
    wait_vm<0>();                                                  // the stage buffers are idle from here on
    __builtin_amdgcn_s_waitcnt(0xc07f);
    wave_barrier_sync();
}

}  // namespace wf
