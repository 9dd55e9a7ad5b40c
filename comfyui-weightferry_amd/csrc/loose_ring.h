// A main loop for small products whose rows start anywhere (an odd row length, a view): DMA into LDS takes aligned 16-byte runs, loads into
// registers any. So three stages are in flight in registers, a stage goes from there into one of two LDS buffers, and no copy of an
// operand is made first. One barrier a stage: behind it stage p is whole, and the other buffer, last read for stage p - 1, is free once
// the next barrier is passed.
//
// A row's last run begins at its 8th value from the end and is shifted down when it is stored, zeros behind it: nothing is read
// past a row. Rows past the last are read as the last one; what they hold reaches no output.
#pragma once

#include "dense_ring.h"

namespace wf {

constexpr int kLoose = 3;

// rows of values p + r row, `rows` of them from the tile's first on, K >= 8 values each
struct LooseTile {
    const uint16_t* p;
    uint32_t row;
    int rows, k;
};
struct LoosePair {
    const uint16_t* p[2];
    uint32_t row;
    int rows, k;
};

// the LDS layout and the reads of DenseAlong, whose lane l of load q also takes row 8 (q NW + wave) + l / 8, chunk swz8
struct LooseLane {
    int base, c, k;
    uint32_t from;                                                 // the run's first byte in a row, of the stage begun
    __device__ __forceinline__ void init(int k_, int lane, int wave, int t0) {
        k = k_;
        c = 8 * swz8(8 * wave + lane / 8, lane % 8);
        const int lr = lane & 31;
        base = (t0 * 32 + lr) * 8 + swz8(lr, lane >> 5);
    }
    __device__ __forceinline__ void begin(int kt) { from = 2u * (uint32_t)min(64 * kt + c, k - 8); }
    // a run of the last stage, shifted to where it belongs
    __device__ __forceinline__ wl_frag place(wl_frag v, int kt) const {
        const int off = 64 * kt + c - (k - 8);                     // values read before the run's place
        if (off <= 0) return v;
        uint64_t w[2];
        __builtin_memcpy(w, &v, 16);
        const int s = 16 * (off & 3);
        if (off & 4) w[0] = w[1], w[1] = 0;
        if (s) w[0] = w[0] >> s | w[1] << (64 - s), w[1] >>= s;
        if (off >= 8) w[0] = w[1] = 0;
        __builtin_memcpy(&v, w, 16);
        return v;
    }
    template <int I>
    __device__ __forceinline__ wl_frag read(const wl_frag* st, int ks) const {
        return (st + (base ^ (2 * ks)))[I * 256];
    }
};
__device__ __forceinline__ wl_frag loose_run(const uint16_t* p, uint32_t at) {
    wl_frag v;
    __builtin_memcpy(&v, reinterpret_cast<const char*>(p) + at, 16);
    return v;
}

template <int NW, int LW>
struct LooseAlong : LooseLane {
    const uint16_t* p;
    uint32_t at[LW];
    __device__ __forceinline__ void init(const LooseTile& t, int lane, int wave, int t0) {
        static_assert(NW % 2 == 0, "the swizzle goes by the wave's parity");
        LooseLane::init(t.k, lane, wave, t0);
        p = t.p;
#pragma unroll
        for (int q = 0; q < LW; q++) at[q] = 2u * t.row * (uint32_t)min(8 * (q * NW + wave) + lane / 8, t.rows - 1);
    }
    template <int Q>
    __device__ __forceinline__ wl_frag load() const {
        return loose_run(p, at[Q] + from);
    }
};
// load q covers rows 8 wave .. 8 wave + 7 of fragment q of the tile, rows 32 (q / 2) on of matrix q % 2
template <int NW, int LW>
struct LooseAlongPair : LooseLane {
    const uint16_t* p[2];
    uint32_t at[LW / 2];
    __device__ __forceinline__ void init(const LoosePair& t, int lane, int wave, int t0) {
        static_assert(NW == 4 && LW % 2 == 0, "a load of each wave is a fragment's rows");
        LooseLane::init(t.k, lane, wave, t0);
        p[0] = t.p[0];
        p[1] = t.p[1];
#pragma unroll
        for (int q = 0; q < LW / 2; q++) at[q] = 2u * t.row * (uint32_t)min(32 * q + 8 * wave + lane / 8, t.rows - 1);
    }
    template <int Q>
    __device__ __forceinline__ wl_frag load() const {
        return loose_run(p[Q & 1], at[Q / 2] + from);
    }
};

// acc over the nk stages from stage s0, as dense_loop
template <typename S, typename LA, typename LB, typename TA, typename TB, typename Mma>
__device__ __forceinline__ void loose_loop(const TA& ta, const TB& tb, int s0, int nk, int wave, int lane, wl_frag* sb0, wl_frag* sb1,
                                           f32x16v (&acc)[S::WM][S::WN], Mma&& mma) {
    constexpr int WM = S::WM, WN = S::WN, AW = S::AW, BW = S::BW, IPW = AW + BW;
    LA a;
    LB b;
    a.init(ta, lane, wave, wave / S::VN * WM);
    b.init(tb, lane, wave, wave % S::VN * WN);
    const int last = (ta.k - 1) / 64;
    wl_frag v[kLoose][IPW];
    auto issue = [&](wl_frag (&r)[IPW], int kt) {
        a.begin(kt);
        b.begin(kt);
        static_for<AW>([&](auto q) { r[decltype(q)::value] = a.template load<decltype(q)::value>(); });
        static_for<BW>([&](auto q) { r[AW + decltype(q)::value] = b.template load<decltype(q)::value>(); });
    };
    static_for<kLoose>([&](auto i) { issue(v[decltype(i)::value], s0 + decltype(i)::value); });
    auto step = [&](int p, wl_frag (&r)[IPW], wl_frag* st) {
        if (p == last)
#pragma unroll
            for (int q = 0; q < IPW; q++) r[q] = a.place(r[q], p);
#pragma unroll
        for (int q = 0; q < IPW; q++) (st + (q < AW ? 64 * (q * S::NW + wave) : S::ASLOTS + 64 * ((q - AW) * S::NW + wave)))[lane] = r[q];
        issue(r, p + kLoose);
        __builtin_amdgcn_s_waitcnt(0xc07f);                        // lgkmcnt(0): this wave's part of stage p is stored
        wave_barrier_sync();                                       // ... and every wave's
        static_for<4>([&](auto ks) {
            wl_frag fa[WM], fb[WN];
            static_for<WM>([&](auto i) { fa[decltype(i)::value] = a.template read<decltype(i)::value>(st, decltype(ks)::value); });
            static_for<WN>([&](auto j) {
                fb[decltype(j)::value] = b.template read<decltype(j)::value>(st + S::ASLOTS, decltype(ks)::value);
            });
#pragma unroll
            for (int i = 0; i < WM; i++)
#pragma unroll
                for (int j = 0; j < WN; j++) acc[i][j] = mma(acc[i][j], fa[i], fb[j]);
        });
    };
    int p = 0;
    for (; p + 2 * kLoose <= nk; p += 2 * kLoose)
        static_for<2 * kLoose>([&](auto i) {
            constexpr int I = decltype(i)::value;
            step(s0 + p + I, v[I % kLoose], I % 2 ? sb1 : sb0);
        });
    static_for<2 * kLoose - 1>([&](auto i) {
        constexpr int I = decltype(i)::value;
        if (p + I < nk) step(s0 + p + I, v[I % kLoose], I % 2 ? sb1 : sb0);
    });
    __builtin_amdgcn_s_waitcnt(0xc07f);                            // the stage buffers are idle from here on
    wave_barrier_sync();
}

}  // namespace wf
