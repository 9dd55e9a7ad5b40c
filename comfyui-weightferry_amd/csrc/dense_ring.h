// Main loop of the 16-bit linear's GEMM (dense_gemm.h): C[BM x BN] += A[BM rows, K] . B[BN rows, K]^T through two LDS stage
// buffers -- a stage is 64 values of K of every row, four K steps of the MFMA, loaded global -> LDS; stage p + 1 flies while
// stage p is computed.
//
// Eight waves (256 x 320): the barrier discipline of wl_ring.h, one barrier a stage, before its last K step's MFMAs, behind
// which the loads of stage p + 2 and the first fragment reads of stage p + 1 go out between those MFMAs.
//
// Four waves, one a SIMD with twice the registers: larger wave tiles read fewer bytes of LDS a MFMA (128 x 128: 8 fragments
// for 16 MFMAs, against 7 for 10 of 64 x 160), but a lone wave's MFMAs stop whenever it does, and 16 loads behind one K step
// queue up at the load unit, which takes as long for a stage's loads as the matrix unit for half the stage. So the
// fragments of a whole stage are in registers (four sets): step 0 multiplies and reads steps 2 and 3; behind a barrier the
// buffer is free, and the loads of stage p + 2 spread over steps 1 to 3; a second barrier behind step 1 certifies stage p +
// 1, whose steps 0 and 1 are read during steps 2 and 3. us, eight waves by one barrier / four waves by one / by two: 8192 x
// 8192 x 8192 in 256 x 256 tiles 841 / 831 / 763; 1560 x 13824 x 5120 in 256 x 192 tiles 220 / - / 197; 2048 x 5120 x 5120
// 118 / - / 85.
//
// What differs from wl_ring.h besides: each operand lies in memory one of two ways, with a row length of its own, and K need
// not be whole stages.
//
// Along K (DenseAlong): a row's K values are consecutive. A 1 KiB load covers 8 rows of a stage's 128 bytes; the chunks of
// the last stage that lie past K load zeros. Across K (DenseAcross): value (r, k) is at k * row + r -- the operands of a
// linear's backward products, which would otherwise have to be transposed through memory first. A stage is then 64 rows of
// memory of B values each, and ds_read_b64_tr_b16 turns 4 (of K) x 16 (rows) blocks into the MFMA's fragments on the way
// out of LDS. Rows of memory past K lie past the buffer's end and load zeros; chunks past the operand's last row hold
// other values, which only reach outputs that are not stored.
#pragma once

#include "wl_ring.h"

namespace wf {

typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef short s16x4v __attribute__((ext_vector_type(4)));

template <int VM_, int VN_, int WM_, int WN_>
struct DenseShape {
    static constexpr int VM = VM_, VN = VN_, WM = WM_, WN = WN_;
    static constexpr int NT = 64 * VM * VN, NW = NT / 64;
    static constexpr int BM = VM * WM * 32, BN = VN * WN * 32;
    static constexpr bool DEEP = NW == 4;                         // four sets of fragments and two barriers a stage
    static constexpr int AW = BM / 8 / NW, BW = BN / 8 / NW;      // 1 KiB loads of each operand a wave and stage
    static constexpr int ASLOTS = BM * 8, SLOTS = (BM + BN) * 8;  // 16-byte slots of a stage buffer, A's first
    static constexpr int WAVES = DEEP ? (160 * 1024) / (2 * SLOTS * 16) : 2;   // a SIMD, as many as LDS lets share a CU
    static_assert(AW * NW * 8 == BM && BW * NW * 8 == BN, "whole loads for every wave");
    static_assert(2 * SLOTS * 16 <= 160 * 1024, "two stage buffers fit the LDS");
};

// an operand's tile: the buffer from its first value on, bytes between rows (of the operand, or of memory where it lies
// across K), and the bytes of K to load of a row (along K)
struct DenseTile {
    __amdgpu_buffer_rsrc_t r;
    uint32_t row, k;
};

// B rows of an operand, LW loads a wave and stage for NW waves, W fragments of 32 rows a wave from fragment t0 on
template <int B, int NW, int LW, int W>
struct DenseAlong {
    __amdgpu_buffer_rsrc_t r;
    uint32_t lane_at, tail, step;
    int base, last;

    // load q is number g = q NW + wave of the stage and covers rows 8 g .. 8 g + 7: lane l takes row 8 g + l / 8, chunk
    // swz8(row, l % 8). NW is even, so g's parity, all that the swizzle sees of it, is the wave's.
    __device__ __forceinline__ void init(const DenseTile& t, int lane, int wave, int t0) {
        static_assert(NW % 2 == 0, "the swizzle goes by the wave's parity");
        const int row = 8 * wave + lane / 8;
        const uint32_t c = 16u * (uint32_t)swz8(row, lane % 8);
        r = t.r;
        lane_at = (uint32_t)row * t.row + c;
        step = (uint32_t)(8 * NW) * t.row;
        last = (int)((t.k - 1) / 128);
        tail = (uint32_t)last * 128u + c < t.k ? lane_at : 0x80000000u;      // past every buffer's end: zeros
        const int lr = lane & 31;
        base = (t0 * 32 + lr) * 8 + swz8(lr, lane >> 5);          // (the swizzle depends on the row mod 16)
    }
    // before the loads of stage kt; the stages past the last are not read, whatever they hold
    __device__ __forceinline__ void begin(int kt) {
        if (kt >= last) lane_at = tail;
    }
    template <int Q>
    __device__ __forceinline__ void load(wl_frag* st, int wave, int kt) const {
        lds_dma16(r, st + 64 * (Q * NW + wave), lane_at + (Q * step + (uint32_t)kt * 128u));
    }
    template <int I>
    __device__ __forceinline__ wl_frag read(const wl_frag* st, int ks) const {
        return (st + (base ^ (2 * ks)))[I * 256];
    }
};

template <int B, int NW, int LW, int W>
struct DenseAcross {
    // chunk c of memory row k of the stage sits at slot k CPR + (c ^ swz(k)): the four memory rows that a transposing read
    // takes 32 bytes of each then lie in different quarters of the banks
    static constexpr int CPR = B / 8;
    static constexpr int FOLD = CPR % 16 == 0 ? 3 : CPR % 8 == 0 ? 2 : 0;
    __device__ static constexpr int swz(int k) { return FOLD == 3 ? 2 * (k & 3) : FOLD == 2 ? k & 2 : 0; }
    // loads in strides of NW keep one lane pattern where that is whole rows of memory; else each wave takes LW in a row
    static constexpr bool STRIDED = 64 * NW % CPR == 0;
    static constexpr int PATTERNS = STRIDED ? 1 : LW;
    static_assert(STRIDED || 64 * LW % CPR == 0, "a wave's loads are whole rows of memory");

    __amdgpu_buffer_rsrc_t r;
    uint32_t lane_at[PATTERNS], step, stage;
    int base[2];

    __device__ __forceinline__ void init(const DenseTile& t, int lane, int wave, int t0) {
        r = t.r;
#pragma unroll
        for (int q = 0; q < PATTERNS; q++) {
            const int slot = 64 * (STRIDED ? wave : wave * LW + q) + lane, k = slot / CPR, c = slot % CPR;
            lane_at[q] = (uint32_t)k * t.row + 16u * (uint32_t)(c ^ swz(k));
        }
        step = (uint32_t)(64 * NW / CPR) * t.row;
        stage = 64u * t.row;
        const int kr = 8 * (lane >> 5) + ((lane >> 2) & 3), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        const int f = swz(kr), across = f & 4 ? 64 : 0;           // the swizzle's third bit exchanges neighbour fragments
#pragma unroll
        for (int i = 0; i < 2; i++)
            base[i] = kr * CPR * 16 + (c ^ (f & 2)) * 16 + (lane & 1) * 8 + t0 * 64 + ((t0 + i) & 1 ? -across : across);
    }
    __device__ __forceinline__ void begin(int) {}
    template <int Q>
    __device__ __forceinline__ void load(wl_frag* st, int wave, int kt) const {
        if constexpr (STRIDED) lds_dma16(r, st + 64 * (Q * NW + wave), lane_at[0] + (Q * step + (uint32_t)kt * stage));
        else lds_dma16(r, st + 64 * (wave * LW + Q), lane_at[Q] + (uint32_t)kt * stage);
    }
    template <int I>
    __device__ __forceinline__ wl_frag read(const wl_frag* st, int ks) const {
        wl_frag v = {};
#if defined(__HIP_DEVICE_COMPILE__)
        typedef __attribute__((address_space(3))) const char* lds_bytes;
        typedef __attribute__((address_space(3))) s16x4v* lds_quad;
        lds_bytes p = (lds_bytes)(const char*)st + base[I & 1];
        const s16x4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(p + (ks * 16) * CPR * 16 + I * 64));
        const s16x4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_quad)(p + (ks * 16 + 4) * CPR * 16 + I * 64));
        v = __builtin_bit_cast(wl_frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#endif
        return v;
    }
};

// acc[i][j] over the nk stages from stage s0. AX, BX: whether A and B lie across K. mma(acc, a, b) returns acc + a . b.
template <typename S, bool AX, bool BX, typename Mma>
__device__ __forceinline__ void dense_mainloop(const DenseTile& ta, const DenseTile& tb, int s0, int nk, int wave,
                                               int lane, wl_frag* sb0, wl_frag* sb1, f32x16v (&acc)[S::WM][S::WN],
                                               Mma&& mma) {
    constexpr int WM = S::WM, WN = S::WN, AW = S::AW, BW = S::BW, IPW = AW + BW;
    constexpr int READS = WM + WN, MFMAS = WM * WN;
    std::conditional_t<AX, DenseAcross<S::BM, S::NW, AW, WM>, DenseAlong<S::BM, S::NW, AW, WM>> a;
    std::conditional_t<BX, DenseAcross<S::BN, S::NW, BW, WN>, DenseAlong<S::BN, S::NW, BW, WN>> b;
    a.init(ta, lane, wave, wave / S::VN * WM);
    b.init(tb, lane, wave, wave % S::VN * WN);
    auto issue = [&](wl_frag* st, int kt, auto qc) {               // load q of this wave's IPW of stage kt
        constexpr int q = decltype(qc)::value;
        if constexpr (q < AW) a.template load<q>(st, wave, kt);
        else b.template load<q - AW>(st + S::ASLOTS, wave, kt);
    };
    constexpr int SETS = S::DEEP ? 4 : 2;
    wl_frag fa[SETS][WM], fb[SETS][WN];
    auto fread = [&](const wl_frag* st, int ks, int set, auto rc) {    // read rc of a K step: a0, the b's, the other a's
        constexpr int r = decltype(rc)::value;
        if constexpr (r == 0) fa[set][0] = a.template read<0>(st, ks);
        else if constexpr (r <= WN) fb[set][r - 1] = b.template read<r - 1>(st + S::ASLOTS, ks);
        else fa[set][r - WN] = a.template read<r - WN>(st, ks);
    };
    // The MFMAs of `set`, between them NR steps' fragment reads -- K step ks of st into set rs, then ks + 1 into rs + 1 -- and
    // the loads [L0, L1) of stage kt into `free_`. Two steps' reads are done by three quarters of the MFMAs, so that none
    // is waited for at the barrier behind them.
    auto kstep = [&](auto nr, auto l0, auto l1, int set, const wl_frag* st, int ks, int rs, wl_frag* free_, int kt) {
        constexpr int NR = decltype(nr)::value * READS, L0 = decltype(l0)::value, L = decltype(l1)::value - L0;
        constexpr int OVER = decltype(nr)::value == 2 && MFMAS > 4 ? MFMAS * 3 / 4 : MFMAS;
        static_for<MFMAS>([&](auto mc) {
            constexpr int m = decltype(mc)::value;
            acc[m / WN][m % WN] = mma(acc[m / WN][m % WN], fa[set][m / WN], fb[set][m % WN]);
            constexpr int r0 = m < OVER ? m * NR / OVER : NR, r1 = m + 1 < OVER ? (m + 1) * NR / OVER : NR;
            static_for<r1 - r0>([&](auto x) {
                constexpr int r = r0 + decltype(x)::value;
                fread(st, ks + r / READS, rs + r / READS, std::integral_constant<int, r % READS>{});
            });
            constexpr int q0 = L0 + m * L / MFMAS, q1 = L0 + (m + 1) * L / MFMAS;
            static_for<q1 - q0>([&](auto x) {
                issue(free_, kt, std::integral_constant<int, q0 + decltype(x)::value>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    constexpr std::integral_constant<int, 0> none{};
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, IPW / 3> third{};
    constexpr std::integral_constant<int, 2 * IPW / 3> thirds{};
    constexpr std::integral_constant<int, IPW> all{};
    auto begin = [&](int kt) {
        a.begin(kt);
        b.begin(kt);
    };
    begin(s0);
    static_for<IPW>([&](auto q) { issue(sb0, s0, q); });
    begin(s0 + 1);
    static_for<IPW>([&](auto q) { issue(sb1, s0 + 1, q); });
    wait_vm<IPW>();                                      // the first stage landed; the second may be in flight
    wave_barrier_sync();
    static_for<READS>([&](auto rc) { fread(sb0, 0, 0, rc); });
    if constexpr (S::DEEP) static_for<READS>([&](auto rc) { fread(sb0, 1, 1, rc); });
    // stage p in cur (its first fragments already read), stage p + 1 flying into oth
    auto step = [&](int p, wl_frag* cur, wl_frag* oth) {
        if constexpr (S::DEEP) {
            kstep(two, none, none, 0, cur, 2, 2, nullptr, 0);
            begin(p + 2);
            __builtin_amdgcn_s_waitcnt(0xc07f);          // lgkmcnt(0): this wave's reads of cur are done
            wave_barrier_sync();                         // ... and every wave's: cur is free
            kstep(none, none, third, 1, nullptr, 0, 0, cur, p + 2);
            wait_vm<IPW / 3>();                          // stage p + 1 landed (this wave's loads, all but the newest)
            wave_barrier_sync();                         // ... and every wave's: p + 1 is whole
            kstep(one, third, thirds, 2, oth, 0, 0, cur, p + 2);
            kstep(one, thirds, all, 3, oth, 1, 1, cur, p + 2);
        } else {
            kstep(one, none, none, 0, cur, 1, 1, nullptr, 0);
            kstep(one, none, none, 1, cur, 2, 0, nullptr, 0);
            kstep(one, none, none, 0, cur, 3, 1, nullptr, 0);
            begin(p + 2);
            wait_vm<0>();                                // stage p + 1 landed (this wave's loads)
            __builtin_amdgcn_s_waitcnt(0xc07f);
            wave_barrier_sync();                         // cur is free, p + 1 is whole
            kstep(one, none, all, 1, oth, 0, 0, cur, p + 2);
        }
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
