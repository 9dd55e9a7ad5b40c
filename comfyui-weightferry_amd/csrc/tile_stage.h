// Epilogues as loops: a wave's sums go through the idle stage buffers in float32, 16 to 64 rows at a time, and come back as runs of
// consecutive values, which a loop of a few hundred instructions finishes. Straight from the accumulators every value has code of its own:
// an epilogue of any arithmetic on 256 of them is a hundred kilobytes, which take longer to fetch than to run.
#pragma once

#include "dense_ring.h"

namespace wf {

template <typename S>
struct TileStage {
    static constexpr int TC = S::WN * 32;                         // a wave's columns
    static constexpr int PART = S::SLOTS * 2 / S::NW;             // a wave's slots, half the waves in each buffer
    static constexpr int ROWS = S::WM % 2 == 0 && 64 * TC * 4 <= PART * 16 ? 64 : 32 * TC * 4 <= PART * 16 ? 32 : 16;
    static constexpr int PHASES = S::WM * 32 / ROWS;
    static_assert(ROWS * TC * 4 <= PART * 16, "a phase's rows fit a wave's slots");

    __device__ __forceinline__ static float* region(wl_frag* sb0, wl_frag* sb1, int wave) {
        return reinterpret_cast<float*>((wave < S::NW / 2 ? sb0 : sb1) + wave % (S::NW / 2) * PART);
    }
    // rows ROWS P .. of the wave's tile, row-major; the wave's own LDS accesses are in order
    template <int P>
    __device__ __forceinline__ static void put(float* t, const f32x16v (&acc)[S::WM][S::WN], int lane) {
        const int lr = lane & 31, lk = lane >> 5;
#pragma unroll
        for (int h = 0; h < ROWS / 16; h++)                       // 16 rows: half an accumulator
#pragma unroll
            for (int x = 0; x < 8; x++)
#pragma unroll
                for (int j = 0; j < S::WN; j++) {
                    constexpr int H0 = P * (ROWS / 16);
                    t[(16 * h + 8 * (x >> 2) + 4 * lk + (x & 3)) * TC + j * 32 + lr] = acc[(H0 + h) / 2][j][8 * ((H0 + h) & 1) + x];
                }
    }
};

// 8 consecutive staged values
__device__ __forceinline__ void staged_run(float (&v)[8], const float* p) {
    __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 32);
}

}  // namespace wf
