// What the kernels over rows of values share (layer_norm.hip, block_norm.hip): a row lives in the registers of one team of waves,
// a workgroup is one or more teams that walk the rows.
#pragma once

#include <algorithm>
#include <type_traits>

#include "values.h"

namespace wf {

// the sums of a and b over a team's W waves, in every lane. red: 2 x 2 floats a wave, used alternately (phase) so that one
// barrier a call is enough
__device__ __forceinline__ float2 team_sum2(float a, float b, int W, float* red, int phase) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (W > 1) {
        const int wave = threadIdx.x >> 6, first = wave / W * W;
        float2* r = reinterpret_cast<float2*>(red) + phase * 16;
        if ((threadIdx.x & 63) == 0) r[wave] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
        for (int i = 0; i < W; i++) {
            a += r[first + i].x;
            b += r[first + i].y;
        }
    }
    return make_float2(a, b);
}

struct RowShape {
    int waves, packs, teams, parts;      // a row's waves, a lane's packs, a workgroup's teams, workgroups a group of rows
};
// packs of a lane, if a row had one wave
inline int64_t row_packs(int64_t K, int dt) { return (K * value_bytes(dt) + 1023) / 1024; }
// lane_packs packs a lane, then more waves (up to 16); teams up to team_waves waves a workgroup, fewer where that would leave CUs
// idle; workgroups over all groups: as many a CU as make cu_waves waves of it, at most per_cu.
inline RowShape row_shape(int64_t M, int64_t K, int64_t rows_per_group, int dt, int lane_packs, int team_waves, int cu_waves,
                          int per_cu) {
    const int64_t packs = row_packs(K, dt);
    RowShape s;
    s.waves = (int)std::min<int64_t>(16, (packs + lane_packs - 1) / lane_packs);
    s.packs = (int)((packs + s.waves - 1) / s.waves);
    s.teams = (int)std::max<int64_t>(1, std::min<int64_t>(team_waves / s.waves, M / 256));
    const int64_t wgs = 256 * std::max(1, std::min(per_cu, cu_waves / (s.waves * s.teams)));
    s.parts = (int)std::min<int64_t>((rows_per_group + s.teams - 1) / s.teams,
                                     std::max<int64_t>(1, wgs * rows_per_group / std::max<int64_t>(1, M)));
    return s;
}
template <typename F>
inline void by_dtype(int dt, F&& f) {
    if (dt == WF_F16) f(std::integral_constant<int, WF_F16>{});
    else if (dt == WF_BF16) f(std::integral_constant<int, WF_BF16>{});
    else f(std::integral_constant<int, WF_F32>{});
}

}  // namespace wf
