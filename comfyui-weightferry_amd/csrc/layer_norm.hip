// LayerNorm over rows of K values for gfx950, forward and backward, with affine weights or a DiT block's modulation.
//
//   xh = (x - mean) rstd,  y = xh s + b,  s = w (or 1 + w), row r taking parameter row r / rows_per_group
//   g = dy s,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over a group's rows of dy xh,  db = the sum of dy
//
// What bounds it is memory: the forward pass reads and writes each value once, the backward pass reads two and writes
// one. A row lives in the registers of one team of waves (16-byte packs, C a lane) from its only load to its only store,
// so mean and variance are two passes over registers, not the one-pass difference of large sums. Statistics and all sums
// are float32.
//
// The parameters' gradient is a sum over rows for every column: a lane keeps the sums of its own columns in registers
// over all the rows its team walks, a workgroup's teams meet in LDS and write one row of partial sums, and a second
// kernel adds those in a fixed order (no atomics: the same bits on every run). The next row's loads go out before the
// current row's sums are awaited.

#include <algorithm>
#include <type_traits>

#include "column_sums.h"
#include "row_teams.h"

namespace wf {

struct LnParams {
    const void* w;
    const void* b;
    int dt;                        // type of w and b
    float plus;                    // 1: the scale is 1 + w
    int64_t rows_per_group;
};

// W waves a row, C packs a lane. Workgroup (i, g) walks the rows of group g: team t takes rows i T + t, then every
// gridDim.x T further, T = blockDim.x / (64 W) teams. The group's parameters stay in registers (HOLD, up to 16 values a
// lane; beyond that they are read for each row), and the next row is loaded before this one's sums are awaited.
template <int D, int C>
__global__ __launch_bounds__(1024) void ln_fwd(const value_t<D>* __restrict__ x, int64_t ldx, LnParams q, float eps,
                                               value_t<D>* __restrict__ y, float2* __restrict__ stats, int K, int W) {
    constexpr int VEC = Pack<D>::VEC;
    constexpr bool HOLD = C * VEC <= 16;
    __shared__ float red[64];
    const int wave = threadIdx.x >> 6, teams = (int)blockDim.x / (64 * W), team = wave / W;
    const int t = (wave % W) * 64 + (threadIdx.x & 63);
    const int64_t g = blockIdx.y, rows = q.rows_per_group, first = g * rows, stride = (int64_t)gridDim.x * teams;
    Pack<D> next[C];
    auto fetch = [&](int64_t r) {                          // row r of the group, or its last
        const value_t<D>* xr = x + (first + min(r, rows - 1)) * ldx;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            next[c].zero();
            if (col < K) next[c].load(xr + col, K - col);
        }
    };
    int64_t r0 = (int64_t)blockIdx.x * teams;
    fetch(r0 + team);
    float sc[HOLD ? C : 1][VEC], sh[HOLD ? C : 1][VEC];
    auto params = [&](float (&s)[VEC], float (&b)[VEC], int c) {
        const int col = (c * 64 * W + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) s[i] = 1.0f, b[i] = 0.0f;
        if (col >= K) return;
        if (q.w) {
            load_params<VEC>(s, q.w, g * K + col, K - col, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] += q.plus;
        }
        if (q.b) load_params<VEC>(b, q.b, g * K + col, K - col, q.dt);
    };
    if (HOLD)
#pragma unroll
        for (int c = 0; c < C; c++) params(sc[HOLD ? c : 0], sh[HOLD ? c : 0], c);
    for (int phase = 0; r0 < rows; r0 += stride) {
        const int64_t r = r0 + team;
        Pack<D> p[C];
#pragma unroll
        for (int c = 0; c < C; c++) p[c] = next[c];
        if (r0 + stride < rows) fetch(r + stride);
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) s += p[c].get(i);
        const float mean = team_sum2(s, 0.0f, W, red, phase).x / (float)K;
        phase ^= 1;
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int n = K - (c * 64 * W + t) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = p[c].get(i) - mean;
                ss += i < n ? d * d : 0.0f;
            }
        }
        const float var = team_sum2(ss, 0.0f, W, red, phase).x / (float)K;
        phase ^= 1;
        const float rstd = 1.0f / sqrtf(var + eps);
        if (r >= rows) continue;
        if (stats && t == 0) stats[first + r] = make_float2(mean, rstd);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            if (col >= K) continue;
            if (!HOLD) params(sc[0], sh[0], c);
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++)
                v[i] = (p[c].get(i) - mean) * rstd * sc[HOLD ? c : 0][i] + sh[HOLD ? c : 0][i];
            Pack<D> o;
            o.put(v);
            o.store_streamed(y + (first + r) * K + col, K - col);
        }
    }
}

// Workgroup (i, g) walks the rows of group g: team t takes rows i T + t, then every gridDim.x T further, T = blockDim.x /
// (64 W) teams. wparts, bparts: [G * gridDim.x, K] float32 partial sums, a row a workgroup (either may be NULL). Dynamic
// LDS: T - 1 teams' sums of both.
template <int D, int C>
__global__ __launch_bounds__(1024) void ln_bwd(const value_t<D>* __restrict__ x, int64_t ldx,
                                               const value_t<D>* __restrict__ dy, int64_t ldd, LnParams q,
                                               const float2* __restrict__ stats, value_t<D>* __restrict__ dx,
                                               float* __restrict__ wparts, float* __restrict__ bparts, int K, int W) {
    constexpr int VEC = Pack<D>::VEC;
    extern __shared__ float sums[];
    __shared__ float red[64];
    const int wave = threadIdx.x >> 6, teams = (int)blockDim.x / (64 * W), team = wave / W;
    const int t = (wave % W) * 64 + (threadIdx.x & 63);
    // up to 16 values a lane the scale stays in registers and the next row is loaded ahead; beyond, neither fits
    constexpr bool HOLD = C * VEC <= 16;
    float sc[HOLD ? C : 1][VEC], aw[C][VEC], ab[C][VEC];
    const int64_t g = blockIdx.y;
    auto scale = [&](float (&s)[VEC], int c) {
        const int col = (c * 64 * W + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) s[i] = 1.0f;
        if (q.w && col < K) {
            load_params<VEC>(s, q.w, g * K + col, K - col, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] += q.plus;
        }
    };
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) aw[c][i] = ab[c][i] = 0.0f;
        if (HOLD) scale(sc[HOLD ? c : 0], c);
    }
    const int64_t rows = q.rows_per_group, first = g * rows, stride = (int64_t)gridDim.x * teams;
    Pack<D> nx[C], nd[C];
    float2 ns;
    auto fetch = [&](int64_t r) {                          // row r of the group, or its last
        const int64_t m = first + min(r, rows - 1);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            nx[c].zero();
            nd[c].zero();
            if (col < K) {
                nx[c].load(x + m * ldx + col, K - col);
                nd[c].load(dy + m * ldd + col, K - col);
            }
        }
        ns = stats[m];
    };
    int64_t r0 = (int64_t)blockIdx.x * teams;
    if (HOLD) fetch(r0 + team);
    for (int phase = 0; r0 < rows; r0 += stride, phase ^= 1) {
        const int64_t r = r0 + team;
        const bool on = r < rows;
        if (!HOLD) fetch(r);
        Pack<D> px[C], pd[C];
#pragma unroll
        for (int c = 0; c < C; c++) px[c] = nx[c], pd[c] = nd[c];
        const float mean = ns.x, rstd = ns.y;
        if (HOLD && r0 + stride < rows) fetch(r + stride);
        float s1 = 0.0f, s2 = 0.0f;
        if (on) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                if (!HOLD) scale(sc[0], c);
#pragma unroll
                for (int i = 0; i < VEC; i++) {            // (past the row's end dy is zero, so every term is)
                    const float d = pd[c].get(i), xh = (px[c].get(i) - mean) * rstd, gi = d * sc[HOLD ? c : 0][i];
                    s1 += gi;
                    s2 += gi * xh;
                    aw[c][i] += d * xh;
                    ab[c][i] += d;
                }
            }
        }
        if (!dx) continue;
        const float2 s = team_sum2(s1, s2, W, red, phase);
        if (!on) continue;
        const float m1 = s.x / (float)K, m2 = s.y / (float)K;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            if (col >= K) continue;
            if (!HOLD) scale(sc[0], c);
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float xh = (px[c].get(i) - mean) * rstd;
                v[i] = rstd * (pd[c].get(i) * sc[HOLD ? c : 0][i] - m1 - xh * m2);
            }
            Pack<D> o;
            o.put(v);
            o.store_streamed(dx + (first + r) * K + col, K - col);
        }
    }
    if (!wparts && !bparts) return;
    // the other teams' sums, in their order: [team][value of a lane][lane of the team]
    const int lanes = 64 * W;
    if (team > 0)
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                float* o = sums + ((int64_t)(team - 1) * 2 * C * VEC + 2 * (c * VEC + i)) * lanes + t;
                o[0] = aw[c][i];
                o[lanes] = ab[c][i];
            }
    __syncthreads();
    if (team > 0) return;
    const int64_t row = g * gridDim.x + blockIdx.x;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC;
        for (int k = 0; k < teams - 1; k++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float* o = sums + ((int64_t)k * 2 * C * VEC + 2 * (c * VEC + i)) * lanes + t;
                aw[c][i] += o[0];
                ab[c][i] += o[lanes];
            }
        if (col >= K) continue;
        auto put = [&](float* p, const float (&v)[VEC]) {
            if (col + VEC <= K) __builtin_memcpy(p, v, sizeof(v));
            else
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (col + i < K) p[i] = v[i];
        };
        if (wparts) put(wparts + row * K + col, aw[c]);
        if (bparts) put(bparts + row * K + col, ab[c]);
    }
}

constexpr int kLnMaxWidth = 32768;

// Forward: workgroups of up to 5 waves. us at 4096 x 5120 bfloat16 (84 MB; 5 waves a workgroup) with 2 / 3 / 4 a CU: 21.8 /
// 19.6 / 22.8; one row a workgroup, without loading ahead, 31. 5152 x 2048 in workgroups of 4 waves 11.9, of 8 waves 16.4;
// 3000 x 8192 float32 (16 waves) with one a CU 32.8, with three 35.6. 16384 x 5120 takes 64 us, 5.2 TB/s. Rows of one pack a
// lane use half the registers: 30000 x 256 in three workgroups of 8 waves a CU 13.0, in three of 5 14.4.
static RowShape ln_fwd_shape(int64_t M, int64_t K, int64_t rows_per_group, int dt) {
    return K <= 64 * (dt == WF_F32 ? 4 : 8) ? row_shape(M, K, rows_per_group, dt, 2, 8, 24, 3)
                                            : row_shape(M, K, rows_per_group, dt, 2, 5, 16, 8);
}
// Backward: one workgroup of up to 16 waves a CU, since every workgroup writes a row of partial sums: 4096 x 5120 takes
// 35.7 us with 256, 37.9 with 512 of half the teams, 42.4 with 512 whole ones. 16384 x 5120: 98 us, 5.2 TB/s.
static RowShape ln_bwd_shape(int64_t M, int64_t K, int64_t rows_per_group, int dt) {
    return row_shape(M, K, rows_per_group, dt, 2, 16, 16, 1);
}

// f with a lane's packs as a constant: the next of 1, 2, 3, 4, 6, 8 (a row of 32768 values over 16 waves has 4, or 8 of
// float32)
template <int D, typename F>
static void ln_packs(int packs, F&& f) {
    using std::integral_constant;
    if (packs <= 1) f(integral_constant<int, 1>{});
    else if (packs <= 2) f(integral_constant<int, 2>{});
    else if (packs <= 3) f(integral_constant<int, 3>{});
    else if (D != WF_F32 || packs <= 4) f(integral_constant<int, 4>{});
    else if (packs <= 6) f(integral_constant<int, D == WF_F32 ? 6 : 4>{});
    else f(integral_constant<int, D == WF_F32 ? 8 : 4>{});
}

static int ln_check(const char* who, int64_t M, int64_t K, int64_t rows_per_group, int dt, int param_dt) {
    if (M < 0 || K <= 0 || rows_per_group <= 0 || M % rows_per_group) {
        set_error("%s: M, K, rows_per_group = %lld, %lld, %lld", who, (long long)M, (long long)K,
                  (long long)rows_per_group);
        return WF_EINVAL;
    }
    if (!known_dtype(dt) || (param_dt != dt && param_dt != WF_F32)) {
        set_error("%s: dtype codes %d, %d", who, dt, param_dt);
        return WF_EUNSUPPORTED;
    }
    if (K > kLnMaxWidth || M >= (1LL << 31) || M / rows_per_group > 65535) {
        set_error("%s: rows of at most %d values, 2^31 rows, 65535 groups", who, kLnMaxWidth);
        return WF_EUNSUPPORTED;
    }
    return WF_OK;
}

}  // namespace wf

extern "C" int wf_layer_norm(const void* x, int64_t ldx, int dt, const void* w, const void* b, int param_dt,
                             int plus_one, int64_t rows_per_group, float eps, void* y, float* stats, int64_t M,
                             int64_t K, void* stream) {
    using namespace wf;
    if (const int rc = ln_check("wf_layer_norm", M, K, rows_per_group, dt, param_dt)) return rc;
    if (M == 0) return WF_OK;
    if (!x || !y || ldx < 0) { set_error("wf_layer_norm: null pointer or row stride %lld", (long long)ldx); return WF_EINVAL; }
    const LnParams q = {w, b, param_dt, plus_one ? 1.0f : 0.0f, rows_per_group};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    by_dtype(dt, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const RowShape p = ln_fwd_shape(M, K, rows_per_group, dt);
        ln_packs<D>(p.packs, [&](auto c) {
            ln_fwd<D, decltype(c)::value>
                <<<dim3(p.parts, (uint32_t)(M / rows_per_group)), 64 * p.waves * p.teams, 0, s>>>(
                    static_cast<const value_t<D>*>(x), ldx, q, eps, static_cast<value_t<D>*>(y),
                    reinterpret_cast<float2*>(stats), (int)K, p.waves);
        });
    });
    WF_LAUNCH_CHECK("wf_layer_norm launch");
    return WF_OK;
}

extern "C" int wf_layer_norm_bwd_workspace(int64_t M, int64_t K, int64_t rows_per_group, int dt, int64_t* bytes) {
    using namespace wf;
    if (!bytes || M < 0 || K <= 0 || rows_per_group <= 0 || M % rows_per_group || !known_dtype(dt)) {
        set_error("wf_layer_norm_bwd_workspace: bad arguments");
        return WF_EINVAL;
    }
    *bytes = M ? 2 * (M / rows_per_group) * ln_bwd_shape(M, std::min<int64_t>(K, kLnMaxWidth), rows_per_group, dt).parts * K * 4
               : 0;
    return WF_OK;
}

extern "C" int wf_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t ldd, int dt, const void* w,
                                 int param_dt, int plus_one, int64_t rows_per_group, const float* stats, void* dx,
                                 void* dw, void* db, int64_t M, int64_t K, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
    using namespace wf;
    if (const int rc = ln_check("wf_layer_norm_bwd", M, K, rows_per_group, dt, param_dt)) return rc;
    if (M == 0) return WF_OK;                                   // (no rows: the caller's empty or zero gradients)
    if (!x || !dy || !stats || ldx < 0 || ldd < 0) {
        set_error("wf_layer_norm_bwd: null pointer or negative row stride");
        return WF_EINVAL;
    }
    const RowShape p = ln_bwd_shape(M, K, rows_per_group, dt);
    const int n = p.parts;
    const int64_t groups = M / rows_per_group, plane = groups * n * K;
    float* parts = static_cast<float*>(workspace);
    if ((dw || db) && (!workspace || workspace_bytes < 2 * plane * 4 || !aligned(workspace, 4))) {
        set_error("wf_layer_norm_bwd: a workspace of %lld bytes is required", (long long)(2 * plane * 4));
        return WF_EINVAL;
    }
    const LnParams q = {w, nullptr, param_dt, plus_one ? 1.0f : 0.0f, rows_per_group};
    float *wparts = dw ? parts : nullptr, *bparts = db ? parts + plane : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    by_dtype(dt, [&](auto d) {
        constexpr int D = decltype(d)::value;
        ln_packs<D>(p.packs, [&](auto c) {
            constexpr int C = decltype(c)::value;
            const uint32_t lds = (uint32_t)(p.teams - 1) * 2 * C * Pack<D>::VEC * 64 * p.waves * 4;
            ln_bwd<D, C><<<dim3(n, (uint32_t)groups), 64 * p.waves * p.teams, dw || db ? lds : 0, s>>>(
                static_cast<const value_t<D>*>(x), ldx, static_cast<const value_t<D>*>(dy), ldd, q,
                reinterpret_cast<const float2*>(stats), static_cast<value_t<D>*>(dx), wparts, bparts, (int)K, p.waves);
        });
    });
    WF_LAUNCH_CHECK("wf_layer_norm_bwd launch");
    if (dw || db) {
        const ColumnSums sw = {wparts, dw, param_dt, n}, sb = {bparts, db, param_dt, n};
        column_sums<<<dim3((uint32_t)((K + 63) / 64), (uint32_t)groups, dw && db ? 2 : 1), 1024, 0, s>>>(dw ? sw : sb, sb,
                                                                                                         (int)K);
        WF_LAUNCH_CHECK("wf_layer_norm_bwd sums launch");
    }
    return WF_OK;
}
