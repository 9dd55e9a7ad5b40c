// The norms after and before two sub-layers of a block, with the gated residual between them, for gfx950, forward and backward.
// Rows of K values:
//
//   hh = h, h / sqrt(mean h^2 + eps) or (h - mean) / sqrt(var + eps)          the norm after a sub-layer (none, RMS, LayerNorm)
//   r = scale x + gate pw hh                                                  the residual stream behind it
//   rh = the norm of r (RMS or LayerNorm),  y = rh s + b,  s = w or 1 + w     what the next sub-layer reads
//
//   dR = dr + through(dy s; rh),  dx = scale dR,  dh = through(dR gate pw; hh),  where for a norm z = (t - m) / d of a row
//   through(g; z) = (g - mean(g) - z mean(g z)) / d, without mean(g) for RMS; and, summed over the rows that share a parameter,
//   dgate = sum dR pw hh,  dpw = sum dR gate hh,  dw = sum dy rh,  db = sum dy
//
// What bounds it is memory: two values in and two out a place, four in and two out in the backward pass, which reads x and h
// again and not r, so that r is as exact there as it was. A row lives in the registers of one team of waves from its only
// load to its only store: variances are a second pass over registers, and y comes from the r that no rounding has touched.
// Statistics and all sums are float32.
//
// Few groups of many rows are what this is made for. Where every row is a group (a gate row a token) a workgroup has one row, writes as
// many partial sums as it reads values, and a shared parameter's 16384 rows of them are added by 32 workgroups: training 16384 x 2048
// takes 2380 us against 187 with one group, the sums 2000 of it; forward 69 against 47.
//
// A workgroup's rows share one row of every parameter. So the lanes keep one sum of dR hh a column, for gate and pw both, which
// become their own by a multiplication when the workgroup is done; it writes a row of partial sums for each parameter and a
// second kernel adds those in a fixed order (no atomics).

#include <algorithm>

#include "column_sums.h"
#include "row_teams.h"

namespace wf {

enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

struct BlockNorm {
    const void *pw, *gate, *w, *b;         // any may be NULL
    int pw_dt, gate_dt, dt;                // dt: of w and b
    int post, norm;
    float plus, scale, eps;                // plus: 1 where s is 1 + w
    int64_t rows;                          // of a group, a workgroup's stretch
    int64_t gate_step, step;               // values from one group's gate, w and b to the next's; 0 where all share one
};

// W waves a row, C packs a lane; workgroup (i, g) walks the rows of group g as in layer_norm.hip: team t takes rows i T + t, then
// every gridDim.x T further, the next row loaded ahead. With up to 16 values a lane the parameters stay in registers.
template <int D, int C, bool CENTER>
__global__ __launch_bounds__(1024) void bn_fwd(const value_t<D>* __restrict__ x, int64_t ldx,
                                             const value_t<D>* __restrict__ h, int64_t ldh, BlockNorm q,
                                             value_t<D>* __restrict__ r, value_t<D>* __restrict__ y,
                                             float4* __restrict__ stats, int K, int W) {
    constexpr int VEC = Pack<D>::VEC;
    __shared__ float red[64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), teams = (int)blockDim.x / (64 * W), team = wave / W;
    const int t = (wave % W) * 64 + (threadIdx.x & 63);
    const int64_t g = blockIdx.y, rows = q.rows, first = g * rows, stride = (int64_t)gridDim.x * teams;
    Pack<D> nx[C], nh[C];
    auto fetch = [&](int64_t i) {                          // row i of the group, or its last
        const int64_t m = first + min(i, rows - 1);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            nx[c].zero();
            nh[c].zero();
            if (col < K) {
                nx[c].load(x + m * ldx + col, K - col);
                if (h) nh[c].load(h + m * ldh + col, K - col);
            }
        }
    };
    int64_t r0 = (int64_t)blockIdx.x * teams;
    fetch(r0 + team);
    float gp[C][VEC], sc[C][VEC], sh[C][VEC];              // gate pw, s, b; past the row's end gp is zero
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC, n = K - col;
        float u[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) gp[c][i] = i < n ? 1.0f : 0.0f, sc[c][i] = 1.0f, sh[c][i] = 0.0f;
        if (col >= K) continue;
        if (q.gate) load_params<VEC>(gp[c], q.gate, g * q.gate_step + col, n, q.gate_dt);
        if (q.pw) {
            load_params<VEC>(u, q.pw, col, n, q.pw_dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) gp[c][i] *= u[i];
        }
        if (q.w) {
            load_params<VEC>(sc[c], q.w, g * q.step + col, n, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) sc[c][i] += q.plus;
        }
        if (q.b) load_params<VEC>(sh[c], q.b, g * q.step + col, n, q.dt);
    }
    int phase = 0;
    // mean (0 for RMS) and 1 / sqrt(mean square about it + eps) of a row's values v, zero past its end
    auto moments = [&](const float (&v)[C][VEC], int kind) {
        float mean = 0.0f, ss = 0.0f;
        if (CENTER && kind == NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < VEC; i++) s += v[c][i];
            mean = team_sum2(s, 0.0f, W, red, phase).x / (float)K;
            phase ^= 1;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int n = K - (c * 64 * W + t) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = i < n ? v[c][i] - mean : 0.0f;
                    ss = fmaf(d, d, ss);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < VEC; i++) ss = fmaf(v[c][i], v[c][i], ss);
        }
        const float var = team_sum2(ss, 0.0f, W, red, phase).x / (float)K;
        phase ^= 1;
        return make_float2(mean, 1.0f / sqrtf(var + q.eps));
    };
    for (; r0 < rows; r0 += stride) {
        const int64_t i0 = r0 + team;
        Pack<D> px[C];
        float v[C][VEC];
#pragma unroll
        for (int c = 0; c < C; c++) {
            px[c] = nx[c];
#pragma unroll
            for (int i = 0; i < VEC; i++) v[c][i] = nh[c].get(i);
        }
        if (r0 + stride < rows) fetch(i0 + stride);
        float2 a = make_float2(0.0f, 1.0f);
        if (q.post != NORM_NONE) a = moments(v, q.post);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++)
                v[c][i] = fmaf(CENTER ? (v[c][i] - a.x) * a.y : v[c][i] * a.y, gp[c][i], q.scale * px[c].get(i));
        const float2 b = moments(v, q.norm);
        if (i0 >= rows) continue;
        if (stats && t == 0) stats[first + i0] = make_float4(a.x, a.y, b.x, b.y);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            if (col >= K) continue;
            Pack<D> o;
            if (r) {
                o.put(v[c]);
                o.store_streamed(r + (first + i0) * K + col, K - col);
            }
            float z[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) z[i] = fmaf(CENTER ? (v[c][i] - b.x) * b.y : v[c][i] * b.y, sc[c][i], sh[c][i]);
            o.put(z);
            o.store_streamed(y + (first + i0) * K + col, K - col);
        }
    }
}

struct BlockNormSums {
    float *gate, *pw, *w, *b;              // [G * gridDim.x, K], a row a workgroup; any may be NULL
};

// The same walk. One pack a lane leaves room for the parameters and the next row; two (rows of more than 16 KiB) for neither.
// Dynamic LDS: T - 1 teams' sums.
template <int D, int C, bool CENTER>
__global__ __launch_bounds__(1024) void bn_bwd(const value_t<D>* __restrict__ x, int64_t ldx, const value_t<D>* __restrict__ h,
                                             int64_t ldh, const value_t<D>* __restrict__ dr, int64_t ldr,
                                             const value_t<D>* __restrict__ dy, int64_t ldy, BlockNorm q,
                                             const float4* __restrict__ stats, value_t<D>* __restrict__ dx,
                                             value_t<D>* __restrict__ dh, BlockNormSums sums, int K, int W) {
    constexpr int VEC = Pack<D>::VEC;
    constexpr bool HOLD = C == 1;
    extern __shared__ float others[];
    __shared__ float red[64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), teams = (int)blockDim.x / (64 * W), team = wave / W;
    const int t = (wave % W) * 64 + (threadIdx.x & 63);
    const int64_t g = blockIdx.y, rows = q.rows, first = g * rows, stride = (int64_t)gridDim.x * teams;
    Pack<D> nx[C], nh[C], nr[C], ny[C];
    float4 ns;
    auto fetch = [&](int64_t i) {                          // row i of the group, or its last
        const int64_t m = first + min(i, rows - 1);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            nx[c].zero();
            nh[c].zero();
            nr[c].zero();
            ny[c].zero();
            if (col < K) {
                nx[c].load(x + m * ldx + col, K - col);
                if (h) nh[c].load(h + m * ldh + col, K - col);
                if (dr) nr[c].load(dr + m * ldr + col, K - col);
                if (dy) ny[c].load(dy + m * ldy + col, K - col);
            }
        }
        ns = stats[m];
    };
    int64_t r0 = (int64_t)blockIdx.x * teams;
    if (HOLD) fetch(r0 + team);
    float gp[HOLD ? C : 1][VEC], sc[HOLD ? C : 1][VEC];
    auto params = [&](float (&gv)[VEC], float (&sv)[VEC], int c) {
        const int col = (c * 64 * W + t) * VEC, n = K - col;
        float u[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) gv[i] = i < n ? 1.0f : 0.0f, sv[i] = 1.0f;
        if (col >= K) return;
        if (q.gate) load_params<VEC>(gv, q.gate, g * q.gate_step + col, n, q.gate_dt);
        if (q.pw) {
            load_params<VEC>(u, q.pw, col, n, q.pw_dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) gv[i] *= u[i];
        }
        if (q.w) {
            load_params<VEC>(sv, q.w, g * q.step + col, n, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) sv[i] += q.plus;
        }
    };
    float ah[C][VEC], aw[C][VEC], ab[C][VEC];              // sums of dR hh, dy rh, dy
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) ah[c][i] = aw[c][i] = ab[c][i] = 0.0f;
        if (HOLD) params(gp[HOLD ? c : 0], sc[HOLD ? c : 0], c);
    }
    const bool back = dh || dx || sums.gate || sums.pw;    // (whether dR is wanted: dw and db go without)
    for (; r0 < rows; r0 += stride) {
        const int64_t i0 = r0 + team;
        const bool on = i0 < rows;
        if (!HOLD) fetch(i0);
        Pack<D> px[C], ph[C], pr[C], py[C];
#pragma unroll
        for (int c = 0; c < C; c++) px[c] = nx[c], ph[c] = nh[c], pr[c] = nr[c], py[c] = ny[c];
        const float4 st = ns;
        if (HOLD && r0 + stride < rows) fetch(i0 + stride);
        // (a mean that is taken off comes off first; RMS has none)
        auto hh = [&](int c, int i) { return CENTER ? (ph[c].get(i) - st.x) * st.y : ph[c].get(i) * st.y; };
        float rh[C][VEC];                                  // then dR
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            if (!HOLD) params(gp[0], sc[0], c);
#pragma unroll
            for (int i = 0; i < VEC; i++) {                // (past the row's end dy is zero, so every term is)
                const float rv = fmaf(hh(c, i), gp[HOLD ? c : 0][i], q.scale * px[c].get(i));
                rh[c][i] = CENTER ? (rv - st.z) * st.w : rv * st.w;
                const float gi = py[c].get(i) * sc[HOLD ? c : 0][i];
                if (CENTER) s1 += gi;
                s2 = fmaf(gi, rh[c][i], s2);
            }
        }
        if (on)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = py[c].get(i);
                    aw[c][i] = fmaf(d, rh[c][i], aw[c][i]);
                    ab[c][i] += d;
                }
        if (!back) continue;
        const float2 s = team_sum2(s1, s2, W, red, 0);
        // dR = dr + w g - w m1 - w m2 rh, w = 1 / r's root
        const float m1 = CENTER && q.norm == NORM_LAYER ? st.w * (s.x / (float)K) : 0.0f, m2 = st.w * (s.y / (float)K);
        float s3 = 0.0f, s4 = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            if (!HOLD) params(gp[0], sc[0], c);
#pragma unroll
            for (int i = 0; i < VEC; i++) {                // (past the row's end gp is zero, and nothing else is kept)
                float d = fmaf(-m2, rh[c][i], fmaf(py[c].get(i) * sc[HOLD ? c : 0][i], st.w, pr[c].get(i)));
                if (CENTER) d -= m1;
                const float tv = d * gp[HOLD ? c : 0][i];
                rh[c][i] = d;
                if (CENTER) s3 += tv;
                s4 = fmaf(tv, hh(c, i), s4);
            }
            if (dx && on && col < K) {
                float v[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i++) v[i] = q.scale * rh[c][i];
                Pack<D> o;
                o.put(v);
                o.store_streamed(dx + (first + i0) * K + col, K - col);
            }
        }
        if (on)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int i = 0; i < VEC; i++) ah[c][i] = fmaf(rh[c][i], hh(c, i), ah[c][i]);
        float m3 = 0.0f, m4 = 0.0f;                        // (both by 1 / h's root)
        if (q.post != NORM_NONE) {
            const float2 u = team_sum2(s3, s4, W, red, 1);
            m3 = CENTER && q.post == NORM_LAYER ? st.y * (u.x / (float)K) : 0.0f;
            m4 = st.y * (u.y / (float)K);
        } else if (W > 1) {
            __syncthreads();                               // (red is written again before the next row's other barrier)
        }
        if (!dh || !on) continue;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            if (col >= K) continue;
            if (!HOLD) params(gp[0], sc[0], c);
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                v[i] = fmaf(-m4, hh(c, i), st.y * (rh[c][i] * gp[HOLD ? c : 0][i]));
                if (CENTER) v[i] -= m3;
            }
            Pack<D> o;
            o.put(v);
            o.store_streamed(dh + (first + i0) * K + col, K - col);
        }
    }
    if (!sums.gate && !sums.pw && !sums.w && !sums.b) return;
    // the other teams' sums, in their order: [team][value of a lane][lane of the team]
    const int lanes = 64 * W;
    if (team > 0)
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                float* o = others + ((int64_t)(team - 1) * 3 * C * VEC + 3 * (c * VEC + i)) * lanes + t;
                o[0] = ah[c][i];
                o[lanes] = aw[c][i];
                o[2 * lanes] = ab[c][i];
            }
    __syncthreads();
    if (team > 0) return;
    const int64_t row = g * gridDim.x + blockIdx.x;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC, n = K - col;
        for (int k = 0; k < teams - 1; k++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float* o = others + ((int64_t)k * 3 * C * VEC + 3 * (c * VEC + i)) * lanes + t;
                ah[c][i] += o[0];
                aw[c][i] += o[lanes];
                ab[c][i] += o[2 * lanes];
            }
        if (col >= K) continue;
        auto put = [&](float* p, const float (&v)[VEC]) {
            if (col + VEC <= K) __builtin_memcpy(p, v, sizeof(v));
            else
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (i < n) p[i] = v[i];
        };
        // dR hh times the other of gate and pw
        auto put_by = [&](float* p, const void* by, int64_t at, int dt) {
            float v[VEC], u[VEC];
            if (by) load_params<VEC>(u, by, at + col, n, dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) v[i] = by ? ah[c][i] * u[i] : ah[c][i];
            put(p, v);
        };
        if (sums.gate) put_by(sums.gate + row * K + col, q.pw, 0, q.pw_dt);
        if (sums.pw) put_by(sums.pw + row * K + col, q.gate, g * q.gate_step, q.gate_dt);
        if (sums.w) put(sums.w + row * K + col, aw[c]);
        if (sums.b) put(sums.b + row * K + col, ab[c]);
    }
}

constexpr int kBlockNormRow = 32768;     // bytes

// (A lane has two packs at most: 16 waves then hold 32 KiB.)
// Forward. Rows up to 4 KiB: one pack a lane, 24 waves a CU; wider ones two packs, 12 waves. us (the same with the other):
// 5152 x 2048 bfloat16 18.7 (20.3), 20000 x 1024 33.1 (33.8), 16384 x 5120 131 (134): 5.1 TB/s, 3000 x 8192 40.3 (44),
// 2048 x 5120 float32 33.5 (34.4). Three workgroups of 5 waves a CU, of which two fit at a time: 16384 x 5120 204.
static RowShape bn_fwd_shape(int64_t M, int64_t K, int64_t rows, int dt) {
    return row_packs(K, dt) <= 4 ? row_shape(M, K, rows, dt, 1, 4, 24, 6) : row_shape(M, K, rows, dt, 2, 4, 12, 4);
}
// Backward. One pack a lane, and one workgroup of 8 waves or a row's a CU, since each writes a row of partial sums and the more of
// its registers hold data in flight the fewer waves it takes: 16384 x 5120 bfloat16 184 us (5.5 TB/s), 192 with two packs, 197
// with two workgroups; 5152 x 2048 35 (40, 38); 20000 x 1024 54 (59, 56). Rows of one pack: two workgroups, 30000 x 256 29.2 against
// 31.6.
static RowShape bn_bwd_shape(int64_t M, int64_t K, int64_t rows, int dt) {
    const int64_t packs = row_packs(K, dt);
    return row_shape(M, K, rows, dt, packs <= 16 ? 1 : 2, 8, packs == 1 ? 16 : 8, 2);
}

// f(packs a lane, whether a mean is taken off) as constants
template <typename F>
static void bn_forms(const RowShape& z, bool center, F&& f) {
    using std::integral_constant;
    auto by = [&](auto c) {
        if (z.packs == 1) f(integral_constant<int, 1>{}, c);
        else f(integral_constant<int, 2>{}, c);
    };
    if (center) by(std::true_type{});
    else by(std::false_type{});
}

static int bn_check(const char* who, const wf_block_norm* q, int64_t M, int64_t K) {
    if (!q || M < 0 || K <= 0 || q->groups <= 0 || M % q->groups || (q->post < NORM_NONE || q->post > NORM_LAYER) ||
        (q->norm != NORM_RMS && q->norm != NORM_LAYER)) {
        set_error("%s: M, K = %lld, %lld, or no parameters, groups or norms that fit", who, (long long)M, (long long)K);
        return WF_EINVAL;
    }
    auto other = [&](int dt) { return dt != q->dt && dt != WF_F32; };
    if (!known_dtype(q->dt) || other(q->post_weight_dt) || other(q->gate_dt) || other(q->weight_dt)) {
        set_error("%s: dtype codes %d, %d, %d, %d", who, q->dt, q->post_weight_dt, q->gate_dt, q->weight_dt);
        return WF_EUNSUPPORTED;
    }
    if (K * value_bytes(q->dt) > kBlockNormRow || M >= (1LL << 31) || q->groups > 65535) {
        set_error("%s: rows of at most %d bytes, 2^31 rows, 65535 groups", who, kBlockNormRow);
        return WF_EUNSUPPORTED;
    }
    return WF_OK;
}

static BlockNorm bn_of(const wf_block_norm* q, const void* pw, const void* gate, const void* w, const void* b, int64_t M, int64_t K) {
    return {pw, gate, w, b, q->post_weight_dt, q->gate_dt, q->weight_dt, q->post, q->norm,
            q->plus_one ? 1.0f : 0.0f, q->scale, q->eps, M / q->groups, q->gate_groups > 1 ? K : 0, q->weight_groups > 1 ? K : 0};
}

}  // namespace wf

extern "C" int wf_block_norm_fwd(const wf_block_norm* q, const void* x, int64_t x_row, const void* h, int64_t h_row,
                                 const void* post_weight, const void* gate, const void* weight, const void* bias, void* r, void* y,
                                 float* stats, int64_t M, int64_t K, void* stream) {
    using namespace wf;
    if (const int rc = bn_check("wf_block_norm_fwd", q, M, K)) return rc;
    auto one_or_all = [&](int64_t n) { return n == 1 || n == q->groups; };
    if (!one_or_all(q->gate_groups) || !one_or_all(q->weight_groups) || x_row < 0 || h_row < 0) {
        set_error("wf_block_norm_fwd: a parameter has one row or one a group; row strides are not negative");
        return WF_EINVAL;
    }
    if (M == 0) return WF_OK;
    if (!x || !y) { set_error("wf_block_norm_fwd: null pointer"); return WF_EINVAL; }
    const BlockNorm p = bn_of(q, post_weight, gate, weight, bias, M, K);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    by_dtype(q->dt, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const RowShape z = bn_fwd_shape(M, K, p.rows, D);
        auto go = [&](auto c, auto center) {
            bn_fwd<D, decltype(c)::value, decltype(center)::value><<<dim3(z.parts, (uint32_t)q->groups), 64 * z.waves * z.teams, 0, s>>>(
                static_cast<const value_t<D>*>(x), x_row, static_cast<const value_t<D>*>(h), h_row, p,
                static_cast<value_t<D>*>(r), static_cast<value_t<D>*>(y), reinterpret_cast<float4*>(stats), (int)K, z.waves);
        };
        bn_forms(z, q->post == NORM_LAYER || q->norm == NORM_LAYER, go);
    });
    WF_LAUNCH_CHECK("wf_block_norm_fwd launch");
    return WF_OK;
}

extern "C" int wf_block_norm_bwd_workspace(const wf_block_norm* q, int64_t M, int64_t K, int sums, int64_t* bytes) {
    using namespace wf;
    if (!bytes || sums < 0 || sums > 4) { set_error("wf_block_norm_bwd_workspace: null pointer or %d sums", sums); return WF_EINVAL; }
    if (const int rc = bn_check("wf_block_norm_bwd_workspace", q, M, K)) return rc;
    *bytes = M ? (int64_t)sums * q->groups * bn_bwd_shape(M, K, M / q->groups, q->dt).parts * K * 4 : 0;
    return WF_OK;
}

extern "C" int wf_block_norm_bwd(const wf_block_norm* q, const void* x, int64_t x_row, const void* h, int64_t h_row,
                                 const void* post_weight, const void* gate, const void* weight, const void* dr, int64_t dr_row,
                                 const void* dy, int64_t dy_row, const float* stats, void* dx, void* dh, void* dpost_weight,
                                 void* dgate, void* dweight, void* dbias, int64_t M, int64_t K, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = bn_check("wf_block_norm_bwd", q, M, K)) return rc;
    auto one_or_all = [&](int64_t n) { return n == 1 || n == q->groups; };
    if (!one_or_all(q->gate_groups) || !one_or_all(q->weight_groups) || x_row < 0 || h_row < 0 || dr_row < 0 || dy_row < 0) {
        set_error("wf_block_norm_bwd: a parameter has one row or one a group; row strides are not negative");
        return WF_EINVAL;
    }
    if (M == 0) return WF_OK;                                   // (no rows: the caller's empty or zero gradients)
    if (!x || !stats || (!dr && !dy)) { set_error("wf_block_norm_bwd: null pointer"); return WF_EINVAL; }
    const BlockNorm p = bn_of(q, post_weight, gate, weight, nullptr, M, K);
    const RowShape z = bn_bwd_shape(M, K, p.rows, q->dt);
    const int64_t plane = q->groups * z.parts * K;
    const int count = (dpost_weight ? 1 : 0) + (dgate ? 1 : 0) + (dweight ? 1 : 0) + (dbias ? 1 : 0);
    if (count && (!workspace || workspace_bytes < count * plane * 4 || !aligned(workspace, 4))) {
        set_error("wf_block_norm_bwd: a workspace of %lld bytes is required", (long long)(count * plane * 4));
        return WF_EINVAL;
    }
    float* at = static_cast<float*>(workspace);
    ColumnSums4 sums = {};
    int n = 0;
    int64_t most = 1;
    auto take = [&](void* out, int dt, int64_t groups) -> float* {
        if (!out) return nullptr;
        float* parts = at + n * plane;
        sums.q[n] = {parts, out, dt, (int)(q->groups / groups * z.parts)};
        sums.groups[n++] = (int)groups;
        most = std::max(most, groups);
        return parts;
    };
    const BlockNormSums b = {take(dgate, q->gate_dt, q->gate_groups), take(dpost_weight, q->post_weight_dt, 1),
                             take(dweight, q->weight_dt, q->weight_groups), take(dbias, q->weight_dt, q->weight_groups)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    by_dtype(q->dt, [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto go = [&](auto c, auto center) {
            constexpr int C = decltype(c)::value;
            const uint32_t lds = (uint32_t)(z.teams - 1) * 3 * C * Pack<D>::VEC * 64 * z.waves * 4;
            bn_bwd<D, C, decltype(center)::value><<<dim3(z.parts, (uint32_t)q->groups), 64 * z.waves * z.teams, count ? lds : 0, s>>>(
                static_cast<const value_t<D>*>(x), x_row, static_cast<const value_t<D>*>(h), h_row,
                static_cast<const value_t<D>*>(dr), dr_row, static_cast<const value_t<D>*>(dy), dy_row, p,
                reinterpret_cast<const float4*>(stats), static_cast<value_t<D>*>(dx), static_cast<value_t<D>*>(dh), b, (int)K,
                z.waves);
        };
        bn_forms(z, q->post == NORM_LAYER || q->norm == NORM_LAYER, go);
    });
    WF_LAUNCH_CHECK("wf_block_norm_bwd launch");
    if (count) {
        column_sums4<<<dim3((uint32_t)((K + 63) / 64), (uint32_t)most, count), 1024, 0, s>>>(sums, (int)K);
        WF_LAUNCH_CHECK("wf_block_norm_bwd sums launch");
    }
    return WF_OK;
}
