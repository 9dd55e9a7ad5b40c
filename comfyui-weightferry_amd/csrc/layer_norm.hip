// LayerNorm over rows of K values for gfx950, forward and backward, with affine weights or a DiT block's modulation.
//
//   xh = (x - mean) rstd,  y = xh s + b,  s = w (or 1 + w), row r taking parameter row r / rows_per_group
//   g = dy s,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over a group's rows of dy xh,  db = the sum of dy
//
// What bounds it is memory: the forward pass reads and writes each value once, the backward pass reads two and writes
// one. A row lives in the registers of one team of W waves (16-byte packs, at most 32 values a lane) from its only load
// to its only store, so mean and variance are two passes over registers, not the one-pass difference of large sums.
// Statistics and all sums are float32.
//
// The parameters' gradient is a sum over rows for every column: a lane keeps the sums of its own columns in registers
// over all the rows its workgroup walks, the workgroup writes one row of partial sums, and a second kernel adds those
// in a fixed order (no atomics: the same bits on every run).

#include <algorithm>
#include <type_traits>

#include "column_sums.h"

namespace wf {

// the sums of a and b over a team's W waves (one team per workgroup when W > 1), in every lane. red: 2 x 2 x W floats of
// LDS, used alternately (phase) so that one barrier a call is enough.
template <int W>
__device__ __forceinline__ float2 team_sum2(float a, float b, float* red, int phase) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (W > 1) {
        float* r = red + phase * 2 * W;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            r[2 * wave] = a;
            r[2 * wave + 1] = b;
        }
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) {
            a += r[2 * i];
            b += r[2 * i + 1];
        }
    }
    return make_float2(a, b);
}

struct LnParams {
    const void* w;
    const void* b;
    int dt;                        // type of w and b
    float plus;                    // 1: the scale is 1 + w
    int64_t rows_per_group;
};

template <int D, int W, int C>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void ln_fwd(const value_t<D>* __restrict__ x, int64_t ldx,
                                                                LnParams q, float eps, value_t<D>* __restrict__ y,
                                                                float2* __restrict__ stats, int64_t M, int K) {
    constexpr int VEC = Pack<D>::VEC, TEAMS = W == 1 ? 4 : 1;
    __shared__ float red[W == 1 ? 1 : 4 * W];
    const int t = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t m = (int64_t)blockIdx.x * TEAMS + (W == 1 ? threadIdx.x >> 6 : 0);
    if (m >= M) return;                            // (a whole wave; with W > 1 there is one row a workgroup)
    const value_t<D>* xr = x + m * ldx;
    Pack<D> p[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC;
        p[c].zero();
        if (col < K) p[c].load(xr + col, K - col);
    }
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < VEC; i++) s += p[c].get(i);
    const float mean = team_sum2<W>(s, 0.0f, red, 0).x / (float)K;
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
    const float var = team_sum2<W>(ss, 0.0f, red, 1).x / (float)K;
    const float rstd = 1.0f / sqrtf(var + eps);
    if (stats && t == 0) stats[m] = make_float2(mean, rstd);
    const int64_t base = m / q.rows_per_group * K;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC;
        if (col >= K) continue;
        float v[VEC], u[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = (p[c].get(i) - mean) * rstd;
        if (q.w) {
            load_params<VEC>(u, q.w, base + col, K - col, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) v[i] = v[i] * (u[i] + q.plus);
        }
        if (q.b) {
            load_params<VEC>(u, q.b, base + col, K - col, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) v[i] = v[i] + u[i];
        }
        Pack<D> o;
        o.put(v);
        o.store(y + m * K + col, K - col);
    }
}

// Workgroup (i, g) walks rows i, i + gridDim.x, ... of group g. parts: the workgroup's row of partial sums, weights'
// first, then biases', each [G * gridDim.x, K] float32 (either may be NULL).
template <int D, int W, int C>
__global__ __launch_bounds__(64 * W) void ln_bwd(const value_t<D>* __restrict__ x, int64_t ldx,
                                                 const value_t<D>* __restrict__ dy, int64_t ldd, LnParams q,
                                                 const float2* __restrict__ stats, value_t<D>* __restrict__ dx,
                                                 float* __restrict__ wparts, float* __restrict__ bparts, int64_t M,
                                                 int K) {
    constexpr int VEC = Pack<D>::VEC;
    __shared__ float red[W == 1 ? 1 : 4 * W];
    const int t = threadIdx.x;
    float sc[C][VEC], aw[C][VEC], ab[C][VEC];
    const int64_t g = blockIdx.y;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) sc[c][i] = 1.0f, aw[c][i] = ab[c][i] = 0.0f;
        if (q.w && col < K) {
            load_params<VEC>(sc[c], q.w, g * K + col, K - col, q.dt);
#pragma unroll
            for (int i = 0; i < VEC; i++) sc[c][i] += q.plus;
        }
    }
    int phase = 0;
    for (int64_t r = blockIdx.x; r < q.rows_per_group; r += gridDim.x, phase ^= 1) {
        const int64_t m = g * q.rows_per_group + r;
        Pack<D> px[C], pd[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            px[c].zero();
            pd[c].zero();
            if (col < K) {
                px[c].load(x + m * ldx + col, K - col);
                pd[c].load(dy + m * ldd + col, K - col);
            }
        }
        const float2 st = stats[m];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {               // (past the row's end dy is zero, so every term is)
                const float d = pd[c].get(i), xh = (px[c].get(i) - st.x) * st.y, gi = d * sc[c][i];
                s1 += gi;
                s2 += gi * xh;
                aw[c][i] += d * xh;
                ab[c][i] += d;
            }
        if (!dx) continue;
        const float2 s = team_sum2<W>(s1, s2, red, phase);
        const float m1 = s.x / (float)K, m2 = s.y / (float)K;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = (c * 64 * W + t) * VEC;
            if (col >= K) continue;
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float xh = (px[c].get(i) - st.x) * st.y;
                v[i] = st.y * (pd[c].get(i) * sc[c][i] - m1 - xh * m2);
            }
            Pack<D> o;
            o.put(v);
            o.store(dx + m * K + col, K - col);
        }
    }
    const int64_t row = g * gridDim.x + blockIdx.x;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int col = (c * 64 * W + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            if (col + i >= K) continue;
            if (wparts) wparts[row * K + col + i] = aw[c][i];
            if (bparts) bparts[row * K + col + i] = ab[c][i];
        }
    }
}

constexpr int kLnMaxWidth = 32768;

// waves a row (a lane keeps at most 32 values) and 16-byte packs a lane, as <W, C> of f
template <int D, typename F>
static void ln_shape(int K, F&& f) {
    constexpr int VEC = Pack<D>::VEC;
    const int packs = (K + VEC - 1) / VEC;                       // of the row
    int W = 1;
    while (packs > W * 64 * (32 / VEC)) W *= 2;
    const int C = (packs + 64 * W - 1) / (64 * W);
    auto with_c = [&](auto w) {
        constexpr int WW = decltype(w)::value;
        if (C <= 1) f(w, std::integral_constant<int, 1>{});
        else if (C <= 2) f(w, std::integral_constant<int, 2>{});
        else if (C <= 3) f(w, std::integral_constant<int, 3>{});
        else if (VEC == 8 || C <= 4) f(w, std::integral_constant<int, 4>{});
        else if (VEC == 4 && C <= 6) f(w, std::integral_constant<int, VEC == 4 ? 6 : 4>{});
        else f(w, std::integral_constant<int, VEC == 4 ? 8 : 4>{});
        (void)WW;
    };
    switch (W) {
    case 1: with_c(std::integral_constant<int, 1>{}); break;
    case 2: with_c(std::integral_constant<int, 2>{}); break;
    case 4: with_c(std::integral_constant<int, 4>{}); break;
    case 8: with_c(std::integral_constant<int, 8>{}); break;
    default: with_c(std::integral_constant<int, 16>{}); break;
    }
}

template <typename F>
static void by_dtype(int dt, F&& f) {
    if (dt == WF_F16) f(std::integral_constant<int, WF_F16>{});
    else if (dt == WF_BF16) f(std::integral_constant<int, WF_BF16>{});
    else f(std::integral_constant<int, WF_F32>{});
}

// workgroups a group of rows in the backward pass
static int ln_bwd_parts(int64_t M, int64_t rows_per_group) {
    if (M == 0) return 0;
    const int64_t groups = M / rows_per_group;
    return (int)std::min<int64_t>(rows_per_group, std::max<int64_t>(1, 512 / groups));
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
        ln_shape<D>((int)K, [&](auto w_, auto c_) {
            constexpr int W = decltype(w_)::value, C = decltype(c_)::value;
            const int64_t wgs = W == 1 ? (M + 3) / 4 : M;
            ln_fwd<D, W, C><<<dim3((uint32_t)wgs), W == 1 ? 256 : 64 * W, 0, s>>>(
                static_cast<const value_t<D>*>(x), ldx, q, eps, static_cast<value_t<D>*>(y),
                reinterpret_cast<float2*>(stats), M, (int)K);
        });
    });
    WF_LAUNCH_CHECK("wf_layer_norm launch");
    return WF_OK;
}

extern "C" int wf_layer_norm_bwd_workspace(int64_t M, int64_t K, int64_t rows_per_group, int64_t* bytes) {
    using namespace wf;
    if (!bytes || M < 0 || K <= 0 || rows_per_group <= 0 || M % rows_per_group) {
        set_error("wf_layer_norm_bwd_workspace: bad arguments");
        return WF_EINVAL;
    }
    *bytes = 2 * (M / rows_per_group) * ln_bwd_parts(M, rows_per_group) * K * 4;
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
    const int n = ln_bwd_parts(M, rows_per_group);
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
        ln_shape<D>((int)K, [&](auto w_, auto c_) {
            constexpr int W = decltype(w_)::value, C = decltype(c_)::value;
            ln_bwd<D, W, C><<<dim3(n, (uint32_t)groups), 64 * W, 0, s>>>(
                static_cast<const value_t<D>*>(x), ldx, static_cast<const value_t<D>*>(dy), ldd, q,
                reinterpret_cast<const float2*>(stats), static_cast<value_t<D>*>(dx), wparts, bparts, M, (int)K);
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
