// The 16-bit linear for gfx950: y = resid + gate * act(x w^T + bias) on bfloat16 or float16, float32 accumulation, one
// rounding at the end; and the products of its backward pass, which are the same product on other operands.
//
// 2 M N K operations: v_mfma_f32_32x32x16 tiles fed through the two-buffer LDS ring of dense_ring.h. A product with too
// few tiles to fill the 256 CUs runs as slices of K that write float32 partial sums; a second kernel adds them in slice
// order and runs the epilogue. Operands whose rows are not 16-byte runs along K (odd widths, transposed views) are first
// copied into rows of whole 128-byte stages.
//
// The epilogue works on runs of 8 outputs of a row: the accumulators (16 rows x 1 column a lane) pass through the idle
// stage buffers in float32, so bias, activation, gate and residual are computed on the unrounded sums and every global
// access is 16 bytes.

#include <algorithm>
#include <type_traits>

#include "dense_gemm.h"

namespace wf {

// the slices' sums in slice order, then the epilogue: one run of 8 outputs a thread
template <int D>
__global__ __launch_bounds__(256) void dense_sum(const float* __restrict__ parts, int slices, int M, int N,
                                                 DenseEpilogue e) {
    const int runs = (N + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)M * runs) return;
    const int64_t m = i / runs;
    const int n = (int)(i - m * runs) * 8, cnt = N - n;
    const EpilogueAhead<D> r = epilogue_ahead<D>(e, m, n, N, cnt);
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = 0; s < slices; s++) {
        const float* p = parts + ((int64_t)s * M + m) * N + n;
        float u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (cnt >= 8) __builtin_memcpy(u, p, 32);
        else
#pragma unroll
            for (int x = 0; x < 8; x++)
                if (x < cnt) u[x] = p[x];
#pragma unroll
        for (int x = 0; x < 8; x++) v[x] += u[x];
    }
    epilogue_run<D, true>(e, v, r, m, n, N, cnt);
}

// rows of a strided operand (values row apart along its rows, col apart along K) as [R, KP] rows of whole stages, zeros
// past K: 64 x 64 tiles through LDS, read along whichever of the two is the shorter step
__global__ __launch_bounds__(256) void dense_pack(const uint16_t* __restrict__ p, int64_t row, int64_t col, int R, int K,
                                                  int KP, uint16_t* __restrict__ out) {
    __shared__ uint16_t t[64][66];
    const int64_t r0 = (int64_t)blockIdx.y * 64;
    const int k0 = blockIdx.x * 64, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const bool along_rows = row < col;
#pragma unroll 4
    for (int i = w; i < 64; i += 4) {
        const int r = along_rows ? lane : i, k = along_rows ? i : lane;
        t[r][k] = r0 + r < R && k0 + k < K ? p[(r0 + r) * row + (k0 + k) * col] : (uint16_t)0;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = w; i < 64; i += 4)
        if (r0 + i < R) out[(r0 + i) * KP + k0 + lane] = t[i][lane];
}

// ------------------------------------------------------------------------------------------------- host side
// the tilings, each with its outputs per modelled time (per mille of the largest's)
struct DenseTiling {
    int bm, bn, eff;
};
constexpr DenseTiling kDense[] = {{256, 320, 1000}, {256, 256, 900}, {256, 192, 820}, {256, 128, 700},
                                  {128, 160, 650},  {128, 128, 560}, {64, 128, 380},  {32, 128, 220}};
constexpr int kDenseTilings = sizeof(kDense) / sizeof(kDense[0]);

static DensePlan dense_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t stages = (K + 63) / 64;
    DensePlan best = {0, 1, (int)stages};
    double least = 1e300;
    for (int t = 0; t < kDenseTilings; t++) {
        const int64_t tiles = ((M + kDense[t].bm - 1) / kDense[t].bm) * ((N + kDense[t].bn - 1) / kDense[t].bn);
        const double stage = (double)kDense[t].bm * kDense[t].bn / kDense[t].eff;
        for (int64_t s = 1; s <= 16 && s <= stages; s++) {
            const int64_t per = (stages + s - 1) / s, slices = (stages + per - 1) / per;
            if (slices != s || (s > 1 && (per < 8 || tiles * s > 1024))) continue;
            const int64_t rounds = (tiles * s + 255) / 256;
            double c = (double)rounds * stage * (per + 8);
            if (s > 1) c += 1200 + (double)M * N * (s + 1) * 0.0006;
            if (c < least) least = c, best = {t, (int)s, (int)per};
        }
    }
    return best;
}

static void dense_run(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                      float* parts, const DenseEpilogue& e, hipStream_t s) {
    (a.x ? dense_gemm_across : b.x ? dense_gemm_b_across : dense_gemm_along)(dt, a, b, M, N, K, p, parts, e, s);
    if (p.slices > 1) {
        const int64_t runs = (int64_t)M * ((N + 7) / 8);
        const dim3 grid((uint32_t)((runs + 255) / 256));
        if (dt == WF_BF16) dense_sum<WF_BF16><<<grid, 256, 0, s>>>(parts, p.slices, M, N, e);
        else dense_sum<WF_F16><<<grid, 256, 0, s>>>(parts, p.slices, M, N, e);
    }
}

// whether an operand can be loaded as it is, along K or across it: 16-byte runs, offsets inside 31 bits
static bool dense_along(const void* p, int64_t row, int64_t col, int64_t K) {
    return col == 1 && row % 8 == 0 && K % 8 == 0 && row >= K && row <= (1 << 20) && aligned(p, 16);
}
static bool dense_across(const void* p, int64_t row, int64_t col, int64_t R, int64_t K) {
    return row == 1 && col % 8 == 0 && col >= R && aligned(p, 16) && (K + 128) * col * 2 < (1LL << 31);
}

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct DenseNeeds {
    bool across_x, across_w, copy_x, copy_w;
    int64_t kp, w_at, parts_at, bytes;                // a copy's row; offsets into the workspace, x's copy first
};
static DenseNeeds dense_needs(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col,
                              int64_t M, int64_t N, int64_t K, const DensePlan& p) {
    DenseNeeds d;
    const bool along_x = dense_along(x, x_row, x_col, K), along_w = dense_along(w, w_row, w_col, K);
    d.across_w = !along_w && dense_across(w, w_row, w_col, N, K);
    d.across_x = !along_x && d.across_w && dense_across(x, x_row, x_col, M, K);   // (x across and w along: x is copied)
    d.copy_x = !along_x && !d.across_x;
    d.copy_w = !along_w && !d.across_w;
    d.kp = up(K, 64);
    d.w_at = d.copy_x ? up(M * d.kp * 2, 256) : 0;
    d.parts_at = d.w_at + (d.copy_w ? up(N * d.kp * 2, 256) : 0);
    d.bytes = d.parts_at + (p.slices > 1 ? (int64_t)p.slices * M * N * 4 : 0);
    return d;
}

static int dense_check(const char* who, int dt, int64_t M, int64_t N, int64_t K, int64_t x_row, int64_t x_col,
                       int64_t w_row, int64_t w_col) {
    if (M < 0 || N < 0 || K <= 0 || x_row < 0 || x_col < 0 || w_row < 0 || w_col < 0) {
        set_error("%s: M, N, K = %lld, %lld, %lld or a negative stride", who, (long long)M, (long long)N, (long long)K);
        return WF_EINVAL;
    }
    if (dt != WF_BF16 && dt != WF_F16) {
        set_error("%s: dtype code %d (float16 and bfloat16 are handled)", who, dt);
        return WF_EUNSUPPORTED;
    }
    if (M > (1 << 24) || N > (1 << 24) || K > (1 << 20)) {
        set_error("%s: M or N above 2^24, or K above 2^20", who);
        return WF_EUNSUPPORTED;
    }
    return WF_OK;
}

}  // namespace wf

extern "C" int wf_dense_workspace(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col,
                                  int dt, int64_t M, int64_t N, int64_t K, int64_t* bytes) {
    using namespace wf;
    if (!bytes) { set_error("wf_dense_workspace: null pointer"); return WF_EINVAL; }
    if (const int rc = dense_check("wf_dense_workspace", dt, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    *bytes = M && N ? dense_needs(x, x_row, x_col, w, w_row, w_col, M, N, K, dense_plan(M, N, K)).bytes : 0;
    return WF_OK;
}

extern "C" int wf_dense(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt,
                        int64_t M, int64_t N, int64_t K, const void* bias, int bias_dt, int act, const void* gate,
                        int gate_dt, int64_t rows_per_group, const void* resid, int64_t resid_row, void* y, void* h,
                        void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = dense_check("wf_dense", dt, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    if (act < ACT_NONE || act > ACT_RELU || (bias && bias_dt != dt && bias_dt != WF_F32) ||
        (gate && ((gate_dt != dt && gate_dt != WF_F32) || rows_per_group <= 0)) || (resid && resid_row < 0)) {
        set_error("wf_dense: activation %d, dtype codes %d, %d, rows_per_group %lld", act, bias_dt, gate_dt,
                  (long long)rows_per_group);
        return WF_EINVAL;
    }
    if (M == 0 || N == 0) return WF_OK;
    if (!x || !w || !y) { set_error("wf_dense: null pointer"); return WF_EINVAL; }
    if (!aligned(x, 2) || !aligned(w, 2) || !aligned(y, 2) || !aligned(h, 2) || !aligned(resid, 2) ||
        !aligned(bias, bias_dt == WF_F32 ? 4 : 2) || !aligned(gate, gate_dt == WF_F32 ? 4 : 2)) {
        set_error("wf_dense: a pointer is not aligned to its values");
        return WF_EINVAL;
    }
    const DensePlan p = dense_plan(M, N, K);
    const DenseNeeds d = dense_needs(x, x_row, x_col, w, w_row, w_col, M, N, K, p);
    if (d.bytes && (!workspace || workspace_bytes < d.bytes || !aligned(workspace, 256))) {
        set_error("wf_dense: a workspace of %lld bytes is required", (long long)d.bytes);
        return WF_EINVAL;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    auto operand = [&](const void* v, int64_t row, int64_t col, int64_t R, bool across, bool copy, int64_t at) {
        const uint16_t* q = static_cast<const uint16_t*>(v);
        if (!copy) return DenseOperand{q, across ? col : row, (int)K, (int)R, across};
        uint16_t* out = reinterpret_cast<uint16_t*>(ws + at);
        for (int64_t r = 0; r < R; r += 65535 * 64) {                        // (a grid's second dimension ends there)
            const int64_t n = std::min<int64_t>(R - r, 65535 * 64);
            dense_pack<<<dim3((uint32_t)(d.kp / 64), (uint32_t)((n + 63) / 64)), 256, 0, s>>>(
                q + r * row, row, col, (int)n, (int)K, (int)d.kp, out + r * d.kp);
        }
        return DenseOperand{out, d.kp, (int)d.kp, (int)R, false};
    };
    const DenseOperand a = operand(x, x_row, x_col, M, d.across_x, d.copy_x, 0);
    const DenseOperand b = operand(w, w_row, w_col, N, d.across_w, d.copy_w, d.w_at);
    const DenseEpilogue e = {bias, gate, resid, bias_dt, gate_dt, act, gate ? rows_per_group : 1, resid_row, y, h};
    float* parts = reinterpret_cast<float*>(ws + d.parts_at);
    dense_run(dt, a, b, (int)M, (int)N, (int)K, p, parts, e, s);
    WF_LAUNCH_CHECK("wf_dense launch");
    return WF_OK;
}
