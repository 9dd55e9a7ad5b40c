// Orthogonalised updates (the Muon optimizer's step) for gfx950: of a matrix's momentum, or of a given matrix, every singular value is
// moved towards one by a few steps of an odd polynomial, without the decomposition:
//
//   m = mu m + (1 - mu) g,  u = (1 - mu) g + mu m (or m),  X = u / max(|u|, eps)          |u| the Frobenius norm
//   steps times: A = X X^T,  X = a X + (b A + c A A) X                                    sigma -> a sigma + b sigma^3 + c sigma^5
//   p = keep p - rate X
//
// With the shorter side m and the longer n that is steps (m^2 n + m^3 + 2 m^2 n) operations, A and its square being symmetric: matrix
// instructions bound it. Matrices of one shape go through every launch together.
//
// Shorter side above 64: float16 tiles (muon_gemm.hip). Everything there is bounded (sigma <= 2, which the host checks), so float16's 11 bits
// serve where bfloat16's 8 would: the direction is off by 1e-3 of its norm against 1e-2, and in gradients whose singular values
// fall off fast, where X is carried with the remainder of its rounding until the last two steps, by 1e-3 against 5e-2. The five steps
// multiply a singular value's relative error by up to 10, and each adds roundings: the fewer singular values hold a matrix, the less they
// average, up to 4e-3 where a few directions do, 1.5e-2 for two or three entries alone. That is so for float32 matrices too: float32
// matrix instructions have a sixteenth of the rate. Powers of two keep the small entries of X and A in float16's normal range.
//
// Up to 64: the steps run on the Gram matrix, in float64. G = u u^T is summed from the float32 u, then P = the product of the steps'
// polynomials of G / |u|^2, each a 64 x 64 matrix product in one workgroup's LDS, then O = P u / |u|. That is two reads of u and three
// launches in place of 17, and nothing is rounded to 16 bits; in float32 G would lose singular values below 2^-12 of the largest, in
// float64 it keeps 2^-26.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "grids.h"
#include "muon.h"

namespace wf {

// -------------------------------------------------------------------------------------------------- a matrix's update u
// 8 places of a matrix's g and m from i on, the first cnt of them (zeros for the others)
struct MuonRun {
    float g[8], m[8];
    __device__ __forceinline__ void load(const MuonTensors& t, int b, int64_t i, int cnt) {
        load_params<8>(g, t.g[b], i, cnt, t.dt);
        if (t.m[b]) load_params<8>(m, t.m[b], i, cnt, WF_F32);
    }
    // u; STEP: m is stepped first, and stored
    template <bool STEP>
    __device__ __forceinline__ void finish(float (&u)[8], const MuonTensors& t, int b, int64_t i, int cnt) const {
        float* p = t.m[b];
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d = t.nu * g[k];
            v[k] = STEP ? fmaf(t.mu, m[k], d) : m[k];
            u[k] = !p ? g[k] : t.nesterov ? fmaf(t.mu, v[k], d) : v[k];
        }
        if (!STEP || !p) return;
        if (cnt >= 8) __builtin_memcpy(p + i, v, 32);
        else
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < cnt) p[i + k] = v[k];
    }
};
template <bool STEP>
__device__ __forceinline__ void muon_u(float (&u)[8], const MuonTensors& t, int b, int64_t i, int cnt) {
    MuonRun r;
    r.load(t, b, i, cnt);
    r.finish<STEP>(u, t, b, i, cnt);
}

__device__ __forceinline__ double wave_sum_f64(double v) {         // by halves: a fixed order
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ double block_sum_f64(double v, double (&red)[4]) {
    v = wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// Steps m and sums u^2 (in float64: float32 squares of 1e-20 are zero, of 1e20 infinite): workgroup (i, matrix) takes `chunk` values.
__global__ __launch_bounds__(256) void muon_norm(MuonTensors t, int64_t size, int64_t chunk, double* __restrict__ parts) {
    __shared__ double red[4];
    const int b = blockIdx.y;
    const int64_t first = blockIdx.x * chunk, end = min(size, first + chunk);
    double s = 0.0;
    for (int64_t i = first + threadIdx.x * 8; i < end; i += 2048) {
        float u[8];
        muon_u<true>(u, t, b, i, (int)min<int64_t>(8, end - i));
#pragma unroll
        for (int k = 0; k < 8; k++) s = fma((double)u[k], (double)u[k], s);
    }
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) parts[(int64_t)b * gridDim.x + blockIdx.x] = s;
}

// X scale = u scale / max(|u|, eps) in float16, the remainder of that rounding times 2048 to lo (may be NULL); [rows, ld], zeros past cols.
__global__ __launch_bounds__(256) void muon_scale(MuonTensors t, int rows, int cols, int ld, const double* __restrict__ parts, int n_parts,
                                                  double scale, double eps, uint16_t* __restrict__ x, uint16_t* __restrict__ lo) {
    __shared__ double red[4];
    const int b = blockIdx.y;
    double s = 0.0;
    for (int i = threadIdx.x; i < n_parts; i += 256) s += parts[(int64_t)b * n_parts + i];
    const double norm = sqrt(block_sum_f64(s, red));
    const float f = (float)fmin(scale / (norm > eps ? norm : norm == norm ? eps : norm), 3.0e38);
    const uint32_t across = (uint32_t)ld / 8, runs = (uint32_t)rows * across;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < runs; i += gridDim.x * 256) {
        const uint32_t r = i / across, c = (i - r * across) * 8;
        float u[8], v[8];
        muon_u<false>(u, t, b, (int64_t)r * cols + c, min(8, cols - (int)c));
        Pack<WF_F16> h, l;
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = u[k] * f;
        h.put(v);
        const int64_t at = ((int64_t)b * rows + r) * ld + c;
        h.store(x + at, 8);
        if (!lo) continue;
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (v[k] - h.get(k)) * 2048.0f;
        l.put(v);
        l.store(lo + at, 8);
    }
}

// ------------------------------------------------------------------------------------------ shorter side up to 64
typedef double f64x4 __attribute__((ext_vector_type(4)));
constexpr int kNarrow = 64, kStretch = 256;                        // the longer side in stretches

// Element (i of the shorter side, k of the longer) of a matrix is at i n + k, or where it is tall at k m + i. In LDS a stretch is
// u[i][k], zeros past n and past the matrix's m rows, rows 4 banks apart (16 rows x 4 k of a matrix instruction's operand: all 64 banks).
constexpr int kStretchRow = kStretch + 4;

// The runs of 8 consecutive values of a stretch's memory, f(place in LDS of the first, offset in the matrix, count, u) each: G runs' loads
// go out together, whatever load() does, before finish() does anything.
struct NarrowRuns {
    int m, len, runs;
    int64_t n, k0;
    bool tall;
    __device__ __forceinline__ NarrowRuns(int m_, int64_t n_, bool tall_, int64_t k0_)
        : m(m_), len((int)min<int64_t>(kStretch, n_ - k0_)), n(n_), k0(k0_), tall(tall_) {
        runs = tall ? (len * m + 7) / 8 : m * (kStretch / 8);
    }
    // run i: its offset in the matrix, values (0: none), and its first value's place (r, k)
    __device__ __forceinline__ int at(int i, int64_t& offset, int& r, int& k) const {
        if (i >= runs) return 0;
        if (tall) {                                                // (the stretch is one run of values)
            offset = k0 * m + i * 8;
            k = i * 8 / m;
            r = i * 8 - k * m;
            return min(8, len * m - i * 8);
        }
        r = i / (kStretch / 8);
        k = i % (kStretch / 8) * 8;
        offset = r * n + k0 + k;
        return min(8, len - k);
    }
    // f(x, place) for the run's 8 places from (r, k) on
    template <typename F>
    __device__ __forceinline__ void places(int r, int k, F&& f) const {
#pragma unroll
        for (int x = 0; x < 8; x++) {
            f(x, r * kStretchRow + k);
            if (!tall) k++;
            else if (++r == m) r = 0, k++;
        }
    }
};
constexpr int kRunsAhead = 4;

template <int MT, bool STEP>
__device__ __forceinline__ void narrow_load(float* us, const MuonTensors& t, int b, const NarrowRuns& q) {
    if (q.m != 16 * MT || q.len != kStretch) {
        for (int i = threadIdx.x; i < 16 * MT * kStretchRow; i += 256) us[i] = 0.0f;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < q.runs; i += 256 * kRunsAhead) {
        MuonRun v[kRunsAhead];
#pragma unroll
        for (int h = 0; h < kRunsAhead; h++) {
            int64_t offset;
            int r, k;
            const int cnt = q.at(i + 256 * h, offset, r, k);
            if (cnt > 0) v[h].load(t, b, offset, cnt);
        }
#pragma unroll
        for (int h = 0; h < kRunsAhead; h++) {
            int64_t offset;
            int r, k;
            const int cnt = q.at(i + 256 * h, offset, r, k);
            if (cnt <= 0) continue;
            float u[8];
            v[h].template finish<STEP>(u, t, b, offset, cnt);
            q.places(r, k, [&](int x, int place) {
                if (x < cnt) us[place] = u[x];
            });
        }
    }
    __syncthreads();
}

// Steps m and sums u u^T over a stretch: workgroup (stretch, matrix). parts: [batch, stretches, tiles, 64 lanes, 4], the 16 x 16 tiles on and
// below the diagonal.
template <int MT>
__global__ __launch_bounds__(256, (MT <= 2 ? 4 : 2)) void narrow_gram(MuonTensors t, int m, int64_t n, int tall, f64x4* __restrict__ parts) {
    constexpr int TILES = MT * (MT + 1) / 2;
    __shared__ float us[16 * MT * kStretchRow];
    __shared__ f64x4 red[3][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    narrow_load<MT, true>(us, t, blockIdx.y, NarrowRuns(m, n, tall != 0, (int64_t)blockIdx.x * kStretch));
    f64x4 acc[TILES];
#pragma unroll
    for (int i = 0; i < TILES; i++) acc[i] = f64x4{0.0, 0.0, 0.0, 0.0};
    const float* p = us + (lane & 15) * kStretchRow + (lane >> 4);
    for (int k = wave * (kStretch / 4); k < (wave + 1) * (kStretch / 4); k += 4) {
        double a[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) a[i] = (double)p[i * 16 * kStretchRow + k];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j <= i; j++)
                acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[i], a[j], acc[i * (i + 1) / 2 + j], 0, 0, 0);
    }
    f64x4* out = parts + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * TILES * 64 + lane;
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        if (wave) red[wave - 1][lane] = acc[i];
        __syncthreads();
        if (!wave) out[i * 64] = (acc[i] + red[0][lane]) + (red[1][lane] + red[2][lane]);
        __syncthreads();
    }
}

// D = alpha A B + beta C + gamma I of [16 MT]^2 float64 matrices in LDS (rows ROW apart), all of them polynomials of one symmetric matrix:
// they commute and are symmetric, so the tiles on and below the diagonal are computed and stored twice. C may be NULL; D may be any of
// them: everything is read before anything is written. The jobs' tiles go over the workgroup's 16 waves.
struct NarrowJob {
    const double *A, *B, *C;
    double* D;
    double alpha, beta, gamma;
};
template <int MT, int ROW, int JOBS>
__device__ __forceinline__ void narrow_products(const NarrowJob (&jobs)[JOBS]) {
    constexpr int TILES = MT * (MT + 1) / 2, EACH = (TILES * JOBS + 15) / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    f64x4 d[EACH];
    auto each = [&](auto&& f) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int job = wave + 16 * e, tile = job % TILES;
            if (job >= TILES * JOBS) continue;
            int ti = 0;
            while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
            f(jobs[JOBS > 1 && job >= TILES ? JOBS - 1 : 0], d[e], 16 * ti, 16 * (tile - ti * (ti + 1) / 2));
        }
    };
    each([&](const NarrowJob& q, f64x4& d, int i0, int j0) {
        f64x4 acc[2] = {};                                         // (two chains: each product waits for the one before)
#pragma unroll
        for (int k = 0; k < 4 * MT; k++) {                         // (A's column k is its row k)
            const int at = (4 * k + g) * ROW + c;
            acc[k & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64(q.A[at + i0], q.B[at + j0], acc[k & 1], 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int r = i0 + 4 * v + g, s = j0 + c;
            d[v] = q.alpha * (acc[0][v] + acc[1][v]);
            if (q.C) d[v] += q.beta * q.C[r * ROW + s];
            if (r == s) d[v] += q.gamma;
        }
    });
    __syncthreads();
    each([&](const NarrowJob& q, f64x4& d, int i0, int j0) {
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int r = i0 + 4 * v + g, s = j0 + c;
            q.D[r * ROW + s] = d[v];
            if (i0 != j0) q.D[s * ROW + r] = d[v];
        }
    });
    __syncthreads();
}

struct MuonSteps {
    int steps;
    double a, b, c, eps;
};
// (a norm of float32 values is zero or above 1e-45: a smaller eps means the same, and 1 / eps^2 has to be finite)
static MuonSteps muon_steps(int steps, const double* abc, double eps) { return {steps, abc[0], abc[1], abc[2], std::max(eps, 1e-60)}; }

// From the sums to P / max(|u|, eps): a workgroup a matrix, which adds its stretches in turn: 16 us at 8 of them (32 rows), 49 at 54 (64 rows),
// but 1080 at 4096, the longest side there is, where orthogonalising 64 x 2^20 takes 1550. out: [batch, 16 MT, 16 MT].
template <int MT>
__global__ __launch_bounds__(1024) void narrow_steps(const f64x4* __restrict__ parts, int stretches, MuonSteps s, double* __restrict__ out) {
    constexpr int TILES = MT * (MT + 1) / 2, M = 16 * MT, ROW = M + 2;      // (two rows' lanes then lie in different banks)
    __shared__ double A[M * ROW], Q[M * ROW], P[M * ROW], trace;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int tile = wave; tile < TILES; tile += 16) {
        f64x4 g = {0.0, 0.0, 0.0, 0.0};
        const f64x4* p = parts + ((int64_t)b * stretches * TILES + tile) * 64 + lane;
#pragma unroll 4
        for (int i = 0; i < stretches; i++) g += p[(int64_t)i * TILES * 64];
        int ti = 0;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
        const int tj = tile - ti * (ti + 1) / 2;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int r = 16 * ti + 4 * v + (lane >> 4), c = 16 * tj + (lane & 15);
            A[r * ROW + c] = g[v];
            if (ti != tj) A[c * ROW + r] = g[v];
        }
    }
    __syncthreads();
    if (wave == 0) {
        double d = lane < M ? A[lane * ROW + lane] : 0.0;
        d = wave_sum_f64(d);
        if (lane == 0) trace = d;
    }
    __syncthreads();
    const double norm = sqrt(trace), inv = 1.0 / (norm > s.eps ? norm : norm == norm ? s.eps : norm);
    for (int i = threadIdx.x; i < M * M; i += 1024) {
        const int at = i / M * ROW + i % M;
        A[at] *= inv * inv;
        P[at] = i / M == i % M ? inv : 0.0;
    }
    __syncthreads();
    for (int k = 0; k < s.steps; k++) {
        narrow_products<MT, ROW>({{A, A, A, Q, s.c, s.b, s.a}});   // Q = a + b A + c A^2
        if (k + 1 == s.steps) {
            narrow_products<MT, ROW>({{Q, P, nullptr, P, 1.0, 0.0, 0.0}});
        } else {                                                   // P = Q P; A = Q A Q
            narrow_products<MT, ROW>({{Q, P, nullptr, P, 1.0, 0.0, 0.0}, {Q, A, nullptr, A, 1.0, 0.0, 0.0}});
            narrow_products<MT, ROW>({{Q, A, nullptr, A, 1.0, 0.0, 0.0}});
        }
    }
    for (int i = threadIdx.x; i < M * M; i += 1024) out[(int64_t)b * M * M + i] = P[i / M * ROW + i % M];
}

// 8 places of a parameter from `at` on, the first cnt of them: keep old - rate v (keep 0: old is not looked at)
__device__ __forceinline__ void muon_store(const MuonTensors& t, int b, int64_t at, const float (&old)[8], const float (&v)[8], int cnt) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = fmaf(-t.rate, v[i], t.keep != 0.0f ? t.keep * old[i] : 0.0f);
    if (t.dt == WF_F32) {
        float* p = static_cast<float*>(t.p[b]) + at;
        if (cnt >= 8) __builtin_memcpy(p, w, 32);
        else
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < cnt) p[i] = w[i];
    } else if (t.dt == WF_BF16) {
        Pack<WF_BF16> o;
        o.put(w);
        o.store(static_cast<uint16_t*>(t.p[b]) + at, cnt);
    } else {
        Pack<WF_F16> o;
        o.put(w);
        o.store(static_cast<uint16_t*>(t.p[b]) + at, cnt);
    }
}

// O = P u over a stretch, and the parameter's step: workgroup (stretch, matrix).
template <int MT>
__global__ __launch_bounds__(256, (MT <= 2 ? 4 : 2)) void narrow_apply(MuonTensors t, int m, int64_t n, int tall, const double* __restrict__ parts) {
    constexpr int M = 16 * MT;
    __shared__ float us[M * kStretchRow];
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    double p[MT][4 * MT];                                          // P's operands: P is symmetric, so row 16 i + c is column
    const double* pp = parts + (int64_t)b * M * M;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int k = 0; k < 4 * MT; k++) p[i][k] = pp[(4 * k + q) * M + 16 * i + c];
    const NarrowRuns runs(m, n, tall != 0, (int64_t)blockIdx.x * kStretch);
    narrow_load<MT, false>(us, t, b, runs);
    // a wave's 64 columns, 16 at a time; its outputs take their place (no other wave reads them)
#pragma unroll 1
    for (int j = wave * 64; j < wave * 64 + 64; j += 16) {
        f64x4 acc[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) acc[i] = f64x4{0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int k = 0; k < 4 * MT; k++) {
            const double u = (double)us[(4 * k + q) * kStretchRow + j + c];
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(p[i][k], u, acc[i], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int v = 0; v < 4; v++) us[(16 * i + 4 * v + q) * kStretchRow + j + c] = (float)acc[i][v];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < runs.runs; i += 256 * kRunsAhead) {
        float old[kRunsAhead][8];
#pragma unroll
        for (int h = 0; h < kRunsAhead; h++) {
            int64_t offset;
            int r, k;
            const int cnt = runs.at(i + 256 * h, offset, r, k);
            if (cnt > 0 && t.keep != 0.0f) load_params<8>(old[h], t.p[b], offset, cnt, t.dt);
        }
#pragma unroll
        for (int h = 0; h < kRunsAhead; h++) {
            int64_t offset;
            int r, k;
            const int cnt = runs.at(i + 256 * h, offset, r, k);
            if (cnt <= 0) continue;
            float v[8];
            runs.places(r, k, [&](int x, int place) { v[x] = x < cnt ? us[place] : 0.0f; });
            muon_store(t, b, offset, old[h], v, cnt);
        }
    }
}

// ------------------------------------------------------------------------------------------------- host side
// How matrices of a shape are stepped: `batch` at a time, and where what they need is in the workspace.
struct MuonPlan {
    bool narrow;
    int batch, mt, stretches;
    int64_t parts, chunk;                              // of muon_norm
    double scale;
    MuonShape s;
    int64_t x_at, y_at, lo_at, a_at, b_at, sums_at, bytes;
};
static MuonPlan muon_plan(int64_t rows, int64_t cols, int64_t count) {
    MuonPlan p = {};
    const int64_t side = std::min(rows, cols), n = std::max(rows, cols), size = rows * cols;
    p.narrow = side <= kNarrow;
    if (p.narrow) {
        p.batch = (int)std::min<int64_t>(count, kMuonBatch);
        p.mt = (int)(side + 15) / 16;
        p.stretches = (int)((n + kStretch - 1) / kStretch);
        p.sums_at = up((int64_t)p.batch * p.stretches * p.mt * (p.mt + 1) / 2 * 64 * 32, 256);
        p.bytes = p.sums_at + (int64_t)p.batch * 256 * p.mt * p.mt * 8;
        return p;
    }
    // as many matrices at a time as fill the chip a few times over: more would only take more memory
    const int64_t tiles = ((rows + 127) / 128) * ((cols + 127) / 128);
    p.batch = (int)std::min<int64_t>(std::min<int64_t>(count, kMuonBatch), std::max<int64_t>(1, 4096 / tiles));
    p.chunk = up(std::max<int64_t>(8192, (size + 1023) / 1024), 8);
    p.parts = (size + p.chunk - 1) / p.chunk;
    p.scale = std::exp2(std::floor(0.5 * std::log2((double)side)) - 1.0);
    p.s = {(int)rows, (int)cols, (int)up(cols, 8), (int)side, (int)up(side, 8), p.batch, rows > cols};
    const int64_t x = up((int64_t)p.batch * rows * p.s.ld * 2, 256), a = up((int64_t)p.batch * side * p.s.sld * 2, 256);
    p.x_at = up((int64_t)p.batch * p.parts * 8, 256);
    p.y_at = p.x_at + x;
    p.lo_at = p.y_at + x;
    p.a_at = p.lo_at + x;
    p.b_at = p.a_at + a;
    p.sums_at = p.b_at + a;
    p.bytes = p.sums_at;
    for (int batch : {p.batch, (int)(count % p.batch)}) {          // (the last batch may be smaller, and sliced otherwise)
        if (batch == 0) continue;
        MuonShape s = p.s;
        s.batch = batch;
        p.bytes = std::max(p.bytes, p.sums_at + std::max(muon_symmetric_bytes(s, false), muon_symmetric_bytes(s, true)));
    }
    return p;
}

static void muon_narrow(const MuonPlan& p, int batch, int64_t rows, int64_t cols, const MuonSteps& s, const MuonTensors& t, char* ws,
                        hipStream_t st) {
    const int m = (int)std::min(rows, cols), tall = rows > cols;
    const int64_t n = std::max(rows, cols);
    f64x4* parts = reinterpret_cast<f64x4*>(ws);
    double* out = reinterpret_cast<double*>(ws + p.sums_at);
    auto go = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        narrow_gram<MT><<<dim3(p.stretches, batch), 256, 0, st>>>(t, m, n, tall, parts);
        narrow_steps<MT><<<dim3(batch), 1024, 0, st>>>(parts, p.stretches, s, out);
        narrow_apply<MT><<<dim3(p.stretches, batch), 256, 0, st>>>(t, m, n, tall, out);
    };
    if (p.mt == 1) go(std::integral_constant<int, 1>{});
    else if (p.mt == 2) go(std::integral_constant<int, 2>{});
    else if (p.mt == 3) go(std::integral_constant<int, 3>{});
    else go(std::integral_constant<int, 4>{});
}

static void muon_wide(const MuonPlan& p, int batch, const MuonSteps& s, const MuonTensors& t, char* ws, hipStream_t st) {
    MuonShape z = p.s;
    z.batch = batch;
    auto at = [&](int64_t o) { return reinterpret_cast<uint16_t*>(ws + o); };
    double* parts = reinterpret_cast<double*>(ws);
    uint16_t *x = at(p.x_at), *y = at(p.y_at), *lo = at(p.lo_at), *A = at(p.a_at), *B = at(p.b_at);
    float* sums = reinterpret_cast<float*>(ws + p.sums_at);
    const int64_t size = (int64_t)z.rows * z.cols;
    const int carried = std::max(0, s.steps - 2);                  // steps that take a X from X and its remainder
    muon_norm<<<dim3((uint32_t)p.parts, batch), 256, 0, st>>>(t, size, p.chunk, parts);
    const int64_t runs = (int64_t)z.rows * z.ld / 8;
    muon_scale<<<dim3((uint32_t)std::min<int64_t>((runs + 255) / 256, 2048), batch), 256, 0, st>>>(
        t, z.rows, z.cols, z.ld, parts, (int)p.parts, p.scale, s.eps, x, carried ? lo : nullptr);
    const float back = (float)(1.0 / (p.scale * p.scale));
    for (int k = 0; k < s.steps; k++) {
        const bool carry = k < carried;
        const float a = carry ? 0.0f : (float)(s.a * p.scale * p.scale);           // a I goes into B, or a X beside the product
        muon_symmetric(z, {x, false, nullptr, A, 1.0f, 0.0f, 0.0f}, sums, st);
        muon_symmetric(z, {A, true, A, B, (float)s.c * back, (float)s.b, a}, sums, st);
        const bool last = k + 1 == s.steps;
        // (the last X is scaled back with the product)
        muon_update(z, {x, B, carry ? lo : nullptr, last ? nullptr : y, last ? back / (float)p.scale : back, (float)s.a}, t, st);
        std::swap(x, y);
    }
}

static int muon_check(const char* who, int64_t count, int64_t rows, int64_t cols, int dt, int steps, const double* abc) {
    if (count < 0 || rows < 0 || cols < 0 || steps < 1 || steps > 32 || !abc) {
        set_error("%s: count, rows, cols = %lld, %lld, %lld, %d steps (1 to 32)", who, (long long)count, (long long)rows, (long long)cols,
                  steps);
        return WF_EINVAL;
    }
    if (!known_dtype(dt)) { set_error("%s: dtype code %d", who, dt); return WF_EUNSUPPORTED; }
    if (std::min(rows, cols) > 16384 || std::max(rows, cols) > (1 << 20) || (rows + 256) * (cols + 8) >= (1LL << 30)) {
        set_error("%s: the shorter side above 16384, the longer above 2^20 or 2^30 values", who);
        return WF_EUNSUPPORTED;
    }
    // float16 holds what the steps pass through only while singular values stay small. (A maximum drops a NaN, so those are asked for.)
    if (!std::isfinite(abc[0]) || !std::isfinite(abc[1]) || !std::isfinite(abc[2])) {
        set_error("%s: coefficients %g, %g, %g", who, abc[0], abc[1], abc[2]);
        return WF_EINVAL;
    }
    double top = 1.0;
    for (int k = 0; k < steps; k++) {
        double next = 0.0, most = 0.0;
        for (int i = 0; i <= 128; i++) {
            const double v = top * i / 128, q = abc[1] * v * v + abc[2] * v * v * v * v;
            next = std::max(next, std::fabs(v * (abc[0] + q)));
            most = std::max(most, std::fabs(q));
        }
        if (!(next <= 1.9) || !(most + std::fabs(abc[0]) <= 12.0)) {
            set_error("%s: coefficients %g, %g, %g take singular values up to %g past 1.9 or multiply by more than 12", who, abc[0],
                      abc[1], abc[2], top);
            return WF_EINVAL;
        }
        top = std::max(1.0, 1.02 * next);
    }
    return WF_OK;
}

// table: param, grad, momentum (0: none) of each matrix
static int muon_run(const char* who, const int64_t* table, int64_t count, int64_t rows, int64_t cols, MuonTensors t, const MuonSteps& s,
                    void* workspace, int64_t workspace_bytes, hipStream_t st) {
    if (count == 0 || rows == 0 || cols == 0) return WF_OK;
    const int bytes = value_bytes(t.dt);
    if (!table) { set_error("%s: null pointer", who); return WF_EINVAL; }
    for (int64_t i = 0; i < count; i++)
        if (!table[3 * i] || !table[3 * i + 1] || table[3 * i] % bytes || table[3 * i + 1] % bytes || table[3 * i + 2] % 4) {
            set_error("%s: matrix %lld: a null pointer, or one not aligned to its values", who, (long long)i);
            return WF_EINVAL;
        }
    const MuonPlan p = muon_plan(rows, cols, count);
    char* ws = static_cast<char*>(workspace);
    if (!ws || workspace_bytes < p.bytes || !aligned(ws, 256)) {
        set_error("%s: a workspace of %lld bytes is required", who, (long long)p.bytes);
        return WF_EINVAL;
    }
    for (int64_t first = 0; first < count; first += p.batch) {
        const int batch = (int)std::min<int64_t>(p.batch, count - first);
        for (int i = 0; i < batch; i++) {
            const int64_t* q = table + 3 * (first + i);
            t.p[i] = reinterpret_cast<void*>(q[0]);
            t.g[i] = reinterpret_cast<const void*>(q[1]);
            t.m[i] = reinterpret_cast<float*>(q[2]);
        }
        if (p.narrow) muon_narrow(p, batch, rows, cols, s, t, ws, st);
        else muon_wide(p, batch, s, t, ws, st);
    }
    if (const hipError_t e = hipGetLastError()) return hip_fail(e, who);
    return WF_OK;
}

}  // namespace wf

extern "C" int wf_muon_workspace(int64_t count, int64_t rows, int64_t cols, int64_t* bytes) {
    using namespace wf;
    const double abc[3] = {1.0, 0.0, 0.0};
    if (!bytes) { set_error("wf_muon_workspace: null pointer"); return WF_EINVAL; }
    if (const int rc = muon_check("wf_muon_workspace", count, rows, cols, WF_F32, 1, abc)) return rc;
    *bytes = count && rows && cols ? muon_plan(rows, cols, count).bytes : 0;
    return WF_OK;
}

extern "C" int wf_muon_plan(int64_t count, int64_t rows, int64_t cols, int* plan) {
    using namespace wf;
    const double abc[3] = {1.0, 0.0, 0.0};
    if (!plan) { set_error("wf_muon_plan: null pointer"); return WF_EINVAL; }
    if (const int rc = muon_check("wf_muon_plan", count, rows, cols, WF_F32, 1, abc)) return rc;
    for (int i = 0; i < 7; i++) plan[i] = 0;
    if (!count || !rows || !cols) return WF_OK;
    const MuonPlan p = muon_plan(rows, cols, count);
    plan[0] = p.batch;
    plan[1] = p.mt;
    if (p.narrow) return WF_OK;
    muon_symmetric_form(p.s, false, plan[2], plan[3]);
    muon_symmetric_form(p.s, true, plan[4], plan[5]);
    plan[6] = muon_update_tiling(p.s);
    return WF_OK;
}

extern "C" int wf_muon(const int64_t* table, int64_t count, int64_t rows, int64_t cols, int dt, double momentum, int nesterov,
                       double keep, double rate, int steps, const double* coefficients, double eps, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = muon_check("wf_muon", count, rows, cols, dt, steps, coefficients)) return rc;
    if (!(momentum >= 0.0 && momentum < 1.0) || !(eps > 0.0) || !std::isfinite(keep) || !std::isfinite(rate)) {
        set_error("wf_muon: momentum %g, eps %g, keep %g, rate %g", momentum, eps, keep, rate);
        return WF_EINVAL;
    }
    MuonTensors t = {};
    t.dt = dt;
    t.keep = (float)keep;
    t.rate = (float)rate;
    t.mu = (float)momentum;
    t.nu = (float)(1.0 - momentum);
    t.nesterov = nesterov;
    return muon_run("wf_muon", table, count, rows, cols, t, muon_steps(steps, coefficients, eps), workspace,
                    workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int wf_orthogonalize(const int64_t* table, int64_t count, int64_t rows, int64_t cols, int dt, int steps,
                                const double* coefficients, double eps, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = muon_check("wf_orthogonalize", count, rows, cols, dt, steps, coefficients)) return rc;
    if (!(eps > 0.0)) { set_error("wf_orthogonalize: eps %g", eps); return WF_EINVAL; }
    MuonTensors t = {};
    t.dt = dt;
    t.rate = -1.0f;
    return muon_run("wf_orthogonalize", table, count, rows, cols, t, muon_steps(steps, coefficients, eps),
                    workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
