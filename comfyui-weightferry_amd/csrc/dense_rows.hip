// The 16-bit linear at few rows of x (both operands along K): the weight streams through the chip once, straight from
// memory into v_mfma_f32_16x16x32 operands, without LDS -- at these rows the product is bound by the weight's bytes and by
// how many of them are in flight. 1 x 13824 x 5120 takes 30 us (4.7 TB/s), 1 x 5120 x 5120 14.4.
//
// The weight's rows are the MFMA's 16 rows, x's rows its 16 columns, so a lane holds a row's 8 consecutive values of K for
// either. A workgroup owns 16 RT weight rows and 16 rows of x; its four waves split K and meet in LDS (8 and 16 waves were
// no faster at any of 19 shapes, nor were 32 rows of x); where that leaves the chip without enough waves, K is split over
// workgroups too (float32 partial sums, dense_sum). Each wave keeps
// the next STEPS steps of 32 values in flight while it multiplies the current ones (ordinary loads: a load takes half of each
// row's cache line, and streamed past the caches the other half came from memory again, 36 against 30 us). Loads are 16 bytes at any alignment, so
// odd row lengths need no copy; rows past the ends repeat the last one and their sums are dropped.

#include <algorithm>

#include "dense_gemm.h"
#include "dense_rows.h"

namespace wf {

typedef float f32x4v __attribute__((ext_vector_type(4)));

template <int D>
__device__ __forceinline__ f32x4v mma_rows(const f32x4v& c, const Pack<D>& a, const Pack<D>& b) {
    if constexpr (D == WF_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8v, a), __builtin_bit_cast(f16x8v, b), c, 0, 0,
                                                      0);
}

// workgroup (16 RT weight rows, slice of K, 16 rows of x). PAIR (RT = 2): the gated linear's 16 rows of the gate and the 16 of
// the other half that go with them, N rows further on, with its epilogue and partial sums [slices, M, 2 N].
template <int D, int RT, bool PAIR, typename Epilogue>
__global__ __launch_bounds__(256) void dense_rows(const uint16_t* __restrict__ x, int64_t ldx,
                                                     const uint16_t* __restrict__ w, int64_t ldw, int M, int N, int K,
                                                     float* __restrict__ parts, Epilogue e) {
    constexpr int STEPS = 4, W = 4;
    static_assert(!PAIR || RT == 2, "a tile of each half");
    constexpr int ROW = 16 * RT + 4;                              // (a lane's 4 sums are one store; rows apart by 4 banks)
    __shared__ float red[W][16][ROW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * (PAIR ? 1 : RT), m0 = blockIdx.z * 16, r = lane & 15, q = lane >> 4;
    const int steps = (K + 31) / 32, per = (steps + W * gridDim.y - 1) / (W * (int)gridDim.y);
    const int s0 = min(steps, ((int)blockIdx.y * W + wave) * per), s1 = min(steps, s0 + per);
    const int whole = min(s1, K / 32);                            // steps of 32 values; at most one, the last, is short
    const uint16_t* wp[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) wp[i] = w + (PAIR ? i * N + min(n0 + r, N - 1) : min(n0 + 16 * i + r, N - 1)) * ldw + 8 * q;
    const uint16_t* xp = x + min(m0 + r, M - 1) * ldx + 8 * q;
    f32x4v acc[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) acc[i] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
    Pack<D> a[STEPS][RT], b[STEPS];
    auto load = [&](int u, int s, int cnt) {
#pragma unroll
        for (int i = 0; i < RT; i++) a[u][i].load(wp[i] + s * 32, cnt);
        b[u].load(xp + s * 32, cnt);
    };
    auto mul = [&](int u) {
#pragma unroll
        for (int i = 0; i < RT; i++) acc[i] = mma_rows<D>(acc[i], a[u][i], b[u]);
    };
    int s = s0;
    if (s + STEPS <= whole) {
#pragma unroll
        for (int u = 0; u < STEPS; u++) load(u, s + u, 8);
        for (; s + 2 * STEPS <= whole; s += STEPS) {
#pragma unroll
            for (int u = 0; u < STEPS; u++) {                     // a step's registers are free once its MFMAs are issued
                mul(u);
                load(u, s + STEPS + u, 8);
            }
        }
#pragma unroll
        for (int u = 0; u < STEPS; u++) mul(u);
        s += STEPS;
    }
    for (; s < whole; s++) {
        load(0, s, 8);
        mul(0);
    }
    if (s < s1) {
        load(0, s, K - s * 32 - 8 * q);
        mul(0);
    }
    // lane: weight rows 4 q .. 4 q + 3 of a tile, x row r
#pragma unroll
    for (int i = 0; i < RT; i++) *reinterpret_cast<f32x4v*>(&red[wave][r][16 * i + 4 * q]) = acc[i];
    __syncthreads();
    auto sum = [&](float (&v)[8], int m, int c) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] += red[i][m][c + k];
    };
    if constexpr (PAIR) {
        if (threadIdx.x < 32) {
            const int m = threadIdx.x / 2, c = 8 * (threadIdx.x % 2), n = n0 + c, cnt = N - n;
            if (m0 + m >= M || cnt <= 0) return;
            float g[8], u[8];
            sum(g, m, c);
            sum(u, m, 16 + c);
            if (!parts) {
                gated_run<D, true>(e, g, u, m0 + m, n, N, cnt);
                return;
            }
            float* o = parts + ((int64_t)blockIdx.y * M + m0 + m) * 2 * N + n;
            store_run(o, g, cnt);
            store_run(o + N, u, cnt);
        }
        return;
    } else {
        constexpr int RUNS = 2 * RT;
        if (threadIdx.x < 16 * RUNS) {
            const int m = threadIdx.x / RUNS, c = 8 * (threadIdx.x % RUNS), n = n0 + c, cnt = N - n;
            if (m0 + m >= M || cnt <= 0) return;
            float v[8];
            sum(v, m, c);
            if (!parts) {
                epilogue_run<D, true>(e, v, epilogue_ahead<D>(e, m0 + m, n, N, cnt), m0 + m, n, N, cnt);
                return;
            }
            store_run(parts + ((int64_t)blockIdx.y * M + m0 + m) * N + n, v, cnt);
        }
    }
}

template <int D>
static void launch(const DenseRowsPlan& p, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int M, int N, int K,
                   float* parts, const DenseEpilogue& e, hipStream_t s) {
    auto go = [&](auto rt) {
        constexpr int RT = decltype(rt)::value;
        const dim3 grid((uint32_t)((N + 16 * RT - 1) / (16 * RT)), p.slices, (uint32_t)((M + 15) / 16));
        dense_rows<D, RT, false><<<grid, 256, 0, s>>>(x, ldx, w, ldw, M, N, K, parts, e);
    };
    if (p.tiles == 1) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
}

void dense_rows_run(int dt, const DenseRowsPlan& p, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int M,
                    int N, int K, float* parts, const DenseEpilogue& e, hipStream_t s) {
    if (dt == WF_BF16) launch<WF_BF16>(p, x, ldx, w, ldw, M, N, K, parts, e, s);
    else launch<WF_F16>(p, x, ldx, w, ldw, M, N, K, parts, e, s);
}

void gated_rows_run(int dt, int slices, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int M, int N, int K,
                    float* parts, const GatedEpilogue& e, hipStream_t s) {
    const dim3 grid((uint32_t)((N + 15) / 16), slices, (uint32_t)((M + 15) / 16));
    if (dt == WF_BF16) dense_rows<WF_BF16, 2, true><<<grid, 256, 0, s>>>(x, ldx, w, ldw, M, N, K, parts, e);
    else dense_rows<WF_F16, 2, true><<<grid, 256, 0, s>>>(x, ldx, w, ldw, M, N, K, parts, e);
}

}  // namespace wf
