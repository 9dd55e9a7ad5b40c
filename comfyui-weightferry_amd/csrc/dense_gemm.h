// The tiled kernel of the 16-bit linear and its launch; dense.hip chooses how a product runs.
#pragma once

#include "dense.h"
#include "dense_ring.h"

namespace wf {

typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));

template <int D>
__device__ __forceinline__ f32x16v mma16(const f32x16v& c, const wl_frag& a, const wl_frag& b) {
    if constexpr (D == WF_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8v, a), __builtin_bit_cast(f16x8v, b), c, 0, 0,
                                                      0);
}

// An operand as the kernel loads it, 16-byte runs throughout: along K, value (r, k) at r * row + k and k values to load of
// a row (a copied row's zeros among them); or across K (x set), at k * row + r, r up to `rows`.
struct DenseOperand {
    const uint16_t* p;
    int64_t row;
    int k, rows;
    bool x;
};

// the buffer of rows r0.. of an operand: it ends with the last value's 16-byte run
template <bool X>
__device__ __forceinline__ DenseTile dense_tile(const DenseOperand& o, int r0) {
    const int64_t at = X ? r0 : r0 * o.row;
    const int64_t end = X ? (o.k - 1) * o.row + ((o.rows + 7) & ~7) : (o.rows - 1) * o.row + o.k;
    return {tile_rsrc(o.p + at, (end - at) * 2), (uint32_t)o.row * 2u, (uint32_t)o.k * 2u};
}

// Workgroup (tile, slice). parts: [slices, M, N] float32 partial sums, or NULL: one slice, and the outputs. PLAIN: the
// epilogue is at most a bias.
template <int D, bool AX, bool BX, bool PLAIN, typename S>
__global__ __launch_bounds__(S::NT, S::WAVES) void dense_gemm(DenseOperand a, DenseOperand b, int M, int N, int K, int slice_stages,
                                                    float* __restrict__ parts, DenseEpilogue e) {
    constexpr int WM = S::WM, WN = S::WN, TC = WN * 32;
    __shared__ wl_frag sb0[S::SLOTS], sb1[S::SLOTS];
    const int ntm = (M + S::BM - 1) / S::BM, ntn = (N + S::BN - 1) / S::BN;
    int tm, tn;
    tile_order(blockIdx.x, ntm * ntn, ntm, ntn, tm, tn);
    const int m0 = __builtin_amdgcn_readfirstlane(tm * S::BM), n0 = __builtin_amdgcn_readfirstlane(tn * S::BN);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int stages = (K + 63) / 64, s0 = blockIdx.y * slice_stages, nk = min(slice_stages, stages - s0);
    const DenseTile ta = dense_tile<AX>(a, m0), tb = dense_tile<BX>(b, n0);
    // the sums start from the bias
    f32x16v acc[WM][WN];
#pragma unroll
    for (int j = 0; j < WN; j++) {
        const int n = n0 + wave % S::VN * TC + j * 32 + (lane & 31);
        const float bn = !parts && e.bias && n < N ? load_value(e.bias, n, e.bias_dt) : 0.0f;
#pragma unroll
        for (int i = 0; i < WM; i++)
#pragma unroll
            for (int x = 0; x < 16; x++) acc[i][j][x] = bn;
    }
    dense_mainloop<S, AX, BX>(ta, tb, s0, nk, wave, lane, sb0, sb1, acc,
                              [](const f32x16v& c, const wl_frag& x, const wl_frag& y) { return mma16<D>(c, x, y); });
    const int mw = m0 + wave / S::VN * WM * 32, nw = n0 + wave % S::VN * TC;
    const int lr = lane & 31, lk = lane >> 5;
    // Outputs of whole 16-byte runs whose tile lies in one group of the gate are computed in the accumulators: the residual
    // comes through LDS into their layout, the outputs go out through it rounded, the pre-activations, where they are
    // kept, before them. 4096 x 5120 x 5120 with a gated residual takes 171 us, 183 by the loop over runs below; with GELU 167
    // against 174.
    uint16_t* o16 = wl_out_region<S>(sb0, sb1, wave);
    auto store = [&](void* out, auto&& f) {
        wl_store_tile<WM, WN>(o16, static_cast<uint16_t*>(out), M, N, mw, nw, lane,
                              [&](int i, int j, int x) { return from_f32<D>(f(acc[i][j][x])); });
    };
    if constexpr (PLAIN) {
        if (!parts) {
            store(e.y, [](float v) { return v; });
            return;
        }
    } else {
        const uint32_t rpg = (uint32_t)e.rows_per_group, group = (uint32_t)m0 / rpg;
        const bool one_group = !e.gate || group == (uint32_t)(min(m0 + S::BM, M) - 1) / rpg;
        if (!parts && one_group && ((N & 7) == 0 || (!e.gate && !e.resid))) {
            constexpr int ROW_RUNS = TC / 8;                       // (16 rows at a time: their runs are WN a lane)
            Pack<D> res[WN];
            auto fetch = [&](int half) {
#pragma unroll
                for (int it = 0; it < WN; it++) {
                    const int q = it * 64 + lane, m = mw + 16 * half + q / ROW_RUNS, n = nw + 8 * (q % ROW_RUNS);
                    res[it].zero();
                    if (m < M && n < N) res[it].load(static_cast<const value_t<D>*>(e.resid) + m * e.ldr + n, 8);
                }
            };
            if (e.resid) fetch(0);
            float gj[WN];
#pragma unroll
            for (int j = 0; j < WN; j++) {
                const int n = nw + j * 32 + lr;
                gj[j] = e.gate && n < N ? load_value(e.gate, (int64_t)group * N + n, e.gate_dt) : 1.0f;
            }
            if (e.h) store(e.h, [](float v) { return keep_finite<D>(v); });
            by_act(e.act, [&](auto k) {
                auto act = [&](int i, int j, int x) { return act_of<decltype(k)::value>(acc[i][j][x]) * gj[j]; };
                if (!e.resid) {
                    wl_store_tile<WM, WN>(o16, static_cast<uint16_t*>(e.y), M, N, mw, nw, lane,
                                          [&](int i, int j, int x) { return from_f32<D>(act(i, j, x)); });
                    return;
                }
                auto run_at = [&](int q) { return static_cast<uint16_t*>(__builtin_assume_aligned(o16 + 8 * q, 16)); };
#pragma unroll
                for (int half = 0; half < 2 * WM; half++) {
#pragma unroll
                    for (int it = 0; it < WN; it++)
                        __builtin_memcpy(run_at(it * 64 + lane), res[it].w, 16);
                    if (half + 1 < 2 * WM) fetch(half + 1);
#pragma unroll
                    for (int x = 0; x < 8; x++)                    // each value in its place, by the lane that has its sum
#pragma unroll
                        for (int j = 0; j < WN; j++) {
                            uint16_t& at = o16[(8 * (x >> 2) + 4 * lk + (x & 3)) * TC + j * 32 + lr];
                            at = from_f32<D>(act(half / 2, j, 8 * (half & 1) + x) + to_f32<D>(at));
                        }
#pragma unroll
                    for (int it = 0; it < WN; it++) {
                        const int q = it * 64 + lane, m = mw + 16 * half + q / ROW_RUNS, n = nw + 8 * (q % ROW_RUNS);
                        Pack<D> v;
                        __builtin_memcpy(v.w, run_at(q), 16);
                        if (m < M && n < N) v.store(static_cast<value_t<D>*>(e.y) + (int64_t)m * N + n, 8);
                    }
                }
            });
            return;
        }
    }
    // the wave's region: 16 rows x TC float32
    constexpr int PER_BUF = S::SLOTS * 16 / (16 * TC * 4);
    static_assert(2 * PER_BUF >= S::NW, "the output rows fit in the stage buffers");
    float* ot = reinterpret_cast<float*>(wave < PER_BUF ? sb0 : sb1) + (wave % PER_BUF) * 16 * TC;
    constexpr int RUNS = TC / 8;
    // (the loop over runs stays a loop: unrolled, the epilogue's code took longer to fetch than to run. What a run needs
    // from memory is loaded two runs ahead.)
    // WHOLE: every run is 8 outputs.
    auto body = [&](auto whole) {
        auto at_run = [&](int half, int it, auto&& f) {
            const int over = it >= WN, q = (over ? it - WN : it) * 64 + lane;
            const int m = mw + (half + over) * 16 + q / RUNS, n = nw + 8 * (q % RUNS);
            return f(q, m, n, m < M && n < N ? (decltype(whole)::value ? 8 : N - n) : 0);
        };
        auto ahead = [&](int half, int it) {
            return at_run(half, it, [&](int, int m, int n, int cnt) {
                EpilogueAhead<D> a = {};
                if (cnt > 0) a = epilogue_ahead<D>(e, m, n, N, decltype(whole)::value ? 8 : cnt);
                return a;
            });
        };
        EpilogueAhead<D> next[2];
        if (!PLAIN && !parts) next[0] = ahead(0, 0), next[1] = ahead(0, 1);
#pragma unroll
        for (int half = 0; half < 2 * WM; half++) {
            if (mw + half * 16 >= M) break;
#pragma unroll
            for (int x = 0; x < 8; x++)
#pragma unroll
                for (int j = 0; j < WN; j++)
                    ot[(8 * (x >> 2) + 4 * lk + (x & 3)) * TC + j * 32 + lr] = acc[half / 2][j][8 * (half & 1) + x];
#pragma unroll 1
            for (int it = 0; it < WN; it++) {
                EpilogueAhead<D> now;
                if (!PLAIN && !parts) {
                    now = next[0];
                    next[0] = next[1];
                    next[1] = ahead(half, it + 2);
                }
                at_run(half, it, [&](int q, int m, int n, int count) {
                    const float4 lo = reinterpret_cast<const float4*>(ot)[2 * q], hi = reinterpret_cast<const float4*>(ot)[2 * q + 1];
                    float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                    if (count <= 0) return;
                    const int cnt = decltype(whole)::value ? 8 : count;
                    if (!PLAIN && !parts) {
                        epilogue_run<D, false>(e, v, now, m, n, N, cnt);
                        return;
                    }
                    float* o = parts + ((int64_t)blockIdx.y * M + m) * N + n;
                    if (cnt >= 8) __builtin_memcpy(o, v, 32);
                    else
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (i < cnt) o[i] = v[i];
                });
            }
        }
    };
    if ((N & 7) == 0) body(std::true_type{});
    else body(std::false_type{});
}

struct DensePlan {
    int tiling, slices, slice_stages;
};

template <int D, bool AX, bool BX, bool PLAIN, int VM, int VN, int WM, int WN>
static void dense_launch(const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                         float* parts, const DenseEpilogue& e, hipStream_t s) {
    using S = DenseShape<VM, VN, WM, WN>;
    const int tiles = ((M + S::BM - 1) / S::BM) * ((N + S::BN - 1) / S::BN);
    dense_gemm<D, AX, BX, PLAIN, S><<<dim3(tiles, p.slices), S::NT, 0, s>>>(a, b, M, N, K, p.slice_stages, parts, e);
}

// the tilings by number; kDense in dense.hip has their sizes
template <int D, bool AX, bool BX, bool PLAIN>
static void dense_tiling(const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p, float* parts,
                         const DenseEpilogue& e, hipStream_t s) {
    switch (p.tiling) {
    case 0: dense_launch<D, AX, BX, PLAIN, 4, 2, 2, 5>(a, b, M, N, K, p, parts, e, s); break;
    case 1: dense_launch<D, AX, BX, PLAIN, 2, 2, 4, 4>(a, b, M, N, K, p, parts, e, s); break;
    case 2: dense_launch<D, AX, BX, PLAIN, 2, 2, 4, 3>(a, b, M, N, K, p, parts, e, s); break;
    case 3: dense_launch<D, AX, BX, PLAIN, 2, 2, 2, 3>(a, b, M, N, K, p, parts, e, s); break;
    case 4: dense_launch<D, AX, BX, PLAIN, 4, 1, 1, 5>(a, b, M, N, K, p, parts, e, s); break;
    case 5: dense_launch<D, AX, BX, PLAIN, 2, 2, 2, 2>(a, b, M, N, K, p, parts, e, s); break;
    case 6: dense_launch<D, AX, BX, PLAIN, 1, 4, 2, 1>(a, b, M, N, K, p, parts, e, s); break;
    default: dense_launch<D, AX, BX, PLAIN, 1, 4, 1, 1>(a, b, M, N, K, p, parts, e, s); break;
    }
}

// One source each: both operands along K with a plain and with any epilogue, B across, both across (plain, or into parts).
// parts: NULL where the outputs are stored.
void dense_gemm_along(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                      float* parts, const DenseEpilogue& e, hipStream_t s);
void dense_gemm_along_full(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                           float* parts, const DenseEpilogue& e, hipStream_t s);
void dense_gemm_b_across(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                         float* parts, const DenseEpilogue& e, hipStream_t s);
void dense_gemm_across(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                       float* parts, const DenseEpilogue& e, hipStream_t s);

}  // namespace wf
