// The gated feed-forward layer's first half for gfx950: y = act(x wg^T + bg) * (x wu^T + bu), both projections, the activation and
// the product in one kernel, and its backward pass. The weight is [2 N, K], the gate's N rows first.
//
//   g, u = the two halves of x w^T + bias,  y = act(g) u
//   dg = dy u act'(g),  du = dy act(g),  dx = [dg du] w,  dw = [dg du]^T x,  dbias = the column sums of [dg du]
//
// 4 M N K operations forward. The tiles are those of the 16-bit linear (dense_gemm.h), but a tile's rows of the weight are fragments of 32
// from the gate's half and from the other in turn, so that a wave's accumulators hold g and u of the same outputs: the epilogue
// is arithmetic on registers, and neither g nor u goes to memory unless the backward pass will want them (gated.h has the format). A
// product with too few tiles runs as slices of K, whose float32 sums a second kernel adds before the epilogue; few rows of x take
// the form of dense_rows.hip with a tile of each half a workgroup. Operands whose rows are no aligned 16-byte runs are copied into rows
// that are, or, where that would cost more, loaded as they lie (loose_ring.h).
//
// Backward: one element-wise kernel from dy and the kept g and u to [dg du], [M, 2 N], rounded to the operands' type because it is the
// operand of the two products behind it, which are the 16-bit linear's own on a weight of 2 N rows.
//
// In float16 a product of dy and u leaves the type's range where neither they nor the gradients do: past 65504 dx and dw would be
// infinity minus infinity, below 2^-24 zero. So that kernel also finds the largest finite magnitude of [dg du], and where it is past
// 65504 or below 2^-8 (a rounding in steps of 2^-24 is then no longer small beside 2^-11 of it) a second one writes [dg du] again times
// the power of two that brings it to 2^14, which the products' epilogues take back in float32. Elsewhere the second kernel ends after
// reading those magnitudes: 4.7 us at 1560 x 13824, 45 where it writes.

#include <algorithm>
#include <type_traits>

#include "column_sums.h"
#include "deep_ring.h"
#include "dense_call.h"
#include "grids.h"
#include "loose_ring.h"
#include "tile_stage.h"

namespace wf {

// a, b: x and the weight's first half, along K; half: values from a row of the first half to the same of the second. Workgroup
// (tile, slice); parts: [slices, M, 2 N] float32 partial sums, or NULL: one slice, and the outputs.
enum { RING_TWO, RING_DEEP, RING_LOOSE };                          // two stage buffers, four, rows that start anywhere
template <int D, typename S, int RING>
__global__ __launch_bounds__(S::NT, (RING == RING_TWO ? S::WAVES : 1)) void gated_gemm(DenseOperand a, DenseOperand b, int64_t half,
                                                                                       int M, int N, int K, int slice_stages,
                                                                                       float* __restrict__ parts, GatedEpilogue e) {
    constexpr int WM = S::WM, WN = S::WN, TC = WN * 16, BO = S::BN / 2;    // outputs of a wave's row, of a tile's
    static_assert(WN % 2 == 0, "a fragment of each half");
    constexpr int MORE = RING == RING_DEEP ? S::SLOTS : 1;
    __shared__ wl_frag sb0[S::SLOTS], sb1[S::SLOTS], sb2[MORE], sb3[MORE];
    const int ntm = (M + S::BM - 1) / S::BM, ntn = (N + BO - 1) / BO;
    int tm, tn;
    tile_order(blockIdx.x, ntm * ntn, ntm, ntn, tm, tn);
    const int m0 = __builtin_amdgcn_readfirstlane(tm * S::BM), n0 = __builtin_amdgcn_readfirstlane(tn * BO);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int stages = (K + 63) / 64, s0 = blockIdx.y * slice_stages, nk = min(slice_stages, stages - s0);
    const int mw = m0 + wave / S::VN * WM * 32, nw = n0 + wave % S::VN * TC;
    const int lr = lane & 31, lk = lane >> 5;
    // the sums start from the bias
    f32x16v acc[WM][WN];
#pragma unroll
    for (int j = 0; j < WN; j++) {
        const int n = nw + j / 2 * 32 + lr;
        const float bn = !parts && e.bias && n < N ? load_value(e.bias, (int64_t)(j & 1) * N + n, e.bias_dt) : 0.0f;
#pragma unroll
        for (int i = 0; i < WM; i++)
#pragma unroll
            for (int x = 0; x < 16; x++) acc[i][j][x] = bn;
    }
    auto mma = [](const f32x16v& c, const wl_frag& x, const wl_frag& y) { return mma16<D>(c, x, y); };
    if constexpr (RING == RING_LOOSE) {
        const uint16_t* w = b.p + n0 * b.row;
        const LooseTile ta = {a.p + m0 * a.row, (uint32_t)a.row, M - m0, K};
        const LoosePair tb = {{w, w + half}, (uint32_t)b.row, N - n0, K};
        loose_loop<S, LooseAlong<S::NW, S::AW>, LooseAlongPair<S::NW, S::BW>>(ta, tb, s0, nk, wave, lane, sb0, sb1, acc, mma);
    } else {
        using LA = DenseAlong<S::BM, S::NW, S::AW, WM>;
        using LB = DenseAlongPair<S::BN, S::NW, S::BW, WN>;
        const DenseTile ta = dense_tile<false>(a, m0), tg = dense_tile<false>(b, n0);
        b.p += half;
        const DensePair tb = {{tg.r, dense_tile<false>(b, n0).r}, tg.row, tg.k};
        if constexpr (RING == RING_DEEP) {
            wl_frag* const sb[kDeep] = {sb0, sb1, sb2, sb3};
            deep_loop<S, LA, LB>(ta, tb, s0, nk, wave, lane, sb, acc, mma);
        } else {
            dense_loop<S, LA, LB>(ta, tb, s0, nk, wave, lane, sb0, sb1, acc, mma);
        }
    }
    if (parts) {                                                   // (32 lanes store 128 bytes of a row)
        float* o = parts + (int64_t)blockIdx.y * M * 2 * N;
#pragma unroll
        for (int i = 0; i < WM; i++)
#pragma unroll
            for (int x = 0; x < 16; x++) {
                const int m = mw + 32 * i + 8 * (x >> 2) + 4 * lk + (x & 3);
                if (m >= M) continue;
#pragma unroll
                for (int j = 0; j < WN; j++) {
                    const int n = nw + j / 2 * 32 + lr;
                    if (n < N) o[((int64_t)m * 2 + (j & 1)) * N + n] = acc[i][j][x];
                }
            }
        return;
    }
    using Stage = TileStage<S>;
    constexpr int RUNS = TC / 8;
    float* t = Stage::region(sb0, sb1, wave);
    static_for<Stage::PHASES>([&](auto pc) {
        constexpr int P = decltype(pc)::value;
        if (mw + P * Stage::ROWS >= M) return;
        Stage::template put<P>(t, acc, lane);
#pragma unroll 1
        for (int it = 0; it < Stage::ROWS * RUNS / 64; it++) {
            const int q = it * 64 + lane, r = q / RUNS, c = 8 * (q % RUNS), m = mw + P * Stage::ROWS + r, n = nw + c;
            const float* p = t + r * Stage::TC + (c & ~31) * 2 + (c & 31);
            float g[8], u[8];
            staged_run(g, p);
            staged_run(u, p + 32);
            if (m < M && n < N) gated_run<D, false>(e, g, u, m, n, N, N - n);
        }
    });
}

// the slices' sums in slice order, then the epilogue: one run of 8 outputs a thread, from workgroup `wg` of the whole on
template <int D>
__global__ __launch_bounds__(256) void gated_sum(int64_t wg, const float* __restrict__ parts, int slices, int M, int N,
                                                 GatedEpilogue e) {
    const int runs = (N + 7) / 8;
    const int64_t i = (wg + blockIdx.x) * 256 + threadIdx.x;
    if (i >= (int64_t)M * runs) return;
    const int64_t m = i / runs;
    const int n = (int)(i - m * runs) * 8, cnt = N - n;
    const float* p = parts + m * 2 * N + n;
    const int64_t plane = (int64_t)M * 2 * N;
    auto load = [&](float (&v)[8], const float* q) {
        if (cnt >= 8) __builtin_memcpy(v, q, 32);
        else
#pragma unroll
            for (int x = 0; x < 8; x++) v[x] = x < cnt ? q[x] : 0.0f;
    };
    float g[8] = {0, 0, 0, 0, 0, 0, 0, 0}, u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = 0; s < slices; s += 2) {                          // two slices' loads in flight, added in order
        float a[2][8], b[2][8];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int64_t at = min(s + k, slices - 1) * plane;
            load(a[k], p + at);
            load(b[k], p + at + N);
        }
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (s + k < slices)
#pragma unroll
                for (int x = 0; x < 8; x++) g[x] += a[k][x], u[x] += b[k][x];
    }
    gated_run<D, true>(e, g, u, m, n, N, cnt);
}

// The backward pass's element-wise part: workgroup (512 columns, i) walks rows 4 i + wave, + 4 gridDim.y, ...; bparts:
// [gridDim.y, 2 N] float32 sums of the unrounded dg and du, or NULL. dh: [M, ldh], ldh a multiple of 8, zeros past 2 N, or NULL.
// range (float16; NULL without dh): [0] what the products are to be multiplied by, then the largest finite magnitude of each workgroup.
// AGAIN: the second kernel, which does nothing where [0] is 1.
template <int D, bool AGAIN>
__global__ __launch_bounds__(256) void gated_dact(const value_t<D>* __restrict__ dy, int64_t ldd, const uint16_t* __restrict__ kept,
                                                  int64_t plane, int act, value_t<D>* __restrict__ dh, int64_t ldh,
                                                  float* __restrict__ bparts, float* __restrict__ range, int M, int N) {
    __shared__ float red[4][2][512], tops[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = blockIdx.x * 512 + lane * 8, cnt = N - n;
    const bool first = blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0;
    auto largest = [&](float v) {                                  // of the workgroup's, in every thread
        v = wave_max_bits(v);
        if (lane == 0) tops[wave] = v;
        __syncthreads();
        return fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    };
    float top = 0.0f, scale = 1.0f;
    if constexpr (AGAIN) {
        const int parts = gridDim.x * gridDim.y;
        for (int i = threadIdx.x; i < parts; i += 256) top = fmaxf(top, range[1 + i]);
        top = largest(top);
        const bool fits = top == 0.0f || (top <= 65504.0f && top >= 0.00390625f);
        const int up = fits ? 0 : min(126, 14 - ilogbf(top));      // (2^126 and its reciprocal are normal numbers)
        if (first) range[0] = ldexpf(1.0f, -up);
        if (fits) return;
        scale = ldexpf(1.0f, up);
    }
    float sg[8], su[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sg[i] = su[i] = 0.0f;
    for (int64_t m = blockIdx.y * 4 + wave; m < M && cnt > 0; m += gridDim.y * 4) {
        const int64_t at = m * N + n;
        Pack<D> pd;
        Pack<WF_BF16> pg, pu, pl;
        pd.load(dy + m * ldd + n, cnt);
        pg.load(kept + at, cnt);
        pu.load(kept + plane + at, cnt);
        pl.load(kept + 2 * plane + at, cnt);
        float g[8], a[8], slope[8], dg[8], du[8];
        auto half = [](const Pack<WF_BF16>& p, int i) { return i & 1 ? p.w[i / 2] >> 16 : p.w[i / 2] & 0xffffu; };
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] = kept_g(half(pg, i), half(pl, i));
        act_slope_run(act, g, a, slope);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float d = pd.get(i);
            dg[i] = d * kept_u(half(pu, i), half(pl, i)) * slope[i];
            du[i] = d * a[i];
            if constexpr (!AGAIN) sg[i] += dg[i], su[i] += du[i];
            if constexpr (AGAIN) dg[i] *= scale, du[i] *= scale;
            if constexpr (D == WF_F16 && !AGAIN) {
                const float a = fabsf(dg[i]), b = fabsf(du[i]);    // (infinity and NaN are what they are at any scale)
                top = fmaxf(top, fmaxf(a <= 3.4028235e38f ? a : 0.0f, b <= 3.4028235e38f ? b : 0.0f));
            }
        }
        if (!dh) continue;
        Pack<D> o;
        value_t<D>* row = dh + m * ldh;
        o.put(dg);
        o.store(row + n, cnt);
        o.put(du);
        o.store(row + N + n, cnt);
        if (cnt <= 8)                                              // a row's last run writes its padding too
            for (int64_t k = 2 * (int64_t)N; k < ldh; k++) row[k] = from_f32<D>(0.0f);
    }
    if constexpr (AGAIN) return;
    if constexpr (D == WF_F16)
        if (range) {
            top = largest(top);
            if (threadIdx.x == 0) range[1 + blockIdx.y * gridDim.x + blockIdx.x] = top;
        }
    if (!bparts) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        red[wave][0][lane * 8 + i] = sg[i];
        red[wave][1][lane * 8 + i] = su[i];
    }
    __syncthreads();
    float* out = bparts + (int64_t)blockIdx.y * 2 * N;
    for (int c = threadIdx.x; c < 512; c += 256) {
        const int col = blockIdx.x * 512 + c;
        if (col >= N) continue;
        out[col] = red[0][0][c] + red[1][0][c] + red[2][0][c] + red[3][0][c];
        out[N + col] = red[0][1][c] + red[1][1][c] + red[2][1][c] + red[3][1][c];
    }
}

// ------------------------------------------------------------------------------------------------- host side
// Rows of x and of the weight (both halves) a tile, and its times, chosen so that the model picks well among 380 measured launches (20
// shapes of 40-16384 rows, 1000-13824 outputs and K 512-8192, weights not in the caches, with and without the halves kept): what it takes
// is 2 % longer than the best on average. Where a tile has a CU to itself a ring of four stages waits less than two buffers: us in 128
// x 128 tiles, two buffers / four, 128 x 13824 x 5120 79.5 / 70.5, 700 x 2048 x 5120 43.7 (two slices) / 40.2, 77 x 2608 x 1536 16.9 /
// 15.2; 512 x 8192 x 2048, two tiles a CU, 38.6 / 43.6. 4096 x 13824 x 5120 in these tilings: 827 / 1244 / 1092 / 1273 / 2669.
constexpr DenseTiling kGated[] = {{256, 256, 1, 6.1f, 1.09f, 1.09f}, {128, 256, 1, 3.0f, 0.70f, 0.70f},
                                  {128, 128, 2, 0.4f, 0.60f, 0.56f}, {128, 128, 1, 0.8f, 0.432f, 0.432f},
                                  {32, 256, 1, 1.3f, 0.426f, 0.426f}};
// The same for rows that start anywhere: us with copies of both operands and the tilings above (or few rows) / as they lie, of 22 shapes:
// 77 x 2607 x 1531 28 / 19.7, 300 x 1000 x 1025 22.9 / 14.6, 40 x 8191 x 2047 50 / 28, 1 x 13823 x 5119 138 / 67, 2000 x 2047 x 333 22.8 / 19.3;
// but 128 x 5121 x 5119 74 / 76, 700 x 2047 x 2559 38.4 / 40.6: odd places halve the loads' rate, and long sums pay for that more than
// once a copy. The way the model chooses among the two and their slices takes 3 % longer than the best on average.
constexpr DenseTiling kLooseTiles[] = {{128, 128, 2, 2.5f, 0.863f, 0.979f}, {64, 128, 3, 1.3f, 0.556f, 0.67f}};

template <int D>
static void gated_tiling(const DenseOperand& a, const DenseOperand& b, int64_t half, int M, int N, int K, const DensePlan& p, bool loose,
                         float* parts, const GatedEpilogue& e, hipStream_t s) {
    auto go = [&](auto shape, auto ring) {
        using S = decltype(shape);
        const int tiles = ((M + S::BM - 1) / S::BM) * ((N + S::BN / 2 - 1) / (S::BN / 2));
        gated_gemm<D, S, decltype(ring)::value><<<dim3(tiles, p.slices), S::NT, 0, s>>>(a, b, half, M, N, K, p.slice_stages, parts, e);
    };
    const std::integral_constant<int, RING_TWO> two{};
    const std::integral_constant<int, RING_DEEP> four{};
    const std::integral_constant<int, RING_LOOSE> any{};
    if (loose) {
        if (p.tiling == 0) go(DenseShape<2, 2, 2, 2>{}, any);
        else go(DenseShape<2, 2, 1, 2>{}, any);
        return;
    }
    switch (p.tiling) {
    case 0: go(DenseShape<2, 2, 4, 4>{}, two); break;
    case 1: go(DenseShape<2, 2, 2, 4>{}, two); break;
    case 2: go(DenseShape<2, 2, 2, 2>{}, two); break;
    case 3: go(DenseShape<2, 2, 2, 2>{}, four); break;
    default: go(DenseShape<1, 4, 1, 2>{}, four); break;
    }
}

// How a call runs: few rows, or tiles in slices of K, of rows that start anywhere if loose; where the copies of operands that cannot be
// loaded as they lie and the partial sums are in the workspace.
struct GatedCall {
    bool few, loose;
    int slices;
    DensePlan tiles;
    int how_x, how_w;
    int64_t w_at, parts_at, bytes;
};
static GatedCall gated_call(const DenseView& x, const DenseView& w, int64_t M, int64_t N, int64_t K, bool keep) {
    GatedCall c = {};
    float us;
    c.tiles = dense_plan_tiles(kGated, (int)(sizeof(kGated) / sizeof(kGated[0])), M, 2 * N, K, EPI_ACT | (keep ? EPI_KEEP : 0), 5.5f, us);
    c.slices = c.tiles.slices;
    c.how_x = dense_how(x, M, K, false);
    c.how_w = dense_how(w, 2 * N, K, false);
    c.w_at = dense_copy_bytes(c.how_x, M, K);
    c.parts_at = c.w_at + dense_copy_bytes(c.how_w, 2 * N, K);
    if (c.w_at) us += 3.0f + (float)c.w_at * 0.5e-6f;
    if (c.parts_at > c.w_at) us += 3.0f + (float)(c.parts_at - c.w_at) * 0.5e-6f;
    auto rows = [](int how, const DenseView& v, int64_t R) {
        return how == LIES_ALONG || (how == COPY_ALONG && (R == 1 || v.row <= (1 << 20)));
    };
    if (c.parts_at && K >= 8 && rows(c.how_x, x, M) && rows(c.how_w, w, 2 * N)) {
        float any;
        const DensePlan p = dense_plan_tiles(kLooseTiles, (int)(sizeof(kLooseTiles) / sizeof(kLooseTiles[0])), M, 2 * N, K,
                                             EPI_ACT | (keep ? EPI_KEEP : 0), 7.0f, any);
        if (any < us) {
            us = any;
            c.loose = true;
            c.tiles = p;
            c.slices = p.slices;
            c.w_at = c.parts_at = 0;
        }
    }
    if (M <= 256 && x.col == 1 && w.col == 1) {
        const int slices = (N + 15) / 16 * ((M + 15) / 16) < 128 && K >= 4096 ? 4 : 1;
        float few = dense_rows_time(M, 2 * N, K, ((x.row | w.row) & 1) != 0);
        // (loads at odd places, one after the other: us in this form / in tiles of such rows 20 x 600 x 4001 31.7 / 16.5, 1 x 600 x 4001
        // 23.1 / 15.8, 8 x 1000 x 2047 20.9 / 15.9, 100 x 700 x 1025 21.8 / 14.3; 3 x 2607 x 1531 12.6 / 13.5. Over 70 other shapes, 1 to 256
        // rows, 64 to 13824 outputs, odd and even K up to 8192, what is chosen of the three forms takes 1 % longer than the best of them
        // on average, 26 % at most: 3 x 4737 x 6036 42 in this form, 33.5 in tiles)
        if (c.loose) few = std::max(few * (M > 16 ? 1.25f : 1.0f), 4.0f + (4.5e-3f + 0.4e-3f * std::min<int64_t>(M, 8)) * (K / slices));
        if (few < us) {
            c.few = true;
            c.loose = false;
            c.slices = slices;
            c.w_at = c.parts_at = 0;
        }
    }
    c.bytes = c.parts_at + (c.slices > 1 ? (int64_t)c.slices * M * 2 * N * 4 : 0);
    return c;
}

struct GatedBackward {
    int64_t dh_row, range_at, sums_at, product_at, bytes;
    bool ranged;                                       // float16, and dh is wanted
    int rows;                                          // of partial sums
    DenseView dh_along, w_turned, dh_turned, x_turned;
    DenseCall dx, dw;
};
static GatedBackward gated_backward(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, int dt, int64_t M,
                                    int64_t N, int64_t K, bool dx, bool dw, bool db, char* ws) {
    GatedBackward b = {};
    b.dh_row = up(2 * N, 8);
    const int64_t across = (N + 511) / 512;
    b.rows = (int)std::min<int64_t>((M + 3) / 4, std::max<int64_t>(1, 2048 / across));
    b.ranged = dt == WF_F16 && (dx || dw);
    b.range_at = dx || dw ? up(M * b.dh_row * 2, 256) : 0;
    b.sums_at = b.range_at + (b.ranged ? up((1 + across * b.rows) * 4, 256) : 0);
    b.product_at = b.sums_at + (db ? up((int64_t)b.rows * 2 * N * 4, 256) : 0);
    b.dh_along = {ws, b.dh_row, 1, true};              // (a workspace not yet there is as aligned as it will be)
    b.w_turned = {w, w_col, w_row, false};
    b.dh_turned = {ws, 1, b.dh_row, false};
    b.x_turned = {x, 1, x_row, false};
    if (dx) b.dx = dense_call(b.dh_along, b.w_turned, M, K, 2 * N, 0);      // (epilogue 0, which may be a factor)
    if (dw) b.dw = dense_call(b.dh_turned, b.x_turned, 2 * N, K, M, 0);
    b.bytes = b.product_at + std::max(b.dx.bytes, b.dw.bytes);
    return b;
}

static int gated_check(const char* who, int dt, int act, int64_t M, int64_t N, int64_t K, int64_t x_row, int64_t x_col,
                       int64_t w_row, int64_t w_col) {
    if (const int rc = dense_check(who, dt, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    if (act < ACT_NONE || act > ACT_RELU) { set_error("%s: activation %d", who, act); return WF_EINVAL; }
    if (M > (1 << 20) || N > (1 << 19)) {
        set_error("%s: M above 2^20 or N above 2^19", who);
        return WF_EUNSUPPORTED;
    }
    return WF_OK;
}

}  // namespace wf

extern "C" int wf_gated_dense_plan(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col,
                                   int dt, int64_t M, int64_t N, int64_t K, int keep, int* plan, int64_t* bytes) {
    using namespace wf;
    if (!plan || !bytes) { set_error("wf_gated_dense_plan: null pointer"); return WF_EINVAL; }
    if (const int rc = gated_check("wf_gated_dense_plan", dt, 0, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    *bytes = 0;
    plan[0] = plan[1] = plan[2] = plan[3] = plan[4] = 0;
    if (M == 0 || N == 0) return WF_OK;
    const GatedCall c = gated_call({x, x_row, x_col, false}, {w, w_row, w_col, false}, M, N, K, keep);
    plan[0] = c.few ? 0 : c.loose ? 2 : 1;
    plan[1] = c.few ? 0 : c.tiles.tiling;
    plan[2] = c.slices;
    plan[3] = c.few || c.loose ? LIES_ALONG : c.how_x;
    plan[4] = c.few || c.loose ? LIES_ALONG : c.how_w;
    *bytes = c.bytes;
    return WF_OK;
}

extern "C" int wf_gated_dense(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt,
                              int64_t M, int64_t N, int64_t K, const void* bias, int bias_dt, int act, void* y, void* kept,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = gated_check("wf_gated_dense", dt, act, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    if (bias && bias_dt != dt && bias_dt != WF_F32) { set_error("wf_gated_dense: dtype code %d of the bias", bias_dt); return WF_EINVAL; }
    if (M == 0 || N == 0) return WF_OK;
    if (!x || !w || !y) { set_error("wf_gated_dense: null pointer"); return WF_EINVAL; }
    if (!aligned(x, 2) || !aligned(w, 2) || !aligned(y, 2) || !aligned(kept, 2) || !aligned(bias, bias_dt == WF_F32 ? 4 : 2)) {
        set_error("wf_gated_dense: a pointer is not aligned to its values");
        return WF_EINVAL;
    }
    const DenseView xv = {x, x_row, x_col, false}, wv = {w, w_row, w_col, false};
    const GatedCall c = gated_call(xv, wv, M, N, K, kept != nullptr);
    char* ws = static_cast<char*>(workspace);
    if (c.bytes && (!ws || workspace_bytes < c.bytes || !aligned(ws, 256))) {
        set_error("wf_gated_dense: a workspace of %lld bytes is required", (long long)c.bytes);
        return WF_EINVAL;
    }
    const GatedEpilogue e = {bias, bias_dt, act, y, static_cast<uint16_t*>(kept), M * N};
    float* parts = c.slices > 1 ? reinterpret_cast<float*>(ws + c.parts_at) : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (c.few) {
        gated_rows_run(dt, c.slices, static_cast<const uint16_t*>(x), x_row, static_cast<const uint16_t*>(w), w_row, (int)M, (int)N,
                       (int)K, parts, e, s);
    } else {
        DenseOperand a, b;
        if (c.loose) {
            a = {static_cast<const uint16_t*>(x), x_row, (int)K, (int)M, false};
            b = {static_cast<const uint16_t*>(w), w_row, (int)K, (int)N, false};
        } else {
            dense_operands(xv, c.how_x, M, ws, wv, c.how_w, 2 * N, ws + c.w_at, K, a, b, s);
        }
        b.rows = (int)N;
        if (dt == WF_BF16) gated_tiling<WF_BF16>(a, b, N * b.row, (int)M, (int)N, (int)K, c.tiles, c.loose, parts, e, s);
        else gated_tiling<WF_F16>(a, b, N * b.row, (int)M, (int)N, (int)K, c.tiles, c.loose, parts, e, s);
    }
    if (parts) {
        over_grids((M * ((N + 7) / 8) + 255) / 256, kGridMost, [&](int64_t wg, uint32_t n) {
            if (dt == WF_BF16) gated_sum<WF_BF16><<<dim3(n), 256, 0, s>>>(wg, parts, c.slices, (int)M, (int)N, e);
            else gated_sum<WF_F16><<<dim3(n), 256, 0, s>>>(wg, parts, c.slices, (int)M, (int)N, e);
        });
    }
    WF_LAUNCH_CHECK("wf_gated_dense launch");
    return WF_OK;
}

extern "C" int wf_gated_dense_bwd_workspace(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, int dt,
                                            int64_t M, int64_t N, int64_t K, int dx, int dw, int db, int64_t* bytes) {
    using namespace wf;
    if (!bytes) { set_error("wf_gated_dense_bwd_workspace: null pointer"); return WF_EINVAL; }
    if (const int rc = gated_check("wf_gated_dense_bwd_workspace", dt, 0, M, N, K, x_row, 1, w_row, w_col)) return rc;
    *bytes = M && N ? gated_backward(x, x_row, w, w_row, w_col, dt, M, N, K, dx, dw, db, nullptr).bytes : 0;
    return WF_OK;
}

extern "C" int wf_gated_dense_bwd(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, const void* dy,
                                  int64_t dy_row, const void* kept, int dt, int act, int64_t M, int64_t N, int64_t K, void* dx,
                                  void* dw, void* dbias, int bias_dt, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = gated_check("wf_gated_dense_bwd", dt, act, M, N, K, x_row, dy_row, w_row, w_col)) return rc;
    if (dbias && bias_dt != dt && bias_dt != WF_F32) { set_error("wf_gated_dense_bwd: dtype code %d of the bias", bias_dt); return WF_EINVAL; }
    if (M == 0 || N == 0) return WF_OK;                            // (the caller's empty or zero gradients)
    if (!dy || !kept || (dx && !w) || (dw && !x)) { set_error("wf_gated_dense_bwd: null pointer"); return WF_EINVAL; }
    if (!aligned(x, 2) || !aligned(w, 2) || !aligned(dy, 2) || !aligned(kept, 2) || !aligned(dx, 2) || !aligned(dw, 2) ||
        !aligned(dbias, bias_dt == WF_F32 ? 4 : 2)) {
        set_error("wf_gated_dense_bwd: a pointer is not aligned to its values");
        return WF_EINVAL;
    }
    char* ws = static_cast<char*>(workspace);
    const GatedBackward b = gated_backward(x, x_row, w, w_row, w_col, dt, M, N, K, dx, dw, dbias, ws);
    if (b.bytes && (!ws || workspace_bytes < b.bytes || !aligned(ws, 256))) {
        set_error("wf_gated_dense_bwd: a workspace of %lld bytes is required", (long long)b.bytes);
        return WF_EINVAL;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* sums = dbias ? reinterpret_cast<float*>(ws + b.sums_at) : nullptr;
    float* range = b.ranged ? reinterpret_cast<float*>(ws + b.range_at) : nullptr;
    if (dx || dw || dbias) {
        auto go = [&](auto d, auto again) {
            constexpr int D = decltype(d)::value;
            gated_dact<D, decltype(again)::value><<<dim3((uint32_t)((N + 511) / 512), b.rows), 256, 0, s>>>(
                static_cast<const value_t<D>*>(dy), dy_row, static_cast<const uint16_t*>(kept), M * N, act,
                dx || dw ? reinterpret_cast<value_t<D>*>(ws) : nullptr, b.dh_row, sums, range, (int)M, (int)N);
        };
        if (dt == WF_BF16) go(std::integral_constant<int, WF_BF16>{}, std::false_type{});
        else go(std::integral_constant<int, WF_F16>{}, std::false_type{});
        if (b.ranged) go(std::integral_constant<int, WF_F16>{}, std::true_type{});
    }
    if (dbias) {
        const ColumnSums q = {sums, dbias, bias_dt, b.rows};
        column_sums<<<dim3((uint32_t)((2 * N + 63) / 64), 1, 1), 1024, 0, s>>>(q, q, (int)(2 * N));
    }
    DenseEpilogue e = {};
    e.rows_per_group = 1;
    e.alpha = range;
    e.y = dx;
    if (dx) dense_run(b.dx, b.dh_along, b.w_turned, dt, M, K, 2 * N, ws + b.product_at, e, s);
    e.y = dw;
    if (dw) dense_run(b.dw, b.dh_turned, b.x_turned, dt, 2 * N, K, M, ws + b.product_at, e, s);
    WF_LAUNCH_CHECK("wf_gated_dense_bwd launch");
    return WF_OK;
}
