// The products of a Newton-Schulz step on a batch of float16 matrices, for gfx950, in the tiles of the 16-bit linear (dense_ring.h):
//
//   A = X X^T (or X^T X, whichever is the smaller),  B = b A + c A A,  X = a X + B X (or X B)
//
// A and B are symmetric, so only the tiles on and below the diagonal are computed, half the operations, and each is stored twice, as
// it is and turned: a lane's accumulators are four consecutive rows of a column, which turned are four consecutive values of
// a row. X is read as it lies, along or across the sum.
//
// Where a batch's tiles do not fill the chip a symmetric product runs in slices of K: the accumulators go to memory as they are
// in the registers, and a second launch of the same kernel starts from their sum, in slice order.
//
// X is kept with the remainder of its rounding (lo) while small singular values grow, and a X is taken from both: a X is what they live
// from, and an error in the first X is multiplied by a^5 = 485 there. The products see X itself, 11 bits.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "deep_ring.h"
#include "dense_gemm.h"
#include "muon.h"
#include "tile_stage.h"

namespace wf {

__device__ __forceinline__ float f16_at(uint64_t v, int i) { return f16_bits_to_f32((uint32_t)(v >> (16 * i)) & 0xffffu); }

// Workgroup w of W runs on XCD w % 8: which of the W pieces of work, in an order whose neighbours share operands, it takes so that an XCD
// takes neighbours. The pieces are all matrices' tiles, one matrix after the other: an XCD's L2 then sees one matrix of a batch, or few.
__device__ __forceinline__ int muon_spread(int w, int W) {
    return w < (W & ~7) ? (w & 7) * (W >> 3) + (w >> 3) : w;
}
// tile t of an nt x nt lower triangle: bands of `band` rows, a band's columns one after the other
__device__ __forceinline__ void triangle_tile(int t, int nt, int band, int& tm, int& tn) {
    int r0 = 0, rows = min(band, nt);
    for (;; r0 += rows, rows = min(band, nt - r0)) {
        const int here = rows * r0 + rows * (rows + 1) / 2;
        if (t < here) break;
        t -= here;
    }
    if (t < rows * (r0 + 1)) {                                     // columns left of the diagonal, and its first
        tn = t / rows;
        tm = r0 + t % rows;
        return;
    }
    t -= rows * (r0 + 1);
    for (tn = r0 + 1; t >= rows - (tn - r0); tn++) t -= rows - (tn - r0);
    tm = tn + t;
}

// acc over stages s0 .. s0 + nk of a . b in one of the two main loops: four stage buffers for the small tiles, else two
template <typename S, bool AX, bool BX>
struct MuonLoop {
    static constexpr bool DEEP = S::BM * S::BN <= 64 * 64;
    static constexpr int MORE = DEEP ? S::SLOTS : 1;              // of the third and fourth buffer
    static constexpr int WAVES = DEEP ? 2 : S::WAVES;             // a SIMD
    __device__ __forceinline__ static void run(const DenseTile& ta, const DenseTile& tb, int s0, int nk, int wave, int lane, wl_frag* sb0,
                                               wl_frag* sb1, wl_frag* sb2, wl_frag* sb3, f32x16v (&acc)[S::WM][S::WN]) {
        auto mma = [](const f32x16v& c, const wl_frag& x, const wl_frag& y) { return mma16<WF_F16>(c, x, y); };
        if constexpr (DEEP) {
            using LA = std::conditional_t<AX, DenseAcross<S::BM, S::NW, S::AW, S::WM>, DenseAlong<S::BM, S::NW, S::AW, S::WM>>;
            using LB = std::conditional_t<BX, DenseAcross<S::BN, S::NW, S::BW, S::WN>, DenseAlong<S::BN, S::NW, S::BW, S::WN>>;
            wl_frag* const sb[kDeep] = {sb0, sb1, sb2, sb3};
            deep_loop<S, LA, LB>(ta, tb, s0, nk, wave, lane, sb, acc, mma);
        } else {
            dense_mainloop<S, AX, BX>(ta, tb, s0, nk, wave, lane, sb0, sb1, acc, mma);
        }
    }
};

// Workgroup (tile of a matrix, slice). parts: [batch, slices, tiles, accumulators of a workgroup], NULL without slices. SUM: the second
// launch, its slice the only one.
template <bool X, typename S, bool SUM>
__global__ __launch_bounds__(S::NT, (MuonLoop<S, X, X>::WAVES)) void muon_sym(DenseOperand o, int64_t o_step, MuonSymmetric q, int64_t s_step, int side,
                                                            int sld, int stages, int slice_stages, int slices, int T, int band,
                                                            float* __restrict__ parts) {
    constexpr int WM = S::WM, WN = S::WN, LANES = WM * WN * 16 * S::NT;
    static_assert(S::BM == S::BN && WM == WN, "tiles that turn into tiles");
    using Loop = MuonLoop<S, X, X>;
    __shared__ wl_frag sb0[S::SLOTS], sb1[S::SLOTS], sb2[SUM ? 1 : Loop::MORE], sb3[SUM ? 1 : Loop::MORE];
    const int piece = __builtin_amdgcn_readfirstlane(muon_spread(blockIdx.x, gridDim.x)), tile = piece % T;
    const int64_t b = piece / T;
    int tm, tn;
    triangle_tile(tile, (side + S::BM - 1) / S::BM, band, tm, tn);
    const int m0 = __builtin_amdgcn_readfirstlane(tm * S::BM), n0 = __builtin_amdgcn_readfirstlane(tn * S::BN);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x16v acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
        for (int j = 0; j < WN; j++)
#pragma unroll
            for (int x = 0; x < 16; x++) acc[i][j][x] = 0.0f;
    auto at = [&](int s) { return parts + ((b * slices + s) * T + tile) * LANES + threadIdx.x; };
    if constexpr (SUM) {
        for (int s = 0; s < slices; s++) {
            const float* p = at(s);
#pragma unroll
            for (int i = 0; i < WM; i++)
#pragma unroll
                for (int j = 0; j < WN; j++)
#pragma unroll
                    for (int x = 0; x < 16; x++) acc[i][j][x] += p[((i * WN + j) * 16 + x) * S::NT];
        }
    } else {
        o.p += b * o_step;
        const int s0 = blockIdx.y * slice_stages, nk = min(slice_stages, stages - s0);
        const DenseTile ta = dense_tile<X>(o, m0), tb = dense_tile<X>(o, n0);
        Loop::run(ta, tb, s0, nk, wave, lane, sb0, sb1, sb2, sb3, acc);
        if (parts) {
            float* p = at(blockIdx.y);
#pragma unroll
            for (int i = 0; i < WM; i++)
#pragma unroll
                for (int j = 0; j < WN; j++)
#pragma unroll
                    for (int x = 0; x < 16; x++) p[((i * WN + j) * 16 + x) * S::NT] = acc[i][j][x];
            return;
        }
    }
    const int mw = m0 + wave / S::VN * WM * 32, nw = n0 + wave % S::VN * WN * 32;
    const int lr = lane & 31, lk = lane >> 5;
    uint16_t* out = q.out + b * s_step;
    const uint16_t* in = q.in ? q.in + b * s_step : nullptr;
    // the outputs, rounded, in the accumulators' places: four rows' values in 64 bits
    uint64_t v[WM][WN][4];
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
        for (int j = 0; j < WN; j++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int m = mw + 32 * i + 8 * y + 4 * lk, n = nw + 32 * j + lr;
                uint64_t c = 0;                                    // (in is symmetric: its row n holds column n)
                if (in && n < side && m < sld) __builtin_memcpy(&c, in + (int64_t)n * sld + m, 8);
                float r[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    r[x] = q.alpha * acc[i][j][4 * y + x];
                    if (in) r[x] = fmaf(q.beta, f16_at(c, x), r[x]);
                    if (m0 == n0 && m + x == n && n < side) r[x] += q.gamma;
                }
                v[i][j][y] = pack_f16(r[0], r[1]) | (uint64_t)pack_f16(r[2], r[3]) << 32;
            }
    uint16_t* lds = reinterpret_cast<uint16_t*>(TileStage<S>::region(sb0, sb1, wave));
    wl_store_tile<WM, WN>(lds, out, side, sld, mw, nw, lane,
                          [&](int i, int j, int x) { return (uint16_t)(v[i][j][x >> 2] >> (16 * (x & 3))); });
    if (m0 == n0) return;
    // turned: 32 columns at a time are rows of WM 32 values (8 more apart: the lanes' 8-byte writes then share banks by twos)
    constexpr int ROW = WM * 32 + 8, RUNS = WM * 4;
    static_assert(32 * ROW * 2 <= S::SLOTS * 8, "the turned rows fit a wave's region");
#pragma unroll
    for (int j = 0; j < WN; j++) {
#pragma unroll
        for (int i = 0; i < WM; i++)
#pragma unroll
            for (int y = 0; y < 4; y++)
                __builtin_memcpy(__builtin_assume_aligned(lds + lr * ROW + 32 * i + 8 * y + 4 * lk, 8), &v[i][j][y], 8);
#pragma unroll
        for (int it = 0; it < 32 * RUNS / 64; it++) {
            const int p = it * 64 + lane, n = nw + 32 * j + p / RUNS, m = mw + 8 * (p % RUNS);
            Pack<WF_F16> w;
            __builtin_memcpy(w.w, __builtin_assume_aligned(lds + p / RUNS * ROW + 8 * (p % RUNS), 16), 16);
            if (n < side && m < sld) w.store(out + (int64_t)n * sld + m, 8);
        }
    }
}

// Workgroup: a tile of a matrix's outputs [rows, cols]; BX: b lies across K.
template <bool BX, typename S>
__global__ __launch_bounds__(S::NT, (MuonLoop<S, false, BX>::WAVES)) void muon_upd(DenseOperand a, int64_t a_step, DenseOperand bo,
                                                                                   int64_t b_step, MuonUpdate q, int64_t x_step,
                                                                                   int rows, int cols, int ld, int K, MuonTensors t) {
    constexpr int WM = S::WM, WN = S::WN, TC = WN * 32;
    using Loop = MuonLoop<S, false, BX>;
    __shared__ wl_frag sb0[S::SLOTS], sb1[S::SLOTS], sb2[Loop::MORE], sb3[Loop::MORE];
    const int ntm = (rows + S::BM - 1) / S::BM, ntn = (cols + S::BN - 1) / S::BN;
    const int T = ntm * ntn, piece = __builtin_amdgcn_readfirstlane(muon_spread(blockIdx.x, gridDim.x)), b = piece / T, t0 = piece % T;
    const int first = t0 / (8 * ntn) * 8, high = min(ntm - first, 8);      // bands of 8 rows of tiles, column by column
    const int m0 = (first + (t0 - first * ntn) % high) * S::BM, n0 = (t0 - first * ntn) / high * S::BN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    a.p += b * a_step;
    bo.p += b * b_step;
    f32x16v acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
        for (int j = 0; j < WN; j++)
#pragma unroll
            for (int x = 0; x < 16; x++) acc[i][j][x] = 0.0f;
    const DenseTile ta = dense_tile<false>(a, m0), tb = dense_tile<BX>(bo, n0);
    Loop::run(ta, tb, 0, (K + 63) / 64, wave, lane, sb0, sb1, sb2, sb3, acc);
    const int mw = m0 + wave / S::VN * WM * 32, nw = n0 + wave % S::VN * TC;
    using Stage = TileStage<S>;
    float* st = Stage::region(sb0, sb1, wave);
    if (q.next && !q.lo) {
        wl_store_tile<WM, WN>(reinterpret_cast<uint16_t*>(st), q.next + b * x_step, rows, ld, mw, nw, lane,
                              [&](int i, int j, int x) { return from_f32<WF_F16>(q.alpha * acc[i][j][x]); });
        return;
    }
    constexpr int ROWS = Stage::ROWS, RUNS = ROWS * TC / 8 / 64, U = RUNS % 4 == 0 ? 4 : RUNS;
    // The tile's runs of 8 outputs: what load(ahead, m, n) fetches for U of them goes out before the U before are finished by
    // store(v, ahead, m, n), v the sums. width: the columns that are walked.
    auto walk = [&](auto ahead, int width, auto&& load, auto&& store) {
        using Ahead = decltype(ahead);
        static_for<Stage::PHASES>([&](auto pc) {
            constexpr int P = decltype(pc)::value;
            const int mp = mw + P * ROWS;
            if (mp >= rows) return;
            Ahead next[U];
            auto at = [&](int it, int& m, int& n) {
                const int p = it * 64 + lane;
                m = mp + p / (TC / 8);
                n = nw + 8 * (p % (TC / 8));
                return m < rows && n < width;
            };
            auto fetch = [&](int it) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    int m, n;
                    if (at(it + u, m, n)) load(next[u], m, n);
                }
            };
            fetch(0);
            Stage::template put<P>(st, acc, lane);
#pragma unroll 1
            for (int it = 0; it < RUNS; it += U) {
                Ahead now[U];
#pragma unroll
                for (int u = 0; u < U; u++) now[u] = next[u];
                if (it + U < RUNS) fetch(it + U);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    int m, n;
                    if (!at(it + u, m, n)) continue;
                    float v[8];
                    staged_run(v, st + ((it + u) * 64 + lane) * 8);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] *= q.alpha;
                    store(v, now[u], m, n);
                }
            }
        });
    };
    if (q.next) {                                                  // a x from X and its remainder, the new remainder beside
        struct Both { Pack<WF_F16> x, r; };
        walk(
            Both{}, ld,
            [&](Both& f, int m, int n) {
                f.x.load(q.x + b * x_step + (int64_t)m * ld + n, 8);
                f.r.load(q.lo + b * x_step + (int64_t)m * ld + n, 8);
            },
            [&](float (&v)[8], const Both& f, int m, int n) {
                const int64_t to = b * x_step + (int64_t)m * ld + n;
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = fmaf(q.a, fmaf(f.r.get(i), 1.0f / 2048.0f, f.x.get(i)), v[i]);
                Pack<WF_F16> o;
                o.put(v);
                o.store(q.next + to, 8);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = (v[i] - o.get(i)) * 2048.0f;
                o.put(v);
                o.store(q.lo + to, 8);
            });
        return;
    }
    auto step = [&](auto dt) {                                     // the parameter's step
        constexpr int D = decltype(dt)::value, VEC = Pack<D>::VEC;
        struct Old { Pack<D> p[8 / VEC]; };
        value_t<D>* const p = static_cast<value_t<D>*>(t.p[b]);
        walk(
            Old{}, cols,
            [&](Old& f, int m, int n) {
                if (t.keep == 0.0f) return;
#pragma unroll
                for (int h = 0; h < 8 / VEC; h++) {
                    f.p[h].zero();
                    if (h == 0 || cols - n > h * VEC) f.p[h].load(p + (int64_t)m * cols + n + h * VEC, cols - n - h * VEC);
                }
            },
            [&](float (&v)[8], const Old& f, int m, int n) {
#pragma unroll
                for (int h = 0; h < 8 / VEC; h++) {
                    if (h && cols - n <= h * VEC) break;
                    float w[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        w[i] = fmaf(-t.rate, v[h * VEC + i], t.keep != 0.0f ? t.keep * f.p[h].get(i) : 0.0f);
                    Pack<D> o;
                    o.put(w);
                    o.store(p + (int64_t)m * cols + n + h * VEC, cols - n - h * VEC);
                }
            });
    };
    if (t.dt == WF_BF16) step(std::integral_constant<int, WF_BF16>{});
    else if (t.dt == WF_F16) step(std::integral_constant<int, WF_F16>{});
    else step(std::integral_constant<int, WF_F32>{});
}

// ------------------------------------------------------------------------------------------------- host side
// The times that choose a tiling, in us: of a workgroup, of each 64 values of K, and that where per_cu of them share a CU; least-squares
// fits to 268 measured launches of 17 shapes (64 x 128 x 512 to 13824 x 5120), off by 13 % on average for the symmetric product and by 9 %
// for the update.
struct MuonTile {
    int bm, bn, per_cu;
    float fixed, stage, shared;
};
static float muon_time(const MuonTile& q, int64_t wgs, int64_t stages) {
    const int64_t on = (wgs + 255) / 256, full = on / q.per_cu;
    const int rest = (int)(on % q.per_cu);
    auto together = [&](int n) {
        if (n == 0) return 0.0f;
        const float more = q.per_cu > 1 ? (q.shared * q.per_cu - q.stage) * (n - 1) / (q.per_cu - 1) : 0.0f;
        return q.fixed + (float)stages * (q.stage + more);
    };
    return (float)full * together(q.per_cu) + together(rest);
}

constexpr MuonTile kSymmetric[] = {{256, 256, 1, 14.5f, 1.10f, 1.10f}, {128, 128, 2, 4.0f, 0.53f, 0.52f}, {64, 64, 2, 1.75f, 0.20f, 0.25f}};
struct MuonSlices {
    int tiling, tiles, slices, slice_stages;
};
static MuonSlices muon_symmetric_plan(const MuonShape& s, int64_t K) {
    const int64_t stages = (K + 63) / 64;
    MuonSlices best = {};
    float least = 1e30f;
    for (int t = 0; t < 3; t++) {
        const MuonTile& q = kSymmetric[t];
        const int64_t across = (s.side + q.bm - 1) / q.bm, tiles = across * (across + 1) / 2;
        for (int want : {1, 2, 3, 4, 6, 8, 12, 16}) {
            const int64_t per = (stages + want - 1) / want, slices = (stages + per - 1) / per, wgs = tiles * s.batch * slices;
            if (want > 1 && (t == 0 || slices != want || per < 3 || wgs > 1600)) continue;
            float c = muon_time(q, wgs, per);
            // the sum's launch: 64 x 64 tiles 4 to 8 us, 128 x 128 7 to 20; 256 x 256 up to 150, and they never gain
            if (want > 1) c += 2.0f + (t == 2 ? 3.8f : 7.0f) + 0.8e-6f * (float)(tiles * s.batch * slices) * (float)(q.bm * q.bn);
            if (c < least) least = c, best = {t, (int)tiles, (int)slices, (int)per};
        }
    }
    return best;
}
static int muon_symmetric_k(const MuonShape& s, bool square) { return square ? s.sld : s.tall ? s.rows : s.ld; }

void muon_symmetric_form(const MuonShape& s, bool square, int& tiling, int& slices) {
    const MuonSlices p = muon_symmetric_plan(s, muon_symmetric_k(s, square));
    tiling = p.tiling;
    slices = p.slices;
}

int64_t muon_symmetric_bytes(const MuonShape& s, bool square) {
    const MuonSlices p = muon_symmetric_plan(s, muon_symmetric_k(s, square));
    const int64_t bm = kSymmetric[p.tiling].bm;
    return p.slices > 1 ? (int64_t)s.batch * p.slices * p.tiles * bm * bm * 4 : 0;
}

void muon_symmetric(const MuonShape& s, const MuonSymmetric& q, float* parts, hipStream_t st) {
    const int K = muon_symmetric_k(s, q.square);
    const MuonSlices p = muon_symmetric_plan(s, K);
    const bool across = !q.square && s.tall;
    const DenseOperand o = q.square ? DenseOperand{q.x, s.sld, s.sld, s.side, false}
                           : s.tall ? DenseOperand{q.x, s.ld, s.rows, s.cols, true}
                                    : DenseOperand{q.x, s.ld, s.ld, s.rows, false};
    const int64_t s_step = (int64_t)s.side * s.sld, o_step = q.square ? s_step : (int64_t)s.rows * s.ld;
    auto go = [&](auto x, auto shape) {
        constexpr bool X = decltype(x)::value;
        using S = decltype(shape);
        float* w = p.slices > 1 ? parts : nullptr;
        // (bands about as high as an XCD's share of the tiles is wide)
        const int band = std::max(1, std::min(8, (int)std::sqrt((double)p.tiles * s.batch / 8.0)));
        const dim3 grid(p.tiles * s.batch, p.slices), one(p.tiles * s.batch);
        muon_sym<X, S, false><<<grid, S::NT, 0, st>>>(o, o_step, q, s_step, s.side, s.sld, (K + 63) / 64, p.slice_stages, p.slices,
                                                      p.tiles, band, w);
        if (w) muon_sym<X, S, true><<<one, S::NT, 0, st>>>(o, o_step, q, s_step, s.side, s.sld, 0, 0, p.slices, p.tiles, band, w);
    };
    auto by = [&](auto x) {
        if (p.tiling == 0) go(x, DenseShape<2, 2, 4, 4>{});
        else if (p.tiling == 1) go(x, DenseShape<2, 2, 2, 2>{});
        else go(x, DenseShape<2, 2, 1, 1>{});
    };
    if (across) by(std::true_type{});
    else by(std::false_type{});
}

constexpr MuonTile kUpdate[] = {{256, 320, 1, 12.3f, 1.70f, 1.70f}, {256, 192, 1, 13.3f, 1.12f, 1.12f},
                                {128, 128, 2, 5.5f, 0.57f, 0.50f}, {64, 64, 2, 2.7f, 0.20f, 0.19f}};

int muon_update_tiling(const MuonShape& s) {
    int tiling = 0;
    float least = 1e30f;
    for (int i = 0; i < 4; i++) {
        const MuonTile& z = kUpdate[i];
        const int64_t wgs = (int64_t)((s.rows + z.bm - 1) / z.bm) * ((s.cols + z.bn - 1) / z.bn) * s.batch;
        const float c = muon_time(z, wgs, (s.side + 63) / 64);
        if (c < least) least = c, tiling = i;
    }
    return tiling;
}

void muon_update(const MuonShape& s, const MuonUpdate& q, const MuonTensors& t, hipStream_t st) {
    const int tiling = muon_update_tiling(s);
    const int64_t x_step = (int64_t)s.rows * s.ld, q_step = (int64_t)s.side * s.sld;
    const DenseOperand q_along = {q.q, s.sld, s.sld, s.side, false};
    auto go = [&](auto bx, auto shape) {
        constexpr bool BX = decltype(bx)::value;
        using S = decltype(shape);
        const dim3 grid(((s.rows + S::BM - 1) / S::BM) * ((s.cols + S::BN - 1) / S::BN) * s.batch);
        if constexpr (BX) {                                        // q x: x's columns are rows that lie across the sum
            const DenseOperand x = {q.x, s.ld, s.rows, s.cols, true};
            muon_upd<true, S><<<grid, S::NT, 0, st>>>(q_along, q_step, x, x_step, q, x_step, s.rows, s.cols, s.ld, s.side, t);
        } else {
            const DenseOperand x = {q.x, s.ld, s.ld, s.rows, false};
            muon_upd<false, S><<<grid, S::NT, 0, st>>>(x, x_step, q_along, q_step, q, x_step, s.rows, s.cols, s.ld, s.side, t);
        }
    };
    auto by = [&](auto bx) {
        if (tiling == 0) go(bx, DenseShape<4, 2, 2, 5>{});
        else if (tiling == 1) go(bx, DenseShape<2, 2, 4, 3>{});
        else if (tiling == 2) go(bx, DenseShape<2, 2, 2, 2>{});
        else go(bx, DenseShape<2, 2, 1, 1>{});
    };
    if (s.tall) by(std::false_type{});
    else by(std::true_type{});
}

}  // namespace wf
