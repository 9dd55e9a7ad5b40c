// The 16-bit linear for gfx950: y = resid + gate * act(x w^T + bias) on bfloat16 or float16, float32 accumulation, one
// rounding at the end; and the products of its backward pass, which are the same product on other operands.
//
// 2 M N K operations: v_mfma_f32_32x32x16 tiles fed through the two-buffer LDS ring of dense_ring.h. Each operand is loaded as
// it lies, along K or across it (a transposed view: the backward products read the weight, x and dh so); only one that is
// neither in 16-byte runs (odd row lengths, other strides) is first copied into rows that are. A product with too few tiles
// to fill the 256 CUs runs as slices of K that write float32 partial sums, and so does one with w across K that has more than
// a plain epilogue; a second kernel adds the sums in slice order and runs the epilogue. At few rows of x the product takes a
// form of its own (dense_rows.hip).
//
// The epilogue works on the float32 sums: bias as their start, activation and gate in the accumulators (16 rows x 1 column a
// lane). The residual comes through the idle stage buffers into that layout, and what is stored goes out through them,
// rounded once, in 16-byte runs. A tile that spans two of the gate's groups, and rows of no whole runs with a gate or a residual,
// go through the stage buffers in float32 and are finished run by run (dense.h).

#include <algorithm>
#include <type_traits>

#include "dense_call.h"
#include "dense_grad.h"
#include "dense_rows.h"
#include "grids.h"

namespace wf {

// the slices' sums in slice order, then the epilogue: one run of 8 outputs a thread, from workgroup `wg` of the whole on
template <int D>
__global__ __launch_bounds__(256) void dense_sum(int64_t wg, const float* __restrict__ parts, int slices, int M, int N,
                                                 DenseEpilogue e) {
    const int runs = (N + 7) / 8;
    const int64_t i = (wg + blockIdx.x) * 256 + threadIdx.x;
    if (i >= (int64_t)M * runs) return;
    const int64_t m = i / runs;
    const int n = (int)(i - m * runs) * 8, cnt = N - n;
    const EpilogueAhead<D> r = epilogue_ahead<D>(e, m, n, N, cnt);
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const float* p = parts + m * N + n;
    const int64_t plane = (int64_t)M * N;
    for (int s = 0; s < slices; s += 4) {                          // four slices' loads in flight, added in order
        float u[4][8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t at = min(s + i, slices - 1) * plane;
            if (cnt >= 8) __builtin_memcpy(u[i], p + at, 32);
            else
#pragma unroll
                for (int x = 0; x < 8; x++) u[i][x] = x < cnt ? p[at + x] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (s + i < slices)
#pragma unroll
                for (int x = 0; x < 8; x++) v[x] += u[i][x];
    }
    epilogue_run<D, true>(e, v, r, m, n, N, cnt);
}

// R rows of K consecutive values (of an operand, or of memory where it lies across K), `row` apart, as [R, KP], KP a multiple
// of 8, zeros past K: a run of 8 values a thread, loaded at any alignment. One launch copies both operands (blockIdx.y),
// from workgroup `wg` of the whole on.
struct PackRows {
    const uint16_t* p;
    uint16_t* out;
    int64_t row, runs;                                             // runs: R KP / 8
    int K, KP;
};
__global__ __launch_bounds__(256) void dense_pack_rows(int64_t wg, PackRows a, PackRows b) {
    const PackRows q = blockIdx.y ? b : a;
    const int across = q.KP / 8;
    const int64_t i = (wg + blockIdx.x) * 256 + threadIdx.x;
    if (i >= q.runs) return;
    const int64_t r = i / across;
    const int k = (int)(i - r * across) * 8;
    Pack<WF_BF16> v;                                               // (16 bits are moved, whatever they stand for)
    v.zero();
    if (k < q.K) v.load(q.p + r * q.row + k, q.K - k);
    v.store(q.out + r * q.KP + k, 8);
}

// an operand of any strides (value (r, k) at r row + k col) as such rows, KP a multiple of 64: 64 x 64 tiles through LDS, read along
// whichever of the two is the shorter step
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
// The modelled time of a product in us, fitted to 2,230 measurements (30 shapes of 20-16384 rows, 64-13824 columns and K
// 256-16384, every tiling, 1-16 slices, operands along and across K): a workgroup takes `fixed` and `stage` for each 64
// values of K on a CU of its own, `shared` where `per_cu` of them share one; a last round that fills part of the chip runs
// faster than a whole one, which the power limit holds back; operands stream at 4.6 TB/s, less with few workgroups; a second
// kernel adds the slices. The way it chooses took 3 % longer than the best measured one on average over the 60 (shape,
// order) pairs, at most 21 % (2048 x 2048 x 256, 8.0 against 6.6 us).
constexpr DenseTiling kDense[] = {{256, 320, 1, 2.2f, 1.65f, 1.65f},    {256, 256, 1, 3.0f, 1.252f, 1.252f},
                                  {256, 192, 1, 1.8f, 1.076f, 1.076f},  {128, 192, 2, 0.8f, 0.785f, 0.694f},
                                  {128, 160, 2, 1.6f, 0.72f, 0.606f},   {128, 128, 2, 1.5f, 0.634f, 0.519f},
                                  {64, 128, 3, 0.8f, 0.47f, 0.367f},    {32, 128, 3, 1.6f, 0.435f, 0.315f}};

// What an epilogue adds to a workgroup's time. Eight waves hide more of it than four, and workgroups that share a CU hide each
// other's: 4096 x 13824 x 5120 with GELU 465 us in 256 x 320 tiles, 486 in 256 x 256, which without it are as fast.
static float dense_epilogue_time(const DenseTiling& q, int epilogue) {
    const float us = (epilogue & EPI_ACT ? 5.0f : 0.0f) + (epilogue & EPI_KEEP ? 10.0f : 0.0f) +
                     (epilogue & EPI_MORE ? 8.0f : 0.0f);
    return us * (float)(q.bm * q.bn) / 65536.0f * (q.bn == 320 ? 0.5f : q.per_cu > 1 ? 0.75f : 1.0f);
}

DensePlan dense_plan_tiles(const DenseTiling* tilings, int count, int64_t M, int64_t N, int64_t K, int epilogue, float sum_us,
                           float& us) {
    const int64_t stages = (K + 63) / 64;
    DensePlan best = {0, 1, (int)stages};
    us = 1e30f;
    const float bytes = (float)(M * K + N * K) * 2.0f;
    for (int t = 0; t < count; t++) {
        const DenseTiling& q = tilings[t];
        const int64_t tiles = ((M + q.bm - 1) / q.bm) * ((N + q.bn - 1) / q.bn);
        for (int want : {1, 2, 3, 4, 6, 8, 12, 16}) {
            const int64_t per = (stages + want - 1) / want, slices = (stages + per - 1) / per;
            if (want > 1 && (slices != want || per < 3 || tiles * slices > 1600)) continue;
            // workgroups of the busiest CU: full rounds of per_cu together, then a rest
            const int64_t wgs = tiles * slices, on = (wgs + 255) / 256, full = on / q.per_cu;
            const int rest = (int)(on % q.per_cu);
            const float after = want == 1 ? dense_epilogue_time(q, epilogue) : 0.0f;
            auto together = [&](int n) {
                if (n == 0) return 0.0f;
                const float more = q.per_cu > 1 ? (q.shared * q.per_cu - q.stage) * (n - 1) / (q.per_cu - 1) : 0.0f;
                return q.fixed + after + (float)per * (q.stage + more);
            };
            float busy = (float)full * together(q.per_cu) + together(rest);
            if (on > q.per_cu && want == 1) busy *= 0.65f + 0.35f * (float)wgs / (256.0f * (float)on);
            const float mem = bytes / 4.6e6f * (1.0f + 0.12f * 256.0f / (float)wgs);
            const float hi = std::max(busy, mem), r = std::min(busy, mem) / hi;
            float c = 4.4f + hi * (1.0f + 0.26f * r * r * r);
            if (want > 1) c += sum_us + 1.5e-6f * (float)(M * N) * (float)(slices + 1);
            if (c < us) us = c, best = {t, (int)slices, (int)per};
        }
    }
    return best;
}

// The few-rows form: weight bytes at 5.2 TB/s, up to 1.6 times that time as 16 rows fill up, more with every 16 rows, and
// nearly twice where odd row lengths put the 16-byte loads at odd places (`odd`).
// 1 x 13824 x 5120 30 us, 16 x 2048 x 8192 12 (the tiles 19), 128 x 1000 x 1024 5.1 (8.0), 12 x 5896 x 9106 36 (75 with the
// copies that the tiles need); 16 x 5120 x 5120 20 (17), 77 x 2607 x 1531 24 (20).
float dense_rows_time(int64_t M, int64_t N, int64_t K, bool odd) {
    const float fill = 1.0f + 0.6f * (float)std::min<int64_t>(M - 1, 15) / 15.0f;
    const int64_t groups = (M + 15) / 16;
    return 4.0f + (float)(N * K) * 2.0f / 5.2e6f * fill * (groups > 1 ? 0.87f * (float)groups : 1.0f) * (odd ? 1.9f : 1.0f);
}
// Two weight tiles a workgroup share x's loads (16 x 5120 x 5120 20 against 25 us) where that leaves 128 workgroups; a
// single or double row of a wide weight has little of x to share (1 x 13824 x 5120 30.5 against 32.3). A long K of a narrow
// weight is split over four workgroups (16 x 2048 x 8192 12 against 17).
static DenseRowsPlan dense_plan_rows(int64_t M, int64_t N, int64_t K) {
    const int64_t pairs = (N + 31) / 32 * ((M + 15) / 16);
    if (pairs >= 128) return {M <= 2 && pairs >= 256 ? 1 : 2, 1};
    return K >= 4096 ? DenseRowsPlan{2, 4} : DenseRowsPlan{1, 1};
}

constexpr int64_t kRowsMost = 256;

static bool is_across(int how) { return how == LIES_ACROSS || how == COPY_ACROSS; }

// may_cross: whether the operand may lie across K
int dense_how(const DenseView& v, int64_t R, int64_t K, bool may_cross) {
    const bool a16 = aligned(v.p, 16);
    if (v.col == 1 && (R == 1 || v.row >= K)) {
        return v.row % 8 == 0 && (K % 8 == 0 || v.zeros) && v.row <= (1 << 20) && a16 ? LIES_ALONG : COPY_ALONG;
    }
    if (!may_cross || v.row != 1) return COPY_TURNED;
    if (v.col % 8 == 0 && v.col >= R && a16 && (K + 128) * v.col * 2 < (1LL << 31)) return LIES_ACROSS;
    return (K + 128) * up(R, 8) * 2 < (1LL << 31) ? COPY_ACROSS : COPY_TURNED;
}
static int64_t dense_copy_row(int how, int64_t R, int64_t K) {
    return how == COPY_ALONG ? up(K, 8) : how == COPY_ACROSS ? up(R, 8) : up(K, 64);
}
int64_t dense_copy_bytes(int how, int64_t R, int64_t K) {
    if (how == LIES_ALONG || how == LIES_ACROSS) return 0;
    return up((how == COPY_ACROSS ? K : R) * dense_copy_row(how, R, K) * 2, 256);
}

DenseCall dense_call(const DenseView& x, const DenseView& w, int64_t M, int64_t N, int64_t K, int epilogue) {
    DenseCall d = {};
    d.epilogue = epilogue;
    float us;
    d.tiles = dense_plan_tiles(kDense, (int)(sizeof(kDense) / sizeof(kDense[0])), M, N, K, epilogue, 1.3f, us);
    d.how_w = dense_how(w, N, K, true);
    d.how_x = dense_how(x, M, K, is_across(d.how_w));
    int64_t copies = dense_copy_bytes(d.how_x, M, K);
    if (copies) us += 3.0f + (float)copies * 0.5e-6f;                             // (read and written at 4 TB/s)
    if (const int64_t c = dense_copy_bytes(d.how_w, N, K)) us += 3.0f + (float)c * 0.5e-6f, copies += c;
    if (M <= kRowsMost && x.col == 1 && w.col == 1 && dense_rows_time(M, N, K, ((x.row | w.row) & 1) != 0) < us) {
        d.few = true;
        d.rows = dense_plan_rows(M, N, K);
        copies = 0;
    } else {
        d.w_at = dense_copy_bytes(d.how_x, M, K);
    }
    d.parts_at = copies;
    d.summed = d.slices() > 1 || (!d.few && epilogue && is_across(d.how_w));
    d.bytes = d.parts_at + (d.summed ? (int64_t)d.slices() * M * N * 4 : 0);
    return d;
}

// the operand as the tiles load it; where it has to be copied, to `out`: rows by the job that is filled in, others at once
static DenseOperand dense_operand(const DenseView& v, int how, int64_t R, int64_t K, uint16_t* out, PackRows& job,
                                  hipStream_t s) {
    const uint16_t* p = static_cast<const uint16_t*>(v.p);
    const int64_t to = dense_copy_row(how, R, K);
    auto pack_rows = [&](int64_t row, int64_t n, int64_t values) {
        job = {p, out, row, n * (to / 8), (int)values, (int)to};
    };
    switch (how) {
    case LIES_ALONG: return {p, v.row, (int)(v.zeros ? up(K, 8) : K), (int)R, false};
    case LIES_ACROSS: return {p, v.col, (int)K, (int)R, true};
    case COPY_ALONG: pack_rows(v.row, R, K); return {out, to, (int)to, (int)R, false};
    case COPY_ACROSS: pack_rows(v.col, K, R); return {out, to, (int)K, (int)R, true};
    }
    for (int64_t r = 0; r < R; r += 65535 * 64) {                                 // (a grid's second dimension ends there)
        const int64_t n = std::min<int64_t>(R - r, 65535 * 64);
        dense_pack<<<dim3((uint32_t)(to / 64), (uint32_t)((n + 63) / 64)), 256, 0, s>>>(p + r * v.row, v.row, v.col, (int)n,
                                                                                       (int)K, (int)to, out + r * to);
    }
    return {out, to, (int)to, (int)R, false};
}

void dense_operands(const DenseView& x, int how_x, int64_t M, char* x_out, const DenseView& w, int how_w, int64_t N, char* w_out,
                    int64_t K, DenseOperand& a, DenseOperand& b, hipStream_t s) {
    PackRows jx = {}, jw = {};
    a = dense_operand(x, how_x, M, K, reinterpret_cast<uint16_t*>(x_out), jx, s);
    b = dense_operand(w, how_w, N, K, reinterpret_cast<uint16_t*>(w_out), jw, s);
    over_grids((std::max(jx.runs, jw.runs) + 255) / 256, kGridMost, [&](int64_t wg, uint32_t n) {
        dense_pack_rows<<<dim3(n, jx.runs && jw.runs ? 2 : 1), 256, 0, s>>>(wg, jx.runs ? jx : jw, jw);
    });
}

// the tiled kernel of a call (dense_gemm.h has one source each), as wf_dense_plan numbers them; 0 is the few-rows form
enum { FORM_ROWS, FORM_ALONG, FORM_ALONG_FULL, FORM_B_ACROSS, FORM_ACROSS };
static int dense_form(const DenseCall& d) {
    if (d.few) return FORM_ROWS;
    if (is_across(d.how_x)) return FORM_ACROSS;
    if (is_across(d.how_w)) return FORM_B_ACROSS;
    return d.epilogue && !d.summed ? FORM_ALONG_FULL : FORM_ALONG;
}

void dense_run(const DenseCall& d, const DenseView& x, const DenseView& w, int dt, int64_t M, int64_t N, int64_t K,
                      char* ws, const DenseEpilogue& e, hipStream_t s) {
    float* parts = d.summed ? reinterpret_cast<float*>(ws + d.parts_at) : nullptr;
    if (d.few) {
        dense_rows_run(dt, d.rows, static_cast<const uint16_t*>(x.p), x.row, static_cast<const uint16_t*>(w.p), w.row, (int)M,
                       (int)N, (int)K, parts, e, s);
    } else {
        DenseOperand a, b;
        dense_operands(x, d.how_x, M, ws, w, d.how_w, N, ws + d.w_at, K, a, b, s);
        const int form = dense_form(d);
        auto run = form == FORM_ACROSS ? dense_gemm_across : form == FORM_B_ACROSS ? dense_gemm_b_across
                   : form == FORM_ALONG ? dense_gemm_along : dense_gemm_along_full;
        run(dt, a, b, (int)M, (int)N, (int)K, d.tiles, parts, e, s);
    }
    if (d.summed) {
        over_grids((M * ((N + 7) / 8) + 255) / 256, kGridMost, [&](int64_t wg, uint32_t n) {
            if (dt == WF_BF16) dense_sum<WF_BF16><<<dim3(n), 256, 0, s>>>(wg, parts, d.slices(), (int)M, (int)N, e);
            else dense_sum<WF_F16><<<dim3(n), 256, 0, s>>>(wg, parts, d.slices(), (int)M, (int)N, e);
        });
    }
}

// The backward pass: its two products, and where its parts lie in the workspace (dh, the column sums, then the products',
// one after the other in the same place).
struct DenseBackward {
    bool changed;                                     // dh is not dy
    int64_t dh_row, sums_at, product_at, bytes;
    DenseView dh_along, w_turned, dh_turned, x_turned;
    DenseCall dx, dw;
};
static DenseBackward dense_backward(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, const void* dy,
                                    int64_t dy_row, int act, bool gate, int64_t rows_per_group, int64_t M, int64_t N,
                                    int64_t K, bool dx, bool dw, bool sums, char* ws) {
    DenseBackward b = {};
    b.changed = (act != ACT_NONE || gate) && (dx || dw);
    b.dh_row = b.changed ? up(N, 8) : dy_row;
    b.sums_at = b.changed ? up(M * b.dh_row * 2, 256) : 0;
    b.product_at = b.sums_at + (sums ? up(dense_grad_bytes(M, N, rows_per_group), 256) : 0);
    const void* dh = b.changed ? ws : dy;             // (a workspace not yet there is as aligned as it will be)
    b.dh_along = {dh, b.dh_row, 1, b.changed};
    b.w_turned = {w, w_col, w_row, false};
    b.dh_turned = {dh, 1, b.dh_row, false};
    b.x_turned = {x, 1, x_row, false};
    if (dx) b.dx = dense_call(b.dh_along, b.w_turned, M, K, N, 0);
    if (dw) b.dw = dense_call(b.dh_turned, b.x_turned, N, K, M, 0);
    b.bytes = b.product_at + std::max(b.dx.bytes, b.dw.bytes);
    return b;
}

int dense_check(const char* who, int dt, int64_t M, int64_t N, int64_t K, int64_t x_row, int64_t x_col,
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
                                  int dt, int64_t M, int64_t N, int64_t K, int epilogue, int64_t* bytes) {
    using namespace wf;
    if (!bytes || epilogue < 0 || epilogue > 7) { set_error("wf_dense_workspace: null pointer or epilogue %d", epilogue); return WF_EINVAL; }
    if (const int rc = dense_check("wf_dense_workspace", dt, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    *bytes = M && N ? dense_call({x, x_row, x_col, false}, {w, w_row, w_col, false}, M, N, K, epilogue).bytes : 0;
    return WF_OK;
}

extern "C" int wf_dense_plan(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt,
                             int64_t M, int64_t N, int64_t K, int epilogue, int* plan) {
    using namespace wf;
    if (!plan || epilogue < 0 || epilogue > 7) { set_error("wf_dense_plan: null pointer or epilogue %d", epilogue); return WF_EINVAL; }
    if (const int rc = dense_check("wf_dense_plan", dt, M, N, K, x_row, x_col, w_row, w_col)) return rc;
    if (M == 0 || N == 0) { set_error("wf_dense_plan: no outputs"); return WF_EINVAL; }
    const DenseCall d = dense_call({x, x_row, x_col, false}, {w, w_row, w_col, false}, M, N, K, epilogue);
    plan[0] = dense_form(d);
    plan[1] = d.few ? d.rows.tiles : d.tiles.tiling;
    plan[2] = d.slices();
    plan[3] = d.few ? LIES_ALONG : d.how_x;
    plan[4] = d.few ? LIES_ALONG : d.how_w;
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
    const DenseView xv = {x, x_row, x_col, false}, wv = {w, w_row, w_col, false};
    const int epilogue = (act != ACT_NONE ? EPI_ACT : 0) | (h ? EPI_KEEP : 0) | (gate || resid ? EPI_MORE : 0);
    const DenseCall d = dense_call(xv, wv, M, N, K, epilogue);
    if (d.bytes && (!workspace || workspace_bytes < d.bytes || !aligned(workspace, 256))) {
        set_error("wf_dense: a workspace of %lld bytes is required", (long long)d.bytes);
        return WF_EINVAL;
    }
    // (the kernels divide in 32 bits: a group of more than M rows is one of M)
    const DenseEpilogue e = {bias, gate, resid, bias_dt, gate_dt, act, gate ? std::min(rows_per_group, M) : 1, resid_row, y, h};
    dense_run(d, xv, wv, dt, M, N, K, static_cast<char*>(workspace), e, static_cast<hipStream_t>(stream));
    WF_LAUNCH_CHECK("wf_dense launch");
    return WF_OK;
}

static int dense_bwd_check(const char* who, int dt, int64_t M, int64_t N, int64_t K, int64_t x_row, int64_t w_row,
                           int64_t w_col, int64_t dy_row, int act, int64_t rows_per_group) {
    using namespace wf;
    if (const int rc = dense_check(who, dt, M, N, K, x_row, dy_row, w_row, w_col)) return rc;
    if (rows_per_group <= 0 || M % rows_per_group || act < ACT_NONE || act > ACT_RELU) {
        set_error("%s: M, rows_per_group = %lld, %lld, activation %d", who, (long long)M, (long long)rows_per_group, act);
        return WF_EINVAL;
    }
    if (M / rows_per_group > 65535 || M > (1 << 20) || N > (1 << 20)) {
        set_error("%s: more than 65535 groups, or M or N above 2^20", who);
        return WF_EUNSUPPORTED;
    }
    return WF_OK;
}

extern "C" int wf_dense_bwd_workspace(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col,
                                      const void* dy, int64_t dy_row, int dt, int act, int gated, int64_t rows_per_group,
                                      int64_t M, int64_t N, int64_t K, int dx, int dw, int sums, int64_t* bytes) {
    using namespace wf;
    if (!bytes) { set_error("wf_dense_bwd_workspace: null pointer"); return WF_EINVAL; }
    if (const int rc = dense_bwd_check("wf_dense_bwd_workspace", dt, M, N, K, x_row, w_row, w_col, dy_row, act,
                                       rows_per_group))
        return rc;
    *bytes = M && N ? dense_backward(x, x_row, w, w_row, w_col, dy, dy_row, act, gated, rows_per_group, M, N, K, dx, dw, sums,
                                     nullptr).bytes
                    : 0;
    return WF_OK;
}

extern "C" int wf_dense_bwd(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, const void* dy,
                            int64_t dy_row, const void* h, int dt, int act, const void* gate, int gate_dt,
                            int64_t rows_per_group, int64_t M, int64_t N, int64_t K, void* dx, void* dw, void* dbias,
                            int bias_dt, void* dgate, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (const int rc = dense_bwd_check("wf_dense_bwd", dt, M, N, K, x_row, w_row, w_col, dy_row, act, rows_per_group))
        return rc;
    if ((gate && gate_dt != dt && gate_dt != WF_F32) || (dbias && bias_dt != dt && bias_dt != WF_F32)) {
        set_error("wf_dense_bwd: dtype codes %d, %d", gate_dt, bias_dt);
        return WF_EINVAL;
    }
    if (M == 0 || N == 0) return WF_OK;
    if (!dy || (dx && !w) || (dw && !x) || ((act != ACT_NONE || dgate) && !h) || (dgate && !gate)) {
        set_error("wf_dense_bwd: null pointer");
        return WF_EINVAL;
    }
    if (!aligned(x, 2) || !aligned(w, 2) || !aligned(dy, 2) || !aligned(h, 2) || !aligned(dx, 2) || !aligned(dw, 2) ||
        !aligned(gate, gate_dt == WF_F32 ? 4 : 2) || !aligned(dgate, gate_dt == WF_F32 ? 4 : 2) ||
        !aligned(dbias, bias_dt == WF_F32 ? 4 : 2)) {
        set_error("wf_dense_bwd: a pointer is not aligned to its values");
        return WF_EINVAL;
    }
    char* ws = static_cast<char*>(workspace);
    const bool sums = dbias || dgate;
    const DenseBackward b = dense_backward(x, x_row, w, w_row, w_col, dy, dy_row, act, gate, rows_per_group, M, N, K, dx, dw,
                                           sums, ws);
    if (b.bytes && (!ws || workspace_bytes < b.bytes || !aligned(ws, 256))) {
        set_error("wf_dense_bwd: a workspace of %lld bytes is required", (long long)b.bytes);
        return WF_EINVAL;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (b.changed || sums) {
        const DenseGrad q = {dy, h, gate, dy_row, act, gate_dt, rows_per_group, b.changed ? ws : nullptr, b.dh_row,
                             dbias, bias_dt, dgate};
        dense_grad_run(q, dt, M, N, reinterpret_cast<float*>(ws + b.sums_at), s);
    }
    DenseEpilogue e = {};
    e.rows_per_group = 1;
    e.y = dx;
    if (dx) dense_run(b.dx, b.dh_along, b.w_turned, dt, M, K, N, ws + b.product_at, e, s);
    e.y = dw;
    if (dw) dense_run(b.dw, b.dh_turned, b.x_turned, dt, N, K, M, ws + b.product_at, e, s);
    WF_LAUNCH_CHECK("wf_dense_bwd launch");
    return WF_OK;
}
