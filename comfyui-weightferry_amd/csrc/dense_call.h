// How the 16-bit linear's products are planned and run (dense.hip), for the operators that are made of them.
#pragma once

#include "dense_gemm.h"
#include "dense_rows.h"

namespace wf {

// a tiling in the time model of dense.hip: its outputs, workgroups a CU, us of a workgroup and of each 64 values of K
struct DenseTiling {
    int bm, bn, per_cu;
    float fixed, stage, shared;
};

// what an epilogue adds to it: an activation's arithmetic, the kept pre-activations' stores, the residual's loads
enum { EPI_ACT = 1, EPI_KEEP = 2, EPI_MORE = 4 };
// the tiling and slices of K that the model finds fastest, and its time in us; sum_us: of the second launch that slices need, besides
// the time of its bytes
DensePlan dense_plan_tiles(const DenseTiling* tilings, int count, int64_t M, int64_t N, int64_t K, int epilogue, float sum_us,
                           float& us);
// the few-rows form's
float dense_rows_time(int64_t M, int64_t N, int64_t K, bool odd);

struct DenseView {                                    // value (r, k) at r * row + k * col
    const void* p;
    int64_t row, col;
    bool zeros;                                       // along K: rows hold zeros from K up to the next multiple of 8
};

// How an operand gets to the tiles: as it lies along K or across it, or copied into rows that can be loaded, which keeps
// that order (along, across) or turns it (any strides, to rows along K).
enum { LIES_ALONG, LIES_ACROSS, COPY_ALONG, COPY_ACROSS, COPY_TURNED };
// may_cross: whether the operand may lie across K
int dense_how(const DenseView& v, int64_t R, int64_t K, bool may_cross);
int64_t dense_copy_bytes(int how, int64_t R, int64_t K);
// both operands as the tiles load them; copies go to x_out and w_out
void dense_operands(const DenseView& x, int how_x, int64_t M, char* x_out, const DenseView& w, int how_w, int64_t N, char* w_out,
                    int64_t K, DenseOperand& a, DenseOperand& b, hipStream_t s);

// How a product runs: in the few-rows form, or in tiles.
struct DenseCall {
    bool few;
    DenseRowsPlan rows;
    DensePlan tiles;
    int how_x, how_w;
    int epilogue;                                     // 0: at most a bias
    bool summed;                                      // float32 partial sums first: slices, or operands across K with more
    int64_t w_at, parts_at, bytes;                    // than a plain epilogue. Offsets into the workspace, x's copy first
    int slices() const { return few ? rows.slices : tiles.slices; }
};

DenseCall dense_call(const DenseView& x, const DenseView& w, int64_t M, int64_t N, int64_t K, int epilogue);
void dense_run(const DenseCall& d, const DenseView& x, const DenseView& w, int dt, int64_t M, int64_t N, int64_t K, char* ws,
               const DenseEpilogue& e, hipStream_t s);

int dense_check(const char* who, int dt, int64_t M, int64_t N, int64_t K, int64_t x_row, int64_t x_col, int64_t w_row,
                int64_t w_col);

}  // namespace wf
