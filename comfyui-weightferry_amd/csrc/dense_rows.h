// How the few-rows form of the 16-bit linear runs a product (dense_rows.hip).
#pragma once

#include "dense.h"
#include "gated.h"

namespace wf {

struct DenseRowsPlan {
    int tiles, slices;          // 16-row tiles of the weight a workgroup (1 or 2), slices of K over workgroups
};

void dense_rows_run(int dt, const DenseRowsPlan& p, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int M,
                    int N, int K, float* parts, const DenseEpilogue& e, hipStream_t s);

// the gated linear's (w: [2 N, K]); parts: [slices, M, 2 N], or NULL
void gated_rows_run(int dt, int slices, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int M, int N, int K,
                    float* parts, const GatedEpilogue& e, hipStream_t s);

}  // namespace wf
