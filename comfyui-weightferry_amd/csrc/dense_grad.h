// The element-wise part of the 16-bit linear's backward pass (dense_grad.hip).
#pragma once

#include "dense.h"

namespace wf {

struct DenseGrad {
    const void *dy, *h, *gate;             // h may be NULL without an activation and dgate; gate may be
    int64_t dy_row;
    int act, gate_dt;
    int64_t rows_per_group;
    void* dh;                              // may be NULL; rows dh_row (a multiple of 8) values apart, zeros past N
    int64_t dh_row;
    void* dbias;                           // may be NULL, as dgate may
    int bias_dt;
    void* dgate;
};

// bytes of the partial sums, and the launches
int64_t dense_grad_bytes(int64_t M, int64_t N, int64_t rows_per_group);
void dense_grad_run(const DenseGrad& q, int dt, int64_t M, int64_t N, float* parts, hipStream_t s);

}  // namespace wf
