// Second step of the sums over rows (parameter gradients): out[g, k] = sum of group g's n rows of partial sums, in a
// fixed order. 64 columns a workgroup, its 16 waves walk the rows, then meet in LDS.
#pragma once

#include "values.h"

namespace wf {

struct ColumnSums {
    const float* parts;      // [groups * n, K]
    void* out;               // [groups, K] of type dt
    int dt, n;
};

// workgroup: 64 columns (blockIdx.x) of group blockIdx.y
__device__ __forceinline__ void column_sum(const ColumnSums& q, int K, float (&red)[16][64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane;
    const int64_t g = blockIdx.y;
    float s = 0.0f;
    if (col < K)
#pragma unroll 8                                              // (the loads go out together; the order of the sum stays)
        for (int i = wave; i < q.n; i += 16) s += q.parts[(g * q.n + i) * K + col];
    red[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < K) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) s += red[i][lane];
        store_value(q.out, g * K + col, q.dt, s);
    }
}

// blockIdx.z: which of two arrays of partial sums (both with the same groups)
static __global__ __launch_bounds__(1024) void column_sums(ColumnSums a, ColumnSums b, int K) {
    __shared__ float red[16][64];
    column_sum(blockIdx.z ? b : a, K, red);
}

// the same for up to four arrays, each with groups of its own
struct ColumnSums4 {
    ColumnSums q[4];
    int groups[4];
};
static __global__ __launch_bounds__(1024) void column_sums4(ColumnSums4 a, int K) {
    __shared__ float red[16][64];
    if ((int)blockIdx.y < a.groups[blockIdx.z]) column_sum(a.q[blockIdx.z], K, red);
}

}  // namespace wf
