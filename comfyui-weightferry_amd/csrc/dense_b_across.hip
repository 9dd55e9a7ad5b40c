// Tiled kernels of the 16-bit linear, the second operand across K: a linear's dx = dh w.
#include "dense_gemm.h"

namespace wf {

void dense_gemm_b_across(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                         float* parts, const DenseEpilogue& e, hipStream_t s) {
    if (dt == WF_BF16) dense_tiling<WF_BF16, false, true, true>(a, b, M, N, K, p, parts, e, s);
    else dense_tiling<WF_F16, false, true, true>(a, b, M, N, K, p, parts, e, s);
}

}  // namespace wf
