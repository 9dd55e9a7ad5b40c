// Tiled kernels of the 16-bit linear, both operands across K: a linear's dw = dh^T x.
#include "dense_gemm.h"

namespace wf {

void dense_gemm_across(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                       float* parts, const DenseEpilogue& e, hipStream_t s) {
    if (dt == WF_BF16) dense_tiling<WF_BF16, true, true, true>(a, b, M, N, K, p, parts, e, s);
    else dense_tiling<WF_F16, true, true, true>(a, b, M, N, K, p, parts, e, s);
}

}  // namespace wf
