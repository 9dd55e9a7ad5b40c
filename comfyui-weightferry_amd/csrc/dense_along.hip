// Tiled kernels of the 16-bit linear, both operands along K, a plain epilogue.
#include "dense_gemm.h"

namespace wf {

void dense_gemm_along(int dt, const DenseOperand& a, const DenseOperand& b, int M, int N, int K, const DensePlan& p,
                      float* parts, const DenseEpilogue& e, hipStream_t s) {
    if (dt == WF_BF16) dense_tiling<WF_BF16, false, false, true>(a, b, M, N, K, p, parts, e, s);
    else dense_tiling<WF_F16, false, false, true>(a, b, M, N, K, p, parts, e, s);
}

}  // namespace wf
