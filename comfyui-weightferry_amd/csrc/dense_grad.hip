// The element-wise part of the 16-bit linear's backward pass for gfx950. With y = resid + gate * a, a = act(h), h = x w^T +
// bias (dense.hip), and the gradient dy of y:
//   dh = dy gate act'(h),  dbias = sum over all rows of dh,  dgate = sum over a group's rows of dy a
// (dx = dh w and dw = dh^T x are products of dense.hip). One pass over dy and h that writes dh: bound by memory. A lane keeps the
// sums of its 8 columns in registers over the rows its workgroup walks; column_sums.h adds the workgroups' rows in a fixed
// order.
//
// Two values have fewer bits than the sums they come from. dh is rounded to the operands' type because it is the next products'
// operand, and their matrix instructions take 16 bits (rows padded with zeros to 16-byte runs). h was rounded so when the
// forward pass kept it: float32 would double the 113 MB (4096 x 13824) that are written there and read here. In bfloat16 dx and
// dw are off by 2.4e-3 of their norm, against 1.7e-3 for exact sums rounded once; dbias and dgate are summed in float32, from dh
// before it is rounded and from act(h).

#include <algorithm>
#include <type_traits>

#include "column_sums.h"
#include "dense_grad.h"

namespace wf {

// workgroup (512 columns, i, g) walks rows 4 i + wave, + 4 gridDim.y, ... of group g
template <int D>
__global__ __launch_bounds__(256) void dense_dact(const value_t<D>* __restrict__ dy, int64_t ldd,
                                                  const value_t<D>* __restrict__ h, int act, const void* gate, int gate_dt,
                                                  int64_t rows_per_group, value_t<D>* __restrict__ dh, int64_t ldh,
                                                  float* __restrict__ bparts, float* __restrict__ gparts, int N) {
    __shared__ float red[4][2][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = blockIdx.x * 512 + lane * 8, cnt = N - n;
    const int64_t g = blockIdx.z;
    float sb[8], sg[8], gv[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sb[i] = sg[i] = 0.0f, gv[i] = 1.0f;
    if (gate && cnt > 0) load_params<8>(gv, gate, g * N + n, cnt, gate_dt);
    for (int64_t r = blockIdx.y * 4 + wave; r < rows_per_group && cnt > 0; r += gridDim.y * 4) {
        const int64_t m = g * rows_per_group + r;
        Pack<D> pd, ph;
        pd.load(dy + m * ldd + n, cnt);
        ph.zero();
        if (h) ph.load(h + m * N + n, cnt);
        float v[8], x[8], a[8], slope[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = ph.get(i);
        act_slope_run(act, x, a, slope);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float d = pd.get(i);
            v[i] = d * gv[i] * slope[i];
            sb[i] += v[i];
            sg[i] += d * a[i];
        }
        if (dh) {
            Pack<D> o;
            o.put(v);
            o.store(dh + m * ldh + n, 8);                          // (ldh is a multiple of 8: the row's padding, zeros)
        }
    }
    if (!bparts && !gparts) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        red[wave][0][lane * 8 + i] = sb[i];
        red[wave][1][lane * 8 + i] = sg[i];
    }
    __syncthreads();
    const int64_t row = g * gridDim.y + blockIdx.y;
    for (int c = threadIdx.x; c < 512; c += 256) {
        const int col = blockIdx.x * 512 + c;
        if (col >= N) continue;
        if (bparts) bparts[row * N + col] = red[0][0][c] + red[1][0][c] + red[2][0][c] + red[3][0][c];
        if (gparts) gparts[row * N + col] = red[0][1][c] + red[1][1][c] + red[2][1][c] + red[3][1][c];
    }
}

// workgroups over a group's rows: about 2048 in all, no fewer than 4 rows each
static int dact_parts(int64_t M, int64_t N, int64_t rows_per_group) {
    const int64_t across = (N + 511) / 512 * (M / rows_per_group);
    return (int)std::min<int64_t>((rows_per_group + 3) / 4, std::max<int64_t>(1, 2048 / across));
}

int64_t dense_grad_bytes(int64_t M, int64_t N, int64_t rows_per_group) {
    return 2 * (M / rows_per_group) * dact_parts(M, N, rows_per_group) * N * 4;
}

void dense_grad_run(const DenseGrad& q, int dt, int64_t M, int64_t N, float* parts, hipStream_t s) {
    const int64_t groups = M / q.rows_per_group;
    const int n = dact_parts(M, N, q.rows_per_group);
    float *bparts = q.dbias ? parts : nullptr, *gparts = q.dgate ? parts + groups * n * N : nullptr;
    const dim3 grid((uint32_t)((N + 511) / 512), n, (uint32_t)groups);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        dense_dact<D><<<grid, 256, 0, s>>>(static_cast<const value_t<D>*>(q.dy), q.dy_row, static_cast<const value_t<D>*>(q.h),
                                           q.act, q.gate, q.gate_dt, q.rows_per_group, static_cast<value_t<D>*>(q.dh),
                                           q.dh_row, bparts, gparts, (int)N);
    };
    if (dt == WF_BF16) go(std::integral_constant<int, WF_BF16>{});
    else go(std::integral_constant<int, WF_F16>{});
    const uint32_t cols = (uint32_t)((N + 63) / 64);
    if (q.dbias) {
        const ColumnSums b = {bparts, q.dbias, q.bias_dt, (int)(groups * n)};      // every group's rows: one sum
        column_sums<<<dim3(cols, 1, 1), 1024, 0, s>>>(b, b, (int)N);
    }
    if (q.dgate) {
        const ColumnSums b = {gparts, q.dgate, q.gate_dt, n};
        column_sums<<<dim3(cols, (uint32_t)groups, 1), 1024, 0, s>>>(b, b, (int)N);
    }
}

}  // namespace wf
