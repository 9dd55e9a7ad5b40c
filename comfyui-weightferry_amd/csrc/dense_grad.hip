// The element-wise part of the 16-bit linear's backward pass for gfx950. With y = resid + gate * a, a = act(h), h = x w^T +
// bias (dense.hip), and the gradient dy of y:
//   dh = dy gate act'(h),  dbias = sum over all rows of dh,  dgate = sum over a group's rows of dy a
// (dx = dh w and dw = dh^T x are products of dense.hip). One pass over dy and h that writes dh, rounded to the operands'
// type because it is the next products' operand: bound by memory. A lane keeps the sums of its 8 columns in registers
// over the rows its workgroup walks; column_sums.h adds the workgroups' rows in a fixed order.

#include <algorithm>
#include <type_traits>

#include "column_sums.h"
#include "dense.h"

namespace wf {

// workgroup (512 columns, i, g) walks rows 4 i + wave, + 4 gridDim.y, ... of group g
template <int D>
__global__ __launch_bounds__(256) void dense_dact(const value_t<D>* __restrict__ dy, int64_t ldd,
                                                  const value_t<D>* __restrict__ h, int act, const void* gate, int gate_dt,
                                                  int64_t rows_per_group, value_t<D>* __restrict__ dh,
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
            o.store(dh + m * N + n, cnt);
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
static int dact_parts(int64_t N, int64_t groups, int64_t rows_per_group) {
    const int64_t across = (N + 511) / 512 * groups;
    return (int)std::min<int64_t>((rows_per_group + 3) / 4, std::max<int64_t>(1, 2048 / across));
}

}  // namespace wf

extern "C" int wf_dense_grad_workspace(int64_t M, int64_t N, int64_t rows_per_group, int64_t* bytes) {
    using namespace wf;
    if (!bytes || M < 0 || N < 0 || rows_per_group <= 0 || M % rows_per_group) {
        set_error("wf_dense_grad_workspace: bad arguments");
        return WF_EINVAL;
    }
    const int64_t groups = M / rows_per_group;
    *bytes = M && N ? 2 * groups * dact_parts(N, groups, rows_per_group) * N * 4 : 0;
    return WF_OK;
}

extern "C" int wf_dense_grad(const void* dy, int64_t dy_row, const void* h, int dt, int act, const void* gate, int gate_dt,
                             int64_t rows_per_group, void* dh, void* dbias, int bias_dt, void* dgate, int64_t M, int64_t N,
                             void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace wf;
    if (M < 0 || N < 0 || dy_row < 0 || rows_per_group <= 0 || M % rows_per_group || act < ACT_NONE || act > ACT_RELU) {
        set_error("wf_dense_grad: M, N, rows_per_group = %lld, %lld, %lld, activation %d", (long long)M, (long long)N,
                  (long long)rows_per_group, act);
        return WF_EINVAL;
    }
    if ((dt != WF_BF16 && dt != WF_F16) || (gate && gate_dt != dt && gate_dt != WF_F32) ||
        (dbias && bias_dt != dt && bias_dt != WF_F32)) {
        set_error("wf_dense_grad: dtype codes %d, %d, %d", dt, gate_dt, bias_dt);
        return WF_EUNSUPPORTED;
    }
    const int64_t groups = M / rows_per_group;
    if (groups > 65535 || M > (1 << 24) || N > (1 << 24)) {
        set_error("wf_dense_grad: more than 65535 groups, or M or N above 2^24");
        return WF_EUNSUPPORTED;
    }
    if (M == 0 || N == 0) return WF_OK;
    if (!dy || ((act != ACT_NONE || dgate) && !h) || (dgate && !gate)) {
        set_error("wf_dense_grad: null pointer");
        return WF_EINVAL;
    }
    const int n = dact_parts(N, groups, rows_per_group);
    const int64_t plane = groups * n * N;
    float* parts = static_cast<float*>(workspace);
    if ((dbias || dgate) && (!workspace || workspace_bytes < 2 * plane * 4 || !aligned(workspace, 4))) {
        set_error("wf_dense_grad: a workspace of %lld bytes is required", (long long)(2 * plane * 4));
        return WF_EINVAL;
    }
    float *bparts = dbias ? parts : nullptr, *gparts = dgate ? parts + plane : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)((N + 511) / 512), n, (uint32_t)groups);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        dense_dact<D><<<grid, 256, 0, s>>>(static_cast<const value_t<D>*>(dy), dy_row, static_cast<const value_t<D>*>(h),
                                           act, gate, gate_dt, rows_per_group, static_cast<value_t<D>*>(dh), bparts,
                                           gparts, (int)N);
    };
    if (dt == WF_BF16) go(std::integral_constant<int, WF_BF16>{});
    else go(std::integral_constant<int, WF_F16>{});
    WF_LAUNCH_CHECK("wf_dense_grad launch");
    const uint32_t cols = (uint32_t)((N + 63) / 64);
    if (dbias) {
        const ColumnSums q = {bparts, dbias, bias_dt, (int)(groups * n)};          // every group's rows: one sum
        column_sums<<<dim3(cols, 1, 1), 1024, 0, s>>>(q, q, (int)N);
    }
    if (dgate) {
        const ColumnSums q = {gparts, dgate, gate_dt, n};
        column_sums<<<dim3(cols, (uint32_t)groups, 1), 1024, 0, s>>>(q, q, (int)N);
    }
    WF_LAUNCH_CHECK("wf_dense_grad sums launch");
    return WF_OK;
}
