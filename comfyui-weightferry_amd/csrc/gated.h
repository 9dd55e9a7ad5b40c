// The epilogue of the gated linear, y = act(g) u, g and u the two halves of x w^T + bias, on runs of 8 consecutive outputs of a
// row, and how g and u are kept for the backward pass.
//
// They are kept in 24 bits, float32 without its last 8, in three planes of 16: the upper 16 bits of g, those of u, and both
// lower 8. The gradients of both are products of both (dg = dy u act'(g), du = dy act(g)), so 16 bits each would put three more
// roundings of bfloat16 into dx and dw beside the two that the matrix instructions and the outputs need: 3e-3 of their norm instead of
// 2.3e-3, at 4 bytes a pair against 6.
#pragma once

#include "dense.h"

namespace wf {

struct GatedEpilogue {
    const void* bias;                      // [2 N] or NULL, of the outputs' type or float32
    int bias_dt, act;
    void* y;                               // [M, N]
    uint16_t* kept;                        // three planes of [M, N], or NULL
    int64_t plane;                         // M N
};

// float32 rounded to 24 bits, which are the upper ones; NaN stays NaN
__device__ __forceinline__ uint32_t kept_bits(float v) { return v != v ? 0x7fc00000u : __float_as_uint(v) + 0x80u; }
// two places' upper halves, and their lower 8 bits of g and u, as 32 bits each
__device__ __forceinline__ uint32_t kept_uppers(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }
__device__ __forceinline__ uint32_t kept_lowers(uint32_t g0, uint32_t u0, uint32_t g1, uint32_t u1) {
    const uint32_t lo = __builtin_amdgcn_perm(u0, g0, 0x0c0c0501), hi = __builtin_amdgcn_perm(u1, g1, 0x05010c0c);
    return lo | hi;
}
// back to float32, and finite (keep_finite's reason)
__device__ __forceinline__ float kept_g(uint32_t upper, uint32_t lower) {
    return keep_finite<WF_BF16>(__uint_as_float(upper << 16 | (lower & 0xffu) << 8));
}
__device__ __forceinline__ float kept_u(uint32_t upper, uint32_t lower) {
    return keep_finite<WF_BF16>(__uint_as_float(upper << 16 | (lower & 0xff00u)));
}

// the first cnt of 8 values
__device__ __forceinline__ void store_run(float* o, const float (&v)[8], int cnt) {
    if (cnt >= 8) __builtin_memcpy(o, v, 32);
    else
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < cnt) o[k] = v[k];
}

// g, u: a run's sums, without the bias when BIAS is set
template <int D, bool BIAS>
__device__ __forceinline__ void gated_run(const GatedEpilogue& e, float (&g)[8], float (&u)[8], int64_t m, int n, int N, int cnt) {
    if (BIAS && e.bias) {
        float b[8];
        load_params<8>(b, e.bias, n, cnt, e.bias_dt);
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] += b[i];
        load_params<8>(b, e.bias, (int64_t)N + n, cnt, e.bias_dt);
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] += b[i];
    }
    const int64_t at = m * N + n;
    if (e.kept) {
        uint32_t bg[8], bu[8];
#pragma unroll
        for (int i = 0; i < 8; i++) bg[i] = kept_bits(g[i]), bu[i] = kept_bits(u[i]);
        Pack<WF_BF16> pg, pu, pl;                                  // (16 bits are moved, whatever they stand for)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            pg.w[i] = kept_uppers(bg[2 * i], bg[2 * i + 1]);
            pu.w[i] = kept_uppers(bu[2 * i], bu[2 * i + 1]);
            pl.w[i] = kept_lowers(bg[2 * i], bu[2 * i], bg[2 * i + 1], bu[2 * i + 1]);
        }
        pg.store(e.kept + at, cnt);
        pu.store(e.kept + e.plane + at, cnt);
        pl.store(e.kept + 2 * e.plane + at, cnt);
    }
    act_run(e.act, g);
#pragma unroll
    for (int i = 0; i < 8; i++) g[i] *= u[i];
    Pack<D> o;
    o.put(g);
    o.store(static_cast<value_t<D>*>(e.y) + at, cnt);
}

}  // namespace wf
