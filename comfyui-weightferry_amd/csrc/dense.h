// What the 16-bit linear's kernels share: the activations and their slopes, and the epilogue
//   y = resid + gate * act(h),  h = sum + bias
// on runs of 8 consecutive outputs of a row.
#pragma once

#include "values.h"

namespace wf {

// Activations. All but the erf form of GELU are h times a factor that is the logistic of z = h (a + b h^2): GELU's tanh
// form, since (1 + tanh z) / 2 is the logistic of 2 z, has a = 2 sqrt(2 / pi), b = 0.044715 a; SiLU a = 1, b = 0.
enum { ACT_NONE = 0, ACT_GELU = 1, ACT_GELU_TANH = 2, ACT_SILU = 3, ACT_RELU = 4 };

struct Act {
    int kind;
    float a, b;
};
inline Act act_of(int kind) {
    const float c = 1.5957691216057308f;                                   // 2 sqrt(2 / pi)
    return kind == ACT_GELU_TANH ? Act{kind, c, 0.044715f * c} : Act{kind, 1.0f, 0.0f};
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_of(float x) { return __builtin_amdgcn_rcpf(x); }

// 1 / (1 + exp(-z)), one ulp of exp2 and of the reciprocal: far below the 16-bit outputs' rounding
__device__ __forceinline__ float logistic(float z) { return rcp_of(1.0f + exp2_of(z * -1.4426950408889634f)); }

// the normal distribution function by formula 7.1.26 of Abramowitz and Stegun (|error| < 1e-7), on the side where it is
// small, and exp(-h^2 / 2) that it needs on the way
__device__ __forceinline__ float normal_cdf(float h, float& e) {
    const float x = fabsf(h) * 0.7071067811865476f;
    const float t = rcp_of(fmaf(0.3275911f, x, 1.0f));
    e = exp2_of(h * h * -0.7213475204444817f);
    const float q = fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t,
                         0.254829592f) * t * e * 0.5f;
    return h < 0.0f ? q : 1.0f - q;
}

// (h^2 is kept finite, so that b = 0 times it stays 0)
__device__ __forceinline__ float act_z(const Act& f, float h) { return h * fmaf(f.b, fminf(h * h, 1e30f), f.a); }

__device__ __forceinline__ float act_value(const Act& f, float h) {
    if (f.kind == ACT_NONE) return h;
    if (f.kind == ACT_RELU) return h < 0.0f ? 0.0f : h;
    float e;
    return h * (f.kind == ACT_GELU ? normal_cdf(h, e) : logistic(act_z(f, h)));
}

__device__ __forceinline__ float act_slope(const Act& f, float h) {
    if (f.kind == ACT_NONE) return 1.0f;
    if (f.kind == ACT_RELU) return h > 0.0f ? 1.0f : 0.0f;
    if (f.kind == ACT_GELU) {
        float e;
        const float phi = normal_cdf(h, e);
        return fmaf(h * 0.3989422804014327f, e, phi);                      // 1 / sqrt(2 pi)
    }
    const float s = logistic(act_z(f, h));
    const float dz = fmaf(3.0f * f.b, fminf(h * h, 1e30f), f.a);
    return fmaf(h * s * (1.0f - s), dz, s);
}

// the pre-activation as it is kept for the backward pass: float16's infinity would make the slope 0 * infinity where the
// float32 value gives a limit, so it stays finite
template <int D>
__device__ __forceinline__ float keep_finite(float h) {
    if constexpr (D == WF_F16) return h > 65504.0f ? 65504.0f : h < -65504.0f ? -65504.0f : h;
    else return h;
}

struct DenseEpilogue {
    const void *bias, *gate, *resid;       // any may be NULL
    int bias_dt, gate_dt;                  // the outputs' type or float32
    Act act;
    int64_t rows_per_group, ldr;           // row m's gate is row m / rows_per_group of gate; resid's row stride
    void *y, *h;                           // [M, N]; h (may be NULL): the pre-activations
};

// the residual's run at (m, n), its first `cnt` values
template <int D>
__device__ __forceinline__ Pack<D> epilogue_prefetch(const DenseEpilogue& e, int64_t m, int n, int cnt) {
    Pack<D> r;
    r.zero();
    if (e.resid && cnt > 0) r.load(static_cast<const value_t<D>*>(e.resid) + m * e.ldr + n, cnt);
    return r;
}

template <int D>
__device__ __forceinline__ void epilogue_run(const DenseEpilogue& e, float (&v)[8], const Pack<D>& r, int64_t m, int n,
                                             int N, int cnt) {
    float u[8];
    if (e.bias) {
        load_params<8>(u, e.bias, n, cnt, e.bias_dt);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += u[i];
    }
    if (e.h) {
        Pack<D> o;
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = keep_finite<D>(v[i]);
        o.put(u);
        o.store(static_cast<value_t<D>*>(e.h) + m * N + n, cnt);
    }
    if (e.act.kind != ACT_NONE)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_value(e.act, v[i]);
    if (e.gate) {
        load_params<8>(u, e.gate, (int64_t)((uint32_t)m / (uint32_t)e.rows_per_group) * N + n, cnt, e.gate_dt);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= u[i];
    }
    if (e.resid)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += r.get(i);
    Pack<D> o;
    o.put(v);
    o.store(static_cast<value_t<D>*>(e.y) + m * N + n, cnt);
}

}  // namespace wf
