// What the 16-bit linear's kernels share: the activations and their slopes, and the epilogue
//   y = resid + gate * act(h),  h = sum + bias
// on runs of 8 consecutive outputs of a row.
#pragma once

#include <type_traits>

#include "values.h"

namespace wf {

enum { ACT_NONE = 0, ACT_GELU = 1, ACT_GELU_TANH = 2, ACT_SILU = 3, ACT_RELU = 4 };

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_of(float x) { return __builtin_amdgcn_rcpf(x); }

// The normal distribution function on the side where it is small, and e = exp(-h^2 / 2) that it needs on the way: e times a
// polynomial of 1 / (1 + 0.3 |h|), which covers the rest's slow fall (it is the scaled complementary error function). The
// coefficients are a weighted least-squares fit to that function over |h| <= 14, good to 3e-7 where h is small and to 2.3e-5 of
// the value itself far out, where GELU is h times it: 0.05 of float16's rounding, so the outputs there are as good as their
// type. exp2 and the reciprocal are the hardware's, one ulp.
__device__ __forceinline__ float normal_cdf(float h, float& e) {
    const float t = rcp_of(fmaf(0.3f, fabsf(h), 1.0f));
    e = exp2_of(h * h * -0.7213475204444817f);
    const float q = fmaf(fmaf(fmaf(fmaf(fmaf(-0.0788607597f, t, 0.22041145f), t, -0.0207132176f), t, 0.145473763f), t,
                              0.113620818f), t, 0.120067716f) * t * e;
    return h < 0.0f ? q : 1.0f - q;
}
// GELU's tanh form is h times the logistic of 2 z, z = sqrt(2 / pi) (h + 0.044715 h^3), since (1 + tanh z) / 2 is that
__device__ __forceinline__ float tanh_factor(float h) {
    return rcp_of(1.0f + exp2_of(h * fmaf(-0.10294324f, h * h, -2.3022082f)));           // - 2 sqrt(2 / pi) log2(e) (...)
}
__device__ __forceinline__ float logistic(float h) { return rcp_of(1.0f + exp2_of(h * -1.4426950408889634f)); }

template <int KIND>
__device__ __forceinline__ float act_of(float h) {
    float e;
    if constexpr (KIND == ACT_GELU) return h * normal_cdf(h, e);
    else if constexpr (KIND == ACT_GELU_TANH) return h * tanh_factor(h);
    else if constexpr (KIND == ACT_SILU) return h * logistic(h);
    else if constexpr (KIND == ACT_RELU) return h < 0.0f ? 0.0f : h;
    else return h;
}

// f with the activation as a constant
template <typename F>
__device__ __forceinline__ void by_act(int kind, F&& f) {
    using std::integral_constant;
    if (kind == ACT_GELU_TANH) f(integral_constant<int, ACT_GELU_TANH>{});
    else if (kind == ACT_GELU) f(integral_constant<int, ACT_GELU>{});
    else if (kind == ACT_SILU) f(integral_constant<int, ACT_SILU>{});
    else if (kind == ACT_RELU) f(integral_constant<int, ACT_RELU>{});
    else f(integral_constant<int, ACT_NONE>{});
}

// v = act(v) on a run of values; one decision a run
__device__ __forceinline__ void act_run(int kind, float (&v)[8]) {
    by_act(kind, [&](auto k) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_of<decltype(k)::value>(v[i]);
    });
}

// a = act(h) and its slope, from finite h (keep_finite)
__device__ __forceinline__ void act_slope_run(int kind, const float (&h)[8], float (&a)[8], float (&slope)[8]) {
    if (kind == ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float s = tanh_factor(h[i]), dz = fmaf(0.21406614f, fminf(h[i] * h[i], 1e30f), 1.5957691f);
            a[i] = h[i] * s;
            slope[i] = fmaf(a[i] * (1.0f - s), dz, s);
        }
    } else if (kind == ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float e;
            const float phi = normal_cdf(h[i], e);
            a[i] = h[i] * phi;
            slope[i] = fmaf(h[i] * 0.3989422804014327f, e, phi);                         // 1 / sqrt(2 pi)
        }
    } else if (kind == ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float s = logistic(h[i]);
            a[i] = h[i] * s;
            slope[i] = fmaf(a[i], 1.0f - s, s);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool on = kind == ACT_NONE || h[i] > 0.0f;
            a[i] = on ? h[i] : h[i] < 0.0f ? 0.0f : h[i];
            slope[i] = on ? 1.0f : 0.0f;
        }
    }
}

// the pre-activation as it is kept for the backward pass: an infinity (float16's, past 65504) would make the slope 0 *
// infinity where its limit is 0 or 1, so it stays finite
template <int D>
__device__ __forceinline__ float keep_finite(float h) {
    constexpr float most = D == WF_F16 ? 65504.0f : 3.38953139e38f;
    return h > most ? most : h < -most ? -most : h;
}

struct DenseEpilogue {
    const void *bias, *gate, *resid;       // any may be NULL
    int bias_dt, gate_dt;                  // the outputs' type or float32
    int act;
    int64_t rows_per_group, ldr;           // row m's gate is row m / rows_per_group of gate; resid's row stride
    void *y, *h;                           // [M, N]; h (may be NULL): the pre-activations
};

// what a run at (m, n) of `cnt` values (8, or fewer at a row's end) needs from memory
template <int D>
struct EpilogueAhead {
    Pack<D> resid;
    float gate[8];
};
template <int D>
__device__ __forceinline__ EpilogueAhead<D> epilogue_ahead(const DenseEpilogue& e, int64_t m, int n, int N, int cnt) {
    EpilogueAhead<D> a;
    a.resid.zero();
    if (e.resid && cnt > 0) a.resid.load(static_cast<const value_t<D>*>(e.resid) + m * e.ldr + n, cnt);
    if (e.gate && cnt > 0) {
        const int64_t at = (int64_t)((uint32_t)m / (uint32_t)e.rows_per_group) * N + n;
        load_params<8>(a.gate, e.gate, at, cnt, e.gate_dt);
    }
    return a;
}

// v: a run's sums, without the bias when BIAS is set
template <int D, bool BIAS>
__device__ __forceinline__ void epilogue_run(const DenseEpilogue& e, float (&v)[8], const EpilogueAhead<D>& a, int64_t m,
                                             int n, int N, int cnt) {
    float u[8];
    if (BIAS && e.bias) {
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
    act_run(e.act, v);
    if (e.gate)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= a.gate[i];
    if (e.resid)
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += a.resid.get(i);
    Pack<D> o;
    o.put(v);
    o.store(static_cast<value_t<D>*>(e.y) + m * N + n, cnt);
}

}  // namespace wf
