// The products of a Newton-Schulz step on a batch of matrices (muon_gemm.hip), and the matrices of a batch.
#pragma once

#include "values.h"

namespace wf {

constexpr int kMuonBatch = 128;             // matrices a launch: their addresses are kernel arguments

// What is stepped, matrix by matrix: p (of type dt) becomes keep p - rate O, O the orthogonalised update.
struct MuonTensors {
    void* p[kMuonBatch];
    const void* g[kMuonBatch];
    float* m[kMuonBatch];                  // NULL: the update is g itself
    int dt;
    float keep, rate;                      // keep 0: p is written only
    float mu, nu;                          // m = mu m + nu g, nu = 1 - mu; the update is mu m + nu g (nesterov), or m
    int nesterov;
};

// 8 places of a parameter from `at` on, the first cnt of them: keep old - rate v (keep 0: old is not looked at)
__device__ __forceinline__ void muon_store(const MuonTensors& t, int b, int64_t at, const float (&old)[8], const float (&v)[8], int cnt) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = fmaf(-t.rate, v[i], t.keep != 0.0f ? t.keep * old[i] : 0.0f);
    if (t.dt == WF_F32) {
        float* p = static_cast<float*>(t.p[b]) + at;
        if (cnt >= 8) __builtin_memcpy(p, w, 32);
        else
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < cnt) p[i] = w[i];
    } else if (t.dt == WF_BF16) {
        Pack<WF_BF16> o;
        o.put(w);
        o.store(static_cast<uint16_t*>(t.p[b]) + at, cnt);
    } else {
        Pack<WF_F16> o;
        o.put(w);
        o.store(static_cast<uint16_t*>(t.p[b]) + at, cnt);
    }
}

// 8 places of a parameter as they lie (float32: in two packs), and what they stand for
__device__ __forceinline__ void muon_raw(const MuonTensors& t, int b, int64_t at, int cnt, Pack<WF_F16>& lo, Pack<WF_F16>& hi) {
    if (t.dt == WF_F32) {
        const float* p = static_cast<const float*>(t.p[b]) + at;
        Pack<WF_F32> a, c;
        a.load(p, cnt);
        c.zero();
        if (cnt > 4) c.load(p + 4, cnt - 4);
        __builtin_memcpy(lo.w, a.w, 16);
        __builtin_memcpy(hi.w, c.w, 16);
    } else {
        lo.load(static_cast<const uint16_t*>(t.p[b]) + at, cnt);
    }
}
__device__ __forceinline__ void muon_values(const MuonTensors& t, const Pack<WF_F16>& lo, const Pack<WF_F16>& hi, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t h = i & 1 ? lo.w[i / 2] >> 16 : lo.w[i / 2] & 0xffffu;
        v[i] = t.dt == WF_F32 ? __uint_as_float(i < 4 ? lo.w[i] : hi.w[i - 4]) : t.dt == WF_BF16 ? __uint_as_float(h << 16) : f16_bits_to_f32(h);
    }
}

// A batch in float16, matrix b at x + b (rows ld), X s with s a power of two; symmetric matrices [side, sld], times s^2; rows' lengths ld, sld are
// multiples of 8, zeros past the matrix.
struct MuonShape {
    int rows, cols, ld, side, sld, batch;
    bool tall;                             // rows > cols: the short side is the columns
};

// out = alpha S + beta in + gamma I, S = x x^T (or x^T x where tall), in may be NULL
struct MuonSymmetric {
    const uint16_t* x;                     // [rows, ld], or a symmetric matrix [side, sld] (square set)
    bool square;
    const uint16_t* in;
    uint16_t* out;
    float alpha, beta, gamma;
};
// next = alpha q x (x q where tall) + a (x + lo / 2048); the remainder of its rounding, times 2048, to lo. lo NULL: next = alpha q x
// alone; next NULL: the tensors' step with it.
struct MuonUpdate {
    const uint16_t *x, *q;
    uint16_t *lo, *next;
    float alpha, a;
};

int64_t muon_symmetric_bytes(const MuonShape& s, bool square);      // of float32 partial sums
void muon_symmetric(const MuonShape& s, const MuonSymmetric& q, float* parts, hipStream_t st);
void muon_update(const MuonShape& s, const MuonUpdate& q, const MuonTensors& t, hipStream_t st);

}  // namespace wf
