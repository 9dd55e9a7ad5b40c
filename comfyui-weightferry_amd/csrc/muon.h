// The products of a Newton-Schulz step on a batch of matrices (muon_gemm.hip), and the matrices of a batch.
#pragma once

#include "values.h"

namespace wf {

constexpr int kMuonBatch = 64;             // matrices a launch: their addresses are kernel arguments

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

// p[i .. i + 8) of a matrix, the first cnt of them, with v = O there
template <int D>
__device__ __forceinline__ void muon_apply(value_t<D>* p, const float (&v)[8], int cnt, float keep, float rate) {
    constexpr int VEC = Pack<D>::VEC;
#pragma unroll
    for (int h = 0; h < 8 / VEC; h++) {
        if (cnt <= h * VEC) break;
        Pack<D> a;
        float w[VEC];
        if (keep != 0.0f) a.load(p + h * VEC, cnt - h * VEC);
        else a.zero();
#pragma unroll
        for (int i = 0; i < VEC; i++) w[i] = fmaf(-rate, v[h * VEC + i], keep != 0.0f ? keep * a.get(i) : 0.0f);
        a.put(w);
        a.store(p + h * VEC, cnt - h * VEC);
    }
}
__device__ __forceinline__ void muon_apply(const MuonTensors& t, int b, int64_t at, const float (&v)[8], int cnt) {
    if (t.dt == WF_BF16) muon_apply<WF_BF16>(static_cast<uint16_t*>(t.p[b]) + at, v, cnt, t.keep, t.rate);
    else if (t.dt == WF_F16) muon_apply<WF_F16>(static_cast<uint16_t*>(t.p[b]) + at, v, cnt, t.keep, t.rate);
    else muon_apply<WF_F32>(static_cast<float*>(t.p[b]) + at, v, cnt, t.keep, t.rate);
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
